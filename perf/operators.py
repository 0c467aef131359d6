"""Timed cases of the paged 8-bit KV cache: page tables, appends, read-back and the attention that reads it.

A server that keeps its requests' caches in pages runs these per step: it gives back what rejected drafts or finished
requests held and hands pages to the new rows (`tables`), every layer writes its new K and V rows into their pages
(`append`: rows as they are; `norm_append`: behind the per-head norm and RoPE), and attends over the pages
(`attention`).  Cached rows come back as numbers through the read-back operator, which the append cases call for the
rows that they wrote and the `read` cases for whole contexts.  Head layouts and lengths are those of this
repository's configurations and of its other timed cases.

The cache: codes [n_pages, n_kv, page, hd] for K and V, one byte a value (int8 or e4m3), and a scale for each page and
KV head; value = code * scale.  An append scales a page by the least power of two that its rows fit under and rounds the
rows that were there before again where that scale grows.

A case is a dict of plain values; `kind` names the operator.  Where `own` is false, `run` computes with elementary
torch operations on the same tensors.
"""
import math
import random

import torch

own = False

HEADER = 8                  # ints in front of a plan: status, rows, jobs, free pages
QMAX = {"i8": 127.0, "e4m3": 448.0}
EPS = 1e-6
THETA = 1e6


def listed():
    return [
        # every running request gets one token: the smallest call of a serving step
        dict(name="tables_8_decode", kind="tables", seqs=8, page=64, ctx=8192, new=1, back=1),
        # a full server: ragged prompts and idle requests, drafts of some turned down
        dict(name="tables_256_ragged", kind="tables", seqs=256, page=16, ctx=4096, new=127, back=40),
        # one new token in each of eight caches, pages half full
        dict(name="append_8_tokens", kind="append", seqs=8, rows=8, page=64, ctx=4096, n_kv=2, hd=256, act="f32", fmt="i8"),
        # ragged prompts of four requests behind what they have
        dict(name="append_2047_rows", kind="append", seqs=4, rows=2047, page=16, ctx=2048, n_kv=8, hd=128, act="f16", fmt="e4m3"),
        # the same behind the norms and RoPE of a layer: one token of each of four requests, and a prompt pass
        dict(name="norm_append_4_tokens", kind="norm_append", seqs=4, rows=4, page=64, ctx=1000, n_q=8, n_kv=1, hd=256, act="f16", fmt="i8"),
        dict(name="norm_append_2048_rows", kind="norm_append", seqs=3, rows=2048, page=64, ctx=3000, n_q=8, n_kv=2, hd=256, act="f16", fmt="e4m3"),
        # whole contexts read back, as a host that moves a request to another server does
        dict(name="read_20000_rows", kind="read", seqs=5, rows=20000, page=64, ctx=8192, n_kv=2, hd=256, act="f16", fmt="i8"),
        # one chat, one token: latency
        dict(name="attention_1_token", kind="attention", lens="700", rows="1", page=64, n_q=8, n_kv=1, hd=256, window=0, act="f32", fmt="i8"),
        # four requests deep into unequal contexts
        dict(name="attention_4_slots", kind="attention", lens="1024,4096,16384,16384", rows="1,1,1,1", page=64, n_q=8, n_kv=2, hd=256, window=0, act="f32", fmt="i8"),
        # a full server that decodes
        dict(name="attention_48_decode", kind="attention", lens=",".join(str(8192 - 61 * i) for i in range(48)), rows=",".join(["1"] * 48), page=16, n_q=32, n_kv=8,
             hd=128, window=0, act="f16", fmt="e4m3"),
        # prompts of two requests beside ones that decode, drafts of three tokens among them, sliding window
        dict(name="attention_mixed_window", kind="attention", lens="900,1777,3000,512,2100,64,1300,4000", rows="517,300,1,1,3,64,1,3", page=32, n_q=8, n_kv=2, hd=256,
             window=512, act="f32", fmt="e4m3"),
        # the second half of a long prompt
        dict(name="attention_4096_rows", kind="attention", lens="8192", rows="4096", page=64, n_q=16, n_kv=4, hd=128, window=0, act="f16", fmt="i8"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["tables", "append", "norm_append", "read", "attention", "attention", "attention"])
    page = rng.choice([16, 32, 64, 128])
    if kind == "tables":
        return dict(kind=kind, seqs=_log(rng, 1, 256), page=page, ctx=_log(rng, 64, 8192), new=_log(rng, 1, 200), back=_log(rng, 1, 64))
    n_kv, hd = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
    act, fmt = rng.choice(["f32", "f16"]), rng.choice(["i8", "e4m3"])
    if kind == "read":
        return dict(kind=kind, seqs=_log(rng, 1, 32), rows=_log(rng, 1, 8000), page=page, ctx=_log(rng, 300, 8192), n_kv=n_kv, hd=hd, act=act, fmt=fmt)
    if kind in ("append", "norm_append"):
        seqs = _log(rng, 1, 32)
        c = dict(kind=kind, seqs=seqs, rows=max(seqs, _log(rng, 1, 2048)), page=page, ctx=_log(rng, 16, 4096), n_kv=n_kv, hd=hd, act=act, fmt=fmt)
        if kind == "norm_append":
            c.update(n_q=n_kv * rng.choice([1, 2, 4]))
        return c
    group = rng.choice([1, 2, 3, 4, 8])
    shape = rng.choice(["decode", "decode", "prompt", "mixed"])
    if shape == "decode":
        n = _log(rng, 1, 40)
        lens = [_log(rng, 1, 8192) for _ in range(n)]
        rows = [min(t, rng.choice([1, 1, 1, 2, 4])) for t in lens]
    elif shape == "prompt":
        n = _log(rng, 1, 4)
        rows = [_log(rng, 20, 2000 // n) for _ in range(n)]
        lens = [r + rng.choice([0, _log(rng, 1, 2000)]) for r in rows]
    else:
        n = _log(rng, 2, 12)
        rows = [rng.choice([1, 1, 3, 0, _log(rng, 5, 300)]) for _ in range(n - 1)] + [_log(rng, 1, 300)]
        lens = [r + _log(rng, 1, 2500) for r in rows]
    return dict(kind=kind, lens=",".join(map(str, lens)), rows=",".join(map(str, rows)), page=page, n_q=n_kv * group, n_kv=n_kv, hd=hd,
                window=rng.choice([0, 0, _log(rng, 16, 1024)]), act=act, fmt=fmt)


# ---- inputs -------------------------------------------------------------------------------------------

class _State:
    def __init__(self, **kw):
        self.__dict__.update(kw)


def _dtype(act):
    return torch.float32 if act == "f32" else torch.float16


def _round4(n):
    return -(-n // 4) * 4


def _plan_parts(n_seqs, max_rows, page):
    """Where the parts of a plan start: row_start, row_seq, row_pos, row_slot, jobs, and its length."""
    start = HEADER
    seq = start + _round4(n_seqs + 1)
    step = _round4(max_rows)
    return start, seq, seq + step, seq + 2 * step, seq + 3 * step, seq + 3 * step + 4 * (max_rows // page + 2 * n_seqs)


def _codes(gen, fmt, shape):
    """Codes of normally distributed values whose largest fill the format."""
    x = torch.randn(shape, device="cuda", generator=gen)
    if fmt == "i8":
        return (x * 32.0).round_().clamp_(-127, 127).to(torch.int8)
    return (x * 110.0).clamp_(-448, 448).to(torch.float8_e4m3fn)


def _scales(gen, fmt, shape, powers=False):
    """A scale for each page and head that makes values of about one; powers of two where an append wrote them."""
    if powers:
        e = torch.randint(-6, -4, shape, device="cuda", generator=gen).float()
        return torch.exp2(e if fmt == "i8" else e - 2)
    return (0.6 + 0.8 * torch.rand(shape, device="cuda", generator=gen)) / (32.0 if fmt == "i8" else 110.0)


def _spread(rng, total, n):
    """total rows over n requests, one at least each."""
    got = [1] * n
    left = total - n
    for i in range(n - 1):
        take = min(left, int(rng.random() * 2 * left / (n - i)))
        got[i] += take
        left -= take
    got[-1] += left
    return got


def _state_of(lens, page, max_blocks, n_pages, perm):
    """Tables, lengths and free stack of requests of these lengths, whose pages are the first ones of perm."""
    blocks = -(-lens // page)
    first = torch.cumsum(blocks, 0) - blocks
    at = torch.arange(max_blocks, device="cuda")
    held = at[None, :] < blocks[:, None]
    tables = torch.where(held, perm[(first[:, None] + at[None, :]).clamp(max=n_pages - 1)], -1).to(torch.int32)
    used = int(blocks.sum())
    free = torch.zeros(1 + n_pages, dtype=torch.int32, device="cuda")
    free[0] = n_pages - used
    free[1:1 + n_pages - used] = perm[used:].to(torch.int32)
    return lens.to(torch.int32), tables.contiguous(), free


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    kind, page = case["kind"], case["page"]
    dev = dict(device="cuda")
    if kind == "tables":
        n = case["seqs"]
        keep = torch.tensor([rng.randint(1, case["ctx"]) for _ in range(n)], **dev)
        back = torch.tensor([rng.randint(0, case["back"]) for _ in range(n)], **dev)
        new = torch.tensor([rng.randint(0, case["new"]) if case["new"] > 1 else 1 for _ in range(n)], **dev)
        max_rows = _round4(n * case["new"] + 3)
        max_blocks = (case["ctx"] + max(case["new"], case["back"])) // page + 2
        n_pages = n * max_blocks
        perm = torch.randperm(n_pages, generator=gen, **dev)
        lens, tables, free = _state_of(keep + back, page, max_blocks, n_pages, perm)
        plan = torch.zeros(_plan_parts(n, max_rows, page)[-1], dtype=torch.int32, **dev)
        return _State(case=case, kind=kind, n=n, page=page, max_rows=max_rows, max_blocks=max_blocks, n_pages=n_pages, lens=lens, tables=tables, free=free, plan=plan,
                      keep=keep.to(torch.int32), new=new.to(torch.int32), h=None)

    n_kv, hd, fmt, act = case["n_kv"], case["hd"], case["fmt"], _dtype(case["act"])
    if kind == "attention":
        after = [int(v) for v in case["lens"].split(",")]
        rows = [int(v) for v in case["rows"].split(",")]
    elif kind == "read":
        n = case["seqs"]
        rows = after = [min(r, case["ctx"]) for r in _spread(rng, max(case["rows"], n), n)]
    else:
        rows = _spread(rng, max(case["rows"], case["seqs"]), case["seqs"])
        after = [r + rng.randint(0, case["ctx"]) for r in rows]
    n, total = len(rows), sum(rows)
    # buffers go by the case alone
    most = case.get("rows", 0) if kind != "attention" else 0
    max_rows = _round4(max(total, 1) if kind == "attention" else max(most, n))
    max_blocks = max(after) // page + 1 if kind == "attention" else (most + n + case["ctx"]) // page + 2
    n_pages = sum(t // page + 1 for t in after) + n if kind == "attention" else n * (case["ctx"] // page + 2) + (most + n) // page + 1
    perm = torch.randperm(n_pages, generator=gen, **dev)
    before = torch.tensor([a - r for a, r in zip(after, rows)], **dev)
    lens, tables, free = _state_of(before, page, max_blocks, n_pages, perm)
    plan = torch.zeros(_plan_parts(n, max_rows, page)[-1], dtype=torch.int32, **dev)
    new = torch.tensor(rows, dtype=torch.int32, **dev)
    s = _State(case=case, kind=kind, n=n, page=page, max_rows=max_rows, max_blocks=max_blocks, n_pages=n_pages, lens=lens, tables=tables, free=free, plan=plan,
               n_kv=n_kv, hd=hd, fmt=fmt, act=act, rows=total, rows_most=max(rows), ctx_most=max(after), h=None)
    _plain_step(s, new)
    shape = (n_pages, n_kv, page, hd)
    s.K, s.V = _codes(gen, fmt, shape), _codes(gen, fmt, shape)
    s.ks, s.vs = (_scales(gen, fmt, shape[:2], kind in ("append", "norm_append")) for _ in range(2))
    if kind in ("append", "norm_append", "read"):
        s.k_back, s.v_back = (torch.zeros((max_rows, n_kv, hd), dtype=torch.float16 if kind == "norm_append" else act, **dev) for _ in range(2))
    if kind in ("append", "norm_append"):
        s.k, s.v = (torch.randn((max_rows, n_kv, hd), generator=gen, **dev).to(act) for _ in range(2))
    if kind == "norm_append":
        s.n_q = case["n_q"]
        s.q = torch.randn((max_rows, s.n_q, hd), generator=gen, **dev).to(act)
        s.qw, s.kw = ((1.0 + 0.1 * torch.randn(hd, generator=gen, **dev)).to(act) for _ in range(2))
        s.q_out = torch.zeros_like(s.q)
        ang = torch.arange(max_blocks * page, dtype=torch.float64, **dev)[:, None] * THETA ** (-torch.arange(hd // 2, dtype=torch.float64, **dev) * 2 / hd)
        s.rope = torch.cat([ang.cos(), ang.sin()], 1).float().contiguous()
    if kind == "attention":
        s.n_q, s.window, s.scale = case["n_q"], case["window"], hd ** -0.5
        s.q = torch.randn((max_rows, s.n_q, hd), generator=gen, **dev).to(act)
        s.out = torch.zeros_like(s.q)
    return s


# ---- plain forms --------------------------------------------------------------------------------------

def _plain_trim(s, keep):
    """Sequences end at keep; what they held behind that goes back on the stack, the last page first."""
    old = -(-s.lens // s.page)
    kept = torch.where((keep >= 0) & (keep < s.lens), keep, s.lens)
    at = torch.arange(s.max_blocks, device="cuda")
    gone = (at[None, :] >= (-(-kept // s.page))[:, None]) & (at[None, :] < old[:, None])
    rank = torch.cumsum(gone.reshape(-1).to(torch.int64), 0).reshape(gone.shape) - 1
    back = gone.sum()
    where = torch.where(gone, 1 + s.free[0] + back - 1 - rank, 1 + s.n_pages)
    stack = torch.cat([s.free, s.free[:1]])
    stack.scatter_(0, where.reshape(-1), s.tables.reshape(-1))
    s.free[1:] = stack[1:-1]
    s.free[0] += back.to(torch.int32)
    s.tables[:] = torch.where(gone, -1, s.tables)
    s.lens[:] = kept


def _plain_step(s, new):
    """Pages for `new` rows of every sequence and the plan that says where they go (there is room for all of them)."""
    o_start, o_seq, o_pos, o_slot, o_job, end = _plan_parts(s.n, s.max_rows, s.page)
    page = s.page
    old, after = -(-s.lens // page), s.lens + new
    need = -(-after // page) - old
    first = torch.cumsum(need, 0) - need
    at = torch.arange(s.max_blocks, device="cuda")
    fresh = (at[None, :] >= old[:, None]) & (at[None, :] < (old + need)[:, None])
    k = first[:, None] + at[None, :] - old[:, None]
    taken = s.free[torch.where(fresh, s.free[0] - k, 0).long()]
    s.tables[:] = torch.where(fresh, taken, s.tables)
    s.free[0] -= need.sum().to(torch.int32)
    ends = torch.cumsum(new, 0)
    total = ends[-1]
    row = torch.arange(s.max_rows, device="cuda")
    live = row < total
    seq = torch.searchsorted(ends, row, right=True).clamp(max=s.n - 1)
    r = row - (ends - new)[seq]
    pos = s.lens[seq] + r
    slot = s.tables[seq, (pos // page).clamp(0, s.max_blocks - 1)] * page + pos % page
    leads = live & ((r == 0) | (pos % page == 0))
    s.plan.zero_()
    s.plan[o_start + 1:o_start + 1 + s.n] = ends.to(torch.int32)
    for o, v in ((o_seq, seq), (o_pos, pos), (o_slot, slot)):
        s.plan[o:o + _round4(s.max_rows)] = -1
        s.plan[o:o + s.max_rows] = torch.where(live, v, -1).to(torch.int32)
    n_jobs = (end - o_job) // 4
    jobs = torch.full((n_jobs + 1, 4), -1, dtype=torch.int32, device="cuda")
    record = torch.stack([row, torch.minimum(page - pos % page, ends[seq] - row), slot, pos], 1)
    jobs[torch.where(leads, torch.cumsum(leads.long(), 0) - 1, n_jobs)] = torch.where(leads[:, None], record, -1).to(torch.int32)
    s.plan[o_job:end] = jobs[:n_jobs].reshape(-1)
    s.plan[1], s.plan[2], s.plan[3] = total, leads.sum(), s.free[0]
    s.lens[:] = after


def _quantised(x, scale, fmt):
    """Values over their scales, rounded to the format and back; infinities at its ends, NaN as zero."""
    y = torch.nan_to_num(x / scale, nan=0.0, posinf=QMAX[fmt], neginf=-QMAX[fmt]).clamp(-QMAX[fmt], QMAX[fmt])
    return y.round() if fmt == "i8" else y.to(torch.float8_e4m3fn).float()


def _plain_append(s, codes, scales, x):
    """Rows x [max_rows, n_kv, hd] (f32) into their pages."""
    page, n_kv, hd, qmax = s.page, s.n_kv, s.hd, QMAX[s.fmt]
    _, _, o_pos, o_slot, o_job, end = _plan_parts(s.n, s.max_rows, page)
    slot, pos = s.plan[o_slot:o_slot + s.rows].long(), s.plan[o_pos:o_pos + s.rows].long()
    x = x[:s.rows]
    pages = slot // page
    amax = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
    # of each page: the largest of its new rows, and the position in it that the first of them takes
    big = torch.zeros((s.n_pages, n_kv), device="cuda").scatter_reduce_(0, pages[:, None].expand(-1, n_kv), amax, "amax")
    begin = torch.full((s.n_pages,), page, device="cuda").scatter_reduce_(0, pages, pos % page, "amin")
    touched = begin < page
    # the least power of two that the largest fits under
    m, e = torch.frexp(big)
    e = e - int(math.log2(QMAX[s.fmt])) - 1 + (m > qmax / 2.0 ** (int(math.log2(qmax)) + 1)).to(torch.int32)
    want = torch.where(big > 0, torch.exp2(e.double().clamp(-100, 100)), 2.0 ** -100).float()
    grown = torch.where((begin == 0)[:, None], want, torch.maximum(want, scales))
    t = torch.nonzero(touched)[:, 0]
    # what the touched pages held is rounded again
    before = _quantised(codes[t].float() * scales[t][:, :, None, None], grown[t][:, :, None, None], s.fmt)
    codes[t] = torch.where((torch.arange(page, device="cuda") < begin[t][:, None])[:, None, :, None], before.to(codes.dtype).float(), codes[t].float()).to(codes.dtype)
    scales[t] = grown[t]
    codes.transpose(1, 2)[pages, slot % page] = _quantised(x, grown[pages][:, :, None], s.fmt).to(codes.dtype)


def _plain_read(s, codes, scales, out):
    _, _, _, o_slot, _, _ = _plan_parts(s.n, s.max_rows, s.page)
    slot = s.plan[o_slot:o_slot + s.rows].long()
    pages = slot // s.page
    out[:s.rows] = (codes.transpose(1, 2)[pages, slot % s.page].float() * scales[pages][:, :, None]).to(out.dtype)


def _plain_norm(x, w):
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    return x if w is None else x * w.float()


def _plain_rope(s, x):
    _, _, o_pos, o_slot, _, _ = _plan_parts(s.n, s.max_rows, s.page)
    cs = s.rope[s.plan[o_pos:o_pos + s.rows].long()][:, None, :]
    c, sn = cs[..., :s.hd // 2], cs[..., s.hd // 2:]
    u, v = x[:s.rows, :, :s.hd // 2], x[:s.rows, :, s.hd // 2:]
    return torch.cat([u * c - v * sn, u * sn + v * c], -1)


def _plain_attention(s):
    n, n_kv, hd, page = s.n, s.n_kv, s.hd, s.page
    G = s.n_q // n_kv
    start = s.plan[HEADER:HEADER + n + 1].long()
    rows = start[1:] - start[:-1]
    R, blocks = s.rows_most, -(-s.ctx_most // page)
    L = blocks * page
    tab = s.tables[:, :blocks].clamp(min=0).long()
    K = (s.K[tab].float() * s.ks[tab][..., None, None]).permute(0, 2, 1, 3, 4).reshape(n, n_kv, L, hd)
    V = (s.V[tab].float() * s.vs[tab][..., None, None]).permute(0, 2, 1, 3, 4).reshape(n, n_kv, L, hd)
    r = torch.arange(R, device="cuda")
    live = r[None, :] < rows[:, None]
    at = torch.where(live, start[:-1, None] + r[None, :], 0)
    q = s.q[at].float().reshape(n, R, n_kv, G, hd).permute(0, 2, 1, 3, 4).reshape(n, n_kv, R * G, hd)
    score = (q @ K.transpose(2, 3)).mul_(s.scale).reshape(n, n_kv, R, G, L)
    pos = (s.lens.long() - rows)[:, None] + r[None, :]
    key = torch.arange(L, device="cuda")
    seen = key[None, None, :] <= pos[..., None]
    if s.window:
        seen &= key[None, None, :] > pos[..., None] - s.window
    score.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    score.sub_(score.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = score.sum(-1, keepdim=True)
    out = score.reshape(n, n_kv, R * G, L) @ V
    out = out.reshape(n, n_kv, R, G, hd) / total.clamp(min=1e-30)
    out = out.permute(0, 2, 1, 3, 4).reshape(n, R, s.n_q, hd)
    s.out[at[live]] = out[live].to(s.out.dtype)


def _plain(s):
    if s.kind == "tables":
        _plain_trim(s, s.keep)
        _plain_step(s, s.new)
    elif s.kind == "append":
        _plain_append(s, s.K, s.ks, s.k.float())
        _plain_append(s, s.V, s.vs, s.v.float())
    elif s.kind == "norm_append":
        s.q_out[:s.rows] = _plain_rope(s, _plain_norm(s.q, s.qw)).to(s.act)
        _plain_append(s, s.K, s.ks, _plain_rope(s, _plain_norm(s.k, s.kw)))
        _plain_append(s, s.V, s.vs, _plain_norm(s.v, None))
    elif s.kind == "attention":
        _plain_attention(s)
    if s.kind in ("append", "norm_append", "read"):
        _plain_read(s, s.K, s.ks, s.k_back)
        _plain_read(s, s.V, s.vs, s.v_back)


# ---- the framework's operators -------------------------------------------------------------------------

_CTX = []


def _handles(s):
    """What a program keeps with its tensors: the context and the handles of its buffers."""
    from ksearch_b200 import Buffer, CudaContext, E4M3, Eng, F16, F32, I8, PageTables, Q8Cache

    if not _CTX:
        _CTX.append(CudaContext(torch.cuda.current_device(), 1))
    ctx = _CTX[0]

    def buf(t):
        nbytes = t.numel() * t.element_size()
        return Buffer(ctx, ctx.lib.ks_buf_wrap(ctx.h, t.data_ptr(), nbytes), nbytes)

    h = _State(ctx=ctx, eng=Eng(F16 if s.case.get("act") == "f16" else F32), f16=Eng(F16))
    h.tables = PageTables(ctx, s.n, s.max_blocks, s.n_pages, s.page, s.max_rows, lens=buf(s.lens), tables=buf(s.tables), free=buf(s.free), plan=buf(s.plan))
    names = ("keep", "new", "k", "v", "q", "qw", "kw", "q_out", "rope", "k_back", "v_back", "out")
    for name in names:
        if hasattr(s, name):
            setattr(h, name, buf(getattr(s, name)))
    if s.kind != "tables":
        h.cache = Q8Cache(ctx, s.n_pages, s.page, s.n_kv, s.hd, I8 if s.fmt == "i8" else E4M3, k=buf(s.K), v=buf(s.V), k_scale=buf(s.ks), v_scale=buf(s.vs))
    if s.kind == "attention":
        h.tmp = ctx.buffer_empty_f32(h.eng.sdpa_paged_tmp_floats(ctx, h.cache, h.tables, s.n_q, s.rows_most))
    return h


def _framework(s):
    if s.h is None:
        s.h = _handles(s)
    h = s.h
    ctx, eng = h.ctx, h.eng
    if s.kind == "tables":
        eng.pages_trim(ctx, h.tables, h.keep)
        eng.pages_step(ctx, h.tables, h.new)
    elif s.kind == "append":
        eng.kv_append_q8(ctx, h.cache, h.tables, h.k, h.v)
    elif s.kind == "norm_append":
        eng.rmsnorm_per_head_qkv_q8(ctx, h.cache, h.tables, s.n_q, EPS, h.q, h.qw, h.rope, h.k, h.kw, h.v, h.q_out)
    elif s.kind == "attention":
        eng.sdpa_paged_q8(ctx, h.cache, h.tables, s.n_q, s.rows_most, s.ctx_most, h.q, h.tmp, h.out, s.scale, s.window)
    if s.kind in ("append", "norm_append", "read"):
        (h.f16 if s.kind == "norm_append" else eng).kv_read_q8(ctx, h.cache, s.rows, h.tables.plan, h.tables.row_slot, h.k_back, h.v_back)


def run(s):
    if own:
        _framework(s)
    else:
        _plain(s)
    if s.kind == "tables":
        return dict(lens=s.lens, tables=s.tables, free=s.free, plan=s.plan)
    if s.kind == "attention":
        return dict(out=s.out)
    got = dict(k=s.k_back, v=s.v_back)
    if s.kind != "read":
        got.update(k_scale=s.ks, v_scale=s.vs)
    if s.kind == "norm_append":
        got.update(q=s.q_out)
    return got


# ---- what a pass cannot do without ----------------------------------------------------------------------

def work(case):
    kind, page = case["kind"], case["page"]
    if kind == "tables":
        n, rows = case["seqs"], case["seqs"] * (case["new"] if case["new"] == 1 else case["new"] / 2)
        turned = n * (case["new"] + case["back"]) / 2 / page
        # lengths twice, counts twice, the table entries and stack words of the pages that move, three words a row, four a touched page
        return dict(bytes=4 * (5 * n + 4 * turned + 3 * rows + 4 * (rows / page + n)), flops=0)
    n_kv, hd = case["n_kv"], case["hd"]
    size = 4 if case["act"] == "f32" else 2
    if kind == "attention":
        after, rows = ([int(v) for v in case[k].split(",")] for k in ("lens", "rows"))
        w = case["window"]
        seen = pairs = 0
        for t, r in zip(after, rows):
            if r:
                seen += t - (max(0, t - r - w + 1) if w else 0)
                pairs += sum(min(p + 1, w) if w else p + 1 for p in range(t - r, t))
        total = sum(rows)
        return dict(bytes=2 * seen * n_kv * hd + 2 * 4 * (seen / page) * n_kv + 2 * total * case["n_q"] * hd * size, flops=4 * hd * case["n_q"] * pairs)
    rows = max(case["rows"], case["seqs"])
    if kind == "read":
        rows = min(rows, case["seqs"] * case["ctx"])
        return dict(bytes=2 * rows * n_kv * hd * (1 + size) + 8 * rows / page * n_kv, flops=2 * rows * n_kv * hd)
    back = 2 if kind == "norm_append" else size
    # rows in, codes out and in again, values out, scales
    moved = 2 * rows * n_kv * hd * (size + 2 + back) + 16 * (rows / page + case["seqs"]) * n_kv
    if kind == "norm_append":
        moved += 2 * rows * case["n_q"] * hd * size + 4 * rows * hd
    return dict(bytes=moved, flops=4 * rows * n_kv * hd + (10 * rows * case["n_q"] * hd if kind == "norm_append" else 0))


# ---- from the definitions, in 64 bits --------------------------------------------------------------------

def _exact_rows(s, x, codes, scales):
    """Rows x [rows, n_kv, hd] in 64 bits as their pages hold them, and all scales: page by page."""
    qmax = QMAX[s.fmt]
    slots = s.plan[_plan_parts(s.n, s.max_rows, s.page)[3]:][:s.rows].tolist()
    scales = scales.double().clone()
    want = torch.zeros((s.max_rows,) + x.shape[1:], dtype=torch.float64, device="cuda")
    groups = {}
    for r, slot in enumerate(slots):
        groups.setdefault(slot // s.page, []).append(r)
    for p, rows in groups.items():
        here = x[rows]
        big = here.abs().amax((0, 2))
        e = torch.ceil(torch.log2(big / qmax))
        e = torch.where(big <= qmax * torch.exp2(e - 1), e - 1, torch.where(big > qmax * torch.exp2(e), e + 1, e))
        sc = torch.exp2(e)
        if slots[rows[0]] % s.page:
            sc = torch.maximum(sc, scales[p])
        scales[p] = sc
        y = here / sc[None, :, None]
        y = torch.round(y) if s.fmt == "i8" else _e4m3(y)
        want[rows] = y * sc[None, :, None]
    return want, scales


def _e4m3(y):
    """The nearest number of three mantissa bits and exponents from -6 on, ties to even."""
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(y / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    if s.kind == "tables":
        return None
    if s.kind == "read":
        got = []
        slots = s.plan[_plan_parts(s.n, s.max_rows, s.page)[3]:][:s.rows].long()
        for codes, scales in ((s.K, s.ks), (s.V, s.vs)):
            back = torch.zeros((s.max_rows, s.n_kv, s.hd), dtype=torch.float64, device="cuda")
            for h in range(s.n_kv):
                flat = codes[:, h].float().reshape(-1, s.hd)
                back[:s.rows, h] = flat[slots].double() * scales[slots // s.page, h].double()[:, None]
            got.append(back)
        return dict(k=got[0], v=got[1])
    if s.kind in ("append", "norm_append"):
        k, v = s.k[:s.rows].double(), s.v[:s.rows].double()
        got = {}
        if s.kind == "norm_append":
            pos = s.plan[_plan_parts(s.n, s.max_rows, s.page)[2]:][:s.rows].long()
            ang = s.rope[pos].double()
            turn = torch.complex(ang[:, :s.hd // 2], ang[:, s.hd // 2:])[:, None, :]

            def normed(x, w):
                x = x[:s.rows].double()
                return x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / s.hd + EPS) * w

            def turned(x):
                z = torch.complex(x[..., :s.hd // 2], x[..., s.hd // 2:]) * turn
                return torch.cat([z.real, z.imag], -1)

            q = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
            q[:s.rows] = turned(normed(s.q, s.qw.double()))
            k, v = turned(normed(s.k, s.kw.double())), normed(s.v, 1.0)
            got["q"] = q
        got["k"], got["k_scale"] = _exact_rows(s, k, s.K, s.ks)
        got["v"], got["v_scale"] = _exact_rows(s, v, s.V, s.vs)
        return got
    out = torch.zeros(s.out.shape, dtype=torch.float64, device="cuda")
    start = s.plan[HEADER:HEADER + s.n + 1].tolist()
    lens, G = s.lens.tolist(), s.n_q // s.n_kv
    for i in range(s.n):
        r0, r1 = start[i], start[i + 1]
        if r1 == r0:
            continue
        pages = s.tables[i, :-(-lens[i] // s.page)].long()
        first = lens[i] - (r1 - r0)
        p = torch.arange(first, lens[i], device="cuda")[:, None]
        j = torch.arange(lens[i], device="cuda")[None, :]
        seen = (j <= p) & (j > p - s.window) if s.window else j <= p
        for h in range(s.n_kv):
            k = (s.K[pages, h].float().double() * s.ks[pages, h].double()[:, None, None]).reshape(-1, s.hd)[:lens[i]]
            v = (s.V[pages, h].float().double() * s.vs[pages, h].double()[:, None, None]).reshape(-1, s.hd)[:lens[i]]
            for g in range(G):
                sc = s.q[r0:r1, h * G + g].double() @ k.T * s.scale
                out[r0:r1, h * G + g] = torch.softmax(sc.masked_fill(~seen, -math.inf), -1) @ v
    return dict(out=out)
