"""The paged 8-bit cache on the GPU against plain loops and 64 bits (tests/paged_ref.py): tables, appends, read-back, attention, and
all of them together as a decoder uses them."""
import numpy as np
import pytest

from ksearch_b200 import E4M3, F16, F32, I8, CudaContext, Eng, KsError, PageTables, Q8Cache, _lib
from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

NP = {F32: np.float32, F16: np.float16}


def ints(ctx, x):
    return ctx.buffer_bytes(np.asarray(x, np.int32))


class Pair:
    """Tables on the GPU and the restatement beside them."""

    def __init__(self, ctx, n_seqs, max_blocks, n_pages, page, max_rows):
        self.ctx, self.eng = ctx, Eng()
        self.gpu = PageTables(ctx, n_seqs, max_blocks, n_pages, page, max_rows)
        self.cpu = ref.Tables(n_seqs, max_blocks, n_pages, page, max_rows)

    def step(self, new, check=True):
        self.eng.pages_step(self.ctx, self.gpu, ints(self.ctx, new))
        status = self.cpu.step(new)
        if check:
            self.same(status)
        return status

    def trim(self, keep):
        self.eng.pages_trim(self.ctx, self.gpu, ints(self.ctx, keep))
        self.cpu.trim(keep)

    def same(self, status=0):
        g, c = self.gpu, self.cpu
        assert np.array_equal(g.read(g.lens), c.lens)
        assert np.array_equal(g.read(g.tables).reshape(c.tables.shape), c.tables)
        free = g.read(g.free)
        assert free[0] == len(c.stack) and np.array_equal(free[1:1 + len(c.stack)], c.stack)
        plan = g.read(g.plan)
        part = [g.plan_part(p) for p in range(6)]
        assert plan[:8].tolist() == [status, len(c.rows), len(c.jobs), len(c.stack), 0, 0, 0, 0]
        assert np.array_equal(plan[part[0]:part[0] + c.n_seqs + 1], c.row_start)
        rows = np.full((c.max_rows, 3), -1, np.int64)
        rows[:len(c.rows)] = np.array(c.rows, np.int64).reshape(-1, 3)
        for k in range(3):
            assert np.array_equal(plan[part[1 + k]:part[1 + k] + c.max_rows], rows[:, k])
        jobs = np.full(((part[5] - part[4]) // 4, 4), -1, np.int64)
        jobs[:len(c.jobs)] = np.array(c.jobs, np.int64).reshape(-1, 4)
        assert np.array_equal(plan[part[4]:part[5]].reshape(-1, 4), jobs)


# ---- tables ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("n_seqs,page,max_rows,most", [(1, 16, 1, 1), (1, 64, 300, 300), (5, 32, 77, 15), (33, 16, 700, 40), (129, 16, 3000, 20), (256, 64, 30000, 200), (300, 16, 600, 2),
                                                       (1024, 128, 20000, 25)])
def test_steps_and_trims(ctx, n_seqs, page, max_rows, most):
    """Steps of no, one and many rows with trims in between: every table, stack and plan equal.  The larger ones take several blocks."""
    rng = np.random.default_rng(n_seqs * 1000 + page)
    p = Pair(ctx, n_seqs, 6 * most // page + 8, n_seqs * (6 * most // page + 8), page, max_rows)
    p.same()
    for i in range(6):
        new = rng.integers(0, most + 1, n_seqs) if i != 3 else np.zeros(n_seqs, np.int64)
        while new.sum() > max_rows:
            new //= 2
        assert p.step(new) == 0
        keep = np.where(rng.random(n_seqs) < 0.4, rng.integers(-1, p.cpu.lens + 2), p.cpu.lens)
        if i == 4:
            keep[:] = 0
        p.trim(keep)
    assert p.step(np.minimum(1, rng.integers(0, 2, n_seqs)) if n_seqs <= max_rows else np.zeros(n_seqs)) == 0


def test_a_step_is_taken_back_exactly(ctx):
    p = Pair(ctx, 4, 10, 40, 16, 200)
    p.step([20, 0, 7, 33])
    g = p.gpu
    before = [g.read(b).copy() for b in (g.lens, g.tables, g.free)]
    p.step([30, 1, 16, 15])
    p.trim([20, 0, 7, 33])
    after = [g.read(b) for b in (g.lens, g.tables, g.free)]
    assert np.array_equal(before[0], after[0]) and np.array_equal(before[1], after[1]) and np.array_equal(before[2][:1 + before[2][0]], after[2][:1 + after[2][0]])
    p.step([30, 1, 16, 15])


@pytest.mark.parametrize("new,status", [([17, 0, 1], 1), ([0, 0, 65], 2), ([40, 0, 40], 3), ([0, -1, 0], 4), ([71, 0, -5], 4), ([71, 0, 65], 3), ([0, 2 ** 31 - 1, 0], 3), ([17, 0, 50], 2)])
def test_steps_that_do_not_fit_change_nothing(ctx, new, status):
    p = Pair(ctx, 3, 4, 4, 16, 70)
    p.step([16, 0, 30])
    assert p.step(new) == status
    assert p.gpu.status() == status
    p.step([0, 1, 2])
    ctx.synchronize()


def test_lengths_outside_the_table_are_refused(ctx):
    p = Pair(ctx, 3, 4, 20, 16, 70)
    p.step([5, 5, 5])
    ctx.write_buffer(p.gpu.lens, np.array([5, -7, 65], np.int32))
    p.cpu.lens[:] = [5, -7, 65]
    assert p.step([1, 1, 1]) == 4
    p.eng.pages_trim(ctx, p.gpu, ints(ctx, [0, 0, 0]))    # the sound one goes, the others stay and are named
    with pytest.raises(KsError) as e:
        ctx.synchronize()
    assert e.value.code == _lib.ERR_INVALID and "rows of a sequence" in e.value.msg
    assert p.gpu.read(p.gpu.lens).tolist() == [0, -7, 65]
    ctx.synchronize()


def test_a_captured_step_serves_every_count(ctx):
    p = Pair(ctx, 6, 12, 60, 16, 64)
    new = ints(ctx, [0] * 6)
    ctx.graph_begin()
    p.eng.pages_step(ctx, p.gpu, new)
    g = ctx.graph_end()
    rng = np.random.default_rng(8)
    for _ in range(5):
        n = rng.integers(0, 10, 6)
        ctx.write_buffer(new, n.astype(np.int32))
        ctx.graph_launch(g)
        p.cpu.step(n)
        p.same()
    ctx.graph_free(g)


# ---- appends ---------------------------------------------------------------------------------------------

def hard_rows(rng, shape, act):
    """Values of many sizes with infinities, NaN, zeros and rows of nothing but those."""
    x = rng.normal(0, 1, shape) * 10.0 ** rng.uniform(-2, 2, shape[:2] + (1,))
    x[rng.random(shape) < 0.01] = 0.0
    x = x.astype(NP[act])
    for bad in (np.inf, -np.inf, np.nan):
        x[rng.random(shape) < 0.002] = bad
    if shape[0] > 4:
        x[1], x[3, 0] = 0.0, np.nan
    return x


class CachePair:
    def __init__(self, ctx, n_pages, page, n_kv, hd, fmt):
        self.ctx = ctx
        self.gpu, self.cpu = Q8Cache(ctx, n_pages, page, n_kv, hd, fmt), ref.Cache(n_pages, page, n_kv, hd, fmt)
        rng = np.random.default_rng(5)
        for b, c in ((self.gpu.k, self.cpu.codes[0]), (self.gpu.v, self.cpu.codes[1])):   # what nobody writes stays
            c[:] = rng.integers(0, 256, c.shape)
            ctx.write_buffer(b, c)
        for b, c in ((self.gpu.k_scale, self.cpu.scales[0]), (self.gpu.v_scale, self.cpu.scales[1])):
            c[:] = 2.0 ** rng.integers(-9, 9, c.shape)
            ctx.write_buffer(b, c.astype(np.float32))

    def read(self):
        g, c = self.gpu, self.cpu
        return ([self.ctx.read_bytes(b).reshape(c.codes[0].shape) for b in (g.k, g.v)], [self.ctx.read_f32(b, c.scales[0].size).reshape(c.scales[0].shape) for b in (g.k_scale, g.v_scale)])

    def same(self):
        codes, scales = self.read()
        for w in range(2):
            assert np.array_equal(scales[w], self.cpu.scales[w])
            # -0 is the same number as 0
            a, b = ref.decode(codes[w], self.cpu.fmt), ref.decode(self.cpu.codes[w], self.cpu.fmt)
            assert np.array_equal(a, b)


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("fmt", [I8, E4M3])
@pytest.mark.parametrize("page,n_kv,hd", [(16, 1, 256), (32, 3, 64), (64, 2, 128), (128, 2, 256)])
def test_append_is_exact(ctx, act, fmt, page, n_kv, hd):
    """Codes and scales equal to the definition's over several steps: pages begun, continued, grown past, rows behind the last left alone."""
    rng = np.random.default_rng(page + hd)
    p = Pair(ctx, 4, 6, 24, page, 3 * page + 7)
    c = CachePair(ctx, 24, page, n_kv, hd, fmt)
    eng = Eng(act)
    for i, new in enumerate(([page + 5, 1, 0, 3], [1, 1, 1, 1], [0, 0, 2 * page + 1, 2], [3, page - 1, 0, 11], [0, 0, 0, 0], [1, 1, 1, page])):
        p.step(new)
        k, v = (hard_rows(rng, (p.cpu.max_rows, n_kv, hd), act) * NP[act](0.5 ** i if i % 2 else 1) for _ in range(2))
        eng.kv_append_q8(ctx, c.gpu, p.gpu, ctx.buffer_bytes(k), ctx.buffer_bytes(v))
        c.cpu.append(p.cpu, k, v)
        c.same()
        eng.kv_append_q8(ctx, c.gpu, p.gpu, ctx.buffer_bytes(k), ctx.buffer_bytes(v))   # again: the same answer
        c.same()
    ctx.synchronize()


def test_append_of_ragged_rows_out_of_a_wider_buffer(ctx):
    """Rows that lie in a stacked q|k|v buffer: offsets and a row distance."""
    rng = np.random.default_rng(1)
    page, n_kv, hd, rows = 32, 2, 64, 50
    p, c = Pair(ctx, 3, 4, 9, page, rows), CachePair(ctx, 9, page, n_kv, hd, I8)
    ld = 3 * n_kv * hd + 24
    x = rng.normal(0, 1, (rows, ld)).astype(np.float16)
    p.step([31, 0, 19])
    b = ctx.buffer_bytes(x)
    Eng(F16).kv_append_q8(ctx, c.gpu, p.gpu, b, b, 128, 264, ld)
    c.cpu.append(p.cpu, x[:, 128:256].reshape(rows, n_kv, hd), x[:, 264:392].reshape(rows, n_kv, hd))
    c.same()


def test_scales_at_the_ends_of_their_range(ctx):
    p, c = Pair(ctx, 3, 2, 4, 16, 8), CachePair(ctx, 4, 16, 1, 64, E4M3)
    x = np.zeros((8, 1, 64), np.float32)
    x[0, 0, :3] = 1e-45, -3e-39, 1e-33
    x[1, 0, :3] = 3e38, -1e30, 1.0
    x[2, 0, :3] = 448.0, 449.0, -0.001
    for _ in range(2):
        p.step([1, 1, 1])
        Eng().kv_append_q8(ctx, c.gpu, p.gpu, ctx.buffer_bytes(x), ctx.buffer_bytes(-x))
        c.cpu.append(p.cpu, x, -x)
        c.same()


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("fmt", [I8, E4M3])
@pytest.mark.parametrize("n_q,n_kv,hd,page", [(8, 1, 256, 64), (6, 3, 128, 16), (4, 4, 64, 32)])
def test_norm_append(ctx, act, fmt, n_q, n_kv, hd, page):
    """Behind norm and RoPE the values carry f32 roundings (2^-20 of the row's largest covers the norm's sum of 256 and the handful of
    products behind it), so a code may be the neighbour where its value lies that near the middle of two; q as its type rounds it."""
    rng = np.random.default_rng(hd + page)
    p, c = Pair(ctx, 3, 5, 15, page, 90), CachePair(ctx, 15, page, n_kv, hd, fmt)
    eng, eps, rows = Eng(act), 1e-6, 90
    ang = np.arange(5 * page)[:, None] * 1e4 ** (-np.arange(hd // 2) * 2 / hd)
    rope = np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float32)
    qw, kw = (rng.normal(1, 0.2, hd).astype(NP[act]) for _ in range(2))
    for new in ([40, 1, 3], [1, 1, 1], [7, 0, page + 2]):
        p.step(new)
        q, k, v = (rng.normal(0, 3, (rows, n, hd)).astype(NP[act]) for n in (n_q, n_kv, n_kv))
        n = len(p.cpu.rows)
        q[n:], k[n:], v[n:] = np.nan, np.nan, np.nan
        q_out = ctx.buffer_bytes(np.full(q.shape, 7, NP[act]))
        eng.rmsnorm_per_head_qkv_q8(ctx, c.gpu, p.gpu, n_q, eps, ctx.buffer_bytes(q), ctx.buffer_bytes(qw), ctx.buffer_bytes(rope), ctx.buffer_bytes(k), ctx.buffer_bytes(kw), ctx.buffer_bytes(v), q_out)
        cs = rope[[r[1] for r in p.cpu.rows]].astype(np.float64)
        want = ref.norm_rope(q[:n], qw, cs, eps)
        got = ctx.read_act(q_out, q.size, act).reshape(q.shape)
        big = np.abs(want).max(-1, keepdims=True)
        assert (np.abs(got[:n] - want) <= 2.0 ** -20 * big + (np.abs(want) * 2.0 ** -11 + 2.0 ** -25 if act == F16 else 0)).all()
        assert (got[n:] == 7).all()
        rows_of = [np.zeros((rows, n_kv, hd)) for _ in range(2)]
        rows_of[0][:n], rows_of[1][:n] = ref.norm_rope(k[:n], kw, cs, eps), ref.norm_rope(v[:n], None, None, eps)
        before = [x.copy() for x in c.cpu.codes], [x.copy() for x in c.cpu.scales]
        c.cpu.append(p.cpu, *rows_of)
        codes, scales = c.read()
        for w in range(2):
            assert np.array_equal(scales[w], c.cpu.scales[w])     # (no maximum of these seeds lies within 2^-20 of a power of two times qmax)
            for row, m, slot, _ in p.cpu.jobs:
                pg, off = divmod(int(slot), page)
                for h in range(n_kv):
                    y = rows_of[w][row:row + m, h] / c.cpu.scales[w][pg, h]
                    got = ref.decode(codes[w][pg, h, off:off + m], fmt)
                    step = 1.0 if fmt == I8 else np.exp2(np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6))) - 3)
                    assert (np.abs(got - y) <= 0.5 * step + 2.0 ** -20 * np.abs(y).max(-1, keepdims=True)).all()
                    if fmt == I8 and off:   # what was there: exact
                        assert np.array_equal(codes[w][pg, h, :off], c.cpu.codes[w][pg, h, :off])
            touched = {int(j[2]) // page for j in p.cpu.jobs}
            rest = [x for x in range(15) if x not in touched]
            assert np.array_equal(codes[w][rest], before[0][w][rest])
            c.cpu.codes[w][:] = codes[w]
    ctx.synchronize()


def test_rope_table_too_short_for_a_row(ctx):
    p, c = Pair(ctx, 2, 4, 8, 16, 40), CachePair(ctx, 8, 16, 1, 64, I8)
    p.step([20, 4])
    x = np.ones((40, 1, 64), np.float32)
    w, rope = np.ones(64, np.float32), np.zeros((10, 64), np.float32)
    out = ctx.buffer_bytes(np.full(x.shape, 7, np.float32))
    Eng().rmsnorm_per_head_qkv_q8(ctx, c.gpu, p.gpu, 1, 1e-6, *(ctx.buffer_bytes(b) for b in (x, w, rope, x, w, x)), out)
    with pytest.raises(KsError) as e:
        ctx.synchronize()
    assert "RoPE" in e.value.msg
    got = ctx.read_f32(out, x.size).reshape(40, 64)
    assert (got[:10] == 0).all() and (got[10:20] == 7).all() and (got[20:24] == 0).all() and (got[24:] == 7).all()


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("fmt", [I8, E4M3])
@pytest.mark.parametrize("page,n_kv,hd", [(16, 3, 64), (64, 1, 128), (128, 2, 256)])
def test_read_back(ctx, act, fmt, page, n_kv, hd):
    c = CachePair(ctx, 5, page, n_kv, hd, fmt)
    rng = np.random.default_rng(2)
    if fmt == I8:   # -128 is no code of an append; it reads as what it says
        c.cpu.codes[0][0, 0, 0, 0] = 128
        ctx.write_buffer(c.gpu.k, c.cpu.codes[0])
    slots = rng.integers(0, 5 * page, 77)
    slots[[3, 40]] = -1
    out = [ctx.buffer_bytes(np.full((77, n_kv, hd), 3, NP[act])) for _ in range(2)]
    Eng(act).kv_read_q8(ctx, c.gpu, 77, ints(ctx, np.concatenate([[0, 0], slots])), 2, *out)
    for w in range(2):
        got = ctx.read_act(out[w], 77 * n_kv * hd, act).reshape(77, n_kv, hd)
        want = ref.decode(c.cpu.codes[w], fmt)[slots // page, :, slots % page] * c.cpu.scales[w][slots // page][:, :, None]
        want[slots < 0] = 3
        with np.errstate(over="ignore"):
            assert np.array_equal(got, want.astype(NP[act]).astype(np.float32))
    ctx.synchronize()


def test_bad_slots_and_pages_are_named(ctx):
    c = CachePair(ctx, 5, 16, 1, 64, I8)
    out = [ctx.buffer_bytes(np.full((3, 64), 3, np.float32)) for _ in range(2)]
    Eng().kv_read_q8(ctx, c.gpu, 3, ints(ctx, [80, -2, 5]), 0, *out)
    with pytest.raises(KsError) as e:
        ctx.synchronize()
    assert e.value.code == _lib.ERR_INVALID and "slot" in e.value.msg
    assert (ctx.read_f32(out[0], 128) == 3).all()
    p = Pair(ctx, 2, 3, 5, 16, 20)
    p.step([5, 3])
    ctx.write_buffer(p.gpu.tables, np.array([7, -1, -1, 1, -1, -1], np.int32))
    p.eng.pages_step(ctx, p.gpu, ints(ctx, [1, 1]))
    q = np.ones((20, 1, 64), np.float32)
    Eng().kv_append_q8(ctx, c.gpu, p.gpu, ctx.buffer_bytes(q), ctx.buffer_bytes(q))
    with pytest.raises(KsError) as e:
        ctx.synchronize()
    assert "page id" in e.value.msg and "slot" in e.value.msg
    o = ctx.buffer_empty_f32(q.size)
    tmp = ctx.buffer_empty_f32(p.eng.sdpa_paged_tmp_floats(ctx, c.gpu, p.gpu, 1, 1))
    Eng().sdpa_paged_q8(ctx, c.gpu, p.gpu, 1, 1, 40, ctx.buffer_bytes(q), tmp, o)
    with pytest.raises(KsError) as e:
        ctx.synchronize()
    assert "page id" in e.value.msg
    ctx.synchronize()


# ---- attention -------------------------------------------------------------------------------------------

def fill(ctx, rng, n_pages, page, n_kv, hd, fmt, wild=False):
    """A cache of values of about one; wild: scales of very different sizes."""
    c = CachePair(ctx, n_pages, page, n_kv, hd, fmt)
    for w, (b, s) in enumerate(((c.gpu.k, c.gpu.k_scale), (c.gpu.v, c.gpu.v_scale))):
        unit = 32.0 if fmt == I8 else 110.0
        c.cpu.codes[w][:] = ref.encode(rng.normal(0, unit, c.cpu.codes[w].shape), fmt)
        c.cpu.scales[w][:] = (rng.uniform(0.6, 1.4, c.cpu.scales[w].shape) / unit * (2.0 ** rng.integers(-20, 20, c.cpu.scales[w].shape) if wild and w else 1)).astype(np.float32)
        ctx.write_buffer(b, c.cpu.codes[w])
        ctx.write_buffer(s, c.cpu.scales[w].astype(np.float32))
    return c


def run_attention(ctx, rng, lens, rows, page, n_q, n_kv, hd, act, fmt, window=0, wild=False, scale=None, poison=True, slack=0, qs=1.0):
    """Outputs of the plan's rows against 64 bits.

    Tolerance.  f32: q and the probabilities enter as two f16 terms (2^-22 of the row's, each value's, largest) and sums run in f32, so a score is
    off by d <= 2^-19 max_j sum_d |q_d k_jd| scale at most and a probability by e^2d; the sums of p v add as much again.  f16: the probabilities
    and the result are rounded to f16 (2^-11 each), tensor-core sums drop up to 2^-15 of their terms over a long context."""
    scale = hd ** -0.5 if scale is None else scale
    n = len(lens)
    blocks = [-(-t // page) for t in lens]
    n_pages = sum(blocks) + 3
    p = Pair(ctx, n, max(blocks) + 1, n_pages, page, sum(rows) + 3)
    perm = rng.permutation(n_pages)
    tables = np.full((n, max(blocks) + 1), -1, np.int64)
    at = 0
    for s, b in enumerate(blocks):
        tables[s, :b] = perm[at:at + b]
        at += b
    ctx.write_buffer(p.gpu.tables, tables.astype(np.int32))
    ctx.write_buffer(p.gpu.lens, np.array(lens, np.int32))
    start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    ctx.write_buffer(p.gpu.plan, start, 4 * p.gpu.plan_part(0))
    c = fill(ctx, rng, n_pages, page, n_kv, hd, fmt, wild)
    if poison:   # what no row may see: pages of nobody, the ends of last pages
        for w, (b, s) in enumerate(((c.gpu.k, c.gpu.k_scale), (c.gpu.v, c.gpu.v_scale))):
            codes = c.cpu.codes[w].copy()
            scales = c.cpu.scales[w].astype(np.float32)
            codes[perm[at:]], scales[perm[at:]] = 0x7F, np.nan
            for i, t in enumerate(lens):
                if t % page:
                    codes[tables[i, blocks[i] - 1], :, t % page:] = 0x7F
            ctx.write_buffer(b, codes)
            ctx.write_buffer(s, scales)
    total = sum(rows)
    q = (rng.normal(0, 1, (p.cpu.max_rows, n_q, hd)) * qs).astype(NP[act])
    q[total:] = np.nan
    out = ctx.buffer_bytes(np.full(q.shape, 5, NP[act]))
    eng = Eng(act)
    most = max(rows)
    tmp = ctx.buffer_bytes(np.full(eng.sdpa_paged_tmp_floats(ctx, c.gpu, p.gpu, n_q, most) + 4, np.nan, np.float32))
    eng.sdpa_paged_q8(ctx, c.gpu, p.gpu, n_q, most, max(lens) + slack, ctx.buffer_bytes(q), tmp, out, scale, window)
    ctx.synchronize()
    got = ctx.read_act(out, q.size, act).reshape(q.shape).astype(np.float64)
    assert (got[total:] == 5).all()
    for s in range(n):
        if rows[s] == 0:
            continue
        x = q[start[s]:start[s + 1]].astype(np.float64)
        want, spread, weight = ref.attention(c.cpu, tables[s], lens[s], rows[s], x, scale, window)
        d = 2.0 ** -19 * spread[..., None]
        if act == F32:
            tol = weight * (2 * d + 2.0 ** -18) + 1e-30
        else:
            tol = weight * (2 * d + 2.0 ** -11 + 2.0 ** -15) + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
        err = np.abs(got[start[s]:start[s + 1]] - want)
        assert (err <= tol).all(), (s, lens[s], rows[s], float((err / tol).max()), np.argwhere(err > tol)[:3].tolist())
    return got


HEADS = [(8, 1, 256), (8, 2, 256), (16, 4, 128), (3, 1, 64), (4, 4, 128)]


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("fmt", [I8, E4M3])
@pytest.mark.parametrize("n_q,n_kv,hd", HEADS)
def test_attention_of_single_rows(ctx, act, fmt, n_q, n_kv, hd):
    """Lengths of one and around pages and tiles, an idle sequence."""
    rng = np.random.default_rng(n_q * hd)
    lens = [1, 15, 16, 17, 63, 64, 65, 9, 127, 128, 129, 700]
    rows = [1] * len(lens)
    rows[7] = 0
    for page, window in ((16, 0), (64, 0), (128, 50)):
        run_attention(ctx, rng, lens, rows, page, n_q, n_kv, hd, act, fmt, window)


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("fmt", [I8, E4M3])
@pytest.mark.parametrize("n_q,n_kv,hd", HEADS)
def test_attention_of_ragged_rows(ctx, act, fmt, n_q, n_kv, hd):
    """Drafts, prompt pieces and single tokens in one call, causal inside the piece, windows that end inside a tile."""
    rng = np.random.default_rng(n_q + hd)
    lens, rows = [200, 3, 140, 64, 1, 333, 90], [2, 3, 140, 0, 1, 33, 17]
    for page, window in ((32, 0), (16, 37), (128, 1)):
        run_attention(ctx, rng, lens, rows, page, n_q, n_kv, hd, act, fmt, window)


@pytest.mark.parametrize("act,fmt", [(F32, I8), (F16, E4M3)])
def test_attention_over_long_contexts(ctx, act, fmt):
    rng = np.random.default_rng(4)
    run_attention(ctx, rng, [9000, 70, 4097, 1], [1, 1, 2, 1], 64, 8, 2, 256, act, fmt)
    run_attention(ctx, rng, [5000, 300], [1, 5], 16, 16, 1, 128, act, fmt, window=1500)
    run_attention(ctx, rng, [3000], [257], 64, 4, 2, 128, act, fmt)
    run_attention(ctx, rng, [1300, 900], [300, 1], 64, 8, 1, 256, act, fmt, window=700)


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("rows", [1, 40])
def test_attention_scales_far_apart(ctx, act, rows):
    """V scales from 2^-20 to 2^20 beside one another: what carries the sum is exact wherever it lies."""
    rng = np.random.default_rng(6)
    run_attention(ctx, rng, [300, 77], [rows, 1], 16, 8, 2, 128, act, I8 if rows == 1 else E4M3, wild=act == F32, scale=0.5)


def test_attention_of_large_and_small_queries(ctx):
    """f32 queries beyond f16's range and far below it."""
    rng = np.random.default_rng(7)
    for qs in (1e6, 1e-6):
        for rows in (1, 60):
            run_attention(ctx, rng, [200, 60], [rows, 1], 32, 8, 2, 256, F32, I8, scale=0.01 / qs, qs=qs)


def test_more_query_heads_than_a_tile(ctx):
    rng = np.random.default_rng(9)
    for act in (F32, F16):
        run_attention(ctx, rng, [100, 260], [1, 2], 32, 40, 1, 64, act, I8)
        run_attention(ctx, rng, [100, 260], [1, 7], 32, 64, 1, 128, act, E4M3)
        run_attention(ctx, rng, [100, 2, 260], [50, 2, 7], 16, 10, 2, 64, act, I8)


def test_many_sequences(ctx):
    rng = np.random.default_rng(10)
    lens = rng.integers(1, 90, 1024).tolist()
    run_attention(ctx, rng, lens, [1] * 1024, 16, 2, 1, 64, F16, I8)
    rows = [int(min(t, r)) for t, r in zip(lens, rng.integers(0, 4, 1024))]
    run_attention(ctx, rng, lens, rows, 32, 2, 1, 64, F32, E4M3)


def test_rows_that_see_nothing_are_zero(ctx):
    """More rows than positions: those before position 0 have nothing to see; a length of 0 the same."""
    rng = np.random.default_rng(11)
    for rows in ([1, 5], [20, 70]):
        got = run_attention(ctx, rng, [0, 3], rows, 16, 4, 2, 128, F32, I8)
        assert (got[:rows[0] + rows[1] - 3] == 0).all()


def test_sequences_of_more_rows_than_announced_are_left_out(ctx):
    p, c = Pair(ctx, 2, 4, 8, 16, 40), CachePair(ctx, 8, 16, 1, 64, I8)
    p.step([30, 2])
    for most in (2, 29):
        q = np.ones((40, 2, 64), np.float32)
        out = ctx.buffer_bytes(np.full(q.shape, 7, np.float32))
        tmp = ctx.buffer_empty_f32(p.eng.sdpa_paged_tmp_floats(ctx, c.gpu, p.gpu, 2, most))
        Eng().sdpa_paged_q8(ctx, c.gpu, p.gpu, 2, most, 30, ctx.buffer_bytes(q), tmp, out)
        with pytest.raises(KsError) as e:
            ctx.synchronize()
        assert "rows of a sequence" in e.value.msg
        got = ctx.read_f32(out, q.size).reshape(q.shape)
        assert (got[:30] == 7).all() and (got[30:32] != 7).all() and (got[32:] == 7).all()


@pytest.mark.parametrize("lens,rows", [([3000, 900, 17], [1, 1, 1]), ([700, 64], [64, 1])])
def test_attention_repeats_bit_for_bit(ctx, lens, rows):
    a, b = (run_attention(ctx, np.random.default_rng(12), lens, rows, 32, 8, 2, 256, F32, I8) for _ in range(2))
    assert np.array_equal(a, b)


def test_caches_of_more_than_4_gb(ctx):
    """Pages whose byte offsets pass 32 bits: append, read back and attention, few rows and many."""
    page, n_kv, hd = 128, 4, 256
    n_pages = (1 << 32) // (page * n_kv * hd) + 40
    rng = np.random.default_rng(13)
    gpu = Q8Cache(ctx, n_pages, page, n_kv, hd, I8)
    p = Pair(ctx, 2, 3, n_pages, page, 300)
    stack = np.concatenate([[n_pages], rng.permutation(n_pages - 20), np.arange(n_pages - 20, n_pages)]).astype(np.int32)   # the last pages come first
    ctx.write_buffer(p.gpu.free, stack)
    p.cpu.stack = stack[1:].tolist()
    c = ref.Cache(8, page, n_kv, hd, I8)
    eng = Eng()
    for new in ([260, 9], [1, 30]):
        p.step(new)
        k, v = (rng.normal(0, 1, (300, n_kv, hd)).astype(np.float32) for _ in range(2))
        eng.kv_append_q8(ctx, gpu, p.gpu, ctx.buffer_bytes(k), ctx.buffer_bytes(v))
        pages = sorted(set(p.cpu.tables[p.cpu.tables >= 0].tolist()))
        near = {x: i for i, x in enumerate(pages)}          # the same pages in a small cache
        jobs, p.cpu.jobs = p.cpu.jobs, [[r, n, near[s // page] * page + s % page, q] for r, n, s, q in p.cpu.jobs]
        c.append(p.cpu, k, v)
        p.cpu.jobs = jobs
        n = len(p.cpu.rows)
        back = [ctx.buffer_empty_f32(300 * n_kv * hd) for _ in range(2)]
        eng.kv_read_q8(ctx, gpu, n, p.gpu.plan, p.gpu.row_slot, *back)
        slots = np.array([near[s // page] * page + s % page for _, _, s in p.cpu.rows])
        for w in range(2):
            want = ref.decode(c.codes[w], I8)[slots // page, :, slots % page] * c.scales[w][slots // page][:, :, None]
            assert np.array_equal(ctx.read_f32(back[w], n * n_kv * hd).reshape(want.shape), want)
        q = rng.normal(0, 1, (300, 8, hd)).astype(np.float32)
        out, most = ctx.buffer_empty_f32(q.size), max(new)
        tmp = ctx.buffer_empty_f32(eng.sdpa_paged_tmp_floats(ctx, gpu, p.gpu, 8, most))
        eng.sdpa_paged_q8(ctx, gpu, p.gpu, 8, most, 300, ctx.buffer_bytes(q), tmp, out, hd ** -0.5)
        got = ctx.read_f32(out, q.size).reshape(q.shape).astype(np.float64)
        for s in range(2):
            a, b = p.cpu.row_start[s:s + 2]
            table = [near.get(x, 0) for x in p.cpu.tables[s]]
            want, spread, weight = ref.attention(c, table, int(p.cpu.lens[s]), int(b - a), q[a:b].astype(np.float64), hd ** -0.5, 0)
            assert (np.abs(got[a:b] - want) <= weight * (2.0 ** -18 * spread[..., None] + 2.0 ** -18)).all()
    ctx.synchronize()


@pytest.mark.parametrize("hint", [1, 64, 1 << 20])
def test_the_announced_context_is_a_hint(ctx, hint):
    """A context longer or shorter than announced: the same answers."""
    rng = np.random.default_rng(14)
    for rows in ([1, 2, 1], [40, 1, 300], [300, 90, 17]):
        run_attention(ctx, rng, [900, 130, 700], rows, 32, 8, 2, 128, F16, I8, slack=hint - 900)
    run_attention(ctx, rng, [900], [150], 16, 4, 1, 256, F32, E4M3, slack=hint - 900)


@pytest.mark.parametrize("hint", [1, 1 << 20])
@pytest.mark.parametrize("act,fmt", [(F32, E4M3), (F16, I8)])
@pytest.mark.parametrize("n_q,n_kv,hd", HEADS)
def test_pieces_of_rows_by_either_kernel(ctx, act, fmt, n_q, n_kv, hd, hint):
    """Short contexts announced: the kernel of few rows takes up to 512 (row, head) pairs of a sequence; long ones: up to 32."""
    rng = np.random.default_rng(n_q + hd + hint % 7)
    G = n_q // n_kv
    lens, rows = [200, 3, 140, 64, 1, 333, 90], [2, 3, 140, 0, 1, 33, 17]
    for page, window in ((32, 0), (16, 37), (128, 1)):
        run_attention(ctx, rng, lens, rows, page, n_q, n_kv, hd, act, fmt, window, slack=hint - max(lens))
    for many in (32 // G, 32 // G + 1, 512 // G, 512 // G + 1):
        run_attention(ctx, rng, [many + 70], [many], 64, n_q, n_kv, hd, act, fmt, 0, slack=hint - many - 70)
        run_attention(ctx, rng, [many + 270, 77], [many, 1], 16, n_q, n_kv, hd, act, fmt, 100, slack=hint - many - 270)


def test_negative_and_zero_scales(ctx):
    rng = np.random.default_rng(15)
    for scale in (-0.1, 0.0):
        for rows in ([1, 3], [90, 60]):
            run_attention(ctx, rng, [200, 70], rows, 32, 4, 2, 128, F32, I8, scale=scale)
            run_attention(ctx, rng, [200, 70], rows, 16, 4, 2, 64, F16, E4M3, scale=scale)


# ---- together --------------------------------------------------------------------------------------------

@pytest.fixture(scope="module")
def early(ctx):
    """A context whose kernels may start while their predecessors run."""
    c = CudaContext(0, 1)
    yield c
    c.close()


def test_calls_back_to_back_that_start_early(ctx, early):
    """Steps, appends and mixed attention enqueued many times over with nothing in between, plainly and as a captured graph: bit for bit what a
    context without early starts gets, call by call."""
    got = []
    for c, waits in ((ctx, True), (early, False)):
        rng = np.random.default_rng(40)
        n_q, n_kv, hd, page, T = 8, 2, 128, 32, 300
        eng, tables = Eng(F16), PageTables(c, 4, 20, 80, page, T)
        cache = Q8Cache(c, 80, page, n_kv, hd, I8)
        k, v, q = (c.buffer_bytes(rng.normal(0, 1, (T, n, hd)).astype(np.float16)) for n in (n_kv, n_kv, n_q))
        new = [ints(c, x) for x in ([150, 1, 0, 40], [1, 1, 1, 1], [2, 130, 1, 0])]
        keep = ints(c, [0, 0, 0, 0])
        outs = [[c.buffer_bytes(np.zeros((T, n_q, hd), np.float16)) for _ in range(3)] for _ in range(6)]
        tmp = c.buffer_empty_f32(eng.sdpa_paged_tmp_floats(c, cache, tables, n_q, 150))

        def go(out):
            eng.pages_trim(c, tables, keep)
            for step in range(3):
                eng.pages_step(c, tables, new[step])
                eng.kv_append_q8(c, cache, tables, k, v)
                eng.sdpa_paged_q8(c, cache, tables, n_q, 150, 400, q, tmp, out[step], hd ** -0.5)
                if waits:
                    c.synchronize()

        for out in outs[:4]:
            go(out)
        if not waits:
            c.graph_begin()
            go(outs[4])
            g = c.graph_end()
            for _ in range(20):
                c.graph_launch(g)
        go(outs[5])
        c.synchronize()
        got.append([c.read_bytes(b) for out in (outs[:4] + outs[5:] if waits else outs) for b in out])
        if not waits:
            c.graph_free(g)
    for i, x in enumerate(got[1]):
        assert np.array_equal(x, got[0][i % 3]), i


@pytest.mark.parametrize("flags", [0, 1])
@pytest.mark.parametrize("act,fmt,window", [(F32, I8, 0), (F16, E4M3, 40)])
def test_a_decoder_steps_over_pages(ctx, early, flags, act, fmt, window):
    """Two layers over one set of tables, op by op as a host's loop runs them: prompts of three requests, single tokens, a draft that is turned
    down, a request that ends and another that takes its pages; the single-token step as one captured graph.  Every attention against
    64 bits over what the cache holds, every cache row against the norm and RoPE of what went in."""
    ctx = early if flags else ctx
    rng = np.random.default_rng(21)
    n_q, n_kv, hd, page, eps, rows_most = 8, 2, 128, 32, 1e-6, 70
    p = Pair(ctx, 3, 8, 18, page, 120)
    caches = [CachePair(ctx, 18, page, n_kv, hd, fmt) for _ in range(2)]
    eng, T = Eng(act), p.cpu.max_rows
    ang = np.arange(8 * page)[:, None] * 1e4 ** (-np.arange(hd // 2) * 2 / hd)
    rope = np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float32)
    w = rng.normal(1, 0.1, (2, 2, hd)).astype(NP[act])
    brope, bw = ctx.buffer_bytes(rope), [[ctx.buffer_bytes(w[l, i]) for i in range(2)] for l in range(2)]
    bq, bk, bv = (ctx.buffer_bytes(np.zeros((T, n, hd), NP[act])) for n in (n_q, n_kv, n_kv))
    bqo, bo = ([ctx.buffer_bytes(np.zeros((T, n_q, hd), NP[act])) for _ in range(2)] for _ in range(2))
    new_buf = ints(ctx, [0, 0, 0])
    tmp = ctx.buffer_empty_f32(max(eng.sdpa_paged_tmp_floats(ctx, caches[0].gpu, p.gpu, n_q, m) for m in (1, rows_most)))

    def enqueue(most):
        eng.pages_step(ctx, p.gpu, new_buf)
        for l in range(2):
            eng.rmsnorm_per_head_qkv_q8(ctx, caches[l].gpu, p.gpu, n_q, eps, bq, bw[l][0], brope, bk, bw[l][1], bv, bqo[l])
            eng.sdpa_paged_q8(ctx, caches[l].gpu, p.gpu, n_q, most, 8 * page, bqo[l], tmp, bo[l], hd ** -0.5, window)

    enqueue(1)     # no rows: nothing happens
    ctx.graph_begin()
    enqueue(1)
    graph = ctx.graph_end()

    def step(new, captured=False):
        q, k, v = (rng.normal(0, 1, (T, n, hd)).astype(NP[act]) for n in (n_q, n_kv, n_kv))
        for b, x in ((bq, q), (bk, k), (bv, v)):
            ctx.write_buffer(b, x)
        ctx.write_buffer(new_buf, np.array(new, np.int32))
        if captured:
            ctx.graph_launch(graph)
        else:
            enqueue(rows_most)
        assert p.cpu.step(new) == 0
        p.same()
        n = len(p.cpu.rows)
        cs = rope[[r[1] for r in p.cpu.rows]].astype(np.float64)
        for l in range(2):
            c = caches[l]
            codes, scales = c.read()
            for which in range(2):
                c.cpu.codes[which][:], c.cpu.scales[which][:] = codes[which], scales[which]
            x = ref.norm_rope(k[:n], w[l, 1], cs, eps)
            for r, (_, _, slot) in enumerate(p.cpu.rows):
                held = ref.decode(codes[0][slot // page, :, slot % page], fmt) * scales[0][slot // page][:, None]
                assert (np.abs(held - x[r]) <= scales[0][slot // page][:, None] * (0.51 if fmt == I8 else 16.1)).all()
            got_q = ctx.read_act(bqo[l], T * n_q * hd, act).reshape(T, n_q, hd).astype(np.float64)
            got = ctx.read_act(bo[l], T * n_q * hd, act).reshape(T, n_q, hd).astype(np.float64)
            for s in range(3):
                a, b = p.cpu.row_start[s:s + 2]
                if a == b:
                    continue
                want, spread, weight = ref.attention(c.cpu, p.cpu.tables[s], int(p.cpu.lens[s]), int(b - a), got_q[a:b], hd ** -0.5, window)
                d = 2.0 ** -18 * spread[..., None]
                tol = weight * (d + (2.0 ** -18 if act == F32 else 2.0 ** -11 + 2.0 ** -15)) + (np.abs(want) * 2.0 ** -11 + 2.0 ** -25 if act == F16 else 0)
                assert (np.abs(got[a:b] - want) <= tol).all()

    step([70, 20, 5])
    for _ in range(4):
        step([1, 1, 1], captured=True)
    step([3, 0, 4])
    p.trim([75, -1, 10])          # drafts turned down
    step([1, 1, 1], captured=True)
    p.trim([-1, 0, -1])           # a request ends
    step([0, 60, 1])
    step([1, 1, 1], captured=True)
    ctx.synchronize()
    ctx.graph_free(graph)


def test_two_contexts_and_another_current_device_state(ctx):
    """Two contexts, each with its stream, workspace and cache, used in turn."""
    other = CudaContext(0, 1)
    got = []
    for c in (ctx, other, ctx, other):
        got.append(run_attention(c, np.random.default_rng(31), [2000, 130, 40], [1, 1, 40], 32, 8, 2, 128, F32, E4M3))
    assert all(np.array_equal(got[0], g) for g in got[1:])
    other.close()
