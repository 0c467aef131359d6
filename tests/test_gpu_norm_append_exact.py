"""Codes and scales behind norm and RoPE are those of 64 bits: rows made so that a page's maximum lies next to a limit of the scales, and values
next to the middle of two codes; infinities, NaN and products that pass f32's range."""
import numpy as np
import pytest

from ksearch_b200 import E4M3, F16, F32, I8, Eng
from tests import paged_ref as ref
from tests.test_gpu_paged_cache import NP, CachePair, Pair

EPS = float(np.float32(1e-6))
gpu = pytest.mark.gpu


def down_to(x, act):
    """The largest number of the type that x >= 0 does not fall below."""
    y = NP[act](x)
    return float(np.nextafter(y, NP[act](0))) if float(y) > x else float(y)


def fill_up(x, at, total, act):
    """Sets x[at] (zeros) one after the other so that the squares sum up to `total` from below, as near as the type has it."""
    for i in at:
        x[i] = down_to(np.sqrt(max(total - float((x ** 2).sum()), 0.0)), act)
    return x


def limit_row(rng, w, c, s, act, fmt, near):
    """A row whose largest value behind norm, weights and RoPE (half-split cos c and sin s) is qmax 2^e (1 + near)."""
    hd = w.size
    L = ref.QMAX[fmt] * (2.0 ** -7 if fmt == E4M3 else 2.0 ** -5) * (1 + near)
    m = int(rng.integers(0, hd // 2))
    turn = max(abs(c[m]), abs(s[m]))
    assert turn > 0.5
    total = hd * ((abs(float(w[m])) * turn / L) ** 2 - EPS)             # with x[m] = 1
    x = rng.uniform(-1, 1, hd)
    free = rng.permutation([i for i in range(hd) if i % (hd // 2) != m])[:5]
    x[free] = 0
    x[m] = x[m + hd // 2] = 0
    x *= np.sqrt((total - 1) * (1 - 2.0 ** -8) / (x ** 2).sum())
    x = x.astype(NP[act]).astype(np.float64)
    x[m] = 1
    return fill_up(x, free, total, act)


def middle(z, fmt):
    """The middle between the codes around z."""
    if fmt == I8:
        return np.floor(z) + 0.5
    e = np.exp2(np.floor(np.log2(np.maximum(np.abs(z), 2.0 ** -6))) - 3)
    return np.where(z < 0, -1, 1) * (np.floor(np.abs(z) / e) + 0.5) * e


def middle_row(rng, w, act, fmt, near):
    """A row of norm 1 / (1 + near) (nearly) whose values are middles between codes times that; weights are powers of two, RoPE turns by quarters."""
    hd = w.size
    s = 2.0 ** -5 if fmt == I8 else 2.0 ** -7
    total, most = hd * (1 - EPS) * (1 + near), np.sqrt(3 * (hd - 10) / (1 / w ** 2).sum())
    while True:
        free = rng.permutation(hd)[:6]
        x = middle(rng.uniform(-most, most, hd) / s, fmt) * s / w
        x[free] = 0
        x[free[0]] = 3.0 / w[free[0]]                                   # the largest: the scale is s
        if 0 < total - float((x ** 2).sum()) < 1.5:
            return fill_up(x, free[1:], total, act)


def test_rows_are_where_they_claim_to_be():
    rng = np.random.default_rng(0)
    for act in (F32, F16):
        for fmt in (I8, E4M3):
            for hd in (64, 256):
                w = rng.uniform(0.8, 1.2, hd).astype(NP[act]).astype(np.float64)
                ang = rng.uniform(0, 0.6, hd // 2)
                cs = np.concatenate([np.cos(ang), np.sin(ang)]).astype(np.float32).astype(np.float64)
                for near in (-2.0 ** -22, 2.0 ** -23):
                    x = limit_row(rng, w, cs[:hd // 2], cs[hd // 2:], act, fmt, near)
                    assert np.array_equal(x, x.astype(NP[act]))
                    y = np.abs(ref.norm_rope(x[None, None], w, cs[None], EPS)).max()
                    limit = ref.QMAX[fmt] * (2.0 ** -7 if fmt == E4M3 else 2.0 ** -5)
                    assert abs(y / limit - 1 - near) < 2.0 ** -25 and (y > limit) == (near > 0)
                    w2 = 2.0 ** rng.integers(-1, 1, hd)
                    x = middle_row(rng, w2, act, fmt, near)
                    assert np.array_equal(x, x.astype(NP[act]))
                    z = ref.norm_rope(x[None, None], w2, np.repeat([1.0, 0.0], hd // 2)[None], EPS)[0, 0] / (2.0 ** -5 if fmt == I8 else 2.0 ** -7)
                    off = np.abs(z / middle(z, fmt) - 1)
                    assert ((off < 2.0 ** -21) & (off > 2.0 ** -26)).sum() > hd // 2


def run(ctx, act, fmt, hd, n_kv, page, k, v, kw, rope, new, before=None):
    """Appends rows [n, n_kv, hd] to empty sequences; returns codes and scales of the GPU, and the restatement's with the values it rounded."""
    n, n_q = k.shape[0], 2
    p, c = Pair(ctx, len(new), 4, 4 * len(new), page, n), CachePair(ctx, 4 * len(new), page, n_kv, hd, fmt)
    p.step(new)
    eng = Eng(act)
    q, qw = np.ones((n, n_q, hd), NP[act]), np.ones(hd, NP[act])
    eng.rmsnorm_per_head_qkv_q8(ctx, c.gpu, p.gpu, n_q, EPS, *(ctx.buffer_bytes(np.ascontiguousarray(x)) for x in (q, qw, rope, k.astype(NP[act]), kw.astype(NP[act]), v.astype(NP[act]))),
                                ctx.buffer_bytes(q))
    cs = rope[[r[1] for r in p.cpu.rows]].astype(np.float64)
    with np.errstate(invalid="ignore"):
        rows = [ref.norm_rope(k.astype(NP[act]), kw.astype(NP[act]), cs, EPS), ref.norm_rope(v.astype(NP[act]), None, None, EPS)]
    if before:
        before(rows)
    c.cpu.append(p.cpu, *rows)
    got = c.read()
    ctx.synchronize()
    return p, c, rows, got


def same(p, c, rows, got, page, fmt):
    """Scales equal, and codes wherever the value is not within 2^-40 of the middle between two (64 bits do not say more)."""
    codes, scales = got
    near = 0
    for w in range(2):
        assert np.array_equal(scales[w], c.cpu.scales[w]), np.argwhere(scales[w] != c.cpu.scales[w])[:4].tolist()
        for row, m, slot, _ in p.cpu.jobs:
            pg, off = divmod(int(slot), page)
            for h in range(rows[w].shape[1]):
                z = rows[w][row:row + m, h] / c.cpu.scales[w][pg, h]
                a, b = (ref.decode(x[w][pg, h, off:off + m], fmt) for x in (codes, c.cpu.codes))
                with np.errstate(invalid="ignore"):
                    gap = np.abs(z / middle(z, fmt) - 1)
                clear = ~(gap <= 2.0 ** -40)
                near += int((gap < 2.0 ** -20).sum())
                assert np.array_equal(a[clear], b[clear]), (w, row, h, np.argwhere((a != b) & clear)[:4].tolist())
    return near


def quarter_turns(n, hd):
    c, s = np.array([1, 0, -1, 0.0])[np.arange(n) % 4], np.array([0, 1, 0, -1.0])[np.arange(n) % 4]
    return np.concatenate([np.repeat(c[:, None], hd // 2, 1), np.repeat(s[:, None], hd // 2, 1)], 1).astype(np.float32)


HEADS = [(64, 3, 16), (128, 2, 64), (256, 1, 128), (256, 2, 32)]


@gpu
@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("fmt", [I8, E4M3])
@pytest.mark.parametrize("hd,n_kv,page", HEADS)
def test_maxima_next_to_a_limit_of_the_scales(ctx, act, fmt, hd, n_kv, page):
    """Each row's maximum lies within 2^-21 of qmax 2^e, on either side of it, in pages of one row and of many."""
    rng = np.random.default_rng(hd + page)
    new = [1] * 12 + [3, page + 1, 2, 5] * 3
    ang = rng.uniform(0, 0.6, (4 * page, hd // 2))
    rope = np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float32)
    kw = rng.uniform(0.8, 1.2, hd).astype(NP[act]).astype(np.float64)
    n = sum(new)
    k, v = (np.empty((n, n_kv, hd)) for _ in range(2))
    pos = np.concatenate([np.arange(m) for m in new])
    one, none = np.ones(hd), (np.ones(hd // 2), np.zeros(hd // 2))
    for r in range(n):
        cs = rope[pos[r]].astype(np.float64)
        for h in range(n_kv):
            near = float(rng.choice([-1, 1])) * 2.0 ** -rng.uniform(21.5, 25)
            k[r, h] = limit_row(rng, kw, cs[:hd // 2], cs[hd // 2:], act, fmt, near)
            v[r, h] = limit_row(rng, one, *none, act, fmt, -near)
    p, c, rows, got = run(ctx, act, fmt, hd, n_kv, page, k, v, kw, rope, new)
    same(p, c, rows, got, page, fmt)


@gpu
@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("fmt", [I8, E4M3])
@pytest.mark.parametrize("hd,n_kv,page", HEADS)
def test_values_next_to_the_middle_of_two_codes(ctx, act, fmt, hd, n_kv, page):
    rng = np.random.default_rng(hd + page)
    new = [1, 1, 4, page, 2 * page + 1, 7]
    rope, kw, n = quarter_turns(4 * page, hd), 2.0 ** rng.integers(-1, 1, hd), sum(new)
    k, v = (np.empty((n, n_kv, hd)) for _ in range(2))
    for r in range(n):
        for h in range(n_kv):
            near = float(rng.choice([-1, 1])) * 2.0 ** -rng.uniform(21, 26)
            k[r, h] = middle_row(rng, kw, act, fmt, near)
            v[r, h] = middle_row(rng, np.ones(hd), act, fmt, -near)
    p, c, rows, got = run(ctx, act, fmt, hd, n_kv, page, k, v, kw, rope, new)
    assert same(p, c, rows, got, page, fmt) > n * n_kv * hd // 4


@gpu
@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("fmt", [I8, E4M3])
@pytest.mark.parametrize("hd,n_kv,page", HEADS)
def test_infinities_and_nan(ctx, act, fmt, hd, n_kv, page):
    """A row with NaN is NaN behind its norm, which is stored as 0; so is an infinity (infinity over infinity) and what is beside it (0).  A row whose
    squares pass f32's range counts as one with an infinity."""
    rng = np.random.default_rng(hd)
    new = [3, page + 3, 1, 9]
    n = sum(new)
    ang = rng.uniform(0, 6, (4 * page, hd // 2))
    rope = np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float32)
    kw = rng.uniform(0.8, 1.2, hd).astype(NP[act])
    k, v = (rng.normal(0, 2, (n, n_kv, hd)) for _ in range(2))
    for x in (k, v):
        for r, bad in ((0, np.nan), (4, np.inf), (5, -np.inf), (page + 3, np.nan), (page + 6, np.inf), (n - 1, np.inf)):
            x[r, r % n_kv, rng.integers(0, hd)] = bad
        if act == F32:
            x[7, 0] = 1e20
            x[8, n_kv - 1, 3] = -3e38

    def overflow(rows):
        for w in range(2):
            if act == F32:
                rows[w][7, 0], rows[w][8, n_kv - 1] = 0, 0

    p, c, rows, got = run(ctx, act, fmt, hd, n_kv, page, k, v, kw, rope, new, overflow)
    same(p, c, rows, got, page, fmt)


@gpu
@pytest.mark.parametrize("fmt", [I8, E4M3])
@pytest.mark.parametrize("hd,n_kv,page", HEADS)
def test_products_that_pass_the_range_of_f32(ctx, fmt, hd, n_kv, page):
    """A weight of 3e38: its dims and their RoPE partners become infinities, which are the largest code and do not count in the page's scale."""
    rng = np.random.default_rng(hd + 1)
    new = [3, page + 3, 1, 9]
    n, m = sum(new), 5
    ang = rng.uniform(0.2, 1.2, (4 * page, hd // 2))
    rope = np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float32)
    kw = rng.uniform(0.8, 1.2, hd).astype(np.float32)
    kw[m] = 3e38
    k, v = (rng.normal(0, 1, (n, n_kv, hd)) for _ in range(2))
    k[..., m] = rng.choice([-4.0, 4.0], (n, n_kv))
    k[..., m + hd // 2] = 1

    def overflow(rows):        # x w is 3e38 times at least 2: behind cos and sin of 0.2 to 1.2 still an infinity in f32
        for i in (m, m + hd // 2):
            rows[0][..., i] = np.sign(k[..., m]) * np.inf

    p, c, rows, got = run(ctx, F32, fmt, hd, n_kv, page, k, v, kw, rope, new, overflow)
    same(p, c, rows, got, page, fmt)
    held = ref.decode(got[0][0], fmt)
    for (_, pos, slot) in p.cpu.rows:
        assert (np.abs(held[slot // page, :, slot % page][:, [m, m + hd // 2]]) == ref.QMAX[fmt]).all()


@gpu
@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("fmt", [I8, E4M3])
@pytest.mark.parametrize("hd,n_kv,page", HEADS)
def test_pages_that_are_continued(ctx, act, fmt, hd, n_kv, page):
    """Steps that go on in a page, flat rows first and rows with a large value behind them: the scale grows, and the earlier codes are rounded again as
    the definition says."""
    rng = np.random.default_rng(hd * 3 + page)
    p, c = Pair(ctx, 3, 4, 12, page, 2 * page), CachePair(ctx, 12, page, n_kv, hd, fmt)
    eng, T = Eng(act), 2 * page
    ang = rng.uniform(0, 6, (4 * page, hd // 2))
    rope = np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float32)
    kw = rng.uniform(0.8, 1.2, hd).astype(NP[act])
    fixed = [ctx.buffer_bytes(x) for x in (np.ones((T, 1, hd), NP[act]), np.ones(hd, NP[act]), rope)]
    grown = 0
    for i, new in enumerate(([page // 2, 3, 0], [1, page // 4, 2], [2, 1, page // 2], [page // 2, 1, 1], [1, 0, page])):
        p.step(new)
        n = len(p.cpu.rows)
        k, v = (rng.uniform(-1, 1, (T, n_kv, hd)) for _ in range(2))
        if i:
            for x in (k, v):
                x[:n, :, rng.integers(0, hd)] *= 3.0 ** i
        k, v = k.astype(NP[act]), v.astype(NP[act])
        eng.rmsnorm_per_head_qkv_q8(ctx, c.gpu, p.gpu, 1, EPS, *fixed, ctx.buffer_bytes(k), ctx.buffer_bytes(kw), ctx.buffer_bytes(v), ctx.buffer_empty_bytes(4 * T * hd))
        cs = rope[[r[1] for r in p.cpu.rows]].astype(np.float64)
        rows = [ref.norm_rope(k[:n], kw, cs, EPS), ref.norm_rope(v[:n], None, None, EPS)]
        held = [s.copy() for s in c.cpu.scales]
        c.cpu.append(p.cpu, *rows)
        got = c.read()
        same(p, c, rows, got, page, fmt)
        for w in range(2):
            for _, _, slot, _ in p.cpu.jobs:
                pg, off = divmod(int(slot), page)
                assert np.array_equal(ref.decode(got[0][w][pg, :, :off], fmt), ref.decode(c.cpu.codes[w][pg, :, :off], fmt))
                grown += int(off > 0 and (c.cpu.scales[w][pg] > held[w][pg]).any())
            c.cpu.codes[w][:] = got[0][w]
    assert grown >= 4
    ctx.synchronize()
