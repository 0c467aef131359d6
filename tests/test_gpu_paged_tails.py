"""Attention over the paged 8-bit cache where probabilities and V's scales are of very different sizes, in both of its kernels: a first
position that leads by many bits in front of a flat rest, scales far apart in f16, sums over very long contexts."""
import numpy as np
import pytest

from ksearch_b200 import E4M3, F16, F32, I8, Eng
from tests import paged_ref as ref
from tests.test_gpu_paged_cache import NP, CachePair, Pair

pytestmark = pytest.mark.gpu

FEW, MANY = 1, 64       # rows of a sequence: the kernel of few rows, and (with a long context announced) the wide one


def tables_of(ctx, rng, lens, rows, page, n_pages):
    blocks = [-(-t // page) for t in lens]
    p = Pair(ctx, len(lens), max(blocks), n_pages, page, sum(rows))
    perm, tables, at = rng.permutation(n_pages), np.full((len(lens), max(blocks)), -1, np.int64), 0
    for s, b in enumerate(blocks):
        tables[s, :b] = perm[at:at + b]
        at += b
    ctx.write_buffer(p.gpu.tables, tables.astype(np.int32))
    ctx.write_buffer(p.gpu.lens, np.array(lens, np.int32))
    ctx.write_buffer(p.gpu.plan, np.concatenate([[0], np.cumsum(rows)]).astype(np.int32), 4 * p.gpu.plan_part(0))
    return p, tables


def upload(ctx, c):
    for b, x in zip((c.gpu.k, c.gpu.v, c.gpu.k_scale, c.gpu.v_scale), (*c.cpu.codes, *(s.astype(np.float32) for s in c.cpu.scales))):
        ctx.write_buffer(b, x)


def attend(ctx, p, c, n_q, act, q, most, announced, scale):
    eng = Eng(act)
    out = ctx.buffer_bytes(np.full(q.shape, 5, NP[act]))
    tmp = ctx.buffer_bytes(np.full(eng.sdpa_paged_tmp_floats(ctx, c.gpu, p.gpu, n_q, most), np.nan, np.float32))
    eng.sdpa_paged_q8(ctx, c.gpu, p.gpu, n_q, most, announced, ctx.buffer_bytes(q), tmp, out, scale)
    ctx.synchronize()
    return ctx.read_act(out, q.size, act).reshape(q.shape).astype(np.float64)


def least_that_counts(c, table, length, rows, q, scale):
    """Probabilities are stored as f16 with 2^10 in front, relative to the largest exp2(score + log2 of V's scale): one below 2^-14 of the
    format is off by 2^-25 at most, which is 2^-35 of that largest.  Over all codes, and over the sum of exponentials.  V's scales count as 2^-60
    at least in the exponent."""
    n_q, hd = q.shape[1:]
    G = n_q // c.n_kv
    off = np.zeros(q.shape)
    pages = np.asarray(table[:-(-length // c.page)])
    for h in range(c.n_kv):
        K = c.values(0, pages, h)[:length]
        codes = np.abs(ref.decode(c.codes[1][pages, h], c.fmt).reshape(-1, hd)[:length])
        vs = np.log2(np.maximum(np.repeat(c.scales[1][pages, h], c.page)[:length], 2.0 ** -60))
        for r in range(rows):
            seen = length - rows + r + 1
            for g in range(G):
                s = K[:seen] @ q[r, h * G + g] * scale * np.log2(np.e)
                top = (s + vs[:seen]).max()
                off[r, h * G + g] = 2.0 ** -35 * codes[:seen].sum(0) / np.exp2(s - top).sum()
    return off


def check(c, table, length, rows, q, scale, got, act, tiny=1e-30):
    """run_attention's tolerance (tests/test_gpu_paged_cache.py), and what the smallest probabilities add."""
    want, spread, weight = ref.attention(c, table, length, rows, q, scale, 0)
    d = 2.0 ** -19 * spread[..., None]
    tol = weight * (2 * d + (2.0 ** -18 if act == F32 else 2.0 ** -11 + 2.0 ** -15)) + (tiny if act == F32 else np.abs(want) * 2.0 ** -11 + 2.0 ** -25)
    tol = tol + least_that_counts(c, table, length, rows, q, scale)
    err = np.abs(got - want)
    assert (err <= tol).all(), (float((err / tol).max()), np.argwhere(err > tol)[:3].tolist())


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("fmt", [I8, E4M3])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows", [FEW, MANY])
def test_a_first_position_that_leads_a_flat_rest(ctx, act, fmt, hd, rows):
    """The first position leads some 8000 others by 16 to 30 bits and has a V of zero: the answer is what the others have."""
    rng = np.random.default_rng(hd + rows)
    page, n_q, length = 64, 2, 8000 + rows
    n_pages = -(-length // page)
    p, tables = tables_of(ctx, rng, [length], [rows], page, n_pages)
    c = CachePair(ctx, n_pages, page, 1, hd, fmt)
    first = tables[0, 0]
    c.cpu.codes[0][:] = 0
    c.cpu.codes[0][first, 0, 0, 0] = ref.encode(np.array(64.0), fmt)
    c.cpu.scales[0][:] = 2.0 ** -6
    unit = 32.0 if fmt == I8 else 110.0
    v = rng.normal(0, unit, c.cpu.codes[1].shape)
    v[..., ::2] = np.abs(v[..., ::2])
    c.cpu.codes[1][:] = ref.encode(v, fmt)
    c.cpu.codes[1][first, 0, 0] = 0
    c.cpu.scales[1][:] = (rng.uniform(0.6, 1.4, c.cpu.scales[1].shape) / unit).astype(np.float32)
    upload(ctx, c)
    q = rng.normal(0, 1, (rows, n_q, hd))
    q[..., 0] = 1 - np.arange(rows * n_q).reshape(rows, n_q) / 512       # leads of 3/4 of the most to all of it
    q = q.astype(NP[act])
    for lead in (22, 24, 27, 30):
        scale = float(np.float32(lead * np.log(2)))
        got = attend(ctx, p, c, n_q, act, q, rows, 1 << 20, scale)
        check(c.cpu, tables[0], length, rows, q.astype(np.float64), scale, got, act)


@pytest.mark.parametrize("fmt", [I8, E4M3])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows", [FEW, MANY])
def test_v_scales_far_apart_in_f16(ctx, fmt, hd, rows):
    """V scales from 2^-30 to 2^7 beside one another: what carries the sum counts wherever it lies."""
    rng = np.random.default_rng(hd * 2 + rows)
    page, n_q, n_kv, lens, n_rows = 16, 4, 2, [300, 77], [rows, 1]
    n_pages = sum(-(-t // page) for t in lens)
    p, tables = tables_of(ctx, rng, lens, n_rows, page, n_pages)
    c = CachePair(ctx, n_pages, page, n_kv, hd, fmt)
    unit = 32.0 if fmt == I8 else 110.0
    for w in range(2):
        c.cpu.codes[w][:] = ref.encode(rng.normal(0, unit, c.cpu.codes[w].shape), fmt)
        far = 2.0 ** rng.integers(-30, 8, c.cpu.scales[w].shape) if w else 1.0
        c.cpu.scales[w][:] = (rng.uniform(0.6, 1.4, c.cpu.scales[w].shape) / unit * far).astype(np.float32)
    upload(ctx, c)
    q = rng.normal(0, 1, (sum(n_rows), n_q, hd)).astype(np.float16)
    got = attend(ctx, p, c, n_q, F16, q, rows, 1 << 20, 0.5)
    check(c.cpu, tables[0], lens[0], rows, q[:rows].astype(np.float64), 0.5, got[:rows], F16)
    check(c.cpu, tables[1], lens[1], 1, q[rows:].astype(np.float64), 0.5, got[rows:], F16)


@pytest.mark.parametrize("n_q,hd,rows", [(16, 128, 4096), (8, 256, 2048)])
def test_flat_sums_over_131072_positions(ctx, n_q, hd, rows):
    """Values of one sign and scores that are nearly alike, 131072 positions, enough rows that a block sums tens of thousands of them: single
    rows of the result against 64 bits."""
    rng = np.random.default_rng(hd)
    page, length = 128, 131072
    n_pages = length // page
    p, tables = tables_of(ctx, rng, [length], [rows], page, n_pages)
    c = CachePair(ctx, n_pages, page, 1, hd, E4M3)
    c.cpu.codes[0][:] = ref.encode(rng.normal(0, 110, c.cpu.codes[0].shape), E4M3)
    c.cpu.codes[1][:] = ref.encode(np.abs(rng.normal(0, 110, c.cpu.codes[1].shape)), E4M3)
    for w in range(2):
        c.cpu.scales[w][:] = (rng.uniform(0.6, 1.4, c.cpu.scales[w].shape) / 110.0).astype(np.float32)
    upload(ctx, c)
    q = rng.normal(0, 1, (rows, n_q, hd)).astype(np.float16)
    scale = 0.1 * hd ** -0.5
    got = attend(ctx, p, c, n_q, F16, q, rows, length, scale)
    K, V = (c.cpu.values(w, tables[0], 0) for w in range(2))
    for r, g in ((0, 0), (rows // 3, n_q - 1), (rows - 2, 1), (rows - 1, n_q // 2)):
        seen = length - rows + r + 1
        x = q[r, g].astype(np.float64)
        w = np.exp(K[:seen] @ x * scale)
        want = w @ V[:seen] / w.sum()
        d = 2.0 ** -19 * (np.abs(K[:seen]) @ np.abs(x)).max() * scale
        assert (np.abs(got[r, g] - want) <= want * (2 * d + 2.0 ** -11 + 2.0 ** -15 + 2.0 ** -11)).all(), (r, g, float((np.abs(got[r, g] - want) / want).max()), float(((got[r, g] - want) / want).mean()))


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("fmt", [I8, E4M3])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows", [FEW, MANY])
def test_pages_of_zeros_beside_large_values(ctx, act, fmt, hd, rows):
    """One page of large V among pages whose V is all zero, which an append gives the least scale, 2^-100: the zeros' probabilities count in full.
    f32: values of some 2^35; f16: up to the format's end.  The large page leads by 0 to 18 bits, so that its 16 positions have from 1/128
    to 99 % of the sum."""
    rng = np.random.default_rng(hd + 3 * rows)
    page, n_q, length = 16, 2, 2048 + rows
    n_pages = -(-length // page)
    p, tables = tables_of(ctx, rng, [length], [rows], page, n_pages)
    c = CachePair(ctx, n_pages, page, 1, hd, fmt)
    large = tables[0, 3]
    c.cpu.codes[0][:] = 0
    c.cpu.codes[0][large, 0, :, 0] = ref.encode(np.array(64.0), fmt)
    c.cpu.scales[0][:] = 2.0 ** -6
    c.cpu.codes[1][:] = 0
    c.cpu.scales[1][:] = 2.0 ** -100
    c.cpu.codes[1][large, 0] = ref.encode(np.abs(rng.normal(0, 16, (page, hd))).clip(1, 60), fmt)
    c.cpu.scales[1][large, 0] = 2.0 ** 30 if act == F32 else 2.0 ** 10
    upload(ctx, c)
    q = rng.normal(0, 1, (rows, n_q, hd))
    q[..., 0] = 1
    q = q.astype(NP[act])
    for lead in (0, 10, 18):
        scale = float(np.float32(lead * np.log(2)))
        got = attend(ctx, p, c, n_q, act, q, rows, 1 << 20, scale)
        check(c.cpu, tables[0], length, rows, q.astype(np.float64), scale, got, act)


@pytest.mark.parametrize("fmt", [I8, E4M3])
@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("rows", [FEW, MANY])
def test_small_values_everywhere_in_f32(ctx, fmt, hd, rows):
    """V of 2^-65 throughout, and beside scales of 2^-60."""
    rng = np.random.default_rng(hd)
    page, n_q, length = 32, 2, 700
    n_pages = -(-length // page)
    p, tables = tables_of(ctx, rng, [length], [rows], page, n_pages)
    c = CachePair(ctx, n_pages, page, 1, hd, fmt)
    unit = 32.0 if fmt == I8 else 110.0
    for w in range(2):
        c.cpu.codes[w][:] = ref.encode(rng.normal(0, unit, c.cpu.codes[w].shape), fmt)
    c.cpu.scales[0][:] = 2.0 ** -6
    q = rng.normal(0, 1, (rows, n_q, hd)).astype(np.float32)
    for least, most in ((-70, -70), (-72, -56)):
        c.cpu.scales[1][:] = 2.0 ** rng.integers(least, most + 1, c.cpu.scales[1].shape)
        upload(ctx, c)
        got = attend(ctx, p, c, n_q, F32, q, rows, 1 << 20, hd ** -0.5)
        check(c.cpu, tables[0], length, rows, q.astype(np.float64), hd ** -0.5, got, F32, 0.0)
