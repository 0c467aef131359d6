"""Two plans over one set of tables: a small one for steps that decode and a large one for prompts, as a server keeps them whose kernels'
cost follows what a plan can hold."""
import numpy as np
import pytest

from ksearch_b200 import E4M3, F16, F32, I8, Eng, PageTables
from tests import paged_ref as ref
from tests.test_gpu_paged_cache import NP, CachePair, Pair, ints

pytestmark = pytest.mark.gpu


def other_plan(ctx, t, max_rows):
    return PageTables(ctx, t.n_seqs, t.max_blocks, t.n_pages, t.page, max_rows, lens=t.lens, tables=t.tables, free=t.free)


@pytest.mark.parametrize("fmt", [I8, E4M3])
def test_a_plan_without_a_step_has_no_rows(ctx, fmt):
    """A plan that was allocated beside tables that are in use, before its first step: nothing is written."""
    p, c = Pair(ctx, 3, 4, 8, 16, 40), CachePair(ctx, 8, 16, 2, 64, fmt)
    p.step([20, 4, 9])
    x = ctx.buffer_bytes(np.full((30, 2, 64), 3, np.float32))
    small = other_plan(ctx, p.gpu, 30)
    eng = Eng()
    eng.kv_append_q8(ctx, c.gpu, small, x, x)
    w, rope, out = ctx.buffer_bytes(np.ones(64, np.float32)), ctx.buffer_bytes(np.ones((64, 64), np.float32)), ctx.buffer_bytes(np.full((30, 2, 64), 7, np.float32))
    eng.rmsnorm_per_head_qkv_q8(ctx, c.gpu, small, 2, 1e-6, x, w, rope, x, w, x, out)
    tmp = ctx.buffer_empty_f32(eng.sdpa_paged_tmp_floats(ctx, c.gpu, small, 2, 30))
    eng.sdpa_paged_q8(ctx, c.gpu, small, 2, 30, 40, x, tmp, out)
    ctx.synchronize()
    c.same()
    p.same()
    assert (ctx.read_f32(out, 30 * 128) == 7).all()


@pytest.mark.parametrize("act,fmt", [(F32, I8), (F16, E4M3)])
def test_prompts_and_tokens_by_plans_of_their_own(ctx, act, fmt):
    """Prompts through a plan of 300 rows, tokens through one of 4, in turn: tables, codes and attention as of a single set of tables."""
    rng = np.random.default_rng(3)
    n_q, n_kv, hd, page = 4, 2, 128, 32
    p, c = Pair(ctx, 4, 12, 48, page, 300), CachePair(ctx, 48, page, n_kv, hd, fmt)
    small, eng = other_plan(ctx, p.gpu, 4), Eng(act)
    for new in ([150, 3, 0, 40], [1, 1, 0, 1], [1, 0, 1, 1], [0, 100, 33, 0], [1, 1, 1, 1]):
        n = sum(new)
        t = small if n <= 4 else p.gpu
        eng.pages_step(ctx, t, ints(ctx, new))
        assert p.cpu.step(new) == 0 and t.status() == 0
        assert np.array_equal(t.read(t.lens), p.cpu.lens) and np.array_equal(t.read(t.tables).reshape(4, 12), p.cpu.tables)
        q, k, v = (rng.normal(0, 1, (t.max_rows, h, hd)).astype(NP[act]) for h in (n_q, n_kv, n_kv))
        eng.kv_append_q8(ctx, c.gpu, t, ctx.buffer_bytes(k), ctx.buffer_bytes(v))
        c.cpu.append(p.cpu, k, v)
        c.same()
        out, tmp = ctx.buffer_bytes(np.full(q.shape, 5, NP[act])), ctx.buffer_empty_f32(eng.sdpa_paged_tmp_floats(ctx, c.gpu, t, n_q, max(new)))
        eng.sdpa_paged_q8(ctx, c.gpu, t, n_q, max(new), 300, ctx.buffer_bytes(q), tmp, out, hd ** -0.5)
        got = ctx.read_act(out, q.size, act).reshape(q.shape).astype(np.float64)
        assert (got[n:] == 5).all()
        for s in range(4):
            a, b = p.cpu.row_start[s:s + 2]
            if a == b:
                continue
            want, spread, weight = ref.attention(c.cpu, p.cpu.tables[s], int(p.cpu.lens[s]), int(b - a), q[a:b].astype(np.float64), hd ** -0.5, 0)
            tol = weight * (2.0 ** -18 * spread[..., None] + (2.0 ** -18 if act == F32 else 2.0 ** -11 + 2.0 ** -15)) + (np.abs(want) * 2.0 ** -11 + 2.0 ** -25 if act == F16 else 0)
            assert (np.abs(got[a:b] - want) <= tol).all()
    ctx.synchronize()
