"""Page tables with entries that no pool has: what a trim gives back, and what the steps behind it hand out."""
import numpy as np
import pytest

from ksearch_b200 import KsError, _lib
from tests.test_gpu_paged_cache import Pair, ints

pytestmark = pytest.mark.gpu


def spoil(ctx, p, where):
    """Entries (sequence, block, id) into the GPU's table; the restatement's keeps the good ones."""
    g = p.gpu
    tables = g.read(g.tables).reshape(p.cpu.tables.shape).copy()
    for s, b, bad in where:
        tables[s, b] = bad
    ctx.write_buffer(g.tables, tables.astype(np.int32))


def named(ctx):
    with pytest.raises(KsError) as e:
        ctx.synchronize()
    assert e.value.code == _lib.ERR_INVALID and "page id" in e.value.msg


@pytest.mark.parametrize("bad", [-1, 40, 2 ** 31 - 1, -2 ** 31])
def test_a_bad_entry_is_not_given_back(ctx, bad):
    """Sequence 1 ends with one of its four entries bad: three pages go back, the bad id is handed out to nobody."""
    p = Pair(ctx, 3, 8, 12, 16, 100)
    assert p.step([20, 60, 5]) == 0
    spoil(ctx, p, [(1, 2, bad)])
    lost = int(p.cpu.tables[1, 2])
    p.trim([-1, 0, -1])
    p.cpu.stack.remove(lost)
    named(ctx)
    g = p.gpu
    free = g.read(g.free)
    assert free[0] == len(p.cpu.stack) and np.array_equal(free[1:1 + free[0]], p.cpu.stack)
    assert np.array_equal(g.read(g.tables).reshape(3, 8), p.cpu.tables) and g.read(g.lens).tolist() == [20, 0, 5]
    assert p.step([0, 60, 0]) == 0                  # all pages that are left but four
    assert p.step([0, 0, 16 * len(p.cpu.stack) + 16 + 11 + 1]) == 1
    assert p.step([0, 0, 11 + 16 * min(len(p.cpu.stack), 7)]) == 0
    ctx.synchronize()


@pytest.mark.parametrize("n_seqs,blocks,share", [(1, 1, 1.0), (5, 7, 0.3), (300, 40, 0.01), (1024, 9, 0.5), (40, 300, 1.0)])
def test_many_bad_entries(ctx, n_seqs, blocks, share):
    """Bad ids anywhere among the pages of a large trim: the good ones come back in the order that a trim without the others has."""
    rng = np.random.default_rng(n_seqs)
    page, n_pages = 16, n_seqs * blocks
    p = Pair(ctx, n_seqs, blocks, n_pages, page, n_seqs * page * blocks)
    assert p.step(rng.integers(1, page * blocks + 1, n_seqs)) == 0
    used = np.argwhere(p.cpu.tables >= 0)
    used = used[rng.random(len(used)) < share]
    spoil(ctx, p, [(s, b, int(rng.choice([-1, n_pages, n_pages + 7, 2 ** 31 - 1]))) for s, b in used])
    keep = np.where(rng.random(n_seqs) < 0.7, 0, rng.integers(-1, page * blocks, n_seqs))
    gone = [int(p.cpu.tables[s, b]) for s, b in used if 0 <= keep[s] < p.cpu.lens[s] and b >= -(-keep[s] // page)]
    p.trim(keep)
    p.cpu.stack = [x for x in p.cpu.stack if x not in set(gone)]
    g = p.gpu
    free = g.read(g.free)
    assert free[0] == len(p.cpu.stack) and np.array_equal(free[1:1 + free[0]], p.cpu.stack)
    assert np.array_equal(g.read(g.lens), p.cpu.lens)
    if gone:
        named(ctx)
    ctx.synchronize()
