"""Paged 8-bit cache without a GPU: plan layout, refusals of every entry point, and the NumPy restatement against itself."""
import ctypes as C

import numpy as np
import pytest

from ksearch_b200 import E4M3, F16, F32, I8, Q40, _lib
from tests import paged_ref as ref


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.fixture()
def cpu(lib):
    c = lib.ks_debug_ctx_checks_only()
    yield c
    lib.ks_ctx_destroy(c)


class Args:
    """Arguments that every check accepts; the addresses are never touched."""

    def __init__(self, lib, ctx):
        self.lib, self.ctx, self.at = lib, ctx, 1 << 20
        self.t = dict(n_seqs=3, max_blocks=4, n_pages=10, page=32, max_rows=20)
        self.c = dict(n_pages=10, page=32, n_kv=2, hd=128, dtype=I8)
        self.n_q = 4
        self.bytes = {}

    def buf(self, name, nbytes, align=0):
        over = self.bytes.get(name)
        if over == "null":
            return None
        nbytes, align = (nbytes + over, 0) if isinstance(over, int) else (nbytes, over[1] if over else 0)
        self.at += (nbytes + 511) & ~255
        return self.lib.ks_buf_wrap(self.ctx, self.at + align, max(nbytes, 0))

    def tables(self):
        t = self.t
        words = lambda n: max(0, 4 * n)  # noqa: E731
        return _lib.PageTablesStruct(*t.values(), self.buf("lens", words(t["n_seqs"])), self.buf("tables", words(t["n_seqs"] * t["max_blocks"])),
                                     self.buf("free", words(1 + t["n_pages"])), self.buf("plan", words(self.lib.ks_pages_plan_ints(t["n_seqs"], t["max_rows"], t["page"]))))

    def cache(self):
        c = self.c
        codes, scales = c["n_pages"] * c["page"] * c["n_kv"] * c["hd"], 4 * c["n_pages"] * c["n_kv"]
        return _lib.Q8CacheStruct(*c.values(), self.buf("kc", codes), self.buf("vc", codes), self.buf("ks", scales), self.buf("vs", scales))

    def call(self, name, **kw):
        lib, t, c = self.lib, C.byref(self.tables()), C.byref(self.cache())
        act = kw.get("act", F32)
        size = 2 if act == F16 else 4
        rows, hd, n_kv = self.t["max_rows"], self.c["hd"], self.c["n_kv"]
        kv = rows * n_kv * hd * size
        if name in ("step", "trim"):
            return getattr(lib, "ks_pages_" + name)(self.ctx, t, self.buf("n_new", 4 * self.t["n_seqs"]))
        if name == "reset":
            return lib.ks_pages_reset(self.ctx, t)
        if name == "append":
            ld = kw.get("ld", n_kv * hd)
            return lib.ks_kv_append_q8(self.ctx, c, t, act, self.buf("k", kv), kw.get("off", 0), self.buf("v", kv), 0, ld)
        if name == "norm":
            return lib.ks_rmsnorm_per_head_qkv_q8(self.ctx, c, t, self.n_q, 1e-6, act, self.buf("q", rows * self.n_q * hd * size), self.buf("qw", hd * size),
                                                  self.buf("rope", 128 * hd * 4), self.buf("k", kv), self.buf("kw", hd * size), self.buf("v", kv),
                                                  self.buf("q_out", rows * self.n_q * hd * size))
        if name == "read":
            n = kw.get("n_rows", 7)
            return lib.ks_kv_read_q8(self.ctx, c, n, self.buf("slots", 4 * 7), kw.get("off", 0), act, self.buf("k", 7 * n_kv * hd * size), self.buf("v", 7 * n_kv * hd * size))
        most = kw.get("rows_most", rows)
        q = self.buf("q", rows * self.n_q * hd * size)
        out = q if kw.get("alias") else self.buf("out", rows * self.n_q * hd * size)
        tmp = self.buf("tmp", 4 * lib.ks_sdpa_paged_tmp_floats(self.ctx, c, t, self.n_q, most))
        return lib.ks_sdpa_paged_q8(self.ctx, c, t, self.n_q, most, 100, kw.get("window", 0), kw.get("scale", 1.0), act, q, tmp, out)


CALLS = ("step", "trim", "reset", "append", "norm", "read", "attention")


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("name", CALLS)
def test_good_arguments_get_as_far_as_the_device(lib, cpu, name, act):
    assert Args(lib, cpu).call(name, act=act) == _lib.ERR_UNSUPPORTED and b"no device" in lib.ks_last_error(cpu)


TABLE_CALLS = ("step", "trim", "reset", "append", "norm", "attention")
CACHE_CALLS = ("append", "norm", "read", "attention")


@pytest.mark.parametrize("name,change", [(n, c) for n in TABLE_CALLS for c in (
    dict(n_seqs=0), dict(n_seqs=1025), dict(max_rows=0), dict(max_rows=(1 << 20) + 1), dict(page=48), dict(page=0), dict(page=256), dict(page=8), dict(n_pages=0),
    dict(max_blocks=0), dict(n_pages=1 << 27), dict(max_blocks=1 << 25), dict(max_blocks=1 << 62), dict(n_pages=1 << 62))])
def test_table_sizes_are_refused(lib, cpu, name, change):
    a = Args(lib, cpu)
    before = a.call(name)
    assert before == _lib.ERR_UNSUPPORTED
    good = a.tables
    a.tables = lambda: _changed(good(), change)
    assert a.call(name) == _lib.ERR_INVALID


def _changed(struct, change):
    for k, v in change.items():
        setattr(struct, k, v)
    return struct


@pytest.mark.parametrize("name,change,code", [(n, c, e) for n in CACHE_CALLS for c, e in (
    (dict(dtype=Q40), _lib.ERR_UNSUPPORTED), (dict(dtype=F16), _lib.ERR_UNSUPPORTED), (dict(hd=96), _lib.ERR_UNSUPPORTED), (dict(hd=512), _lib.ERR_UNSUPPORTED),
    (dict(hd=0), _lib.ERR_UNSUPPORTED), (dict(page=24), _lib.ERR_INVALID), (dict(n_kv=0), _lib.ERR_INVALID), (dict(n_kv=1025), _lib.ERR_INVALID),
    (dict(n_pages=0), _lib.ERR_INVALID), (dict(n_pages=11), _lib.ERR_INVALID), (dict(n_pages=1 << 61), _lib.ERR_INVALID), (dict(hd=256), _lib.ERR_INVALID),
    (dict(n_kv=3), _lib.ERR_INVALID))])
def test_cache_sizes_are_refused(lib, cpu, name, change, code):
    a = Args(lib, cpu)
    good = a.cache
    a.cache = lambda: _changed(good(), change)
    assert a.call(name) == code and b"no device" not in lib.ks_last_error(cpu)


BUFFERS = {"step": ("lens", "tables", "free", "plan", "n_new"), "trim": ("lens", "tables", "free", "plan", "n_new"), "reset": ("lens", "tables", "free", "plan"),
           "append": ("plan", "kc", "vc", "ks", "vs", "k", "v"), "norm": ("plan", "kc", "vc", "ks", "vs", "q", "qw", "k", "kw", "v", "q_out"),
           "read": ("kc", "vc", "ks", "vs", "slots", "k", "v"), "attention": ("lens", "tables", "plan", "kc", "vc", "ks", "vs", "q", "tmp", "out")}


@pytest.mark.parametrize("how", ["null", -4, (0, 2)])
@pytest.mark.parametrize("name,buf", [(n, b) for n, bs in BUFFERS.items() for b in bs])
def test_buffers_are_checked(lib, cpu, name, buf, how):
    """Missing, a word short, off their alignment."""
    a = Args(lib, cpu)
    a.bytes[buf] = how
    assert a.call(name) == _lib.ERR_INVALID


@pytest.mark.parametrize("name,kw", [("append", dict(ld=248)), ("append", dict(ld=260)), ("append", dict(ld=264)), ("append", dict(off=4)), ("append", dict(off=8)), ("append", dict(off=1 << 62)),
                                     ("append", dict(ld=1 << 62)), ("append", dict(act=I8)), ("norm", dict(act=E4M3)), ("read", dict(act=Q40)), ("read", dict(n_rows=0)), ("read", dict(n_rows=8)),
                                     ("read", dict(off=1)), ("read", dict(off=1 << 62)), ("read", dict(n_rows=1 << 40)), ("attention", dict(rows_most=21)), ("attention", dict(alias=True)),
                                     ("attention", dict(window=1 << 31)), ("attention", dict(scale=float("nan"))), ("attention", dict(scale=float("inf"))), ("attention", dict(act=I8))])
def test_arguments_are_refused(lib, cpu, name, kw):
    assert Args(lib, cpu).call(name, **kw) == _lib.ERR_INVALID


@pytest.mark.parametrize("n_q,code", [(0, _lib.ERR_INVALID), (3, _lib.ERR_INVALID), (130, _lib.ERR_UNSUPPORTED), (65538, _lib.ERR_INVALID), (6, _lib.ERR_UNSUPPORTED), (128, _lib.ERR_UNSUPPORTED)])
def test_head_counts(lib, cpu, n_q, code):
    a = Args(lib, cpu)
    a.n_q = n_q
    assert a.call("attention") == code
    assert (b"no device" in lib.ks_last_error(cpu)) == (n_q in (6, 128))


@pytest.mark.parametrize("name", TABLE_CALLS)
def test_more_table_entries_than_32_bits_count(lib, cpu, name):
    """Lengths that lie could make a sum over all tables' pages pass 2^32."""
    a = Args(lib, cpu)
    good = a.tables
    a.tables = lambda: _changed(good(), dict(n_seqs=1024, max_blocks=1 << 21))
    assert a.call(name) == _lib.ERR_INVALID and b"entries: below 2^31" in lib.ks_last_error(cpu)


def test_more_work_than_one_call_counts(lib, cpu):
    a = Args(lib, cpu)
    a.t.update(n_seqs=1024, max_blocks=1 << 20)
    a.c.update(n_kv=4)
    assert a.call("attention") == _lib.ERR_UNSUPPORTED and b"too much for one call" in lib.ks_last_error(cpu)
    a.t.update(max_blocks=1 << 14)
    assert a.call("attention") == _lib.ERR_UNSUPPORTED and b"no device" in lib.ks_last_error(cpu)


def test_no_rows_are_no_work(lib, cpu):
    assert Args(lib, cpu).call("attention", rows_most=0) == 0


def test_null_structs(lib, cpu):
    for name, args in (("ks_pages_reset", (None,)), ("ks_pages_step", (None, None)), ("ks_pages_trim", (None, None)), ("ks_kv_append_q8", (None, None, F32, None, 0, None, 0, 8)),
                       ("ks_rmsnorm_per_head_qkv_q8", (None, None, 1, 1e-6, F32) + (None,) * 7), ("ks_kv_read_q8", (None, 1, None, 0, F32, None, None)),
                       ("ks_sdpa_paged_q8", (None, None, 1, 1, 1, 0, 1.0, F32, None, None, None))):
        assert getattr(lib, name)(cpu, *args) == _lib.ERR_INVALID
        assert getattr(lib, name)(None, *args) == _lib.ERR_INVALID
    assert lib.ks_sdpa_paged_tmp_floats(cpu, None, None, 1, 1) == 0


@pytest.mark.parametrize("n_seqs,max_rows,page", [(1, 1, 16), (7, 130, 32), (1024, 1 << 20, 128), (3, 4, 64)])
def test_plan_layout(lib, n_seqs, max_rows, page):
    at = [lib.ks_pages_plan_offset(n_seqs, max_rows, page, p) for p in range(6)]
    up = lambda n: -(-n // 4) * 4  # noqa: E731
    assert at[0] == 8 and at[1] == 8 + up(n_seqs + 1) and [b - a for a, b in zip(at[1:], at[2:5])] == [up(max_rows)] * 3
    assert at[5] == at[4] + 4 * (max_rows // page + 2 * n_seqs) == lib.ks_pages_plan_ints(n_seqs, max_rows, page)
    assert lib.ks_pages_plan_offset(n_seqs, max_rows, page, 6) == 0 and lib.ks_pages_plan_offset(n_seqs, max_rows, page, -1) == 0
    assert lib.ks_pages_plan_ints(0, 1, 16) == 0 and lib.ks_pages_plan_ints(1, 1, 17) == 0


def test_touched_pages_fit_the_plan(lib):
    """max_rows / page + 2 n_seqs records hold any step."""
    rng = np.random.default_rng(3)
    for _ in range(300):
        page, n = int(rng.choice([16, 32])), int(rng.integers(1, 6))
        t = ref.Tables(n, 20, 400, page, 10 ** 6)
        t.step(rng.integers(0, 70, n))
        new = rng.integers(0, 90, n)
        assert t.step(new) == 0
        assert len(t.jobs) <= int(new.sum()) // page + 2 * n and sum(j[1] for j in t.jobs) == new.sum()


def test_codes_of_the_restatement():
    for fmt in (I8, E4M3):
        codes = np.arange(256, dtype=np.uint8)
        codes = codes[(codes & 127) != 127] if fmt == E4M3 else codes[codes != 128]
        v = ref.decode(codes, fmt)
        assert np.array_equal(ref.decode(ref.encode(v, fmt), fmt), v)
        x = np.random.default_rng(1).uniform(-ref.QMAX[fmt], ref.QMAX[fmt], 4000)
        y = ref.decode(ref.encode(x, fmt), fmt)
        every = np.unique(v)
        assert np.allclose(np.abs(x - y), np.abs(x[:, None] - every[None, :]).min(1))
    assert ref.scale_for(127.0, I8) == 1 and ref.scale_for(np.nextafter(127.0, 200), I8) == 2 and ref.scale_for(448.0, E4M3) == 1 and ref.scale_for(0.0, I8) == 2.0 ** -100
    torch = pytest.importorskip("torch")
    x = np.random.default_rng(2).normal(0, 100, 5000).clip(-448, 448)
    want = torch.from_numpy(x).float().to(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(ref.decode(ref.encode(x.astype(np.float32).astype(np.float64), E4M3), E4M3), want)
