"""The word that kernels leave index errors in: cleared before anything that is enqueued behind the report."""
import glob
import os
import re

import pytest

from ksearch_b200 import I8, Eng, KsError, Q8Cache, _lib
from tests.test_gpu_paged_cache import ints


def test_device_memory_is_cleared_on_a_stream():
    """cudaMemset works on the default stream and may return before it has run; the contexts' streams do not wait for that stream, so what it
    clears could be cleared after later kernels have written to it."""
    sources = glob.glob(os.path.join(_lib.PKG, "csrc", "*.cu*")) + glob.glob(os.path.join(_lib.PKG, "csrc", "*.h"))
    assert sources
    for path in sources:
        assert not re.search(r"\bcudaMemset\s*\(", open(path).read()), path


@pytest.mark.gpu
def test_an_error_right_behind_a_report_is_reported_too(ctx):
    c, out = Q8Cache(ctx, 2, 16, 1, 64, I8), ctx.buffer_empty_f32(64)
    slots = ints(ctx, [32])
    ctx.synchronize()
    for _ in range(200):
        Eng().kv_read_q8(ctx, c, 1, slots, 0, out, out)
        with pytest.raises(KsError) as e:
            ctx.synchronize()
        assert e.value.code == _lib.ERR_INVALID
    ctx.synchronize()
