"""The row cache's calls next to what else a caller's program does."""
import ctypes as C

import numpy as np
import pytest

from redisearch_amd import rows as R
from redisearch_amd import vecsim as V

from . import rows_plain as P
from .test_gpu_rows import Cache, as64, stream, values

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def hip():
    torch.cuda.synchronize()
    with open("/proc/self/maps") as maps:
        return C.CDLL(next(line.split()[-1] for line in maps if "libamdhip64" in line))


def test_an_error_left_by_an_earlier_call_is_not_this_ones():
    """A call of the runtime that failed before (here a device that there is not) leaves its error with the thread: the calls do their
    work, say so, and leave the error to whoever asks for it."""
    gen = torch.Generator().manual_seed(1)
    n, dim = 40, 96
    cache = Cache(P.F32, dim, R.INT8, 32, n, zero=True)
    rows, slots, back = values(gen, n, dim, P.F32), torch.arange(n, device="cuda"), torch.zeros((n, dim), device="cuda")
    off, cnt = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, 3], [n]))
    pages, scores = torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.zeros((3, n), device="cuda")
    seen, offsets = torch.tensor([5], dtype=torch.int32, device="cuda"), torch.tensor([0, 1, 1, 1], dtype=torch.int32, device="cuda")
    presence = torch.ones(3, device="cuda")
    rules = R.score_rules(seen_offsets=offsets.data_ptr(), seen_ids=seen.data_ptr(), n_seen=1, presence=presence.data_ptr())
    final = torch.zeros_like(scores)
    at = stream()
    calls = [lambda: cache.c.write(rows.data_ptr(), dim, slots.data_ptr(), n, at),
             lambda: cache.c.read(slots.data_ptr(), n, back.data_ptr(), dim, at),
             lambda: cache.c.partition_scores(rows.data_ptr(), dim, 3, off.data_ptr(), 1, pages.data_ptr(), 1, n, cnt.data_ptr(), R.PRODUCT, scores.data_ptr(), n, at),
             lambda: R.adjust_scores(rules, scores.data_ptr(), final.data_ptr(), 3, n, n, None, at)]
    lib = hip()
    for call in calls:
        failed = lib.hipSetDevice(1 << 20)
        assert failed != 0
        try:
            call()
        finally:
            left = lib.hipGetLastError()
        assert left == failed
    stored = P.dequantise(*cache.plain(), dim, R.INT8, 32)
    want = as64(rows[:3]) @ stored.T
    assert np.abs(as64(back) - stored).max() <= 1e-6 * np.abs(stored).max()
    assert np.abs(as64(scores) - want).max() <= 1e-4 * np.abs(want).max()
    want = as64(scores)
    want[0, 5] = np.float32(want[0, 5]) - np.float32(1)
    assert (as64(final) == want).all()

    index = V.VecSimIndex(P.F32, dim, V.VecSimMetric_IP)
    lib.hipSetDevice(1 << 20)
    try:
        assert cache.c.add_to(index, slots.data_ptr(), n, 1, at) == n
        lib.hipSetDevice(1 << 20)
        cache.c.cache_rows(index, 0, n, slots.data_ptr(), at)
    finally:
        lib.hipGetLastError()
    assert index.index_size() == n and (index.read_rows(0, n) == back.cpu().numpy()).all()
    assert np.abs(P.dequantise(*cache.plain(), dim, R.INT8, 32) - stored).max() <= 1e-6 * np.abs(stored).max()
