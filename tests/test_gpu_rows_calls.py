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


@pytest.mark.parametrize("mode", [0, 1, 2], ids=["identity", "direct", "hash"])
def test_labels_that_would_pass_the_last_one(mode):
    """Labels are 64 bits: a range that would go on at 0 is refused, whatever form the index keeps its labels in; one that ends at the
    last label is not."""
    dim, n = 32, 8
    index = V.VecSimIndex(P.F32, dim, V.VecSimMetric_L2)
    x = np.random.default_rng(mode).standard_normal((12, dim)).astype(np.float32)
    index.add_bulk(x[:4], 1)
    if mode == 1:
        index.delete_vector(2)
    if mode == 2:
        index.add_vector(x[4], 10 ** 15)
    assert index.label_table() == mode
    before = index.index_size()
    cache = Cache(P.F32, dim, R.NATIVE, 0, n, zero=True)
    slots = torch.arange(n, device="cuda")
    cache.write(torch.from_numpy(x[4:]).cuda(), slots)
    for first, many in ((2 ** 64 - 2, 4), (2 ** 64 - 1, 2), (2 ** 64 - 7, 8)):
        with pytest.raises(RuntimeError, match="labels end at"):
            cache.c.add_to(index, slots.data_ptr(), many, first, stream())
    assert index.index_size() == before
    assert cache.c.add_to(index, slots[4:].data_ptr(), 2, 2 ** 64 - 3, stream()) == 2
    assert cache.c.add_to(index, slots[6:].data_ptr(), 1, 2 ** 64 - 1, stream()) == 1
    for first, many in ((2 ** 64 - 4, 2), (2 ** 64 - 2, 2), (2 ** 64 - 1, 1)):
        with pytest.raises(RuntimeError, match="label range overlaps"):
            cache.c.add_to(index, slots.data_ptr(), many, first, stream())
    assert index.index_size() == before + 3
    for row, label in ((8, 2 ** 64 - 3), (9, 2 ** 64 - 2), (10, 2 ** 64 - 1)):
        found, distances = index.topk_query(x[row], 1).results()
        assert found.astype(np.uint64).tolist() == [label] and distances[0] <= 1e-6


@pytest.mark.parametrize("vtype", [P.F32, P.F16, P.BF16], ids={P.F32: "f32", P.F16: "f16", P.BF16: "bf16"}.get)
@pytest.mark.parametrize("metric", [V.VecSimMetric_Cosine, V.VecSimMetric_IP], ids={V.VecSimMetric_Cosine: "cosine", V.VecSimMetric_IP: "ip"}.get)
def test_slots_out_of_range_come_into_an_index_as_rows_of_zeros_do(vtype, metric):
    """A row of zeros has no direction: a cosine index keeps it as NaN, by whichever way it came, and finds it behind every other."""
    dim, n = 48, 9
    rng = np.random.default_rng(4)
    x = rng.standard_normal((n, dim)).astype(np.float32)
    cache = Cache(vtype, dim, R.NATIVE, 0, n, zero=True)
    cache.write(torch.from_numpy(x).to({P.F32: torch.float32, P.F16: torch.float16, P.BF16: torch.bfloat16}[vtype]).cuda(), torch.arange(n, device="cuda"))
    cached, loaded = (V.VecSimIndex(vtype, dim, metric) for _ in range(2))
    slots = torch.tensor([0, -1, 2, 3, n, 5, 6, 2 ** 62, 8], device="cuda")
    assert cache.c.add_to(cached, slots.data_ptr(), n, 1, stream()) == n
    x[[1, 4, 7]] = 0
    as_rows = torch.from_numpy(x).to({P.F32: torch.float32, P.F16: torch.float16, P.BF16: torch.bfloat16}[vtype]).cuda()
    torch.cuda.synchronize()
    loaded.add_device_rows(as_rows.data_ptr(), n, 1)
    a, b = cached.read_rows(0, n), loaded.read_rows(0, n)
    assert a.tobytes() == b.tobytes()
    zeros = torch.from_numpy(a[[1, 4, 7]].astype(np.int32) if vtype == P.BF16 else a[[1, 4, 7]].astype(np.float32))
    assert ((zeros & 0x7fff) > 0x7f80).all() if metric == V.VecSimMetric_Cosine and vtype == P.BF16 else zeros.isnan().all() if metric == V.VecSimMetric_Cosine else not zeros.any()
    q = x[2] + x[3]
    near = [index.topk_query(q, n).results()[0].tolist() for index in (cached, loaded)]
    assert near[0] == near[1]
    if metric == V.VecSimMetric_Cosine:
        assert not {2, 5, 8} & set(near[0][:6])
