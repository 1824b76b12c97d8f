"""The row cache on the GPU against plain numpy in 64 bits (tests/rows_plain.py): codes and scales bit for bit, values within the
roundings that the definitions in include/rsgpu_rows.h name."""
import ctypes as C

import numpy as np
import pytest

from redisearch_amd import rows as R
from redisearch_amd import vecsim as V

from . import rows_plain as P

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {P.F32: torch.float32, P.F16: torch.float16, P.BF16: torch.bfloat16}
FORMATS = [R.INT8, R.E4M3, R.INT4]
ids = {P.F32: "f32", P.F16: "f16", P.BF16: "bf16"}.get
fids = {R.NATIVE: "native", R.INT8: "int8", R.E4M3: "e4m3", R.INT4: "int4"}.get


def stream():
    return torch.cuda.current_stream().cuda_stream


class Cache:
    """A cache on the GPU, its memory filled with a pattern."""

    def __init__(self, vtype, dim, fmt, block, capacity, zero=False):
        self.args = (vtype, dim, fmt, block)
        self.codes = torch.full((capacity, P.row_bytes(vtype, dim, fmt)), 0 if zero else 0xA5, dtype=torch.uint8, device="cuda")
        self.scales = torch.full((capacity, P.row_scales(dim, fmt, block)), 0.0 if zero else -7.0, device="cuda")
        self.c = R.RowCache(vtype, dim, fmt, block, capacity, self.codes.data_ptr(), self.scales.data_ptr() if fmt != R.NATIVE else None)

    def write(self, rows, slots):
        self.c.write(rows.data_ptr(), rows.stride(0), slots.data_ptr(), slots.numel(), stream())

    def plain(self):
        return self.codes.cpu().numpy(), self.scales.cpu().numpy()


def values(gen, n, dim, vtype):
    """Rows of many sizes: blocks of different magnitude, zeros, exact halves of a scale among them."""
    x = torch.randn((n, dim), generator=gen, dtype=torch.float64)
    x *= torch.exp2(torch.randint(-12, 12, (n, 1), generator=gen).double())
    x[:, ::5] *= 0.01
    if dim > 3:
        x[::3, 1] = 0
    return x.to(TYPES[vtype]).cuda()


def as64(t):
    return t.double().cpu().numpy()


def strided(x, gap):
    wide = torch.full((x.shape[0], x.shape[1] + gap), 3.0, dtype=x.dtype, device="cuda")
    wide[:, : x.shape[1]] = x
    return wide[:, : x.shape[1]]


# ---- writing and reading -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("vtype", list(TYPES), ids=ids)
@pytest.mark.parametrize("fmt", FORMATS, ids=fids)
@pytest.mark.parametrize("block", [0, 32, 64, 128])
@pytest.mark.parametrize("dim,n,gap", [(1, 1, 0), (7, 5, 3), (32, 3, 0), (33, 40, 1), (100, 130, 0), (128, 9, 8), (768, 67, 0), (1000, 20, 5), (2049, 3, 0)])
def test_write_and_read(vtype, fmt, block, dim, n, gap):
    gen = torch.Generator().manual_seed(dim * 7 + block + fmt)
    capacity = 2 * n + 3
    cache = Cache(vtype, dim, fmt, block, capacity)
    rows = strided(values(gen, n, dim, vtype), gap)
    slots = torch.randperm(capacity, generator=gen)[:n].cuda()
    if n > 4:
        slots[1], slots[3], slots[4] = -1, capacity, -(2 ** 62)          # left out
    cache.write(rows, slots)
    codes, scales = cache.plain()
    at = slots.cpu().numpy()
    kept = (at >= 0) & (at < capacity)
    want_codes, want_scales = P.quantise(as64(rows), fmt, block)
    assert (codes[at[kept]] == want_codes[kept]).all()
    assert (scales[at[kept]] == want_scales[kept]).all()
    others = np.setdiff1d(np.arange(capacity), at[kept])
    assert (codes[others] == 0xA5).all() and (scales[others] == -7.0).all()

    again = torch.cat([slots, slots[:2]]).contiguous()                   # a slot may be read twice
    out = torch.full((again.numel() + 1, dim + gap), 5.0, dtype=TYPES[vtype], device="cuda")
    cache.c.read(again.data_ptr(), again.numel(), out.data_ptr(), out.stride(0), stream())
    got = as64(out)
    kept = np.concatenate([kept, kept[:2]])
    want = np.zeros((again.numel(), dim))
    want[kept] = P.dequantise(codes[again.cpu().numpy()[kept]], scales[again.cpu().numpy()[kept]], dim, fmt, block)
    # the product code * scale is rounded to fp32, and that to the type: half a step of each
    bound = np.abs(want) * (2.0 ** -24 + P.EPS[vtype] * (1 + 2.0 ** -24)) + P.LEAST[vtype] + 2.0 ** -150
    assert (np.abs(got[:-1, :dim] - want) <= bound).all()
    assert (got[:-1, dim:] == 5.0).all() and (got[-1] == 5.0).all()


@pytest.mark.parametrize("vtype", list(TYPES), ids=ids)
@pytest.mark.parametrize("dim,n,gap", [(1, 3, 0), (33, 40, 1), (100, 9, 4), (768, 30, 0)])
def test_native_rows_are_kept_as_they_are(vtype, dim, n, gap):
    gen = torch.Generator().manual_seed(dim)
    cache = Cache(vtype, dim, R.NATIVE, 0, n + 2)
    rows = strided(values(gen, n, dim, vtype), gap)
    rows[0, 0] = float("inf")
    rows[1, dim // 2] = float("nan")
    slots = torch.randperm(n + 2, generator=gen)[:n].cuda()
    slots[2] = -1
    cache.write(rows, slots)
    kept = (slots >= 0)
    stored = cache.codes[slots[kept]].view(TYPES[vtype])
    assert torch.equal(stored[:, :dim].nan_to_num(7.0), rows[kept].nan_to_num(7.0)) and not stored[:, dim:].any()
    assert torch.equal(torch.isnan(stored[:, :dim]), torch.isnan(rows[kept]))
    out = torch.full((n, dim + gap), 5.0, dtype=TYPES[vtype], device="cuda")
    cache.c.read(slots.data_ptr(), n, out.data_ptr(), out.stride(0), stream())
    assert torch.equal(out[kept][:, :dim].nan_to_num(7.0), rows[kept].nan_to_num(7.0))
    assert not out[2, :dim].any() and (out[:, dim:] == 5.0).all()


@pytest.mark.parametrize("fmt", FORMATS, ids=fids)
@pytest.mark.parametrize("block", [0, 32])
def test_write_special_values(fmt, block):
    # (the values read back never pass the type's range: a row of the largest numbers stays finite)
    """Blocks of zeros, below and at the smallest magnitude that is kept, subnormal, at the largest, with infinities and NaN; and
    quotients that lie on a border between two codes and right beside it."""
    dim = 64
    top = {R.INT8: 127.0, R.INT4: 7.0, R.E4M3: 448.0}[fmt]
    rows = np.zeros((16, dim), np.float32)
    rows[1, :] = -0.0
    rows[2, 5] = 2.0 ** -101
    rows[3, 5] = 2.0 ** -100
    rows[3, 6] = -(2.0 ** -103)
    rows[4, 40] = 1e-45
    rows[5, :] = np.linspace(-1, 1, dim) * np.float32(3.4028235e38)
    rows[6, 3], rows[6, 4] = np.inf, 1
    rows[7, 3] = np.nan
    rows[8, 50] = -np.inf
    for i, scale in enumerate([1.0, 0.75, 2.0 ** 20, 1.2345678e-20]):      # borders: (k + 1/2) scale, and one fp32 step to each side
        s = np.float32(np.float32(scale) * np.float32(top)) / np.float32(top)
        k = (np.arange(dim) % int(min(top, 120))) + 0.5
        x = (k * np.float64(s)).astype(np.float32)
        x[1::3] = np.nextafter(x[1::3], np.float32(0))
        x[2::3] = np.nextafter(x[2::3], np.float32(np.inf))
        x[::2] *= -1
        x[0] = x[32] = np.float32(scale) * np.float32(top)
        rows[9 + i] = x
    rows[13, :] = 448 * 2.0 ** np.arange(-20, 44)[:dim]
    rows[14, ::2], rows[14, 1::2] = 448.00003, 1e-3
    rows[15, :] = np.float32(2.0) ** -np.arange(dim)
    cache = Cache(P.F32, dim, fmt, block, 16)
    t = torch.from_numpy(rows).cuda()
    cache.write(t, torch.arange(16, device="cuda"))
    codes, scales = cache.plain()
    want_codes, want_scales = P.quantise(rows.astype(np.float64), fmt, block)
    np.testing.assert_array_equal(scales, want_scales)
    np.testing.assert_array_equal(codes, want_codes)
    out = torch.zeros((16, dim), device="cuda")
    slots = torch.arange(16, device="cuda")
    cache.c.read(slots.data_ptr(), 16, out.data_ptr(), dim, stream())
    want = np.clip(P.dequantise(codes, scales, dim, fmt, block), -P.LARGEST[P.F32], P.LARGEST[P.F32])
    bad = np.isnan(want)
    assert (np.isnan(out.cpu().numpy()) == bad).all()
    assert bad[6].any() and bad[7].any() and bad[8].any() and not bad[:6].any() and not bad[9:].any()
    ok = ~bad
    assert (np.abs(as64(out)[ok] - want[ok]) <= np.abs(want[ok]) * 2.0 ** -24 + 2.0 ** -149).all()


@pytest.mark.parametrize("vtype", [P.F16, P.BF16], ids=ids)
@pytest.mark.parametrize("fmt", FORMATS, ids=fids)
def test_write_every_16_bit_number(vtype, fmt):
    """Every finite number of the type, in one block with each of a few largest magnitudes."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(TYPES[vtype])
    bits = bits[torch.isfinite(bits)]
    order = torch.argsort(bits.float().abs())
    x = bits[order].cuda()
    n = x.numel() // 96
    rows = torch.zeros((n, 128), dtype=TYPES[vtype], device="cuda")
    rows[:, :96] = x[: n * 96].view(n, 96)
    rows[:, 96:] = rows[:, 95:96]
    cache = Cache(vtype, 128, fmt, 64, n)
    cache.write(rows, torch.arange(n, device="cuda"))
    codes, scales = cache.plain()
    want_codes, want_scales = P.quantise(as64(rows), fmt, 64)
    np.testing.assert_array_equal(scales, want_scales)
    np.testing.assert_array_equal(codes, want_codes)
    back = torch.zeros_like(rows)
    slots = torch.arange(n, device="cuda")
    cache.c.read(slots.data_ptr(), n, back.data_ptr(), 128, stream())
    want = np.clip(P.dequantise(codes, scales, 128, fmt, 64), -P.LARGEST[vtype], P.LARGEST[vtype])
    assert torch.isfinite(back).all()
    assert (np.abs(as64(back) - want) <= np.abs(want) * (2.0 ** -24 + P.EPS[vtype] * (1 + 2.0 ** -24)) + P.LEAST[vtype] + 2.0 ** -150).all()


def test_slots_past_32_bits_of_memory():
    """A cache of more than 4 GiB: the last rows are written, scored and read at their place."""
    dim, capacity = 4096, (1 << 20) + 4096 + 77
    cache = R.RowCache(P.F16, dim, R.INT8, 128)
    codes = torch.empty((capacity, cache.row_bytes), dtype=torch.uint8, device="cuda")
    scales = torch.zeros((capacity, cache.row_scales), device="cuda")
    codes[:4] = 0
    gen = torch.Generator().manual_seed(1)
    x = values(gen, 77, dim, P.F16)
    c = R.RowCache(P.F16, dim, R.INT8, 128, capacity, codes.data_ptr(), scales.data_ptr())
    slots = torch.arange(capacity - 77, capacity, device="cuda")
    c.write(x.data_ptr(), dim, slots.data_ptr(), 77, stream())
    want_codes, want_scales = P.quantise(as64(x), R.INT8, 128)
    assert (codes[-77:].cpu().numpy() == want_codes).all() and (scales[-77:].cpu().numpy() == want_scales).all()
    assert not codes[:4].any()
    out = torch.zeros((77, dim), dtype=torch.float16, device="cuda")
    c.read(slots.data_ptr(), 77, out.data_ptr(), dim, stream())
    rows = P.dequantise(want_codes, want_scales, dim, R.INT8, 128)
    assert (np.abs(as64(out) - rows) <= np.abs(rows) * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -24).all()
    # capacity = 16385 pages of 64 + 13 rows: the last page is cut off by the capacity
    last = capacity // 64
    pages = torch.tensor([[last - 1, last]], dtype=torch.int32, device="cuda")
    check_scores(c, codes, scales, x[:3], [0, 3], pages, 64, [128], R.PRODUCT, 128)


# ---- scores of partitions ------------------------------------------------------------------------------------------------------

def check_scores(c, codes, scales, queries, offsets, pages, page_rows, counts, form, ld, calls=None):
    """One call against the definition; what it has to leave alone is looked at too."""
    st = c.c
    fmt, dim, block, vtype = st.format, st.dim, st.block, st.type
    m = queries.shape[0]
    scores = torch.full((m + 1, ld), 123.0, device="cuda")
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    cnt = torch.tensor(counts, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    c.partition_scores(queries.data_ptr(), queries.stride(0), m, off.data_ptr(), len(counts), pages.data_ptr(), pages.shape[1], page_rows,
                       cnt.data_ptr(), form, scores.data_ptr(), ld, stream())
    got = as64(scores)
    q = as64(queries)
    table = pages.cpu().numpy().astype(np.int64)
    want = np.full((m + 1, ld), 123.0)
    bound = np.zeros((m + 1, ld))
    for g, n in enumerate(counts):
        lo, hi = (min(max(o, 0), m) for o in offsets[g:g + 2])
        n = min(max(n, 0), table.shape[1] * page_rows, ld)
        if hi <= lo or not n:
            continue
        j = np.arange(n)
        slots = table[g, j // page_rows] * page_rows + j % page_rows
        there = (table[g, j // page_rows] >= 0) & (slots < st.capacity)
        at = torch.from_numpy(np.where(there, slots, 0)).cuda()
        cc = codes[at]
        if fmt == R.NATIVE:
            r = as64(cc.view(TYPES[vtype])[:, :dim])
        else:
            r = P.dequantise(cc.cpu().numpy(), scales[at].cpu().numpy(), dim, fmt, block)
        with np.errstate(invalid="ignore"):
            p = q[lo:hi] @ r.T
            size = np.abs(q[lo:hi]) @ np.abs(r).T
        want[lo:hi, :n] = np.where(there, 1 - p if form == R.DISTANCE else p, np.inf if form == R.DISTANCE else -np.inf)
        # every partial sum is at most `size` and is rounded (or cut off) to fp32: dim additions, one product a block, the planes of
        # an fp32 operand that are left out (2^-24 of a product each), and the distance's own rounding
        bound[lo:hi, :n] = np.where(there, size * (dim + 16) * 2.0 ** -23 + (1 + size) * 2.0 ** -23, 0)
    nan = np.isnan(want)
    assert (np.isnan(got) == nan).all()
    inf = np.isinf(want)
    assert (got[inf] == want[inf]).all()
    ok = ~nan & ~inf
    worst = np.max(np.abs(got[ok] - want[ok]) - bound[ok])
    assert worst <= 0, worst
    return scores


def filled(gen, vtype, dim, fmt, block, capacity):
    cache = Cache(vtype, dim, fmt, block, capacity, zero=True)
    for at in range(0, capacity, 8192):
        n = min(8192, capacity - at)
        cache.write(values(gen, n, dim, vtype), torch.arange(at, at + n, device="cuda"))
    return cache


ALL = [(t, f, b) for t in TYPES for f in (R.NATIVE, R.INT8, R.E4M3, R.INT4) for b in (0, 32, 64, 128) if f != R.NATIVE or b == 0]


@pytest.mark.parametrize("vtype,fmt,block", ALL)
@pytest.mark.parametrize("dim", [1, 33, 100, 128, 300, 1000])
def test_scores(vtype, fmt, block, dim):
    gen = torch.Generator().manual_seed(dim + fmt)
    page_rows, capacity = 16, 16 * 40
    cache = filled(gen, vtype, dim, fmt, block, capacity)
    pages = torch.randperm(40, generator=gen).to(torch.int32)[:36].view(4, 9).contiguous().cuda()
    queries = strided(values(gen, 41, dim, vtype), 3 if dim == 100 else 0)
    check_scores(cache.c, cache.codes, cache.scales, queries, [0, 33, 33, 34, 41], pages, page_rows, [130, 5, 144, 1], R.PRODUCT, 150)


@pytest.mark.parametrize("vtype,fmt,block", [(P.F32, R.INT8, 0), (P.F16, R.E4M3, 128), (P.BF16, R.INT4, 32), (P.BF16, R.NATIVE, 0), (P.F32, R.NATIVE, 0)])
@pytest.mark.parametrize("counts,offsets", [([300], [0, 200]), ([300, 300], [3, 260, 390]), ([1, 0, 129], [0, 1, 1, 129]),
                                            ([128, 127], [0, 127, 255])])
@pytest.mark.parametrize("form", [R.PRODUCT, R.DISTANCE])
def test_scores_of_many_queries(vtype, fmt, block, counts, offsets, form):
    gen = torch.Generator().manual_seed(len(counts))
    dim, page_rows = 200, 100
    cache = filled(gen, vtype, dim, fmt, block, 1000)
    pages = torch.randperm(10, generator=gen).to(torch.int32)[: 3 * len(counts)].view(len(counts), 3).contiguous().cuda()
    queries = values(gen, offsets[-1] + 5, dim, vtype)
    check_scores(cache.c, cache.codes, cache.scales, queries, offsets, pages, page_rows, counts, form, 301)


@pytest.mark.parametrize("page_rows", [1, 7, 64, 1000])
@pytest.mark.parametrize("form", [R.PRODUCT, R.DISTANCE])
def test_scores_of_pages_that_are_not_there(page_rows, form):
    gen = torch.Generator().manual_seed(page_rows)
    dim, capacity = 96, 500
    cache = filled(gen, P.F16, dim, R.INT8, 32, capacity)
    many = -(-400 // page_rows)
    pages = torch.randint(0, max(1, capacity // page_rows), (3, many), generator=gen, dtype=torch.int32)   # pages may be shared
    pages[:, ::3] = -1
    pages[1] = -5                                                         # a partition whose pages are all gone
    pages[2, -1] = 2 ** 31 - 1
    check_scores(cache.c, cache.codes, cache.scales, values(gen, 9, dim, P.F16), [0, 3, 6, 9], pages.cuda(), page_rows,
                 [min(400, many * page_rows), 17, min(400, many * page_rows)], form, 400)


def test_scores_of_counts_and_offsets_out_of_range():
    gen = torch.Generator().manual_seed(5)
    cache = filled(gen, P.F32, 64, R.INT8, 64, 256)
    pages = torch.arange(8, dtype=torch.int32).view(4, 2).cuda()
    q = values(gen, 10, 64, P.F32)
    args = (cache.c, cache.codes, cache.scales, q)
    check_scores(*args, [-3, 2, 1, 9, 2 ** 31 - 1], pages, 32, [1000, 5, -4, 40], R.PRODUCT, 50)      # falls: nothing; behind: cut
    check_scores(*args, [0, 0, 0, 0, 0], pages, 32, [64] * 4, R.PRODUCT, 64)                          # nobody asks
    check_scores(*args, [0, 3, 5, 8, 10], pages, 32, [0] * 4, R.DISTANCE, 64)                         # nobody has rows
    check_scores(*args, [10, 10, 10, 10, 10], pages, 32, [64] * 4, R.PRODUCT, 64)


@pytest.mark.parametrize("partitions", [255, 256, 257, 1500])
def test_scores_of_many_partitions(partitions):
    gen = torch.Generator().manual_seed(partitions)
    cache = filled(gen, P.BF16, 40, R.E4M3, 0, 512)
    counts = torch.randint(0, 40, (partitions,), generator=gen).tolist()
    asked = torch.randint(0, 3, (partitions,), generator=gen).tolist()
    offsets = [0] + np.cumsum(asked).tolist()
    pages = torch.randint(0, 64, (partitions, 5), generator=gen, dtype=torch.int32).cuda()
    check_scores(cache.c, cache.codes, cache.scales, values(gen, max(1, offsets[-1]), 40, P.BF16), offsets, pages, 8, counts, R.PRODUCT, 40)


def test_scores_of_one_query_and_one_row():
    gen = torch.Generator().manual_seed(9)
    for vtype, fmt, block in ALL:
        cache = filled(gen, vtype, 17, fmt, block, 1)
        check_scores(cache.c, cache.codes, cache.scales, values(gen, 1, 17, vtype), [0, 1], torch.zeros((1, 1), dtype=torch.int32, device="cuda"), 1, [1], R.PRODUCT, 1)


@pytest.mark.parametrize("vtype,fmt", [(P.F32, R.NATIVE), (P.BF16, R.NATIVE), (P.F16, R.INT8), (P.F32, R.E4M3), (P.F32, R.INT4)])
def test_scores_with_infinities_and_nan(vtype, fmt):
    """A row with a NaN, a block kept as NaN, a query with an infinity: they reach their own scores and no others."""
    gen = torch.Generator().manual_seed(3)
    dim = 70
    rows = values(gen, 64, dim, vtype)
    rows[3, 5] = float("nan")
    rows[40, 69] = float("inf")
    rows[41, 69] = 1e4
    cache = Cache(vtype, dim, fmt, 0 if fmt == R.NATIVE else 32, 64, zero=True)
    cache.write(rows, torch.arange(64, device="cuda"))
    q = values(gen, 6, dim, vtype)
    q[:, 69] = 1.0
    q[2, 0] = float("inf")
    q[4, 7] = float("nan")
    scores = torch.zeros((6, 64), device="cuda")
    off, pages, cnt = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, 6], [[0]], [64]))
    cache.c.partition_scores(q.data_ptr(), dim, 6, off.data_ptr(), 1, pages.data_ptr(), 1, 64, cnt.data_ptr(), R.PRODUCT, scores.data_ptr(), 64, stream())
    got = scores.cpu().numpy()
    codes, scales = cache.plain()
    r = as64(cache.codes.view(TYPES[vtype])[:, :dim]) if fmt == R.NATIVE else P.dequantise(codes, scales, dim, fmt, 32)
    with np.errstate(invalid="ignore"):
        want = (as64(q)[:, None, :] * r[None]).sum(-1)
    assert (np.isnan(got) == np.isnan(want)).all() and (np.isposinf(got) == np.isposinf(want)).all() and (np.isneginf(got) == np.isneginf(want)).all()
    fine = np.isfinite(want)
    assert fine[[0, 1, 3, 5]].sum() >= 4 * 61


def test_scores_past_32_bits_of_cells():
    """Three queries 2^30 cells apart: the last one's scores lie 8 GiB behind the first's."""
    gen = torch.Generator().manual_seed(4)
    cache = filled(gen, P.F16, 64, R.INT8, 0, 64)
    ld = 1 << 30
    scores = torch.empty(2 * ld + 64, device="cuda")
    q = values(gen, 3, 64, P.F16)
    off, pages, cnt = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, 3], [[0]], [64]))
    cache.c.partition_scores(q.data_ptr(), 64, 3, off.data_ptr(), 1, pages.data_ptr(), 1, 64, cnt.data_ptr(), R.PRODUCT, scores.data_ptr(), ld, stream())
    got = np.stack([as64(scores[i * ld: i * ld + 64]) for i in range(3)])
    r = P.dequantise(*cache.plain(), 64, R.INT8, 0)
    size = np.abs(as64(q)) @ np.abs(r).T
    assert (np.abs(got - as64(q) @ r.T) <= size * 81 * 2.0 ** -23).all()


# ---- rules ---------------------------------------------------------------------------------------------------------------------

def check_adjust(arrays, scores, counts, ld_gap=0, in_place=False, form=R.PRODUCT):
    nq, nc = scores.shape
    wide = np.full((nq, nc + ld_gap), 9.0, np.float32)
    wide[:, :nc] = scores
    src = torch.from_numpy(wide).cuda()
    dst = src if in_place else torch.full_like(src, 77.0)
    dev = {k: torch.from_numpy(v).cuda() for k, v in arrays.items() if v is not None and v.size}
    fields = {k: v.data_ptr() for k, v in dev.items()}
    if "mask" in arrays:
        fields.update(mask_words=arrays["mask"].shape[1], n_masks=arrays["mask"].shape[0])
    if "seen_ids" in arrays:
        fields["n_seen"] = arrays["seen_ids"].size
    if "bias_ids" in arrays:
        fields["n_bias"] = arrays["bias_ids"].size
    cnt = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    R.adjust_scores(R.score_rules(form=form, **fields), src.data_ptr(), dst.data_ptr(), nq, nc, nc + ld_gap, cnt.data_ptr() if cnt is not None else None, stream())
    got = dst.cpu().numpy()
    before = wide if in_place else np.full_like(wide, 77.0)
    want, slack = P.adjust(dict(arrays, form=form), scores, before[:, :nc], counts)
    assert (got[:, nc:] == before[:, nc:]).all()
    got = got[:, :nc].astype(np.float64)
    assert (np.isnan(got) == np.isnan(want)).all()
    fine = np.isfinite(want)
    assert (got[~fine & ~np.isnan(want)] == want[~fine & ~np.isnan(want)]).all()
    assert (np.abs(got[fine] - want[fine]) <= slack[fine]).all()
    return got


def lists(rng, nq, nc, most, dup=True):
    lens = rng.integers(0, most + 1, nq)
    lens[0] = most
    idx = rng.integers(0, nc, lens.sum()) if not dup else (rng.random(lens.sum()) ** 3 * nc).astype(np.int64)
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32), idx.astype(np.int32)


@pytest.mark.parametrize("nc", [1, 31, 32, 33, 4095, 4096, 4097, 10001])
@pytest.mark.parametrize("form", [R.PRODUCT, R.DISTANCE])
@pytest.mark.parametrize("in_place", [False, True])
def test_adjust(nc, form, in_place):
    rng = np.random.default_rng(nc)
    nq = 6
    scores = rng.standard_normal((nq, nc)).astype(np.float32)
    so, si = lists(rng, nq, nc, 200)
    bo, bi = lists(rng, nq, nc, 40)
    arrays = dict(mask=rng.integers(0, 2 ** 32, (3, nc // 32 + 2), dtype=np.uint32), mask_rows=np.array([0, 2, -1, 3, 1, 0], np.int32),
                  seen_offsets=so, seen_ids=si, bias_offsets=bo, bias_ids=bi, bias_values=rng.standard_normal(bi.size).astype(np.float32),
                  repetition=(1 + rng.random(nq)).astype(np.float32), frequency=rng.random(nq).astype(np.float32), presence=rng.random(nq).astype(np.float32))
    check_adjust(arrays, scores, [nc, nc // 2, nc, 0, nc + 5, -1], ld_gap=nc % 3, in_place=in_place, form=form)
    for keys in (("mask",), ("seen_offsets", "seen_ids"), ("bias_offsets", "bias_ids", "bias_values"), ("seen_offsets", "seen_ids", "repetition"), ()):
        part = {k: arrays[k] for k in keys}
        if keys == ("mask",):
            part["mask_rows"] = arrays["mask_rows"]
        check_adjust(part, scores, None, in_place=in_place, form=form)


def test_adjust_cells_without_a_rule_keep_their_bits():
    scores = np.random.default_rng(0).integers(0, 2 ** 32, (2, 5000), dtype=np.uint32).view(np.float32)
    src = torch.from_numpy(scores.view(np.int32)).cuda()
    dst = torch.zeros_like(src)
    seen = torch.tensor([10, 4999], dtype=torch.int32, device="cuda")
    off = torch.tensor([0, 2, 2], dtype=torch.int32, device="cuda")
    for form in (R.PRODUCT, R.DISTANCE):
        rules = R.score_rules(form=form, seen_offsets=off.data_ptr(), seen_ids=seen.data_ptr(), n_seen=2)
        R.adjust_scores(rules, src.data_ptr(), dst.data_ptr(), 2, 5000, 5000, None, stream())
        a, b = src.cpu().numpy(), dst.cpu().numpy()
        a[0, [10, 4999]] = b[0, [10, 4999]] = 0
        assert (a == b).all()


def test_adjust_masks_that_leave_nothing_and_one_that_has_no_words_to_spare():
    scores = np.random.default_rng(1).standard_normal((3, 64)).astype(np.float32)
    scores[0, 0], scores[1, 1], scores[2, 2] = np.nan, np.inf, -np.inf
    mask = np.zeros((3, 2), np.uint32)
    mask[1] = 0xFFFFFFFF
    mask[2, 1] = 0x80000000
    for form in (R.PRODUCT, R.DISTANCE):
        check_adjust(dict(mask=mask), scores, None, form=form)


def test_adjust_special_scores_and_penalties():
    """Zeros, infinities, NaN and the type's lowest value under every rule."""
    scores = np.array([[0.0, -0.0, np.inf, -np.inf, np.nan, -3.4028235e38, 3.4028235e38, 1e-45]], np.float32)
    one = np.arange(8, dtype=np.int32)
    off = np.array([0, 8], np.int32)
    for form in (R.PRODUCT, R.DISTANCE):
        check_adjust(dict(seen_offsets=off, seen_ids=one, repetition=np.array([1.5], np.float32)), scores[:, :5] if form else scores[:, [0, 1, 2, 3, 4]], None, form=form)
        check_adjust(dict(bias_offsets=off, bias_ids=one, bias_values=np.ones(8, np.float32)), scores, None, form=form)


def test_adjust_lists_out_of_range():
    rng = np.random.default_rng(2)
    scores = rng.standard_normal((4, 100)).astype(np.float32)
    idx = np.array([-1, 100, 5, 5, 2 ** 31 - 1, -2 ** 31, 99, 0], np.int32)
    arrays = dict(seen_offsets=np.array([0, 8, 3, 2000, 5], np.int32), seen_ids=idx, bias_offsets=np.array([-7, 4, 4, 8, 8], np.int32), bias_ids=idx,
                  bias_values=np.arange(8, dtype=np.float32), frequency=np.ones(4, np.float32))
    check_adjust(arrays, scores, None)


def test_adjust_of_an_id_that_comes_again():
    """Counted as often as it comes; the last boost holds, wherever in the list the two are."""
    scores = np.ones((1, 5000), np.float32)
    seen = np.full(3000, 4500, np.int32)
    bias = np.tile(np.array([4500, 7], np.int32), 700)
    got = check_adjust(dict(seen_offsets=np.array([0, 3000], np.int32), seen_ids=seen, frequency=np.array([0.5], np.float32),
                            bias_offsets=np.array([0, 1400], np.int32), bias_ids=bias, bias_values=np.arange(1400, dtype=np.float32)), scores, None)
    assert got[0, 4500] == 1 - 1500 + 1398 and got[0, 7] == 1 + 1399


# ---- as they are used ------------------------------------------------------------------------------------------------------------

def test_all_calls_in_a_graph():
    """Recorded once, replayed with new inputs between eager work: write, read, scores and rules follow each other on one stream."""
    gen = torch.Generator().manual_seed(11)
    dim, n = 200, 300
    cache = Cache(P.F32, dim, R.INT8, 64, n, zero=True)
    rows, back = torch.zeros((n, dim), device="cuda"), torch.zeros((n, dim), device="cuda")
    slots = torch.randperm(n, generator=gen).cuda()
    q = torch.zeros((7, dim), device="cuda")
    off, cnt = torch.tensor([0, 3, 7], dtype=torch.int32, device="cuda"), torch.tensor([150, 99], dtype=torch.int32, device="cuda")
    pages = torch.randperm(10, generator=gen).to(torch.int32).view(2, 5).contiguous().cuda()
    scores, final = torch.zeros((7, 150), device="cuda"), torch.zeros((7, 150), device="cuda")
    seen, so = torch.tensor([3, 3, 9, 20], dtype=torch.int32, device="cuda"), torch.tensor([0, 2, 3, 4, 4, 4, 4, 4], dtype=torch.int32, device="cuda")
    freq = torch.full((7,), 0.25, device="cuda")
    rules = R.score_rules(seen_offsets=so.data_ptr(), seen_ids=seen.data_ptr(), n_seen=4, frequency=freq.data_ptr())

    def calls():
        cache.write(rows, slots)
        cache.c.read(slots.data_ptr(), n, back.data_ptr(), dim, stream())
        cache.c.partition_scores(q.data_ptr(), dim, 7, off.data_ptr(), 2, pages.data_ptr(), 5, 30, cnt.data_ptr(), R.PRODUCT, scores.data_ptr(), 150, stream())
        R.adjust_scores(rules, scores.data_ptr(), final.data_ptr(), 7, 150, 150, None, stream())

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    for k in range(4):
        rows.copy_(values(gen, n, dim, P.F32))
        q.copy_(values(gen, 7, dim, P.F32))
        scores.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (cache.codes, cache.scales, back, scores, final)]
        for t in (cache.codes, cache.scales, back, scores, final):
            t.zero_()
        calls()
        torch.cuda.synchronize()
        for a, b in zip(got, (cache.codes, cache.scales, back, scores, final)):
            assert torch.equal(a, b)
        assert final.abs().sum() > 0


def test_calls_on_two_streams_at_once():
    """Two callers with their own caches and streams: each gets what it gets alone."""
    gen = torch.Generator().manual_seed(12)
    dim, n = 512, 4096
    work = []
    for fmt in (R.INT8, R.INT4):
        cache = Cache(P.F16, dim, fmt, 128, n, zero=True)
        work.append((cache, values(gen, n, dim, P.F16), torch.randperm(n, generator=gen).cuda(), torch.zeros((n, dim), dtype=torch.float16, device="cuda")))
    alone = []
    for cache, rows, slots, back in work:
        cache.write(rows, slots)
        cache.c.read(slots.data_ptr(), n, back.data_ptr(), dim, stream())
        torch.cuda.synchronize()
        alone.append((cache.codes.clone(), back.clone()))
        cache.codes.zero_()
        back.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, (cache, rows, slots, back) in zip(streams, work):
            with torch.cuda.stream(s):
                cache.write(rows, slots)
                cache.c.read(slots.data_ptr(), n, back.data_ptr(), dim, stream())
    torch.cuda.synchronize()
    for (codes, back), (cache, _, _, b) in zip(alone, work):
        assert torch.equal(codes, cache.codes) and torch.equal(back, b)


def test_host_memory_is_refused():
    host = np.zeros(1 << 16, np.uint8)
    at = (host.ctypes.data + 63) // 64 * 64
    dev = torch.zeros(4096, device="cuda")
    c = R.RowCache(P.F32, 32, R.INT8, 0, 4, at, dev.data_ptr())
    with pytest.raises(RuntimeError, match="not device memory"):
        c.write(dev.data_ptr(), 32, dev.data_ptr(), 1)
    with pytest.raises(RuntimeError, match="not device memory"):
        R.adjust_scores(R.score_rules(), dev.data_ptr(), at, 1, 32, 32)


@pytest.mark.parametrize("vtype,fmt", [(P.F32, R.INT8), (P.F16, R.E4M3), (P.BF16, R.NATIVE)])
@pytest.mark.parametrize("metric", [V.VecSimMetric_Cosine, V.VecSimMetric_IP])
def test_an_index_its_cache_and_a_batch(vtype, fmt, metric):
    """Rows of an index go into a cache, a batch is scored against its partitions, rules are applied, the merge picks the best; and
    an index loaded from the cache answers with the same distances."""
    rng = np.random.default_rng(21)
    n, dim, page = 700, 90, 50
    x = rng.standard_normal((n, dim)).astype(np.float32)
    index = V.VecSimIndex(vtype, dim, metric)
    index.add_bulk(x)
    cache = Cache(vtype, dim, fmt, 0 if fmt == R.NATIVE else 32, n, zero=True)
    slots = torch.from_numpy(rng.permutation(n)).cuda()
    cache.c.cache_rows(index, 0, n, slots.data_ptr(), stream())
    stored = index.read_rows(0, n)
    stored = stored.astype(np.float64) if vtype != P.BF16 else (stored.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    at = slots.cpu().numpy()
    codes, scales = cache.plain()
    if fmt != R.NATIVE:
        wc, ws = P.quantise(stored, fmt, 32)
        assert (codes[at] == wc).all() and (scales[at] == ws).all()

    # partition g: pages g, g + 3, ... ; a batch of 12, four each
    table = torch.tensor([[g + 3 * i if g + 3 * i < n // page else -1 for i in range(5)] for g in range(3)], dtype=torch.int32, device="cuda")
    counts = [250, 230, 200]
    q = torch.from_numpy(rng.standard_normal((12, dim)).astype(np.float32)).cuda()
    q = (q / q.norm(dim=1, keepdim=True)).to(TYPES[vtype])
    scores = check_scores(cache.c, cache.codes, cache.scales, q, [0, 4, 8, 12], table, page, counts, R.DISTANCE, 250)[:12].contiguous()
    mask = rng.integers(0, 2 ** 32, (12, 8), dtype=np.uint32)
    so, si = np.arange(0, 13, dtype=np.int32), rng.integers(0, 200, 12).astype(np.int32)
    per = torch.tensor(np.repeat(counts, 4), dtype=torch.int32, device="cuda")
    dev = {k: torch.from_numpy(v).cuda() for k, v in dict(mask=mask, seen_offsets=so, seen_ids=si, presence=np.full(12, 0.3, np.float32)).items()}
    before = as64(scores)
    R.adjust_scores(R.score_rules(form=R.DISTANCE, mask_words=8, n_masks=12, n_seen=12, **{k: v.data_ptr() for k, v in dev.items()}),
                    scores.data_ptr(), scores.data_ptr(), 12, 250, 250, per.data_ptr(), stream())
    labels = torch.arange(250, device="cuda")
    torch.cuda.synchronize()
    for m in (0, 5, 11):
        nrow = counts[m // 4]
        d = before[m, :nrow].copy()
        d[si[m]] += 0.3
        bits = np.unpackbits(mask[m].view(np.uint8), bitorder="little")[:nrow]
        d = np.where(bits == 1, d, np.inf)
        out_s, out_l = np.zeros(10), np.zeros(10, np.uint64)
        got = V.load().RSGPU_MergeTopK(0, scores[m].data_ptr(), labels.data_ptr(), nrow, 10, out_s.ctypes.data_as(C.c_void_p), out_l.ctypes.data_as(C.c_void_p), stream())
        assert got == 10
        best = np.lexsort((np.arange(nrow), d.astype(np.float32)))[:10]
        assert (np.sort(d)[:10] <= out_s + 1e-6).all() and np.abs(d[out_l.astype(int)] - out_s).max() < 1e-6
        assert np.abs(np.sort(d)[:10] - out_s).max() < 1e-6 and len(set(out_l.tolist())) == 10 and best.size == 10

    loaded = V.VecSimIndex(vtype, dim, metric)
    assert cache.c.add_to(loaded, slots.data_ptr(), n, 1, stream()) == n
    want = P.dequantise(codes[at], scales[at], dim, fmt, 32) if fmt != R.NATIVE else stored
    back = loaded.read_rows(0, n)
    back = back.astype(np.float64) if vtype != P.BF16 else (back.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    if metric == V.VecSimMetric_Cosine:
        want = want / np.linalg.norm(want, axis=1, keepdims=True)
    # the value rounded to the type, the norm's sum and root in fp32, and the quotient rounded to the type again
    assert (np.abs(back - want) <= np.abs(want) * (2 * P.EPS[vtype] + (dim + 4) * 2.0 ** -24) + 2 * P.LEAST[vtype] + 1e-7 * (vtype == P.F16)).all()
    a = loaded.topk_query(as64(q)[0].astype(np.float32), 5).results()
    assert a[0].size == 5


def test_an_index_refuses_another_cache():
    index = V.VecSimIndex(P.F32, 64, V.VecSimMetric_IP)
    index.add_bulk(np.ones((4, 64), np.float32))
    slots = torch.arange(8, device="cuda")
    for vtype, dim in ((P.F16, 64), (P.F32, 65)):
        cache = Cache(vtype, dim, R.INT8, 0, 8)
        with pytest.raises(RuntimeError, match="another type or dim"):
            cache.c.cache_rows(index, 0, 4, slots.data_ptr())
        with pytest.raises(RuntimeError, match="another type or dim"):
            cache.c.add_to(index, slots.data_ptr(), 4)
    cache = Cache(P.F32, 64, R.INT8, 0, 8, zero=True)
    for begin, n in ((0, 5), (5, 0), (4, 1), (2 ** 62, 2)):
        with pytest.raises(RuntimeError, match="range beyond"):
            cache.c.cache_rows(index, begin, n, slots.data_ptr())
    with pytest.raises(RuntimeError, match="label range overlaps"):
        cache.c.add_to(index, slots.data_ptr(), 4, 2)
    assert index.index_size() == 4 and not cache.codes.any()


@pytest.mark.parametrize("vtype,fmt,block", ALL)
@pytest.mark.parametrize("dim,counts,offsets", [(33, [300, 50], [0, 33, 40]), (768, [130, 257], [0, 32, 33]), (1500, [40], [0, 47]), (200, [70, 0, 65], [1, 17, 40, 90])])
def test_scores_of_a_few_dozen_queries(vtype, fmt, block, dim, counts, offsets):
    """13 to 47 queries a partition on average: tiles of 32 queries, one of them cut, rows longer than what LDS holds of the queries."""
    gen = torch.Generator().manual_seed(dim)
    page_rows = 13
    need = -(-max(counts) // page_rows)
    cache = filled(gen, vtype, dim, fmt, block, page_rows * need * len(counts))
    pages = torch.randperm(need * len(counts), generator=gen).to(torch.int32).view(len(counts), need).contiguous().cuda()
    check_scores(cache.c, cache.codes, cache.scales, values(gen, offsets[-1] + 2, dim, vtype), offsets, pages, page_rows, counts, R.DISTANCE, max(counts) + 1)


@pytest.mark.parametrize("vtype,fmt,block", [(P.F32, R.INT8, 128), (P.F16, R.INT4, 64), (P.BF16, R.NATIVE, 0), (P.F32, R.NATIVE, 0)])
def test_scores_where_one_partition_has_all_the_queries(vtype, fmt, block):
    """The average says few queries a partition, one partition has hundreds."""
    gen = torch.Generator().manual_seed(77)
    cache = filled(gen, vtype, 96, fmt, block, 640)
    pages = torch.arange(640 // 16, dtype=torch.int32).view(40, 1).cuda()
    offsets = [0] * 20 + [210] * 21
    check_scores(cache.c, cache.codes, cache.scales, values(gen, 210, 96, vtype), offsets, pages, 16, [16] * 40, R.PRODUCT, 16)


@pytest.mark.parametrize("vtype", list(TYPES), ids=ids)
@pytest.mark.parametrize("dim", [1, 5, 7, 8, 9, 15, 31, 63, 65, 95])
def test_scores_of_many_queries_of_every_odd_width(vtype, dim):
    """The ends of queries that are no multiple of anything, in the kernel that takes a hundred and more a partition; the memory right
    behind the last query is not the caller's."""
    gen = torch.Generator().manual_seed(dim)
    for fmt, block in ((R.INT8, 0), (R.NATIVE, 0), (R.INT4, 32)):
        cache = filled(gen, vtype, dim, fmt, block, 160)
        pages = torch.arange(10, dtype=torch.int32).view(1, 10).cuda()
        q = values(gen, 131, dim, vtype)
        guarded = torch.full((131 * dim + 64,), float("nan"), dtype=q.dtype, device="cuda")
        guarded[: 131 * dim] = q.reshape(-1)
        check_scores(cache.c, cache.codes, cache.scales, guarded[: 131 * dim].view(131, dim), [0, 131], pages, 16, [150], R.PRODUCT, 160)


def test_writes_at_the_end_of_memory():
    """The last row of an array of odd width: what lies behind it (NaN here) does not get into its block."""
    for vtype in TYPES:
        for dim in (3, 9, 33, 100, 515, 1037):
            for block in (0, 32):
                data = torch.full((5 * dim + 16,), float("nan"), dtype=TYPES[vtype], device="cuda")
                data[: 5 * dim] = torch.randn(5 * dim, device="cuda").to(TYPES[vtype])
                rows = data[: 5 * dim].view(5, dim)
                cache = Cache(vtype, dim, R.INT8, block, 5)
                cache.write(rows, torch.arange(5, device="cuda"))
                codes, scales = cache.plain()
                want_codes, want_scales = P.quantise(as64(rows), R.INT8, block)
                np.testing.assert_array_equal(scales, want_scales)
                np.testing.assert_array_equal(codes, want_codes)


def test_a_row_with_nan_leaves_its_neighbours_alone():
    """A full load of a row's end reads into the next row; a NaN there stays out of this one's block."""
    for vtype in TYPES:
        for dim, block in ((33, 0), (100, 32), (517, 0), (1030, 0), (1030, 128)):
            rows = torch.randn((6, dim), device="cuda").to(TYPES[vtype])
            rows[1::2, 0] = float("nan")
            cache = Cache(vtype, dim, R.E4M3, block, 6)
            cache.write(rows, torch.arange(6, device="cuda"))
            codes, scales = cache.plain()
            want_codes, want_scales = P.quantise(as64(rows), R.E4M3, block)
            np.testing.assert_array_equal(scales, want_scales)
            np.testing.assert_array_equal(codes, want_codes)


def test_overlapping_ranges_of_queries_stay_in_bounds():
    """Offsets that fall and rise again: every range that is one is answered."""
    gen = torch.Generator().manual_seed(8)
    cache = filled(gen, P.F16, 64, R.INT8, 0, 64)
    pages = torch.zeros((5, 1), dtype=torch.int32, device="cuda")
    check_scores(cache.c, cache.codes, cache.scales, values(gen, 20, 64, P.F16), [0, 20, 0, 20, 5, 9], pages, 64, [64] * 5, R.PRODUCT, 64)


def check_scores_in_a_wide_table(cache, queries, offsets, pages, page_rows, counts, form, ld):
    """The same call, in a table and an array of scores that allow 70 000 rows a partition, which is what the kernel is chosen by; the
    columns that no partition has are compared on the GPU."""
    wide = -(-70000 // page_rows)
    table = torch.full((len(counts), wide), -1, dtype=torch.int32, device="cuda")
    table[:, : pages.shape[1]] = pages
    out = torch.full((queries.shape[0] + 1, 70001), 123.0, device="cuda")

    class Wide:
        c = cache.c.c

        def partition_scores(self, q, stride, m, off, n, narrow, max_pages, page_rows, cnt, form, scores, ld, s):
            cache.c.partition_scores(q, stride, m, off, n, table.data_ptr(), wide, page_rows, cnt, form, out.data_ptr(), 70001, s)
            # the first columns go where the check looks for them
            there = torch.arange(m + 1, device="cuda")
            kept = out[:, :ld].contiguous()
            R.RowCache(P.F32, ld, R.NATIVE, 0, m + 1, kept.data_ptr(), None).read(there.data_ptr(), m + 1, scores, ld, s)
            torch.cuda.synchronize()

    check_scores(Wide(), cache.codes, cache.scales, queries, offsets, pages, page_rows, counts, form, ld)
    assert (out[:, ld:] == 123).all() and (out[-1] == 123).all()


@pytest.mark.parametrize("vtype,fmt,block", ALL)
@pytest.mark.parametrize("dim", [33, 300, 768])
@pytest.mark.parametrize("offsets", [[0, 0, 4, 7, 20, 22, 23, 24, 40], [0, 17, 20, 20, 33, 49, 60, 72, 100], [0, 40, 41, 90, 90, 100, 101, 133, 180]],
                         ids=["few", "tens", "dozens"])
def test_scores_in_tables_of_many_rows(vtype, fmt, block, dim, offsets):
    """The kernels for long partitions, at partitions of none, one and a tile and a bit."""
    gen = torch.Generator().manual_seed(dim + len(offsets) + fmt)
    counts, page_rows = [33, 600, 1, 0, 257, 1100, 64, 16], 32
    need = [-(-n // page_rows) for n in counts]
    cache = filled(gen, vtype, dim, fmt, block, page_rows * sum(need))
    pages = torch.full((8, max(need)), -1, dtype=torch.int32)
    pages[torch.arange(max(need))[None, :] < torch.tensor(need)[:, None]] = torch.randperm(sum(need), generator=gen).to(torch.int32)
    check_scores_in_a_wide_table(cache, values(gen, offsets[-1], dim, vtype), offsets, pages.cuda(), page_rows, counts, R.PRODUCT, 1120)


@pytest.mark.parametrize("vtype", list(TYPES), ids=ids)
@pytest.mark.parametrize("dim", [1, 2, 3, 4, 5, 7])
def test_narrow_rows_up_to_the_end_of_an_allocation(vtype, dim):
    """Rows of less than eight elements whose array ends where its allocation (32 MiB, a whole number of pages) does."""
    size = torch.empty((), dtype=TYPES[vtype]).element_size()
    whole = torch.zeros(32 * 2 ** 20 // size, dtype=TYPES[vtype], device="cuda")
    rows = whole[whole.numel() - 9 * dim:].view(9, dim)
    rows.copy_(values(torch.Generator().manual_seed(dim), 9, dim, vtype))
    for fmt in FORMATS:
        cache = Cache(vtype, dim, fmt, 0, 9)
        cache.write(rows, torch.arange(9, device="cuda"))
        codes, scales = cache.plain()
        want_codes, want_scales = P.quantise(as64(rows), fmt, 0)
        assert (codes == want_codes).all() and (scales == want_scales).all()


def test_adjust_lists_that_end_at_the_last_entry():
    """Lists of 2^31 - 1 entries, the queries' own at their ends."""
    n = 2 ** 31 - 1
    seen = torch.empty(n, dtype=torch.int32, device="cuda")
    seen[-300:] = torch.arange(300, dtype=torch.int32, device="cuda")
    seen[-1] = 7
    boosts = torch.empty(n, device="cuda")
    boosts[-2:] = torch.tensor([2.0, 4.0], device="cuda")
    scores = torch.ones((2, 400), device="cuda")
    so = torch.tensor([n - 300, n - 1, n], dtype=torch.int32, device="cuda")
    bo = torch.tensor([n - 2, n, n], dtype=torch.int32, device="cuda")
    freq = torch.full((2,), 0.5, device="cuda")
    rules = R.score_rules(seen_offsets=so.data_ptr(), seen_ids=seen.data_ptr(), n_seen=n, bias_offsets=bo.data_ptr(), bias_ids=seen.data_ptr(),
                          bias_values=boosts.data_ptr(), n_bias=n, frequency=freq.data_ptr())
    R.adjust_scores(rules, scores.data_ptr(), scores.data_ptr(), 2, 400, 400, None, stream())
    want = np.ones((2, 400))
    want[0, :299] -= 0.5
    want[0, 298] += 2
    want[0, 7] += 4
    want[1, 7] -= 0.5
    assert (scores.cpu().numpy() == want).all()


@pytest.mark.parametrize("partitions,queries", [(2048, 300), (2049, 5), (2300, 9), (9001, 200), (9001, 12000), (20011, 700), (2050, 2050 * 81)])
def test_scores_of_thousands_of_partitions(partitions, queries):
    """More than a thread of a workgroup takes, a few of them with queries; in the last case all."""
    gen = torch.Generator().manual_seed(partitions + queries)
    cache = filled(gen, P.F16, 16, R.INT8, 0, 512)
    counts = torch.randint(0, 12, (partitions,), generator=gen).tolist()
    counts[-1] = 9
    who = torch.randint(0, partitions, (queries,), generator=gen)
    if queries == 5:
        who[:] = partitions - 1                                    # all of them ask the last partition
    offsets = torch.searchsorted(who.sort().values, torch.arange(partitions + 1)).tolist()
    pages = torch.randint(0, 64, (partitions, 2), generator=gen, dtype=torch.int32).cuda()
    check_scores(cache.c, cache.codes, cache.scales, values(gen, queries, 16, P.F16), offsets, pages, 8, counts, R.PRODUCT, 12)


def test_thousands_of_partitions_with_offsets_out_of_order_stay_in_bounds():
    gen = torch.Generator().manual_seed(3)
    cache = filled(gen, P.BF16, 16, R.INT4, 0, 512)
    n = 5000
    offsets = torch.randint(-50, 400, (n + 1,), generator=gen).to(torch.int32).cuda()
    counts = torch.randint(-5, 40, (n,), generator=gen).to(torch.int32).cuda()
    pages = torch.randint(-2, 70, (n, 2), generator=gen).to(torch.int32).cuda()
    q = values(gen, 300, 16, P.BF16)
    out = torch.full((302, 16), 5.0, device="cuda")
    cache.c.partition_scores(q.data_ptr(), 16, 300, offsets.data_ptr(), n, pages.data_ptr(), 2, 8, counts.data_ptr(), R.PRODUCT, out[1:].data_ptr(), 16, stream())
    torch.cuda.synchronize()
    assert (out[0] == 5).all() and (out[301] == 5).all()


@pytest.mark.parametrize("vtype,fmt,block", ALL)
@pytest.mark.parametrize("dim", [9, 40, 200, 768])
def test_scores_of_many_queries_in_tables_of_many_rows(vtype, fmt, block, dim):
    """The tiles of 256 rows (16-bit queries, rows of one scale or none) and those of 128, at their ends: partitions of one row, of a
    tile but one, of a tile and one, without queries."""
    gen = torch.Generator().manual_seed(dim + fmt)
    counts, page_rows = [255, 1, 700, 257], 48
    need = [-(-n // page_rows) for n in counts]
    cache = filled(gen, vtype, dim, fmt, block, page_rows * sum(need))
    pages = torch.full((4, max(need)), -1, dtype=torch.int32)
    pages[torch.arange(max(need))[None, :] < torch.tensor(need)[:, None]] = torch.randperm(sum(need), generator=gen).to(torch.int32)
    pages[2, 3] = -1                                                   # one that is gone
    check_scores_in_a_wide_table(cache, values(gen, 521, dim, vtype), [0, 129, 257, 257, 520], pages.cuda(), page_rows, counts, R.DISTANCE, 704)
