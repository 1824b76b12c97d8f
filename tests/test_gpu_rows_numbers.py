"""Partition scores on the GPU at the ends of the numbers: queries so large that a sum of codes leaves fp32, products of fp32 numbers to
their last bits, infinities and NaN in every kernel."""
import numpy as np
import pytest

from redisearch_amd import rows as R

from . import rows_plain as P
from .test_gpu_rows import TYPES, Cache, as64, check_scores, check_scores_in_a_wide_table, fids, ids, stream, values

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

# (queries of a partition, a table that allows 70 000 rows): which kernel takes the call goes by these.  In order: four wavefronts; eight
# or sixteen; those with rows that are kept; two tiles of queries (16-bit ones); the tiles of 128 rows; those of 256 (16-bit, one scale).
KERNELS = [(6, False), (6, True), (11, True), (20, True), (131, False), (131, True)]
SIZES = pytest.mark.parametrize("asked,wide", KERNELS, ids=["%d%s" % (m, "w" if w else "") for m, w in KERNELS])


def check(cache, queries, rows, wide, form=R.PRODUCT):
    """One partition, row j in slot j."""
    page_rows = 16
    pages = torch.arange(-(-rows // page_rows), dtype=torch.int32, device="cuda").view(1, -1)
    m, ld = queries.shape[0], -(-rows // 32) * 32       # (the wide table's check takes a whole number of 32 columns)
    if wide:
        check_scores_in_a_wide_table(cache, queries, [0, m], pages, page_rows, [rows], form, ld)
    else:
        check_scores(cache.c, cache.codes, cache.scales, queries, [0, m], pages, page_rows, [rows], form, ld)


@SIZES
@pytest.mark.parametrize("vtype", [P.F32, P.BF16], ids=ids)
@pytest.mark.parametrize("fmt,block", [(R.INT8, 0), (R.INT8, 128), (R.E4M3, 0), (R.E4M3, 32), (R.INT4, 0), (R.INT4, 64)])
def test_scores_of_queries_whose_sums_of_codes_leave_fp32(vtype, fmt, block, asked, wide):
    """Elements of 1e36 against rows of thousandths: the scores are numbers of 1e33 to 1e35, the sums of query times code are not."""
    gen = torch.Generator().manual_seed(fmt * 7 + block)
    dim, rows = 300, 272
    cache = Cache(vtype, dim, fmt, block, rows, zero=True)
    cache.write((torch.randn((rows, dim), generator=gen) * 1e-3).to(TYPES[vtype]).cuda(), torch.arange(rows, device="cuda"))
    q = torch.randn((asked, dim), generator=gen)
    large = 5e37 if fmt == R.INT4 else 1e36
    q[::3] *= large
    q[1::3] = q[1::3].abs() * large                     # of one sign: infinities, not NaN
    check(cache, q.to(TYPES[vtype]).cuda(), rows, wide, R.DISTANCE if block else R.PRODUCT)


# A number with 24 bits is three bf16.  Whichever way it is cut into them, what the products of the planes leave out is of the order of
# 2^-24 at best; a product of single elements shows it, where a sum of hundreds hides it behind its own rounding.
EDGES = [0x3f80ffff, 0x3fffffff, 0x3f7fffff, 0x3f808000, 0x3f818000, 0x3f80807f, 0x3f808080, 0x3f80ff80, 0x3fb504f3, 0x3f800001]


@SIZES
@pytest.mark.parametrize("dim", [40, 200, 768])
def test_products_of_single_fp32_elements(asked, wide, dim):
    """Rows with one element, at every place of a row: each score is one product."""
    gen = torch.Generator().manual_seed(dim + asked)
    rows = 800
    edges = torch.tensor(EDGES, dtype=torch.int32).view(torch.float32)
    x = 1 + torch.rand((rows,), generator=gen)
    x[::3] = edges[torch.arange(rows)[::3] % len(EDGES)]
    x[1::4] *= -2.0 ** torch.randint(-30, 30, (rows,), generator=gen)[1::4]
    q = 1 + torch.rand((asked, dim), generator=gen)
    q.view(-1)[::2] = edges[torch.arange(asked * dim)[::2] // 2 % len(EDGES)]
    q[1::2] *= -1
    where = torch.arange(rows) % dim
    data = torch.zeros((rows, dim))
    data[torch.arange(rows), where] = x
    cache = Cache(P.F32, dim, R.NATIVE, 0, rows, zero=True)
    cache.write(data.cuda(), torch.arange(rows, device="cuda"))
    got = one_partition(cache, q.cuda(), rows, wide)
    want = as64(q)[:, where.numpy()] * as64(x)[None]
    # x = hi + mid + lo, each the nearest bf16: |mid| <= 2^-8, |lo| <= 2^-17 of x's binade.  Left out are mid lo + lo mid + lo lo, no more
    # than 2^-24 + 2^-34 of |x y|.  The six products are exact and added smallest first, each sum rounded or cut off: five sums below
    # 2^-6 |x y| by 2^-23 of themselves, then the whole by 2^-23.  Zeros change nothing.
    assert (np.abs(got - want) <= np.abs(want) * (2.0 ** -23 + 5 * 2.0 ** -29 + 2.0 ** -24 + 2.0 ** -33)).all(), np.max(np.abs(got / want - 1)) * 2.0 ** 24


def one_partition(cache, q, rows, wide, page_rows=16):
    """Scores as float64, the call made in a table of the partition's rows or one that allows 70 000."""
    m, ld = q.shape[0], 70001 if wide else rows
    pages = torch.full((1, -(-ld // page_rows)), -1, dtype=torch.int32, device="cuda")
    have = -(-rows // page_rows)
    pages[0, :have] = torch.arange(have, dtype=torch.int32, device="cuda")
    scores = torch.zeros((m, ld), device="cuda")
    off, cnt = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, m], [rows]))
    cache.c.partition_scores(q.data_ptr(), q.stride(0), m, off.data_ptr(), 1, pages.data_ptr(), pages.shape[1], page_rows, cnt.data_ptr(),
                             R.PRODUCT, scores.data_ptr(), ld, stream())
    return as64(scores[:, :rows])


@SIZES
@pytest.mark.parametrize("fmt", [R.NATIVE, R.INT8, R.E4M3, R.INT4], ids=fids)
def test_products_of_the_largest_fp32_numbers(fmt, asked, wide):
    """Numbers next to the type's end, of which the nearest bf16 is an infinity, one to a row of the queries."""
    dim, rows = 96, 300
    top = torch.tensor([0x7f7fffff, 0x7f7f8000, 0x7f7f7fff, 0x7f7f0001, 0x7f7f8001, 0x7f000000], dtype=torch.int32).view(torch.float32)
    q = torch.zeros((asked, dim))
    at = torch.arange(asked) * 7 % dim
    q[torch.arange(asked), at] = top[torch.arange(asked) % 6] * (1 - 2.0 * (torch.arange(asked) % 2))
    data = torch.full((rows, dim), 2.0 ** -20)
    data[::3] = 1.0
    data[1::3] = -2.0 ** -90
    cache = Cache(P.F32, dim, fmt, 0, rows, zero=True)
    cache.write(data.cuda(), torch.arange(rows, device="cuda"))
    got = one_partition(cache, q.cuda(), rows, wide)
    stored = as64(data) if fmt == R.NATIVE else P.dequantise(*cache.plain(), dim, fmt, 0)
    want = as64(q)[np.arange(asked), at.numpy()][:, None] * stored[:, 0][None]
    # three products whose sum is rounded or cut off twice, and the scale's.  (7 times the fp32 number next to 1 / 7 is more than 1: what
    # passes the largest number by more than half a step, 2^-25 of it, is an infinity.)
    past = np.abs(want) > P.LARGEST[P.F32] * (1 + 2.0 ** -25)
    assert (got[past] == np.sign(want[past]) * np.inf).all()
    assert (np.abs(got - want)[~past] <= np.abs(want[~past]) * (2 * 2.0 ** -23 + 2.0 ** -24)).all()


@SIZES
@pytest.mark.parametrize("vtype,fmt,block", [(P.F32, R.NATIVE, 0), (P.BF16, R.NATIVE, 0), (P.F16, R.NATIVE, 0), (P.F32, R.INT8, 32), (P.BF16, R.INT8, 0),
                                             (P.F16, R.E4M3, 0), (P.BF16, R.E4M3, 128), (P.F16, R.INT4, 0), (P.F32, R.INT4, 0), (P.BF16, R.INT4, 64)])
def test_scores_with_infinities_and_nan_in_every_kernel(vtype, fmt, block, asked, wide):
    """A NaN, an infinity or a block kept as NaN reach the scores of their own row, a query's those of its own line, and no others: at the
    first and the last row, the first and the last element, on both sides of the tiles' borders."""
    gen = torch.Generator().manual_seed(fmt)
    dim, rows = 135, 530
    data = values(gen, rows, dim, vtype)
    inf, nan = float("inf"), float("nan")
    for row, at, value in [(0, 0, nan), (63, dim - 1, inf), (64, 31, -inf), (127, 32, inf), (128, dim - 1, nan), (255, 0, inf), (256, dim - 1, -inf),
                           (257, 64, nan), (511, 127, inf), (512, 128, nan), (rows - 1, dim - 1, inf)]:
        data[row, at] = value
    data[300, 5] = inf
    data[300, 90] = -inf
    q = values(gen, asked, dim, vtype)
    q[0, 0] = inf
    q[1, dim - 1] = -inf
    q[2, 64] = nan
    q[asked - 1, dim - 1] = nan
    if asked > 100:
        q[63, 3], q[64, 133], q[127, 134], q[128, 0] = inf, nan, -inf, inf
    cache = Cache(vtype, dim, fmt, block, rows, zero=True)
    cache.write(data, torch.arange(rows, device="cuda"))
    check(cache, q, rows, wide)


@SIZES
@pytest.mark.parametrize("vtype", [P.F32, P.BF16], ids=ids)
@pytest.mark.parametrize("fmt,block", [(R.NATIVE, 0), (R.INT8, 0), (R.E4M3, 32), (R.INT4, 128)])
def test_scores_of_tiny_queries(vtype, fmt, block, asked, wide):
    """Elements of 2^-60 down to 2^-125 against rows of ordinary size and of 2^60."""
    gen = torch.Generator().manual_seed(fmt + 3)
    dim, rows = 140, 270
    data = torch.randn((rows, dim), generator=gen)
    data[::4] *= 2.0 ** 60
    q = torch.randn((asked, dim), generator=gen) * torch.exp2(-60.0 - 65 * torch.arange(asked)[:, None] / asked)
    cache = Cache(vtype, dim, fmt, block, rows, zero=True)
    cache.write(data.to(TYPES[vtype]).cuda(), torch.arange(rows, device="cuda"))
    q = q.to(TYPES[vtype]).cuda()
    got = one_partition(cache, q, rows, wide)
    stored = as64(cache.codes.view(TYPES[vtype])[:, :dim]) if fmt == R.NATIVE else P.dequantise(*cache.plain(), dim, fmt, block)
    want, size = as64(q) @ stored.T, np.abs(as64(q)) @ np.abs(stored).T
    # fp32's own roundings (dim sums, a product a block, the unit's); an element's bits below 2^-107 are gone: times the row; a product or
    # sum has no bits below 2^-149 times the unit of 2^30, dim and a product a block of them times what the scale makes of it at most
    lost = 2.0 ** -107 * np.abs(stored).sum(1) + (dim + 8) * 2.0 ** -119 * np.maximum(1, np.abs(stored).max(1))
    assert (np.abs(got - want) <= size * (dim + 16) * 2.0 ** -23 + lost[None]).all()
