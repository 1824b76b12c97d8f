"""ctypes binding of include/rsgpu_rows.h: rows kept in 8 or 4 bits, the scores of a batch's queries against their own partitions'
rows, and the rules on a batch's scores.  Thin binding only: arrays are device addresses (ints), strides and leading dimensions
count elements, `stream` is a hipStream_t (None: the device's default stream), a refused call raises with the engine's message."""
import ctypes as C

from . import vecsim as V

_sz, _vp, _i, _u32, _u64 = C.c_size_t, C.c_void_p, C.c_int, C.c_uint32, C.c_uint64

NATIVE, INT8, E4M3, INT4 = 0, 1, 2, 3      # RSGPU_RowFormat
PRODUCT, DISTANCE = 0, 1                   # RSGPU_ScoreForm


class RowCacheStruct(C.Structure):
    _fields_ = [("device", _i), ("type", _i), ("format", _i), ("dim", _u32), ("block", _u32), ("capacity", _u64), ("codes", _vp),
                ("scales", _vp)]


class ScoreRules(C.Structure):
    _fields_ = [("device", _i), ("form", _i), ("mask", _vp), ("mask_words", _sz), ("n_masks", _sz), ("mask_rows", _vp),
                ("bias_offsets", _vp), ("bias_ids", _vp), ("bias_values", _vp), ("n_bias", _sz), ("seen_offsets", _vp), ("seen_ids", _vp),
                ("n_seen", _sz), ("repetition", _vp), ("frequency", _vp), ("presence", _vp)]


ABI = {
    "RSGPU_RowCache_RowBytes": (_sz, [C.POINTER(RowCacheStruct)]),
    "RSGPU_RowCache_RowScales": (_sz, [C.POINTER(RowCacheStruct)]),
    "RSGPU_RowCache_Write": (_i, [C.POINTER(RowCacheStruct), _vp, _sz, _vp, _sz, _vp]),
    "RSGPU_RowCache_Read": (_i, [C.POINTER(RowCacheStruct), _vp, _sz, _vp, _sz, _vp]),
    "RSGPU_RowCache_PartitionScores": (_i, [C.POINTER(RowCacheStruct), _vp, _sz, _sz, _vp, _sz, _vp, _sz, _sz, _vp, _i, _vp, _sz, _vp]),
    "RSGPU_AdjustScores": (_i, [C.POINTER(ScoreRules), _vp, _vp, _sz, _sz, _sz, _vp, _vp]),
    "RSGPU_FlatIndex_CacheRows": (_i, [_vp, _sz, _sz, C.POINTER(RowCacheStruct), _vp, _vp]),
    "RSGPU_FlatIndex_AddCachedRows": (_i, [_vp, C.POINTER(RowCacheStruct), _vp, _sz, _sz, _vp]),
}

_bound = None


def load():
    global _bound
    if _bound is None:
        lib = V.load()
        for name, (res, args) in ABI.items():
            f = getattr(lib, name)
            f.restype, f.argtypes = res, args
        _bound = lib
    return _bound


def _done(code):
    if code < 0:
        raise RuntimeError(V.last_error())
    return code


class RowCache:
    """A cache over the caller's device arrays: `codes` (capacity * row_bytes bytes) and `scales` (capacity * row_scales floats).
    Without them it answers row_bytes and row_scales, for allocating."""

    def __init__(self, vtype, dim, fmt, block=0, capacity=0, codes=None, scales=None, device=-1):
        self.lib = load()
        self.c = RowCacheStruct(device, vtype, fmt, dim, block, capacity, codes, scales)
        self.ref = C.byref(self.c)

    @property
    def row_bytes(self):
        return self.lib.RSGPU_RowCache_RowBytes(self.ref)

    @property
    def row_scales(self):
        return self.lib.RSGPU_RowCache_RowScales(self.ref)

    def write(self, rows, stride, slots, n, stream=None):
        _done(self.lib.RSGPU_RowCache_Write(self.ref, rows, stride, slots, n, stream))

    def read(self, slots, n, rows_out, stride, stream=None):
        _done(self.lib.RSGPU_RowCache_Read(self.ref, slots, n, rows_out, stride, stream))

    def partition_scores(self, queries, stride, n_queries, query_offsets, n_partitions, pages, max_pages, page_rows, row_counts, form,
                         scores, ld, stream=None):
        _done(self.lib.RSGPU_RowCache_PartitionScores(self.ref, queries, stride, n_queries, query_offsets, n_partitions, pages, max_pages,
                                                      page_rows, row_counts, form, scores, ld, stream))

    def cache_rows(self, index, row_begin, n, slots, wait_stream=None):
        """Stored rows of a FLAT index (vecsim.VecSimIndex) into the cache."""
        _done(self.lib.RSGPU_FlatIndex_CacheRows(index.ptr, row_begin, n, self.ref, slots, wait_stream))

    def add_to(self, index, slots, n, first_label=1, wait_stream=None):
        """Rows of the cache appended to a FLAT index."""
        return _done(self.lib.RSGPU_FlatIndex_AddCachedRows(index.ptr, self.ref, slots, n, first_label, wait_stream))


def score_rules(form=PRODUCT, device=-1, **arrays):
    """RSGPU_ScoreRules by field name; what is not given does not apply."""
    return ScoreRules(device=device, form=form, **arrays)


def adjust_scores(rules, scores_in, scores_out, n_queries, n_columns, ld, counts=None, stream=None):
    _done(load().RSGPU_AdjustScores(C.byref(rules), scores_in, scores_out, n_queries, n_columns, ld, counts, stream))
