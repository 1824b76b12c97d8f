// rows_abi.cpp -- the C entry points of include/rsgpu_rows.h: argument checks, device selection, launches.  No exception crosses
// the boundary: a failure is -1 plus RSGPU_LastError(), and a refused call has launched nothing.
#include "flat_index.hpp"
#include "rows.hpp"
#include "rsgpu_rows.h"

using namespace rsgpu;

namespace {

constexpr size_t MOST = 0x7fffffff;   // counts that kernels keep in 32 bits

[[noreturn]] void refuse(const char *what) { throw std::runtime_error(what); }
void need(bool ok, const char *what) {
  if (!ok) refuse(what);
}

// The caller's thread works on `device` (-1: where `at` lives) until the end of the scope.
struct OnDevice {
  int before = -1, now = -1;
  OnDevice(int device, const void *at) {
    HIP_CHECK(hipGetDevice(&before));
    if (device < 0) {
      hipPointerAttribute_t attr;
      if (hipPointerGetAttributes(&attr, at) != hipSuccess || attr.type == hipMemoryTypeHost || attr.type == hipMemoryTypeUnregistered) {
        (void)hipGetLastError();
        refuse("not device memory");
      }
      device = attr.device;
    }
    now = device;
    if (now != before) HIP_CHECK(hipSetDevice(now));
  }
  ~OnDevice() {
    if (now != before && now >= 0) (void)hipSetDevice(before);
  }
};

bool aligned(const void *p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// the shape alone, without the arrays; 0 bytes: not served
size_t row_bytes(const RSGPU_RowCache &c) {
  if (c.type != VecSimType_FLOAT32 && c.type != VecSimType_FLOAT16 && c.type != VecSimType_BFLOAT16) return 0;
  if (c.dim == 0 || c.dim > 65536) return 0;
  const size_t padded = rows_padded(c.dim);
  if (c.format == RSGPU_ROWS_NATIVE) return c.block ? 0 : padded * type_size((VecSimType)c.type);
  if (c.block != 0 && c.block != 32 && c.block != 64 && c.block != 128) return 0;
  if (c.format == RSGPU_ROWS_INT8 || c.format == RSGPU_ROWS_E4M3) return padded;
  return c.format == RSGPU_ROWS_INT4 ? padded / 2 : 0;
}
size_t row_scales(const RSGPU_RowCache &c) {
  if (!row_bytes(c) || c.format == RSGPU_ROWS_NATIVE) return 0;
  return c.block ? (c.dim + c.block - 1) / c.block : 1;
}

int fail(const char *where, const char *what) {
  last_error() = std::string(where) + ": " + what;
  logf(nullptr, VecSimCommonStrings_LOG_WARNING_STRING, "%s", last_error().c_str());
  return -1;
}

template <typename F>
int guarded(const char *where, F &&body) {
  try {
    return body();
  } catch (const std::exception &e) {
    return fail(where, e.what());
  } catch (...) {
    return fail(where, "unknown error");
  }
}

// what a cache and an index must have in common
void check_pair(const VecSimIndex *index, const RowCacheArgs &c) {
  need(index && !index->sharded && index->flat, "the rows of a sharded handle are on several devices: use its shards (RSGPU_ShardedIndex_Shard)");
  need((int)index->flat->type == c.type && index->flat->dim == c.dim, "the cache has another type or dim than the index");
}

}  // namespace

namespace rsgpu {
RowCacheArgs check_row_cache(const RSGPU_RowCache *c) {
  need(c, "no cache");
  const size_t bytes = row_bytes(*c);
  need(bytes != 0, "cache: type FLOAT32 / FLOAT16 / BFLOAT16, dim 1 .. 65536, format NATIVE (block 0) / INT8 / E4M3 / INT4, block 0 / 32 / 64 / 128");
  need(c->codes && c->capacity && aligned(c->codes, 16), "cache: codes are capacity > 0 rows, 16-byte aligned");
  need(c->format == RSGPU_ROWS_NATIVE || (c->scales && aligned(c->scales, 4)), "cache: scales are fp32, 4-byte aligned");
  need(c->capacity <= UINT32_MAX, "cache: at most 2^32 - 1 slots");
  RowCacheArgs a;
  a.codes = static_cast<uint8_t *>(c->codes);
  a.scales = c->scales;
  a.capacity = c->capacity;
  a.dim = c->dim;
  a.block = c->block ? c->block : c->dim;
  a.nb = (uint32_t)row_scales(*c);
  a.row_bytes = (uint32_t)bytes;
  a.type = c->type;
  a.format = c->format;
  return a;
}
}  // namespace rsgpu

extern "C" {

size_t RSGPU_RowCache_RowBytes(const RSGPU_RowCache *cache) { return cache ? row_bytes(*cache) : 0; }
size_t RSGPU_RowCache_RowScales(const RSGPU_RowCache *cache) { return cache ? row_scales(*cache) : 0; }

int RSGPU_RowCache_Write(const RSGPU_RowCache *cache, const void *rows, size_t stride, const int64_t *slots, size_t n, void *stream) {
  return guarded("RSGPU_RowCache_Write", [&] {
    const RowCacheArgs c = check_row_cache(cache);
    if (!n) return 0;
    need(rows && slots, "rows or slots are NULL");
    need(n <= MOST, "at most 2^31 - 1 rows a call");
    need(stride >= c.dim && stride <= MOST, "stride: elements from row to row, dim .. 2^31 - 1");
    need(aligned(rows, type_size((VecSimType)c.type)) && aligned(slots, 8), "rows or slots are not aligned to their elements");
    OnDevice on(cache->device, c.codes);
    launch_row_write(c, rows, (uint32_t)stride, slots, (uint32_t)n, (hipStream_t)stream);
    return 0;
  });
}

int RSGPU_RowCache_Read(const RSGPU_RowCache *cache, const int64_t *slots, size_t n, void *rows_out, size_t stride, void *stream) {
  return guarded("RSGPU_RowCache_Read", [&] {
    const RowCacheArgs c = check_row_cache(cache);
    if (!n) return 0;
    need(rows_out && slots, "rows_out or slots are NULL");
    need(n <= MOST, "at most 2^31 - 1 rows a call");
    need(stride >= c.dim && stride <= MOST, "stride: elements from row to row, dim .. 2^31 - 1");
    need(aligned(rows_out, type_size((VecSimType)c.type)) && aligned(slots, 8), "rows_out or slots are not aligned to their elements");
    OnDevice on(cache->device, c.codes);
    launch_row_read(c, slots, (uint32_t)n, rows_out, (uint32_t)stride, (hipStream_t)stream);
    return 0;
  });
}

int RSGPU_RowCache_PartitionScores(const RSGPU_RowCache *cache, const void *queries, size_t stride, size_t n_queries,
                                   const int32_t *query_offsets, size_t n_partitions, const int32_t *pages, size_t max_pages,
                                   size_t page_rows, const int32_t *row_counts, int form, float *scores, size_t ld, void *stream) {
  return guarded("RSGPU_RowCache_PartitionScores", [&] {
    PartitionArgs a;
    a.c = check_row_cache(cache);
    need(form == RSGPU_SCORES_PRODUCT || form == RSGPU_SCORES_DISTANCE, "form is PRODUCT or DISTANCE");
    need(page_rows > 0 && page_rows <= MOST, "page_rows: 1 .. 2^31 - 1");
    if (!n_queries || !n_partitions || !max_pages || !ld) return 0;
    need(queries && query_offsets && pages && row_counts && scores, "an array is NULL");
    need(n_queries <= MOST && n_partitions <= MOST && max_pages <= MOST, "at most 2^31 - 1 queries, partitions and pages");
    need(stride >= a.c.dim && stride <= SIZE_MAX / 8 / n_queries, "stride: elements from query to query, at least dim");
    need(ld <= SIZE_MAX / 8 / n_queries, "ld");
    need(aligned(queries, type_size((VecSimType)a.c.type)) && aligned(query_offsets, 4) && aligned(pages, 4) && aligned(row_counts, 4) &&
             aligned(scores, 4), "an array is not aligned to its elements");
    a.queries = queries;
    a.stride = stride;
    a.n_queries = (uint32_t)n_queries;
    a.n_partitions = (uint32_t)n_partitions;
    a.query_offsets = query_offsets;
    a.pages = pages;
    a.row_counts = row_counts;
    a.max_pages = (uint32_t)max_pages;
    a.page_rows = (uint32_t)page_rows;
    const size_t rows = page_rows > MOST / max_pages ? MOST : max_pages * page_rows;
    a.most_rows = (uint32_t)(rows < ld ? rows : ld);
    a.form = form;
    a.scores = scores;
    a.ld = ld;
    OnDevice on(cache->device, a.c.codes);
    const auto launch = a.c.type == VecSimType_FLOAT32 ? launch_partition_scores_f32 : a.c.type == VecSimType_FLOAT16 ? launch_partition_scores_f16 : launch_partition_scores_bf16;
    launch(a, (hipStream_t)stream);
    return 0;
  });
}

int RSGPU_AdjustScores(const RSGPU_ScoreRules *rules, const float *scores_in, float *scores_out, size_t n_queries, size_t n_columns,
                       size_t ld, const int32_t *counts, void *stream) {
  return guarded("RSGPU_AdjustScores", [&] {
    need(rules, "no rules");
    const RSGPU_ScoreRules &r = *rules;
    need(r.form == RSGPU_SCORES_PRODUCT || r.form == RSGPU_SCORES_DISTANCE, "form is PRODUCT or DISTANCE");
    if (!n_queries || !n_columns) return 0;
    need(scores_in && scores_out && aligned(scores_in, 4) && aligned(scores_out, 4), "scores are fp32, 4-byte aligned");
    need(n_queries <= MOST && n_columns <= MOST - 4096, "at most 2^31 - 1 queries and 2^31 - 4097 columns");
    need(ld >= n_columns && ld <= SIZE_MAX / 8 / n_queries, "ld: at least n_columns");
    need(!r.mask || r.mask_words >= (n_columns + 31) / 32, "mask_words: a bit for every column");
    need(!r.mask || r.mask_rows || r.n_masks >= n_queries, "without mask_rows there is a mask row for every query");
    need(!r.bias_offsets || !r.n_bias || (r.bias_ids && r.bias_values), "bias_ids or bias_values are NULL");
    need(!r.seen_offsets || !r.n_seen || r.seen_ids, "seen_ids are NULL");
    need(r.n_bias <= MOST && r.n_seen <= MOST, "at most 2^31 - 1 entries of a list");
    need(aligned(r.mask, 4) && aligned(r.mask_rows, 4) && aligned(r.bias_offsets, 4) && aligned(r.bias_ids, 4) && aligned(r.bias_values, 4) &&
             aligned(r.seen_offsets, 4) && aligned(r.seen_ids, 4) && aligned(r.repetition, 4) && aligned(r.frequency, 4) &&
             aligned(r.presence, 4) && aligned(counts, 4), "an array is not aligned to its elements");
    AdjustArgs a{r, scores_in, scores_out, (uint32_t)n_queries, (uint32_t)n_columns, ld, counts};
    OnDevice on(r.device, scores_out);
    launch_adjust_scores(a, (hipStream_t)stream);
    return 0;
  });
}

int RSGPU_FlatIndex_CacheRows(VecSimIndex *index, size_t row_begin, size_t n, const RSGPU_RowCache *cache, const int64_t *slots,
                              void *wait_stream) {
  return guarded("RSGPU_FlatIndex_CacheRows", [&] {
    need(index, "no index");
    const RowCacheArgs c = check_row_cache(cache);
    check_pair(index, c);
    need(n <= MOST, "at most 2^31 - 1 rows a call");
    need(!n || (slots && aligned(slots, 8)), "slots are 8-byte aligned");
    OnDevice on(cache->device, c.codes);
    need(on.now == index->flat->device, "the cache is on another device than the index");
    (void)hipGetLastError();   // the index asks for the last error of its own launches, not for what the caller's thread has left
    HIP_CHECK(hipStreamSynchronize((hipStream_t)wait_stream));
    index->flat->cache_rows(row_begin, n, c, slots);
    return 0;
  });
}

int RSGPU_FlatIndex_AddCachedRows(VecSimIndex *index, const RSGPU_RowCache *cache, const int64_t *slots, size_t n, size_t first_label,
                                  void *wait_stream) {
  return guarded("RSGPU_FlatIndex_AddCachedRows", [&] {
    need(index, "no index");
    const RowCacheArgs c = check_row_cache(cache);
    check_pair(index, c);
    need(n <= MOST, "at most 2^31 - 1 rows a call");
    need(!n || (slots && aligned(slots, 8)), "slots are 8-byte aligned");
    OnDevice on(cache->device, c.codes);
    need(on.now == index->flat->device, "the cache is on another device than the index");
    (void)hipGetLastError();   // the index asks for the last error of its own launches, not for what the caller's thread has left
    HIP_CHECK(hipStreamSynchronize((hipStream_t)wait_stream));
    return index->flat->add_cached_rows(c, slots, n, first_label);
  });
}

}  // extern "C"
