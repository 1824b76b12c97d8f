// rows.hpp -- launchers of the row cache's kernels (rows_kernels.hip, partition_kernels.hpp), called by the C entry points in rows_abi.cpp.
#pragma once
#include <hip/hip_runtime.h>

#include "common.hpp"
#include "rsgpu_rows.h"

namespace rsgpu {

// elements of a row in memory: every kernel works on whole units of 32
__host__ __device__ inline uint32_t rows_padded(uint32_t dim) { return (dim + 31) / 32 * 32; }

struct RowCacheArgs {   // a checked RSGPU_RowCache
  uint8_t *codes;
  float *scales;
  uint64_t capacity;
  uint32_t dim, block, nb;   // block: elements a scale (the whole row: dim), nb: scales a row
  uint32_t row_bytes;
  int type, format;
};

struct PartitionArgs {
  RowCacheArgs c;
  const void *queries;
  size_t stride;
  uint32_t n_queries, n_partitions;
  const int32_t *query_offsets, *pages, *row_counts;
  uint32_t max_pages, page_rows, most_rows;   // most_rows: the smaller of max_pages * page_rows and ld
  int form;
  float *scores;
  size_t ld;
};

struct AdjustArgs {
  RSGPU_ScoreRules r;
  const float *in;
  float *out;
  uint32_t n_queries, n_columns;
  size_t ld;
  const int32_t *counts;
};

// throws std::runtime_error on anything that is not served
RowCacheArgs check_row_cache(const RSGPU_RowCache *c);

void launch_row_write(const RowCacheArgs &c, const void *rows, uint32_t stride, const int64_t *slots, uint32_t n, hipStream_t s);
void launch_row_read(const RowCacheArgs &c, const int64_t *slots, uint32_t n, void *out, uint32_t stride, hipStream_t s);
// by the type of the queries
void launch_partition_scores_f32(const PartitionArgs &a, hipStream_t s);
void launch_partition_scores_f16(const PartitionArgs &a, hipStream_t s);
void launch_partition_scores_bf16(const PartitionArgs &a, hipStream_t s);
void launch_adjust_scores(const AdjustArgs &a, hipStream_t s);

}  // namespace rsgpu
