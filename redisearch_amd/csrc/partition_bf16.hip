// partition_bf16.hip -- partition_kernels.hpp for BFLOAT16 queries.
#include "partition_kernels.hpp"

namespace rsgpu {
void launch_partition_scores_bf16(const PartitionArgs &a, hipStream_t s) { scores_from<BF16>(a, s); }
}  // namespace rsgpu
