// partition_f32.hip -- partition_kernels.hpp for FLOAT32 queries.
#include "partition_kernels.hpp"

namespace rsgpu {
void launch_partition_scores_f32(const PartitionArgs &a, hipStream_t s) { scores_from<F32>(a, s); }
}  // namespace rsgpu
