// partition_f16.hip -- partition_kernels.hpp for FLOAT16 queries.
#include "partition_kernels.hpp"

namespace rsgpu {
void launch_partition_scores_f16(const PartitionArgs &a, hipStream_t s) { scores_from<F16>(a, s); }
}  // namespace rsgpu
