// The score kernels of head dim 64.
#include "paged_mass.cuh"

namespace hqmq {
namespace paged {
const void* scores_kernel_64(int ib, int rb, int nb, bool outl) { return pick_scores_kernel<16>(ib, rb, nb, outl); }
}  // namespace paged
}  // namespace hqmq
