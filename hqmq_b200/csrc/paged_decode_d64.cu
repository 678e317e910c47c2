// The paged decode kernels of head dim 64.
#include "paged_decode.cuh"

namespace hqmq {
namespace paged {
DecodeKernels decode_kernels_64(int ib, int rb, int nb, bool outl) { return pick_kernels<16>(ib, rb, nb, outl); }
}  // namespace paged
}  // namespace hqmq
