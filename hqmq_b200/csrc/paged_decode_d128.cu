// The paged decode kernels of head dim 128.
#include "paged_decode.cuh"

namespace hqmq {
namespace paged {
DecodeKernels decode_kernels_128(int ib, int rb, int nb, bool outl) { return pick_kernels<32>(ib, rb, nb, outl); }
}  // namespace paged
}  // namespace hqmq
