// The paged compressed cache: views of a plan on the device, and what its kernels share.
//
// The 16-token tiles that a kernel has to walk for one KV head form one flat sequence, unit after unit (a unit is a sequence, or
// some of its query rows).  The sequence is cut into equal stretches, one per WARP, the same for every head: a CTA is (head, stretch
// of 16 or 8 warps).  Warps never meet while they walk; a unit that lies in one warp's stretch is finished by it, one that is cut
// leaves partials that the CTA merges at its end and, where it is cut between CTAs, a second kernel.  (Sequences of a serving batch
// differ in length by orders of magnitude, and a window leaves nine tiles of each: units as the work of a whole CTA, with barriers
// and a merge each, kept most of its warps idle there.)
#pragma once
#include "attn_kernel.cuh"

namespace hqmq {
namespace paged {

using namespace attn;

struct Seq { int kv, q, q_off, tab; };          // tokens, new ones, first row of Q, first entry among the tables

// Stretches of the flat sequence: of n warps, as many as there are tiles at most, warp w has [w * total / n, (w + 1) * total / n); the
// others, the last ones, have none.
__host__ __device__ inline int stretch_begin(int w, int total, int n) {
  n = n < total ? n : total;
  return w < n ? (int)((int64_t)w * total / n) : total;
}
__host__ __device__ inline int warp_of(int tile, int total, int n) {
  n = n < total ? n : total;
  return (int)((((int64_t)tile + 1) * n - 1) / total);
}

// Keys [beg, end) of the queries at rows [row0, row1) of a sequence (row = query * G + head of the group).
__host__ __device__ inline void unit_keys(int kv, int q, int G, int window, int row0, int row1, int& beg, int& end) {
  const int p0 = kv - q + row0 / G, p1 = kv - q + (row1 - 1) / G;
  end = p1 + 1;
  beg = window > 0 && p0 + 1 > window ? p0 + 1 - window : 0;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

constexpr int kDecWarps = 16, kDecWarpsWide = 8;     // warps of a decode CTA, for up to 8 and up to 32 rows
constexpr int kMassWarps = 12;
constexpr int kMassRowsWide = 32;                    // rows of a unit of the weights where a sequence has more than 8
// Tokens of a CTA of the weights' second kernel: of 8 rows a token has 32 bytes of scores per unit, of 32 rows 128 (512 tokens either way:
// 46 us for the last 32 tokens of 4 x 8k, whose sequences have four units each, in 360 CTAs).
constexpr int mass_group(int rows) { return rows > 8 ? 128 : 512; }
constexpr int kMaxCodewords = 6144;                   // two tables and the rings of 16 warps in shared memory, whatever the radius bits
constexpr int kMaxPage = 1024;                       // tokens of a page
constexpr int kWarpRecord = 16;                      // words of a warp's record: its stretch, first unit and tile; the unit's end, the
                                                     // sequence's place among the tables, the first tile's page, the unit's first row; its
                                                     // stretch of the flat sequence; the sequence: one load, then the copies and queries
// CTAs of a head that run as one cluster (148 SMs hold fifteen clusters of eight of these CTAs).
constexpr int kClusterMax = 8;
inline bool as_cluster(int ctas, int heads) { return ctas <= kClusterMax && (int64_t)ctas * heads <= 112; }
inline int dec_warps(int rows) { return rows > 8 ? kDecWarpsWide : kDecWarps; }

int check_plan(const hqmq_paged_plan& p);
int check_pool(const hqmq_packed& k, const hqmq_paged_plan& p);
bool chunked(int q, int G);
// The prompt chunks of a call (attn_prefill.cu).
size_t chunk_workspace(const hqmq_paged_attn_args* a);
int chunk_launch(const hqmq_paged_attn_args* a, void* ws, cudaStream_t st);

}  // namespace paged
}  // namespace hqmq
