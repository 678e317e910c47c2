// Tokens on their way to pages: encoded ones of a batch (hqmq_paged_store), and those that an eviction keeps (hqmq_paged_evict).
#include <string.h>

#include "attn_prefill.cuh"
#include "paged.cuh"

namespace hqmq {
namespace paged {
namespace {

__device__ __forceinline__ uint32_t warp_before(uint32_t own, int lane) {       // sum over the lanes before
  uint32_t x = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  return x - own;
}

// ---- store -----------------------------------------------------------------------------------------------------------------------
// blockIdx.x = (sequence, page among those its new tokens touch), y = KV head, z = tensor.  The tokens are neighbours in the staging
// planes, so their flagged values are one run there and stay one run in the page.  Tokens from the first of them on that the page held before are
// gone: a store may begin anywhere in what was stored.
struct StoreParams {
  hqmq_packed src[2], dst[2];
  const int4* seqs; const int* tabs;
  int per, Hkv, page_bits;
};
__global__ void __launch_bounds__(128) paged_store_kernel(const StoreParams p) {
  const int sq = blockIdx.x / p.per, pi = blockIdx.x - sq * p.per, h = blockIdx.y;
  const hqmq_packed& S = p.src[blockIdx.z];
  const hqmq_packed& D = p.dst[blockIdx.z];
  const int4 s4 = __ldg(p.seqs + sq);
  const Seq s{s4.x, s4.y, s4.z, s4.w};
  const int pt = 1 << p.page_bits, t_new = s.kv - s.q, page_i = (t_new >> p.page_bits) + pi;
  const int lo = max(t_new, page_i << p.page_bits), hi = min(s.kv, (page_i + 1) << p.page_bits), n = hi - lo;
  if (n <= 0) return;
  const int64_t ph = (int64_t)__ldg(p.tabs + s.tab + page_i) * p.Hkv + h;
  const int a = lo & (pt - 1), src_t = s.q_off + (lo - t_new);
  const int64_t drow = (ph << p.page_bits) + a, srow = (int64_t)h * S.T_cap + src_t;
  const int words = D.row_bytes >> 2;
  const uint32_t* sc = reinterpret_cast<const uint32_t*>(S.codes) + srow * words;
  uint32_t* dc = reinterpret_cast<uint32_t*>(D.codes) + drow * words;
  for (int i = threadIdx.x; i < n * words; i += 128) dc[i] = __ldg(sc + i);
  for (int i = threadIdx.x; i < n; i += 128)
    reinterpret_cast<uint16_t*>(D.rs)[drow + i] = __ldg(reinterpret_cast<const uint16_t*>(S.rs) + srow + i);
  if (!D.flags || threadIdx.x >= 32) return;
  const int lane = threadIdx.x;
  uint32_t* off = D.out_off + ph * (pt / HQMQ_OUT_BLOCK + 1);
  // Entries of the page's tokens before the first of these: by the block's offset and its flags, not by the page's counter, which still has
  // tokens that the sequence no longer holds (drafted ones that were taken back, a step that is stored again).
  uint32_t held = 0u;
  if (a > 0) {
    const int in_blk = a & (HQMQ_OUT_BLOCK - 1);
    held = off[a / HQMQ_OUT_BLOCK] + __reduce_add_sync(0xffffffffu, lane < in_blk ? __popc(D.flags[drow - in_blk + lane]) : 0u);
  }
  // entries of the staging tensor before the first of these tokens
  uint32_t from = 0u;
  if (S.flags) {
    const int in_blk = src_t & (HQMQ_OUT_BLOCK - 1);
    uint32_t c = lane < in_blk ? __popc(__ldg(S.flags + srow - in_blk + lane)) : 0u;
    c = __reduce_add_sync(0xffffffffu, c);
    from = __ldg(S.out_off + (int64_t)h * (S.T_cap / HQMQ_OUT_BLOCK + 1) + src_t / HQMQ_OUT_BLOCK) + c;
  }
  if (a == 0 && lane == 0) off[0] = 0u;
  uint32_t total = 0u;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t f = S.flags && i < n ? __ldg(S.flags + srow + i) : 0u, c = __popc(f);
    const uint32_t end = held + total + warp_before(c, lane) + c;
    if (i < n) {
      D.flags[drow + i] = f;
      if (((a + i + 1) & (HQMQ_OUT_BLOCK - 1)) == 0 || i == n - 1) off[(a + i) / HQMQ_OUT_BLOCK + 1] = end;
    }
    total += __reduce_add_sync(0xffffffffu, c);
  }
  if (S.flags) {
    const uint2* sv = reinterpret_cast<const uint2*>(S.out_vals) + (int64_t)h * S.out_cap;
    uint2* dv = reinterpret_cast<uint2*>(D.out_vals) + ph * D.out_cap;
    for (uint32_t i = lane; i < total; i += 32)
      if (held + i < (uint32_t)D.out_cap) dv[held + i] = from + i < (uint32_t)S.out_cap ? __ldg(sv + from + i) : make_uint2(0u, 0u);
  }
  if (lane == 0) D.out_count[ph] = held + total;
}

// ---- evict: which tokens stay --------------------------------------------------------------------------------------------------------
// A cluster of C CTAs per (sequence, KV head), each with a stretch of the tokens, their weights as ordered integers in shared memory.
// Radix select of the smallest weight that stays in three steps (11, 11 and 10 bits): a histogram per CTA, summed over the cluster through
// distributed shared memory by every CTA for itself.  Then every warp counts and writes its own stretch, 32 tokens at a time.
// Bound: latencies, of the one read of the weights (16 bytes a thread, four in flight: a float at a time, behind its page's number, took
// 73 us for 8 heads of 131072 tokens) and of four cluster barriers.
constexpr int kSelThreads = 1024, kSelWarps = kSelThreads / 32;
constexpr int kSelCached = 40960;               // tokens of a CTA whose keys are kept in shared memory (160 KB)

struct EvictParams {
  hqmq_packed K, V;
  const float* mass; float* new_mass; int* kept;
  const int4* src_seqs; const int* src_tabs; const int4* dst_seqs; const int* dst_tabs;
  int first, last, kept_stride, Hkv, page_bits, per_page, cached, n_seqs;      // cached: tokens of a CTA that shared memory holds
};

__device__ __forceinline__ uint32_t order_key(float f) {      // larger is heavier; no number: 0, below every number
  if (f != f) return 0u;
  f += 0.f;                                                   // (-0 is 0)
  const uint32_t b = __float_as_uint(f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t peer_u32(const void* at, uint32_t rank) {
  uint32_t a, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(at)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

__device__ __forceinline__ uint2 peer_u64(const void* at, uint32_t rank) {
  uint32_t a;
  uint2 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(at)), "r"(rank));
  asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}

__global__ void __launch_bounds__(kSelThreads, 1) evict_select_kernel(const EvictParams p) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  uint32_t* hist = reinterpret_cast<uint32_t*>(smem_raw);         // [3][2048]
  uint32_t* pub = hist + 3 * 2048;                                // heavier, equal: what other CTAs read
  uint32_t* wsum = pub + 4;                                       // [2][kSelWarps]
  uint32_t* pick = wsum + 2 * kSelWarps;                          // bin, left
  uint32_t* keys = pick + 4;
  const int C = (int)cluster_size(), rank = (int)cluster_rank();
  const int sh = (int)blockIdx.x / C, sq = sh / p.Hkv, h = sh - sq * p.Hkv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int4 s4 = __ldg(p.src_seqs + sq);
  const int n = s4.x, tab = s4.w, keep = min(min(__ldg(&p.dst_seqs[sq].x), n), p.kept_stride);
  const int last = min(p.last, keep), first = min(p.first, keep - last);
  const int per = ((n + C - 1) / C + 31) & ~31, t0 = min(n, rank * per), t1 = min(n, t0 + per);
  const int mine = t1 - t0;
  const bool cached = per <= p.cached;
  for (int i = tid; i < 3 * 2048; i += kSelThreads) hist[i] = 0u;
  const float* mass_h = p.mass + ((int64_t)h << p.page_bits);
  auto quad_of = [&](int t) {                  // the weights of tokens t .. t + 3 (t a multiple of four, so they lie in one page)
    const int page = __ldg(p.src_tabs + tab + (t >> p.page_bits));
    return __ldg(reinterpret_cast<const float4*>(mass_h + (((int64_t)page * p.Hkv) << p.page_bits) + (t & ((1 << p.page_bits) - 1))));
  };
  auto key_at = [&](int i) {
    if (cached) return keys[i];
    const float4 v = quad_of((t0 + i) & ~3);
    const int x = (t0 + i) & 3;
    return order_key(x == 0 ? v.x : x == 1 ? v.y : x == 2 ? v.z : v.w);
  };
  auto free_at = [&](int t) { return t >= first && t < n - last; };       // neither a first nor a last token
  __syncthreads();
  grid_dep_launch();
  const bool all = keep >= n;
  const uint32_t want = (uint32_t)(keep - first - last);                  // of the free ones
  uint32_t prefix = 0u, left = want;
  if (!all) {                                                             // (the same for the whole cluster)
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
      uint32_t* hp = hist + pass * 2048;
      auto count = [&](int i, uint32_t k) {
        if (i < mine && free_at(t0 + i) && (pass == 0 || (k >> (pass == 1 ? 21 : 10)) == prefix)) atomicAdd(hp + ((k >> shift) & (bins - 1)), 1u);
      };
      if (pass == 0 || !cached) {
#pragma unroll 4
        for (int i = 4 * tid; i < mine; i += 4 * kSelThreads) {
          const float4 v = quad_of(t0 + i);
          const uint4 k = make_uint4(order_key(v.x), order_key(v.y), order_key(v.z), order_key(v.w));
          if (cached) *reinterpret_cast<uint4*>(keys + i) = k;
          count(i, k.x); count(i + 1, k.y); count(i + 2, k.z); count(i + 3, k.w);
        }
      } else {
        for (int i = 4 * tid; i < mine; i += 4 * kSelThreads) {
          const uint4 k = *reinterpret_cast<const uint4*>(keys + i);
          count(i, k.x); count(i + 1, k.y); count(i + 2, k.z); count(i + 3, k.w);
        }
      }
      cluster_sync();
      // bins 2 tid and 2 tid + 1, summed over the cluster; then how many lie in higher bins
      uint32_t c[2] = {0u, 0u};
      if (2 * tid < bins) {
        uint2 v[8];                              // (all on their way before any is added)
#pragma unroll
        for (int x = 0; x < 8; ++x) { v[x] = make_uint2(0u, 0u); if (x < C) v[x] = peer_u64(hp + 2 * tid, x); }
#pragma unroll
        for (int x = 0; x < 8; ++x) { c[0] += v[x].x; c[1] += v[x].y; }
      }
      const uint32_t sum = c[0] + c[1];
      const uint32_t wt = __reduce_add_sync(0xffffffffu, sum), below = warp_before(sum, lane);
      if (lane == 0) wsum[warp] = wt;
      __syncthreads();
      uint32_t above = wt - below - sum;
      for (int x = warp + 1; x < kSelWarps; ++x) above += wsum[x];
      // (left is at least 1 where there is a choice; with nothing wanted the highest bin is taken, of which none stays)
#pragma unroll
      for (int b = 1; b >= 0; --b) {
        if (left > 0 ? above < left && above + c[b] >= left : false) { pick[0] = 2 * tid + b; pick[1] = left - above; }
        above += c[b];
      }
      __syncthreads();
      if (left > 0) { prefix = pass == 0 ? pick[0] : (prefix << (pass == 1 ? 11 : 10)) | pick[0]; left = pick[1]; }
      __syncthreads();
    }
  }
  // heavier (or kept anyway) and equal ones of every warp's stretch, then of the CTA, then of the CTAs before it
  const int seg = (mine + kSelWarps * 32 - 1) / (kSelWarps * 32) * 32, i0 = min(mine, warp * seg), i1 = min(mine, i0 + seg);
  auto kind = [&](int i) -> int {              // 2: stays, 1: equal to the least that stays, 0: goes
    if (i >= i1) return 0;
    if (all || !free_at(t0 + i)) return 2;
    if (want == 0u) return 0;
    const uint32_t k = key_at(i);
    return k > prefix ? 2 : k == prefix ? 1 : 0;
  };
  uint32_t sure = 0u, tie = 0u;
  for (int i = i0; i < i1; i += 32) {
    const int kd = kind(i + lane);
    sure += __popc(__ballot_sync(0xffffffffu, kd == 2));
    tie += __popc(__ballot_sync(0xffffffffu, kd == 1));
  }
  if (lane == 0) { wsum[warp] = sure; wsum[kSelWarps + warp] = tie; }
  __syncthreads();
  if (tid == 0) {
    uint32_t a = 0u, b = 0u;
    for (int x = 0; x < kSelWarps; ++x) { a += wsum[x]; b += wsum[kSelWarps + x]; }
    pub[0] = a; pub[1] = b;
  }
  cluster_sync();
  uint32_t at = 0u, ties = 0u;                 // kept and equal ones before this warp's stretch
  for (int x = 0; x < rank; ++x) { at += peer_u32(pub, x); ties += peer_u32(pub + 1, x); }
  for (int x = 0; x < warp; ++x) { at += wsum[x]; ties += wsum[kSelWarps + x]; }
  at += min(ties, left);                       // (of the equal ones the first `left` stay)
  int* out = p.kept + (int64_t)sh * p.kept_stride;
  for (int i = i0; i < i1; i += 32) {
    const int kd = kind(i + lane);
    const uint32_t eq = __ballot_sync(0xffffffffu, kd == 1);
    const bool stays = kd == 2 || (kd == 1 && ties + __popc(eq & ((1u << lane) - 1u)) < left);
    const uint32_t st = __ballot_sync(0xffffffffu, stays);
    const uint32_t pos = at + __popc(st & ((1u << lane) - 1u));
    if (stays && pos < (uint32_t)p.kept_stride) out[pos] = t0 + i + lane;
    at += __popc(st);
    ties += __popc(eq);
  }
  for (int i = keep + rank * kSelThreads + tid; i < p.kept_stride; i += C * kSelThreads) out[i] = -1;
  cluster_sync();                              // (nobody's shared memory goes while another reads it)
}

// ---- evict: their rows go to the new pages ----------------------------------------------------------------------------------------------
// A warp per 64 tokens of a new page, two per lane; page, KV head and tensor by (blockIdx.x, warp), y, z.  The warps of a page meet once, to
// know the entries before theirs.  (A CTA of 256 threads per page, with its scans by block, took 4200 instructions a warp for 64 tokens:
// 67 us for 16 x 2048 tokens of 8 heads.)  Bound: the chain position - page - row - entries, five loads deep, with 32 to 64 warps an SM in it.
constexpr int kMoveWarps = 8;
__global__ void __launch_bounds__(512, 2) evict_move_kernel(const EvictParams p) {
  __shared__ uint32_t s_count[16];
  __shared__ int64_t s_row[16][64];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pt = 1 << p.page_bits, wpp = pt >> 6, slots = (int)(blockDim.x >> 5) / wpp, slot = warp / wpp, part = warp - slot * wpp;
  const int item = blockIdx.x * slots + slot, sq = item / p.per_page, pi = item - sq * p.per_page, h = blockIdx.y;
  const hqmq_packed& X = blockIdx.z ? p.V : p.K;
  int keep = 0, n = 0;
  int4 src = make_int4(0, 0, 0, 0);
  int64_t ph = 0;
  if (sq < p.n_seqs) {
    src = __ldg(p.src_seqs + sq);
    const int4 dst = __ldg(p.dst_seqs + sq);
    keep = min(min(dst.x, src.x), p.kept_stride);
    n = max(0, min(64, keep - (pi * pt + part * 64)));
    if (n > 0) ph = (int64_t)__ldg(p.dst_tabs + dst.w + pi) * p.Hkv + h;
  }
  grid_dep_wait();
  const int64_t drow = (ph << p.page_bits) + part * 64;
  const int* kept = p.kept + ((int64_t)sq * p.Hkv + h) * p.kept_stride + (int64_t)pi * pt + part * 64;
  int t[2];
  int64_t row[2];
  uint32_t fl[2] = {0u, 0u};
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int i = lane + 32 * x;
    t[x] = i < n ? min(max(__ldcg(kept + i), 0), src.x - 1) : 0;        // (written by the kernel ahead: never through the read-only path)
  }
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int i = lane + 32 * x;
    const int page = i < n ? __ldg(p.src_tabs + src.w + (t[x] >> p.page_bits)) : 0;
    t[x] &= pt - 1;
    row[x] = (((int64_t)page * p.Hkv + h) << p.page_bits) + t[x];
  }
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int i = lane + 32 * x;
    if (i < n) {
      if (X.flags) fl[x] = X.flags[row[x]];
      reinterpret_cast<uint16_t*>(X.rs)[drow + i] = reinterpret_cast<const uint16_t*>(X.rs)[row[x]];
      if (blockIdx.z == 0) p.new_mass[drow + i] = p.mass[row[x]];
    }
  }
  // Code rows: the new ones are one stretch of pieces of 16 or 4 bytes, dealt out to the lanes; a piece's row says where it comes from.
  if (n > 0) { s_row[warp][lane] = row[0]; s_row[warp][lane + 32] = row[1]; }
  __syncwarp();
  auto rows = [&](auto zero, int pieces) {
    using T = decltype(zero);
    T* d = reinterpret_cast<T*>(X.codes) + drow * pieces;
    const T* s = reinterpret_cast<const T*>(X.codes);
    const uint32_t inv = 65536u / (uint32_t)pieces + 1u;      // i / pieces = i * inv >> 16 for i < 64 * pieces (pieces <= 32)
    const int all = n * pieces;
    constexpr int U = sizeof(T) == 16 ? 4 : 8;                // pieces of a lane on their way at a time
#pragma unroll 1
    for (int i0 = lane; i0 < all; i0 += 32 * U) {
      T v[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int i = i0 + 32 * k, q = (int)((uint32_t)i * inv >> 16);
        if (i < all) v[k] = s[s_row[warp][q] * pieces + (i - q * pieces)];
      }
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (i0 + 32 * k < all) d[i0 + 32 * k] = v[k];
    }
  };
  if (X.row_bytes % 16 == 0) rows(make_uint4(0u, 0u, 0u, 0u), X.row_bytes / 16);
  else rows(0u, X.row_bytes / 4);
  if (!X.flags) return;                        // (the same for the whole block)
  // side buffer: entries before every token, of this warp's, then of the page's warps before it
  const uint32_t c0 = __popc(fl[0]), c1 = __popc(fl[1]), b0 = warp_before(c0, lane), n0 = __shfl_sync(0xffffffffu, b0 + c0, 31);
  const uint32_t b1 = n0 + warp_before(c1, lane), all = __shfl_sync(0xffffffffu, b1 + c1, 31);
  uint32_t before = 0u, total = all;
  if (wpp > 1) {
    if (lane == 0) s_count[warp] = all;
    __syncthreads();
    total = 0u;
    for (int x = 0; x < wpp; ++x) { const uint32_t y = s_count[slot * wpp + x]; before += x < part ? y : 0u; total += y; }
  }
  if (sq >= p.n_seqs || pi * pt >= keep) return;
  if (n == 0 && !(part * 64 > 0)) return;
  if (n == 0) {                                // blocks of the page behind its last token hold nothing
    uint32_t* off = reinterpret_cast<uint32_t*>(X.out_off);
    const int4 dst = __ldg(p.dst_seqs + sq);
    const int64_t o = ((int64_t)__ldg(p.dst_tabs + dst.w + pi) * p.Hkv + h) * (pt / HQMQ_OUT_BLOCK + 1) + part * 4;
    if (lane >= 1 && lane <= 4) off[o + lane] = total;
    return;
  }
  uint32_t* off = X.out_off + ph * (pt / HQMQ_OUT_BLOCK + 1) + part * 4;
  if (part == 0 && lane == 0) { off[0] = 0u; X.out_count[ph] = total; }
  const uint32_t at[2] = {before + b0, before + b1}, cnt[2] = {c0, c1};
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int i = lane + 32 * x;
    if (i < n) X.flags[drow + i] = fl[x];
    // (the counts of lanes behind the last token are zero: whole blocks end where they would)
    if ((lane & 15) == 15) off[(i >> 4) + 1] = at[x] + cnt[x];
  }
  // a token's entries: the block's offset and the counts of the tokens before it in the block say where they are
  uint32_t from[2] = {0u, 0u};
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    if (cnt[x]) {
      const int in_blk = t[x] & (HQMQ_OUT_BLOCK - 1);
      const uint4* f4 = reinterpret_cast<const uint4*>(X.flags + (row[x] - in_blk));
      uint32_t c = X.out_off[(row[x] >> p.page_bits) * (pt / HQMQ_OUT_BLOCK + 1) + t[x] / HQMQ_OUT_BLOCK];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint4 f = f4[q];
        c += (4 * q < in_blk ? __popc(f.x) : 0) + (4 * q + 1 < in_blk ? __popc(f.y) : 0) + (4 * q + 2 < in_blk ? __popc(f.z) : 0) +
             (4 * q + 3 < in_blk ? __popc(f.w) : 0);
      }
      from[x] = c;
    }
  }
  const uint2* sv = reinterpret_cast<const uint2*>(X.out_vals);
  uint2* dv = reinterpret_cast<uint2*>(X.out_vals) + ph * X.out_cap;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int64_t s0 = (row[x] >> p.page_bits) * X.out_cap;
    for (uint32_t e = 0; e < cnt[x]; ++e)
      if (at[x] + e < (uint32_t)X.out_cap) dv[at[x] + e] = from[x] + e < (uint32_t)X.out_cap ? sv[s0 + from[x] + e] : make_uint2(0u, 0u);
  }
}

int log2_of(int x) { int b = 0; while ((1 << b) < x) ++b; return b; }

}  // namespace
}  // namespace paged
}  // namespace hqmq

using namespace hqmq;
using namespace hqmq::paged;

extern "C" int hqmq_paged_store(const hqmq_paged_store_args* a, void* stream) {
  if (!a || a->struct_size != sizeof(hqmq_paged_store_args) || !a->plan_data) return HQMQ_ERR_ARG;
  int rc = check_plan(a->plan);
  if (rc) return rc;
  const hqmq_packed* src[2] = {&a->src_K, &a->src_V};
  const hqmq_packed* dst[2] = {&a->K, &a->V};
  StoreParams p;
  memset(&p, 0, sizeof(p));
  for (int i = 0; i < 2; ++i) {
    if ((rc = check_pool(*dst[i], a->plan)) != 0 || (rc = check_packed(*src[i], false)) != 0) return rc;
    const hqmq_packed &s = *src[i], &d = *dst[i];
    if (s.B != 1 || s.H != d.H || s.T_cap < a->plan.total_q || s.n_chunks != d.n_chunks || s.S != d.S || s.radius_bits != d.radius_bits) return HQMQ_ERR_SHAPE;
    if (s.scale_dtype != d.scale_dtype || (s.flags && (!d.flags || s.out_dtype != d.out_dtype))) return HQMQ_ERR_DTYPE;
    p.src[i] = s; p.dst[i] = d;
  }
  if (a->plan.total_q == 0) return HQMQ_OK;
  if ((uintptr_t)a->plan_data & 15) return HQMQ_ERR_ALIGN;
  p.seqs = reinterpret_cast<const int4*>(a->plan_data) + a->plan.seqs / 4;
  p.tabs = a->plan_data + a->plan.tabs;
  p.per = (a->plan.most_q - 1) / a->plan.page_tokens + 2; p.Hkv = a->plan.H_kv; p.page_bits = log2_of(a->plan.page_tokens);
  if ((int64_t)p.per * a->plan.n_seqs > 0x7fffffff) return HQMQ_ERR_SHAPE;
  paged_store_kernel<<<dim3(p.per * a->plan.n_seqs, p.Hkv, 2), 128, 0, (cudaStream_t)stream>>>(p);
  HQMQ_LAUNCH_CHECK();
  return HQMQ_OK;
}

extern "C" int hqmq_paged_evict(const hqmq_paged_evict_args* a, void* stream) {
  if (!a || a->struct_size != sizeof(hqmq_paged_evict_args)) return HQMQ_ERR_ARG;
  int rc = check_plan(a->src);
  if (rc || (rc = check_plan(a->dst)) != 0) return rc;
  const hqmq_paged_plan &s = a->src, &d = a->dst;
  if (s.n_seqs != d.n_seqs || s.n_pages != d.n_pages || s.page_tokens != d.page_tokens || s.H_kv != d.H_kv || s.d != d.d) return HQMQ_ERR_SHAPE;
  if ((rc = check_pool(a->K, s)) != 0 || (rc = check_pool(a->V, s)) != 0) return rc;
  if (!a->mass || !a->new_mass || !a->kept || !a->src_data || !a->dst_data || a->first < 0 || a->last < 0) return HQMQ_ERR_ARG;
  if (((uintptr_t)a->src_data | (uintptr_t)a->dst_data | (uintptr_t)a->mass) & 15) return HQMQ_ERR_ALIGN;
  if (a->most_kept < 0 || a->longest < a->most_kept || a->kept_stride < a->most_kept || (int64_t)s.n_seqs * s.H_kv * 8 > 0x7fffffff) return HQMQ_ERR_SHAPE;
  if (a->longest == 0 || a->kept_stride == 0) return HQMQ_OK;
  EvictParams p;
  memset(&p, 0, sizeof(p));
  p.K = a->K; p.V = a->V; p.mass = a->mass; p.new_mass = a->new_mass; p.kept = a->kept;
  p.src_seqs = reinterpret_cast<const int4*>(a->src_data) + s.seqs / 4; p.src_tabs = a->src_data + s.tabs;
  p.dst_seqs = reinterpret_cast<const int4*>(a->dst_data) + d.seqs / 4; p.dst_tabs = a->dst_data + d.tabs;
  p.first = a->first; p.last = a->last; p.kept_stride = a->kept_stride; p.Hkv = s.H_kv; p.page_bits = log2_of(s.page_tokens);
  // CTAs per (sequence, head): while the SMs are not all used and a CTA has 2048 tokens or more
  const int units = s.n_seqs * s.H_kv;
  int C = 1;
  while (C < 8 && units * C * 2 <= 148 && a->longest >= 2 * C * 2048) C *= 2;
  while (C < 8 && (a->longest + C - 1) / C + 32 > kSelCached) C *= 2;
  const int per = ((a->longest + C - 1) / C + 31) & ~31;
  p.cached = per <= kSelCached ? per : kSelCached;      // (a sequence that does not fit reads its weights again, the others of the call need not)
  const size_t smem = (3 * 2048 + 4 + 2 * kSelWarps + 4 + (size_t)p.cached) * 4;
  cudaStream_t st = (cudaStream_t)stream;
  HQMQ_CHECK_CUDA(raise_smem_limit((const void*)&evict_select_kernel, smem));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = C; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
  cfg.gridDim = dim3(units * C); cfg.blockDim = dim3(kSelThreads); cfg.dynamicSmemBytes = smem; cfg.stream = st; cfg.attrs = &at; cfg.numAttrs = 1;
  void* args[] = {&p};
  HQMQ_CHECK_CUDA(cudaLaunchKernelExC(&cfg, (const void*)&evict_select_kernel, args));
  if (a->most_kept == 0) return HQMQ_OK;
  p.per_page = (a->most_kept + s.page_tokens - 1) / s.page_tokens; p.n_seqs = s.n_seqs;
  const int wpp = s.page_tokens / 64, warps = wpp > kMoveWarps ? wpp : kMoveWarps;
  const int64_t items = (int64_t)p.per_page * s.n_seqs;
  if (items > 0x7ffffff0) return HQMQ_ERR_SHAPE;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)((items * wpp + warps - 1) / warps), s.H_kv, 2); cfg.blockDim = dim3(warps * 32); cfg.dynamicSmemBytes = 0;
  HQMQ_CHECK_CUDA(cudaLaunchKernelExC(&cfg, (const void*)&evict_move_kernel, args));
  return HQMQ_OK;
}
