// The softmax weight that every key of a paged cache receives: kernels.
//
//   scores  the decode kernel's K side (paged_decode.cuh): every warp walks its stretch of tiles, writes the scores of its rows, in the
//           exp2 domain and fp32, and keeps their running maxima and sums.  A weight is compared and accumulated over many steps, so
//           products are kept whole: a codeword times its radius code has 17 bits and a flagged value times qmax / rs 24; each is the sum
//           of two fp16 operands, hi + lo, of two products (fp16 alone: relative error of a weight 1e-3; so 1e-6).  Q is fp16 after
//           division by a power of two: exact for fp16 and bf16, but for what is 2^-24 of the row's largest.
//   sum     per 512 or 128 tokens of a sequence: exp2(score - m) / l over the rows, on top of decay * prior.  Every token has one owner, so
//           nothing is added in an order of its own (no atomics).
// The scores go through memory between the two (R rows x 4 bytes a token, against 50 to 80 bytes of codes): a second decoding pass
// would cost the gathers and products again, which bound the first.
#pragma once
#include "attn_tma.cuh"
#include "paged_tile.cuh"

namespace hqmq {
namespace paged {

struct MassParams {
  PoolView pool;
  QueryView q;
  const uint16_t* tblK;
  const float* sinks;
  int table_rows, ib, row_bytes, repk, window;
  float kfac, cap, cap_in;       // cap (exp2 domain) * tanh(x * cap_in)
  float qmaxf;
  int sdt;
  const int4* seqs; const int4* units; const int* base; const int* warps; const int4* groups; const int* tabs; const int* hdr;
  int ctas;
  float* scores;                 // [head][tile of the flat sequence][16][rows of a unit]
  float2* parts;                 // [CTA][warps][2][rows]
  float2* cta_parts;             // [CTA][2][rows]
  float2* stats;                 // [head][unit][rows]: units that no CTA boundary cuts
  const float* prior; float* mass; float decay;
  uint4* wide;                   // [CTA][warps][16 N]: values of a tile with more flagged chunks than a stage holds
};

__device__ __forceinline__ float2 joined(float2 a, float2 b) {        // (m, l) of two parts
  const float m = fmaxf(a.x, b.x), u = m == -INFINITY ? 0.f : m;
  return make_float2(m, a.y * fast_exp2(a.x - u) + b.y * fast_exp2(b.x - u));
}

template <int N, int IB, int RB, int NB, bool OUTL>
__global__ void __launch_bounds__(kMassWarps * 32, 1) paged_scores_kernel(const MassParams p) {
  using FL = FastLoader<N, IB ? IB : 12, IB ? RB : 4, true>;
  constexpr int NKS = Geo<N>::NKS, NW = kMassWarps, THREADS = NW * 32, R = 8 * NB;
  const int ROW = IB ? row_bytes_of<N, IB, RB>() : p.row_bytes;
  const TileLayout L = tile_layout(ROW, false, OUTL);
  extern __shared__ __align__(16) unsigned char smem_raw[];
  const uint32_t strideK = 8u << p.repk;
  unsigned char* tblK = smem_raw;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, j = lane & 3, r = lane >> 2;
  unsigned char* ring = tblK + (size_t)(p.table_rows >> 1) * strideK + (size_t)warp * kTileStages * L.bytes;
  const uint32_t ring32 = smem_u32(ring);
  constexpr bool QREG = NB == 1;               // (queries in registers, or in shared memory as in paged_decode.cuh)
  uint2* q_s = reinterpret_cast<uint2*>(tblK + (size_t)(p.table_rows >> 1) * strideK + (size_t)NW * kTileStages * L.bytes + kPastPay) + warp * (NKS * NB * 32);
  grid_dep_launch();
  const int h = (int)blockIdx.x / p.ctas, k = (int)blockIdx.x - h * p.ctas;
  const int n_units = p.hdr[2], total = p.hdr[3], n_warps = p.ctas * NW;
  const int w = k * NW + warp;
  TileIter it;                       // the tile to be staged next
  const int2 range = it.init(p.warps + w * kWarpRecord);
  const int f0 = range.x, f1 = range.y, n = f1 - f0, u_first = __ldg(p.warps + k * NW * kWarpRecord + 2);
  const int c0 = stretch_begin(k * NW, total, n_warps), c1 = stretch_begin((k + 1) * NW, total, n_warps);
  if (c0 >= c1) return;

  // ---- the first tiles on their way, then the tables -----------------------------------------------------------------------
  Stager<false, OUTL> sg;
  sg.init(p.pool, L, lane);
  auto stage = [&](uint32_t at) {
    sg.template tile<IB ? row_bytes_of<N, IB, RB>() : 0>(p.pool, L, ROW, ring32 + at, ring + at, h, it.page, it.tile, lane);
    it.next(p.units, p.seqs, p.tabs, p.pool.page_bits);
  };
  uint32_t at0 = 0u, at1 = L.bytes, at2 = 2 * L.bytes;
  if (n > 0) stage(at0);
  if (n > 1) stage(at1);
  cp_commit();
  load_table<THREADS>(tblK, p.tblK, h, p.table_rows, p.repk);
  __syncthreads();
  if constexpr (OUTL) {
    cp_wait_all();
    __syncwarp();
    if (n > 0) stage_values<false>(p.pool, L, ring32, ring, lane);
    cp_commit();
  }
  const uint32_t laneK = (uint32_t)(lane & ((1 << p.repk) - 1)) * 8u;
  FL ld;
  ld.row_bytes = ROW; ld.row_words = ROW / 4; ld.j = j; ld.r = r; ld.sdt = p.sdt;
  auto my_wide = [&] { return p.wide + ((size_t)blockIdx.x * NW + (threadIdx.x >> 5)) * (16 * N); };
  float2* my_parts = p.parts + ((size_t)blockIdx.x * NW + warp) * 2 * R;

  int u = __ldg(p.warps + w * kWarpRecord + 2), i = 0;
  bool first_seg = true;
  while (i < n) {
    const Taken un = first_seg ? take_first(p.warps + w * kWarpRecord, f0) : take_unit(p.units, p.seqs, p.base, u);
    const Seq s = un.s;
    const int b0 = un.b0, b1 = un.b1;
    const int rows = s.q * p.q.G, row0 = un.row0;
    uint32_t qb[1][NKS][2];
    float qmul[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const float mul = load_query<NKS>(qb[0], p.q, s.q_off, h, row0 + nb * 8 + r, rows, j);
      if constexpr (!QREG) {
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) q_s[(ks * NB + nb) * 32 + lane] = make_uint2(qb[0][ks][0], qb[0][ks][1]);
      }
      qmul[nb][0] = __shfl_sync(0xffffffffu, mul, 8 * j);
      qmul[nb][1] = __shfl_sync(0xffffffffu, mul, 8 * j + 4);
    }
    const int p_first = s.kv - s.q + row0 / p.q.G, p_last = s.kv - s.q + (min(row0 + R, rows) - 1) / p.q.G;
    const int edge_lo = p.window > 0 ? p_last + 1 - p.window : 0;
    float2 ml[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) ml[nb][0] = ml[nb][1] = make_float2(-INFINITY, 0.f);
    const int i_end = min(n, b1 - f0);
    int tile = un.lo + (f0 + i - b0);
    for (; i < i_end; ++i, ++tile) {
      cp_wait_all();
      __syncwarp();
      if constexpr (OUTL) {
        if (i + 1 < n) stage_values<false>(p.pool, L, ring32 + at1, ring + at1, lane);
      }
      if (i + 2 < n) stage(at2);
      cp_commit();
      unsigned char* sp = ring + at0;
      { const uint32_t x = at0; at0 = at1; at1 = at2; at2 = x; }
      const int t0 = tile * kTile;
      const bool edge = t0 + kTile > p_first + 1 || t0 < edge_lo;
      uint32_t kw[2][FL::KW + 1];
      float rs[2];
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        const int t = nt * 8 + r;
        if constexpr (IB != 0) ld.template load_span<FL::KW, FL::LK>(kw[nt], sp + t * ROW, j, true);
        rs[nt] = key_scale(bits16_to_float(reinterpret_cast<const uint16_t*>(sp + L.rsk)[t], p.sdt));
      }
      uint32_t kcols = 0u, fk_t = 0u, before = 0u;
      bool wide = false;
      if constexpr (OUTL) {
        if (lane < kTile && t0 + lane < s.kv) fk_t = reinterpret_cast<const uint32_t*>(sp + L.flk)[lane];
        kcols = __reduce_or_sync(0xffffffffu, fk_t);
        if (kcols) {
          // Every lane its token's values times qmax / rs in two halves (see paged_decode.cuh).  An entry takes 16 bytes then: all are read
          // before any is written.
          const uint32_t own = __popc(fk_t);
          before = counts_before(own, lane);
          wide = __any_sync(0xffffffffu, before + own > (lane < 16 ? kPayK : 0xffffu) || own > 4u);
          const float rs_t = bits16_to_float(reinterpret_cast<const uint16_t*>(sp + L.rsk)[lane & 15], p.sdt);
          const float inv = rs_t != 0.f ? __fdiv_rn(p.qmaxf, rs_t) : 0.f;
          auto operand = [&](uint2 v) {
            float4 x = values_of(v, p.pool.K.out_dtype);
            x.x *= inv; x.y *= inv; x.z *= inv; x.w *= inv;
            uint4 o;
            o.x = pack_half2(x.x, x.y); o.y = pack_half2(x.z, x.w);
            const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&o.x)), g2 = __half22float2(*reinterpret_cast<const __half2*>(&o.y));
            o.z = pack_half2(x.x - g.x, x.y - g.y); o.w = pack_half2(x.z - g2.x, x.w - g2.y);
            return o;
          };
          if (!wide) {
            uint2 v[4];
            const uint2* e = reinterpret_cast<const uint2*>(sp + L.pay) + before;
            uint4* d = reinterpret_cast<uint4*>(sp + L.pay) + before;
#pragma unroll
            for (int x = 0; x < 4; ++x) if (x < (int)own) v[x] = e[x];
            __syncwarp();
#pragma unroll
            for (int x = 0; x < 4; ++x) if (x < (int)own) d[x] = operand(v[x]);
          } else {
            const int64_t ph = *reinterpret_cast<const int*>(sp + L.off + 16);
            uint32_t from = *reinterpret_cast<const uint32_t*>(sp + L.off) + before;
            for (uint32_t x = 0; x < own; ++x, ++from)
              my_wide()[before + x] = operand(from < (uint32_t)p.pool.K.out_cap ? __ldg(reinterpret_cast<const uint2*>(p.pool.K.out_vals) + ph * p.pool.K.out_cap + from) : make_uint2(0u, 0u));
          }
          __syncwarp();
        }
      }
      // two chains of the high halves' products and one of the low ones': the tensor cores cut a sum's bits with every step
      float sc[NB][4], s2[NB][4], s3[NB][4];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int x = 0; x < 4; ++x) sc[nb][x] = s2[nb][x] = s3[nb][x] = 0.f;
      static_for<0, NKS>([&](auto ks_) {
        constexpr int ks = decltype(ks_)::value;
        uint32_t a[4], b[4];
        static_for<0, 2>([&](auto nt_) {
          constexpr int nt = decltype(nt_)::value;
          uint32_t idx; __half2 rr;
          if constexpr (IB != 0) FL::template cut<ks>(kw[nt], idx, rr);
          else cut_any(reinterpret_cast<const uint32_t*>(sp + (nt * 8 + r) * ROW), j * NKS + ks, p.ib, p.ib + p.pool.K.radius_bits, idx, rr);
          const uint2 cw = *reinterpret_cast<const uint2*>(tblK + (idx * strideK + laneK));
          // hi = fl(c * r), lo = c * r - hi, which an fma gives exactly
          auto split = [&](uint32_t c, uint32_t& hi, uint32_t& lo) {
            const __half2 ch = *reinterpret_cast<const __half2*>(&c), hh = __hmul2(ch, rr), lh = __hfma2(ch, rr, __hneg2(hh));
            hi = *reinterpret_cast<const uint32_t*>(&hh); lo = *reinterpret_cast<const uint32_t*>(&lh);
          };
          split(cw.x, a[nt], b[nt]);
          split(cw.y, a[2 + nt], b[2 + nt]);
        });
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          uint2 q;
          if constexpr (QREG) q = make_uint2(qb[0][ks][0], qb[0][ks][1]);
          else q = q_s[(ks * NB + nb) * 32 + lane];
          mma16816((ks & 1) ? s2[nb] : sc[nb], a[0], a[1], a[2], a[3], q.x, q.y);
          mma16816(s3[nb], b[0], b[1], b[2], b[3], q.x, q.y);
        }
      });
      // flagged chunks: products of their own (see paged_decode.cuh)
      if constexpr (OUTL) {
        if (kcols) {
          uint32_t f[2], at[2];
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) {
            const uint32_t w_ = __shfl_sync(0xffffffffu, fk_t, nt * 8 + r);
            f[nt] = w_ >> (j * NKS);
            at[nt] = __shfl_sync(0xffffffffu, before, nt * 8 + r) + __popc(w_ & ((1u << (j * NKS)) - 1u));
          }
          auto step = [&](int ks, bool some, auto query) {
            uint32_t a[4], b[4];
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
              const bool mine = some && ((f[nt] >> ks) & 1u);
              const uint4 v = wide ? __ldcg(my_wide() + at[nt]) : reinterpret_cast<const uint4*>(sp + L.pay)[at[nt]];
              a[nt] = mine ? v.x : 0u; a[2 + nt] = mine ? v.y : 0u;
              b[nt] = mine ? v.z : 0u; b[2 + nt] = mine ? v.w : 0u;
              at[nt] += mine ? 1u : 0u;
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              const uint2 q = query(nb);
              mma16816(s2[nb], a[0], a[1], a[2], a[3], q.x, q.y);
              mma16816(s3[nb], b[0], b[1], b[2], b[3], q.x, q.y);
            }
          };
          if constexpr (QREG) {
            uint32_t steps = kcols;
            if constexpr (NKS == 8) { steps |= steps >> 16; steps |= steps >> 8; } else { steps |= steps >> 8; steps |= steps >> 4; }
            static_for<0, NKS>([&](auto ks_) {
              constexpr int ks = decltype(ks_)::value;
              if (steps & (1u << ks)) step(ks, true, [&](int) { return make_uint2(qb[0][ks][0], qb[0][ks][1]); });
            });
          } else {
            uint32_t left = (kcols >> (j * NKS)) & ((1u << NKS) - 1u);
            do {
              const int ks = left ? __ffs(left) - 1 : 0;
              const bool some = left != 0u;
              left &= left - 1u;
              step(ks, some, [&](int nb) { return q_s[(ks * NB + nb) * 32 + lane]; });
            } while (__any_sync(0xffffffffu, left != 0u));
          }
        }
      }
      float* dst = p.scores + ((int64_t)h * total + f0 + i) * (kTile * R) + r * R + 2 * j;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          float v = (sc[nb][x] + s2[nb][x] + s3[nb][x]) * (rs[x >> 1] * (p.kfac * qmul[nb][x & 1]));
          if (p.cap > 0.f) v = p.cap * tanhf(v * p.cap_in);
          if (edge) {
            const int t = t0 + (x >> 1) * 8 + r, pos = min(p_first + (row0 % p.q.G + nb * 8 + 2 * j + (x & 1)) / p.q.G, s.kv - 1);
            if (t > pos || (p.window > 0 && t <= pos - p.window)) v = -INFINITY;
          }
          sc[nb][x] = v;
        }
        // (each lane keeps the maximum and sum of its own tokens)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float m = fmaxf(sc[nb][e], sc[nb][2 + e]);
          if (m > ml[nb][e].x) { ml[nb][e].y *= fast_exp2(ml[nb][e].x - m); ml[nb][e].x = m; }
          const float b = ml[nb][e].x == -INFINITY ? 0.f : ml[nb][e].x;
          ml[nb][e].y += fast_exp2(sc[nb][e] - b) + fast_exp2(sc[nb][2 + e] - b);
        }
        *reinterpret_cast<float2*>(dst + nb * 8) = make_float2(sc[nb][0], sc[nb][1]);
        *reinterpret_cast<float2*>(dst + 8 * R + nb * 8) = make_float2(sc[nb][2], sc[nb][3]);
      }
    }
    const bool whole = b0 >= f0 && b1 <= f1;
    float2* dst = whole ? p.stats + ((int64_t)h * n_units + u) * R : my_parts + (first_seg ? 0 : R);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float2 v = ml[nb][e];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) v = joined(v, make_float2(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o)));
        if (r == 0) dst[nb * 8 + 2 * j + e] = v;
      }
    first_seg = false;
    ++u;
  }
  __syncthreads();
  // units cut between the CTA's warps
  const float2* cta = p.parts + (size_t)blockIdx.x * NW * 2 * R;
  for (int v = u_first; v < n_units; ++v) {
    const int b0 = __ldg(p.base + v), b1 = __ldg(p.base + v + 1);
    if (b0 >= c1) break;
    const int wa = warp_of(b0, total, n_warps), wb = warp_of(b1 - 1, total, n_warps);
    if (wa == wb) continue;
    const int la = max(wa - k * NW, 0), lb = min(wb - k * NW, NW - 1);
    const int first_slot = b0 > stretch_begin(k * NW + la, total, n_warps) ? 1 : 0;
    float2* dst = wa >= k * NW && wb < (k + 1) * NW ? p.stats + ((int64_t)h * n_units + v) * R
                                                    : p.cta_parts + ((size_t)blockIdx.x * 2 + (b0 > c0 ? 1 : 0)) * R;
    for (int row = threadIdx.x; row < R; row += THREADS) {
      float2 a = make_float2(-INFINITY, 0.f);
      for (int x = la; x <= lb; ++x) a = joined(a, __ldcg(cta + (x * 2 + (x == la ? first_slot : 0)) * R + row));
      dst[row] = a;
    }
  }
}

// blockIdx.x = a group of tokens of a sequence, blockIdx.y = KV head.
template <int NB>
__global__ void __launch_bounds__(256) paged_mass_kernel(const MassParams p) {
  constexpr int R = 8 * NB, LPT = R / 4, kGroup = mass_group(R), PER = kGroup * LPT / 256;
  __shared__ float2 s_stat[R];
  // (the plan, and what the weights were, are there before the kernel ahead of this one)
  const int n_units = p.hdr[2], total = p.hdr[3];
  const bool mine = (int)blockIdx.x < p.hdr[4];
  const int h = blockIdx.y, n_warps = p.ctas * kMassWarps;
  const int4 gr = __ldg(p.groups + (mine ? blockIdx.x : 0)), sq4 = __ldg(p.seqs + gr.x);
  const Seq s{sq4.x, sq4.y, sq4.z, sq4.w};
  const int rows = s.q * p.q.G, tid = threadIdx.x;
  float acc[PER], was[PER];
  int64_t at[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    acc[i] = was[i] = 0.f;
    at[i] = -1;
    const int t = gr.y + (tid + i * 256) / LPT;
    if (mine && tid % LPT == 0 && t < s.kv) {
      const int page = __ldg(p.tabs + s.tab + (t >> p.pool.page_bits));
      at[i] = (((int64_t)page * p.pool.Hkv + h) << p.pool.page_bits) + (t & ((1 << p.pool.page_bits) - 1));
      if (p.prior) was[i] = p.prior[at[i]];
    }
  }
  grid_dep_wait();
  if (!mine) return;
  for (int u = gr.z; u < gr.w; ++u) {
    const int4 un = __ldg(p.units + u);
    if (un.w * kTile <= gr.y || un.z * kTile >= gr.y + kGroup) continue;      // (the same for all threads)
    const int b0 = __ldg(p.base + u), b1 = __ldg(p.base + u + 1);
    __syncthreads();
    if (tid < R) {
      const int k0 = warp_of(b0, total, n_warps) / kMassWarps, k1 = warp_of(b1 - 1, total, n_warps) / kMassWarps;
      float2 a = make_float2(-INFINITY, 0.f);
      if (k0 == k1) a = __ldcg(p.stats + ((int64_t)h * n_units + u) * R + tid);
      else
        for (int k = k0; k <= k1; ++k) {
          const int slot = k == k0 && b0 > stretch_begin(k * kMassWarps, total, n_warps) ? 1 : 0;
          a = joined(a, __ldcg(p.cta_parts + ((size_t)(h * p.ctas + k) * 2 + slot) * R + tid));
        }
      const int row = un.y + tid;
      float inv = 0.f;
      if (row < rows) {
        bool none = a.x == -INFINITY;
        if (p.sinks && !none) {
          const float sk = __ldg(p.sinks + h * p.q.G + row % p.q.G) * 1.4426950408889634f;
          none = sk - a.x > 126.f;
          a.y += fast_exp2(sk - a.x);
        }
        inv = none ? 0.f : 1.f / a.y;
      }
      s_stat[tid] = make_float2(a.x == -INFINITY ? 0.f : a.x, inv);
    }
    __syncthreads();
    const float4* sc = reinterpret_cast<const float4*>(p.scores + ((int64_t)h * total + b0 - un.z) * (kTile * R));      // of token 0
    const int q4 = (tid % LPT) * 4;
    const float2 s0 = s_stat[q4], s1 = s_stat[q4 + 1], s2 = s_stat[q4 + 2], s3 = s_stat[q4 + 3];
    const int lo = un.z * kTile, hi = min(un.w * kTile, s.kv);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int t = gr.y + (tid + i * 256) / LPT;
      if (t >= lo && t < hi) {
        const float4 v = __ldcg(sc + (int64_t)t * LPT + tid % LPT);
        acc[i] += fast_exp2(v.x - s0.x) * s0.y + fast_exp2(v.y - s1.x) * s1.y + fast_exp2(v.z - s2.x) * s2.y + fast_exp2(v.w - s3.x) * s3.y;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
#pragma unroll
    for (int o = 1; o < LPT; o <<= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
    if (at[i] >= 0) p.mass[at[i]] = p.prior ? fmaf(p.decay, was[i], acc[i]) : acc[i];
  }
}

const void* scores_kernel_128(int ib, int rb, int nb, bool outl);
const void* scores_kernel_64(int ib, int rb, int nb, bool outl);
template <int N, int NB, bool OUTL>
const void* pick_scores(int ib, int rb) {
  if (ib == 10 && rb == 3) return (const void*)&paged_scores_kernel<N, 10, 3, NB, OUTL>;
  if (ib == 12 && rb == 4) return (const void*)&paged_scores_kernel<N, 12, 4, NB, OUTL>;
  if (ib == 13 && rb == 6) return (const void*)&paged_scores_kernel<N, 13, 6, NB, OUTL>;
  return (const void*)&paged_scores_kernel<N, 0, 0, NB, OUTL>;
}
template <int N>
const void* pick_scores_kernel(int ib, int rb, int nb, bool outl) {
  if (nb == 1) return outl ? pick_scores<N, 1, true>(ib, rb) : pick_scores<N, 1, false>(ib, rb);
  return outl ? pick_scores<N, 4, true>(ib, rb) : pick_scores<N, 4, false>(ib, rb);
}

}  // namespace paged
}  // namespace hqmq
