// Attention of a few query rows per sequence over a paged cache: the kernel.
//
// The tile's arithmetic is that of the staged decode kernels (attn_kernel.cuh): S^T = K Q^T with the 16 tokens as rows and the query
// rows as columns, O^T += V^T P^T, operands gathered from shared-memory tables straight into fragments.  What differs:
//   - a warp walks its own stretch of tiles from unit to unit (paged.cuh);
//   - flagged chunks, whose fields decode to zero.  A lane per token turns its values into fp16(x * qmax / rs), what the table would have given.
//     Where the index bits of a field leave room behind the codebook, the values become table entries of the warp's own and the fields of the
//     staged row point to them, so the look-ups below find them and nothing branches on a flag.  Where they do not (13-bit fields, codebooks
//     without room, fields of any width), or a tile has more than the warp has entries, they are products of their own behind
//     the others': a lane, which owns 2 tokens x N / 4 chunks of K and 4 x N / 8 of V, finds its values by counting the flags before them.
//     (16 sequences of 16 to 32 k tokens, two outlier channels a head in K: values put into the fragments by branches 381 us, products of
//     their own 316, table entries 269; 173 without outliers.  Repeated passes of the main products for a tile with too many, in place of the
//     products of their own, took 277 to 299; without either the kernel would take 254);
//   - V's scales enter P relative to the largest one seen, a power of two that the accumulators are rescaled by like by the maximum, so
//     that values of any size keep their bits.
// What bounds it: instructions, 1004 a tile with those outliers and about 690 without, at 60 to 62 % of the issue slots (chains of look-up,
// multiply, product in 16 warps of 128 registers).
#pragma once
#include "attn_tma.cuh"
#include "paged_tile.cuh"

namespace hqmq {
namespace paged {

struct DecodeParams {
  PoolView pool;
  QueryView q;
  void* O; int o_dtype, o_vec; int64_t os_t, os_h;
  const uint16_t* tblK; const uint16_t* tblV;
  const float* sinks;
  int table_rows, ib, row_bytes, repk, repv, window;
  float kfac, cap_log2;          // kfac: what a product is multiplied by beside rs (softmax scale * log2 e / qmax; with a cap over cap_log2)
  float qmaxf, vfac;             // 1 / qmax
  int sdt, pay_bf16;             // type of the scales; whether the flagged chunks' values are bf16 (else fp16)
  const int4* seqs; const int4* units; const int* base; const int* warps; const int4* cuts; const int* tabs; const int* hdr;
  int ctas, fused, ext_k, ext_v; // fused: the CTAs of a head are a cluster; entries of every warp's own that the tables have (0: none)
  float* parts;                  // [CTA][warps][2][part], then [CTA][2][part]
  uint2* wide;                   // [CTA][warps][K, V][16 N]: values of a tile with more flagged chunks than a stage holds
};

// Values of flagged chunks as table entries: where the index bits of a field leave room behind the codebook (2^(bits - 1) sign-folded
// entries; 896 of them at S = 96, 1792 at 192), the warps share it out, up to the entries that a tile has staged: 56 and 32 of K's and V's at
// S = 96 with 16 warps, 64 and 32 at 192.  Less than kExtLeast would not take one chunk column that is flagged in every token.  A tile with more
// has products of their own, as where there is no room.  (16 x 8k, 8 heads of 128, S = 96, one to four such columns in K: 98, 102, 106
// and 118 us; with 36 and 24 entries and tiles with more through global memory 98, 102, 145 and 167.)
constexpr int kExtLeast = 16;
__host__ __device__ constexpr bool has_ext(int ib) { return ib == 12 || ib == 13; }
// Field c of a row: IB + RB bits, the row's words the writing lane's own.
template <int IB, int RB>
__device__ __forceinline__ void put_field(unsigned char* row, int c, uint32_t v) {
  constexpr int CB = IB + RB;
  if constexpr (CB == 16) reinterpret_cast<uint16_t*>(row)[c] = (uint16_t)v;
  else {
    uint32_t* w = reinterpret_cast<uint32_t*>(row) + ((c * CB) >> 5);
    const int sh = (c * CB) & 31;
    constexpr uint32_t mask = (1u << CB) - 1u;
    w[0] = (w[0] & ~(mask << sh)) | (v << sh);
    if (sh + CB > 32) w[1] = (w[1] & ~(mask >> (32 - sh))) | (v >> (32 - sh));
  }
}

template <int N, int NB> __host__ __device__ constexpr int part_floats() { return NB * (N / 4 * 128 + 16); }

// One finished row pair of a lane: value (i, e) of a part is head 2j + (e & 1), dim 4 (r NVG + i / 2) + 2 (i & 1) + e / 2.
template <int N>
__device__ __forceinline__ void emit_pair(const DecodeParams& p, const Seq& s, int h, int row, int rows, int r, int i, float a, float b) {
  constexpr int NVG = Geo<N>::NVG;
  if (row >= rows) return;
  const int qi = row / p.q.G, g = row - qi * p.q.G, x = 4 * (r * NVG + (i >> 1)) + 2 * (i & 1);
  const int64_t o = (int64_t)(s.q_off + qi) * p.os_t + (int64_t)(h * p.q.G + g) * p.os_h + x;
  if (p.o_vec) {
    *reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(p.O) + o) =
        (uint32_t)float_to_bits16(a, p.o_dtype) | ((uint32_t)float_to_bits16(b, p.o_dtype) << 16);
  } else { store_float(p.O, o, a, p.o_dtype); store_float(p.O, o + 1, b, p.o_dtype); }
}
// What a row's sum is with its head's sink: m and l in the exp2 domain; returns 1 / l (0 for a row that saw nothing).
__device__ __forceinline__ float inverse_sum(const DecodeParams& p, int h, int row, int rows, float m, float l) {
  if (p.sinks && row < rows) {
    const float sk = __ldg(p.sinks + h * p.q.G + row % p.q.G) * 1.4426950408889634f;
    if (m == -INFINITY || sk - m > 126.f) return 0.f;
    l += fast_exp2(sk - m);
  }
  return l != 0.f ? 1.f / l : 0.f;
}

// The parts of a unit, element `idx` of [NB][N / 4][32] quadruples: merged value and the row pair's maxima and sums.
template <int N, int NB, typename PartOf>
__device__ __forceinline__ void merge_parts(int idx, int n, const PartOf& part_of, float4& v, float2& m, float2& l) {
  constexpr int PER = N / 4 * 32;
  const int nb = idx / PER, j = idx & 3;
  m = make_float2(-INFINITY, -INFINITY);
  const int at = NB * PER * 4 + nb * 16 + 2 * j;
  v = make_float4(0.f, 0.f, 0.f, 0.f);
  l = make_float2(0.f, 0.f);
  // (one pass with a running maximum: no load waits for another)
#pragma unroll 8
  for (int k = 0; k < n; ++k) {
    const float* pk = part_of(k);
    const float2 mk = __ldcg(reinterpret_cast<const float2*>(pk + at)), lk = __ldcg(reinterpret_cast<const float2*>(pk + at + 8));
    const float4 x = __ldcg(reinterpret_cast<const float4*>(pk) + idx);
    const float nx = fmaxf(m.x, mk.x), ny = fmaxf(m.y, mk.y), ux = nx == -INFINITY ? 0.f : nx, uy = ny == -INFINITY ? 0.f : ny;
    const float ax = fast_exp2(m.x - ux), ay = fast_exp2(m.y - uy), wx = fast_exp2(mk.x - ux), wy = fast_exp2(mk.y - uy);
    l.x = fmaf(lk.x, wx, l.x * ax); l.y = fmaf(lk.y, wy, l.y * ay);
    v.x = fmaf(x.x, wx, v.x * ax); v.y = fmaf(x.y, wy, v.y * ay); v.z = fmaf(x.z, wx, v.z * ax); v.w = fmaf(x.w, wy, v.w * ay);
    m.x = nx; m.y = ny;
  }
}
__device__ __forceinline__ Seq seq_of(const DecodeParams& p, int u) {
  const int4 sq = __ldg(p.seqs + __ldg(&p.units[u].x));
  return Seq{sq.x, sq.y, sq.z, sq.w};
}
template <int N, int NB>
__device__ __forceinline__ void emit_merged(const DecodeParams& p, const Seq& s, int h, int idx, float4 v, float2 m, float2 l) {
  constexpr int PER = N / 4 * 32;
  const int rows = s.q * p.q.G, nb = idx / PER, i = (idx - nb * PER) >> 5, lane = idx & 31, row = nb * 8 + 2 * (lane & 3);
  const float ia = inverse_sum(p, h, row, rows, m.x, l.x), ib = inverse_sum(p, h, row + 1, rows, m.y, l.y);
  emit_pair<N>(p, s, h, row, rows, lane >> 2, i, v.x * ia, v.z * ia);
  emit_pair<N>(p, s, h, row + 1, rows, lane >> 2, i, v.y * ib, v.w * ib);
}

template <int N, int IB, int RB, int NB, bool OUTL>
__global__ void __launch_bounds__((NB == 1 ? kDecWarps : kDecWarpsWide) * 32, 1) paged_decode_kernel(const DecodeParams p) {
  using FL = FastLoader<N, IB ? IB : 12, IB ? RB : 4, true>;
  constexpr int NKS = Geo<N>::NKS, NVG = Geo<N>::NVG, NOT = 2 * NVG;
  constexpr int NW = NB == 1 ? kDecWarps : kDecWarpsWide, THREADS = NW * 32, PART = part_floats<N, NB>();
  const bool ext = OUTL && has_ext(IB) && p.ext_k != 0;
  const int ROW = IB ? row_bytes_of<N, IB, RB>() : p.row_bytes;
  const TileLayout L = tile_layout(ROW, true, OUTL);
  extern __shared__ __align__(16) unsigned char smem_raw[];
  const uint32_t strideK = 8u << p.repk, strideV = 8u << p.repv;
  unsigned char* tblK = smem_raw;
  unsigned char* tblV = smem_raw + (size_t)((p.table_rows >> 1) + (ext ? NW * p.ext_k : 0)) * strideK;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, j = lane & 3, r = lane >> 2;
  unsigned char* rings = tblV + (size_t)((p.table_rows >> 1) + (ext ? NW * p.ext_v : 0)) * strideV;
  unsigned char* ring = rings + (size_t)warp * kTileStages * L.bytes;
  const uint32_t ring32 = smem_u32(ring);
  // (of 32 rows, a warp's queries are 8 KB in shared memory, as the fragments that a lane reads: registers hold the accumulators)
  constexpr bool QREG = NB <= 2;
  uint2* q_s = reinterpret_cast<uint2*>(rings + (size_t)NW * kTileStages * L.bytes + kPastPay) + warp * (NKS * NB * 32);
  grid_dep_launch();
  const int h = (int)blockIdx.x / p.ctas, k = (int)blockIdx.x - h * p.ctas;
  const int n_units = p.hdr[0], total = p.hdr[1], n_warps = p.ctas * NW;
  const int w = k * NW + warp;
  TileIter it;                       // the tile to be staged next
  const int2 range = it.init(p.warps + w * kWarpRecord);
  const int f0 = range.x, f1 = range.y, n = f1 - f0, u_first = __ldg(p.warps + k * NW * kWarpRecord + 2);
  const int c0 = stretch_begin(k * NW, total, n_warps), c1 = stretch_begin((k + 1) * NW, total, n_warps);

  // ---- the first tiles on their way, then the tables -----------------------------------------------------------------------
  Stager<true, OUTL> sg;
  sg.init(p.pool, L, lane);
  auto stage = [&](uint32_t at) {    // the tile that `it` is at, to the stage at `at`
    sg.template tile<IB ? row_bytes_of<N, IB, RB>() : 0>(p.pool, L, ROW, ring32 + at, ring + at, h, it.page, it.tile, lane);
    it.next(p.units, p.seqs, p.tabs, p.pool.page_bits);
  };
  uint32_t at0 = 0u, at1 = L.bytes, at2 = 2 * L.bytes;       // stages of the tile at hand, of the next two
  if (n > 0) stage(at0);
  if (n > 1) stage(at1);
  cp_commit();
  load_table<THREADS>(tblK, p.tblK, h, p.table_rows, p.repk);
  load_table<THREADS>(tblV, p.tblV, h, p.table_rows, p.repv);
  __syncthreads();
  if constexpr (OUTL) {
    cp_wait_all();
    __syncwarp();
    if (n > 0) stage_values<true>(p.pool, L, ring32, ring, lane);
    cp_commit();
  }

  const uint32_t laneK = (uint32_t)(lane & ((1 << p.repk) - 1)) * 8u, laneV = (uint32_t)(lane & ((1 << p.repv) - 1)) * 8u;
  // (rows of 64 bytes: the odd groups of lanes take their pair of V's tokens in the other order, which spreads the loads over the banks)
  constexpr bool kSwz = IB != 0 && row_bytes_of<N, IB, RB>() % 128 == 64;
  const int vswz = kSwz ? (j & 1) : 0;
  FL ld;
  ld.row_bytes = ROW; ld.row_words = ROW / 4; ld.j = j; ld.r = r; ld.sdt = p.sdt;
  const float kfac = p.kfac;
  auto my_wide = [&] { return p.wide + ((size_t)blockIdx.x * NW + (threadIdx.x >> 5)) * (32 * N); };     // (hardly ever asked for: not held)
  float* my_parts = p.parts + ((size_t)blockIdx.x * NW + warp) * 2 * PART;

  int u = __ldg(p.warps + w * kWarpRecord + 2), i = 0;
  bool first_seg = true;
  while (i < n) {
    // ---- a unit, or what the stretch has of it ------------------------------------------------------------------------------
    const Taken un = first_seg ? take_first(p.warps + w * kWarpRecord, f0) : take_unit(p.units, p.seqs, p.base, u);
    const Seq s = un.s;
    const int b0 = un.b0, b1 = un.b1;
    const int rows = s.q * p.q.G;
    uint32_t qb[QREG ? NB : 1][NKS][2];
    float qmul[NB][2];                     // of this lane's two rows
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const float mul = load_query<NKS>(qb[QREG ? nb : 0], p.q, s.q_off, h, nb * 8 + r, rows, j) * kfac;
      qmul[nb][0] = __shfl_sync(0xffffffffu, mul, 8 * j);
      qmul[nb][1] = __shfl_sync(0xffffffffu, mul, 8 * j + 4);
      if constexpr (!QREG) {
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) q_s[(ks * NB + nb) * 32 + lane] = make_uint2(qb[0][ks][0], qb[0][ks][1]);
      }
    }
    const int p_first = s.kv - s.q, edge_lo = p.window > 0 ? s.kv - p.window : 0;    // (the last query sees nothing before edge_lo)
    float m_run[NB][2], l_run[NB][2], o[NB][NOT][4];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      m_run[nb][0] = m_run[nb][1] = -INFINITY;
      l_run[nb][0] = l_run[nb][1] = 0.f;
#pragma unroll
      for (int x = 0; x < NOT; ++x) o[nb][x][0] = o[nb][x][1] = o[nb][x][2] = o[nb][x][3] = 0.f;
    }
    float v_pow = 0.f, v_inv = 0.f;        // the power of two that V's scales are relative to (0: none yet), and one over it
    const int i_end = min(n, b1 - f0);
    int tile = un.lo + (f0 + i - b0);
    for (; i < i_end; ++i, ++tile) {
      cp_wait_all();
      __syncwarp();
      if constexpr (OUTL) {
        if (i + 1 < n) stage_values<true>(p.pool, L, ring32 + at1, ring + at1, lane);
      }
      if (i + 2 < n) stage(at2);
      cp_commit();
      unsigned char* sp = ring + at0;
      { const uint32_t x = at0; at0 = at1; at1 = at2; at2 = x; }
      const int t0 = tile * kTile;
      const bool edge = t0 + kTile > p_first + 1 || t0 < edge_lo;

      uint32_t kcols = 0u, vcols = 0u;       // the columns of chunks that have a flagged one in some token, where those are products of their own
      uint32_t fl = 0u, before = 0u;         // lanes 0..15: K's tokens, 16..31: V's: flags, and entries of the tile's earlier tokens
      bool wide = false;
      if constexpr (OUTL) {
        if (t0 + (lane & 15) < s.kv && (lane < 16 ? p.pool.K.flags : p.pool.V.flags)) fl = reinterpret_cast<const uint32_t*>(sp + L.flk)[lane];
        if (__any_sync(0xffffffffu, fl != 0u)) {
          const uint32_t own = __popc(fl);
          before = counts_before(own, lane);
          const bool as_entries = ext && __all_sync(0xffffffffu, before + own <= (uint32_t)(lane < 16 ? p.ext_k : p.ext_v));
          if (!as_entries) {
            kcols = __reduce_or_sync(0xffffffffu, lane < 16 ? fl : 0u);
            vcols = __reduce_or_sync(0xffffffffu, lane < 16 ? 0u : fl);
            wide = __any_sync(0xffffffffu, before + own > (uint32_t)(lane < 16 ? kPayK : kPayV));
          }
          // every lane its token's values, in place
          const float rs = bits16_to_float(reinterpret_cast<const uint16_t*>(sp + L.rsk)[lane], p.sdt);
          const float inv = rs != 0.f ? __fdividef(p.qmaxf, rs) : 0.f;
          const bool bf = p.pay_bf16 != 0;
          auto operand = [&](uint2 v) { return make_uint2(scaled_pair(v.x, inv, bf), scaled_pair(v.y, inv, bf)); };
          uint2* e = reinterpret_cast<uint2*>(sp + L.pay + (lane < 16 ? 0 : kPayK * 8)) + before;
          if (as_entries) {
            // Entries behind the codebook are this warp's: the value goes where the lane that decodes the chunk will look, and the chunk's
            // field in the staged row becomes that entry's, times one.
            const bool of_v = lane >= 16;
            const int tok = lane & 15;
            uint32_t entry = (uint32_t)(p.table_rows >> 1) + (of_v ? warp * p.ext_v : warp * p.ext_k) + before;
            const uint32_t stride = of_v ? strideV : strideK, mask = (stride >> 3) - 1u;
            uint32_t dst = (of_v ? (uint32_t)(tblV - smem_raw) : 0u) + entry * stride;
            unsigned char* row = sp + (of_v ? L.v : 0) + tok * ROW;
            // (the lane that decodes it: K (token & 7) * 4 + chunk / NKS, V chunk / NVG * 4 + (token & 7) / 2)
            constexpr int kLog = NKS == 8 ? 3 : 2, vLog = NVG == 4 ? 2 : 1;
            const uint32_t rd0 = of_v ? (uint32_t)(tok & 7) >> 1 : (uint32_t)(tok & 7) << 2;
            const int down = of_v ? vLog : kLog, up = of_v ? 2 : 0;
            auto place = [&](auto bf_c) {
              constexpr bool BF = decltype(bf_c)::value;
              for (uint32_t m = fl; m; m &= m - 1u, ++e, ++entry, dst += stride) {
                const int c = __ffs(m) - 1;
                const uint2 v = *e;
                *reinterpret_cast<uint2*>(smem_raw + dst + (((rd0 | (uint32_t)(c >> down) << up) & mask) << 3)) =
                    make_uint2(scaled_pair(v.x, inv, BF), scaled_pair(v.y, inv, BF));
                if constexpr (has_ext(IB)) put_field<IB, RB>(row, c, entry << 1 | 1u << IB);
              }
            };
            if (bf) place(std::true_type{});
            else place(std::false_type{});
          } else if (!wide) {
            for (uint32_t x = 0; x < own; ++x, ++e) *e = operand(*e);
          } else {
            const int64_t ph = *reinterpret_cast<const int*>(sp + L.off + 16);
            const hqmq_packed& pk = lane < 16 ? p.pool.K : p.pool.V;
            uint2* far = my_wide() + (lane < 16 ? 0 : 16 * N) + before;
            uint32_t from = reinterpret_cast<const uint32_t*>(sp + L.off)[lane < 16 ? 0 : 2] + before;
            for (uint32_t x = 0; x < own; ++x, ++far, ++from)
              *far = operand(from < (uint32_t)pk.out_cap ? __ldg(reinterpret_cast<const uint2*>(pk.out_vals) + ph * pk.out_cap + from) : make_uint2(0u, 0u));
          }
          __syncwarp();
        }
      }
      // Operands of flagged chunks at places counted in entries.  No branch per lane: a place is one of this tile's, or the one behind
      // the last, whether the lane has a value there or not.
      auto values_at = [&](uint2* v, const uint32_t* at, int n_, bool of_v) {
        if (!wide) {
#pragma unroll
          for (int x = 0; x < n_; ++x) v[x] = reinterpret_cast<const uint2*>(sp + L.pay + (of_v ? kPayK * 8 : 0))[at[x]];
        } else {
#pragma unroll
          for (int x = 0; x < n_; ++x) v[x] = __ldcg(my_wide() + (of_v ? 16 * N : 0) + at[x]);
        }
      };

      // ---- this lane's fields and scales ------------------------------------------------------------------------------
      uint32_t kw[2][FL::KW + 1], vw[4][FL::VW + 1];
      float ksc[2], vsc[2];
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        const int t = nt * 8 + r;
        if constexpr (IB != 0) ld.template load_span<FL::KW, FL::LK>(kw[nt], sp + t * ROW, j, true);
        ksc[nt] = key_scale(bits16_to_float(reinterpret_cast<const uint16_t*>(sp + L.rsk)[t], p.sdt));
        vsc[nt] = bits16_to_float(reinterpret_cast<const uint16_t*>(sp + L.rsv)[t], p.sdt) * p.vfac;
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int t = 2 * j + ((x & 1) ^ vswz) + (x >> 1) * 8;
        if constexpr (IB != 0) ld.template load_span<FL::VW, FL::LV>(vw[x], sp + L.v + t * ROW, r, !edge || t0 + t < s.kv);
      }
      // ---- S^T = K Q^T ---------------------------------------------------------------------------------------------------------
      float sc[NB][4], s2[NB][4];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int x = 0; x < 4; ++x) sc[nb][x] = s2[nb][x] = 0.f;
      static_for<0, NKS>([&](auto ks_) {
        constexpr int ks = decltype(ks_)::value;
        uint32_t a[4];
        static_for<0, 2>([&](auto nt_) {
          constexpr int nt = decltype(nt_)::value;
          uint32_t idx; __half2 rr;
          if constexpr (IB != 0) FL::template cut<ks>(kw[nt], idx, rr);
          else cut_any(reinterpret_cast<const uint32_t*>(sp + (nt * 8 + r) * ROW), j * NKS + ks, p.ib, p.ib + p.pool.K.radius_bits, idx, rr);
          const uint2 cw = *reinterpret_cast<const uint2*>(tblK + (idx * strideK + laneK));
          a[nt] = hmul2_u32(cw.x, rr);
          a[2 + nt] = hmul2_u32(cw.y, rr);
        });
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          uint2 q;
          if constexpr (QREG) q = make_uint2(qb[nb][ks][0], qb[nb][ks][1]);
          else q = q_s[(ks * NB + nb) * 32 + lane];
          mma16816((ks & 1) ? s2[nb] : sc[nb], a[0], a[1], a[2], a[3], q.x, q.y);
        }
      });

      // Flagged chunks of K that are no table entries: one more product for every step of the others' that has some.  (Put into the fragments above instead, the
      // branches of every step kept the look-ups from being issued ahead: 381 us against 170 without outliers for 16 x 32k, 287 with that part
      // left out.  A column per group of lanes at a time, which takes fewer products, pays where the queries are in shared memory: picked from
      // registers by selects it took 145 instructions a tile, 339 us against 317; of 32 rows it takes 88 us against 102 for 8 x 8111.)
      if constexpr (OUTL) {
        if (kcols) {
          uint32_t f[2], at[2];
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) {
            const uint32_t w_ = __shfl_sync(0xffffffffu, fl, nt * 8 + r);
            f[nt] = w_ >> (j * NKS);
            at[nt] = __shfl_sync(0xffffffffu, before, nt * 8 + r) + __popc(w_ & ((1u << (j * NKS)) - 1u));
          }
          auto step = [&](int ks, bool some, auto query) {
            uint2 v[2];
            values_at(v, at, 2, false);
            uint32_t a[4];
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
              const bool mine = some && ((f[nt] >> ks) & 1u);
              a[nt] = mine ? v[nt].x : 0u; a[2 + nt] = mine ? v[nt].y : 0u;
              at[nt] += mine ? 1u : 0u;
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) { const uint2 q = query(nb); mma16816(s2[nb], a[0], a[1], a[2], a[3], q.x, q.y); }
          };
          if constexpr (QREG) {
            uint32_t steps = kcols;
            if constexpr (NKS == 8) { steps |= steps >> 16; steps |= steps >> 8; } else { steps |= steps >> 8; steps |= steps >> 4; }
            static_for<0, NKS>([&](auto ks_) {
              constexpr int ks = decltype(ks_)::value;
              if (steps & (1u << ks)) step(ks, true, [&](int nb) { return make_uint2(qb[nb][ks][0], qb[nb][ks][1]); });
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

      // ---- scale, cap, mask -----------------------------------------------------------------------------------------------------
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int x = 0; x < 4; ++x) sc[nb][x] = (sc[nb][x] + s2[nb][x]) * (ksc[x >> 1] * qmul[nb][x & 1]);
      if (p.cap_log2 > 0.f) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int x = 0; x < 4; ++x) sc[nb][x] = p.cap_log2 * tanh_of(sc[nb][x]);
      }
      if (edge) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int t = t0 + (x >> 1) * 8 + r, pos = min(p_first + (nb * 8 + 2 * j + (x & 1)) / p.q.G, s.kv - 1);
            if (t > pos || (p.window > 0 && t <= pos - p.window)) sc[nb][x] = -INFINITY;
          }
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
          if (t0 + nt * 8 + r >= s.kv) vsc[nt] = 0.f;
      }

      // ---- maxima: raised, with the accumulators, only where a score exceeds one by 2^4, or V's scale its power ---------------------
      constexpr float kSlack = 4.f;
      bool need = fmaxf(vsc[0], vsc[1]) > v_pow;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 2; ++e) need |= fmaxf(sc[nb][e], sc[nb][2 + e]) > m_run[nb][e] + kSlack;
      if (__any_sync(0xffffffffu, need)) {
        float big = fmaxf(vsc[0], vsc[1]);
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 4));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 8));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 16));
        float vs = 1.f;
        if (big > v_pow) {
          // the next power of two, within 2^-100 .. 2^100
          const int e = min(100, max(-100, (int)(__float_as_uint(big) >> 23) - 126));
          const float np = __uint_as_float((uint32_t)(127 + e) << 23);
          vs = v_pow * __uint_as_float((uint32_t)(127 - e) << 23);
          v_pow = np;
          v_inv = __uint_as_float((uint32_t)(127 - e) << 23);
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float m = fmaxf(sc[nb][e], sc[nb][2 + e]);
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
            const float m_new = fmaxf(m_run[nb][e], m);
            const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_run[nb][e] - m_new);
            m_run[nb][e] = m_new;
            l_run[nb][e] *= alpha;
            const float oa = alpha * vs;
#pragma unroll
            for (int x = 0; x < NOT; ++x) { o[nb][x][e] *= oa; o[nb][x][2 + e] *= oa; }
          }
      }

      // ---- P: fp16(p * scale of V) -----------------------------------------------------------------------------------------------------
      uint32_t pb[NB][2];
      const float vn[2] = {vsc[0] * v_inv, vsc[1] * v_inv};
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float pr[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) pr[x] = fast_exp2(sc[nb][x] - (m_run[nb][x & 1] == -INFINITY ? 0.f : m_run[nb][x & 1]));
        pb[nb][0] = movmatrix_trans(pack_half2(pr[0] * vn[0], pr[1] * vn[0]));
        pb[nb][1] = movmatrix_trans(pack_half2(pr[2] * vn[1], pr[3] * vn[1]));
        l_run[nb][0] += pr[0] + pr[2];
        l_run[nb][1] += pr[1] + pr[3];
        if (vswz) { pb[nb][0] = __byte_perm(pb[nb][0], 0u, 0x1032); pb[nb][1] = __byte_perm(pb[nb][1], 0u, 0x1032); }
      }

      // ---- O^T += V^T P^T ---------------------------------------------------------------------------------------------------------
      static_for<0, NVG>([&](auto g_) {
        constexpr int g = decltype(g_)::value;
        uint32_t lo[4], hi[4];
        static_for<0, 4>([&](auto x_) {
          constexpr int x = decltype(x_)::value;
          uint32_t idx; __half2 rr;
          if constexpr (IB != 0) FL::template cut<g>(vw[x], idx, rr);
          else {
            const int t = 2 * j + (x & 1) + (x >> 1) * 8;
            cut_any(reinterpret_cast<const uint32_t*>(sp + L.v + t * ROW), r * NVG + g, p.ib, p.ib + p.pool.V.radius_bits, idx, rr);
            if (edge && t0 + t >= s.kv) { idx = 0u; rr = __float2half2_rn(0.f); }
          }
          const uint2 cw = *reinterpret_cast<const uint2*>(tblV + (idx * strideV + laneV));
          lo[x] = hmul2_u32(cw.x, rr);
          hi[x] = hmul2_u32(cw.y, rr);
        });
        const uint32_t a0 = __byte_perm(lo[0], lo[1], 0x5410), a1 = __byte_perm(lo[0], lo[1], 0x7632);
        const uint32_t a2 = __byte_perm(lo[2], lo[3], 0x5410), a3 = __byte_perm(lo[2], lo[3], 0x7632);
        const uint32_t e0 = __byte_perm(hi[0], hi[1], 0x5410), e1 = __byte_perm(hi[0], hi[1], 0x7632);
        const uint32_t e2 = __byte_perm(hi[2], hi[3], 0x5410), e3 = __byte_perm(hi[2], hi[3], 0x7632);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          mma16816(o[nb][2 * g], a0, a1, a2, a3, pb[nb][0], pb[nb][1]);
          mma16816(o[nb][2 * g + 1], e0, e1, e2, e3, pb[nb][0], pb[nb][1]);
        }
      });
      // ... of V: two more products for every g that has some
      if constexpr (OUTL) {
        if (vcols) {
          uint32_t f[4], at[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int t = 2 * j + ((x & 1) ^ vswz) + (x >> 1) * 8;
            const uint32_t w_ = __shfl_sync(0xffffffffu, fl, 16 + t);
            f[x] = w_ >> (r * NVG);
            at[x] = __shfl_sync(0xffffffffu, before, 16 + t) + __popc(w_ & ((1u << (r * NVG)) - 1u));
          }
          static_for<0, NVG>([&](auto g_) {
            constexpr int g = decltype(g_)::value;
            if (vcols & ((NVG == 4 ? 0x11111111u : 0x55555555u) << g)) {
              uint2 v[4];
              values_at(v, at, 4, true);
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const bool mine = (f[x] & (1u << g)) != 0u;
                if (!mine) v[x] = make_uint2(0u, 0u);
                at[x] += mine ? 1u : 0u;
              }
              const uint32_t a0 = __byte_perm(v[0].x, v[1].x, 0x5410), a1 = __byte_perm(v[0].x, v[1].x, 0x7632);
              const uint32_t a2 = __byte_perm(v[2].x, v[3].x, 0x5410), a3 = __byte_perm(v[2].x, v[3].x, 0x7632);
              const uint32_t e0 = __byte_perm(v[0].y, v[1].y, 0x5410), e1 = __byte_perm(v[0].y, v[1].y, 0x7632);
              const uint32_t e2 = __byte_perm(v[2].y, v[3].y, 0x5410), e3 = __byte_perm(v[2].y, v[3].y, 0x7632);
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) {
                mma16816(o[nb][2 * g], a0, a1, a2, a3, pb[nb][0], pb[nb][1]);
                mma16816(o[nb][2 * g + 1], e0, e1, e2, e3, pb[nb][0], pb[nb][1]);
              }
            }
          });
        }
      }
    }

    // ---- the unit's result, or a part of it --------------------------------------------------------------------------------------
    const bool whole = b0 >= f0 && b1 <= f1;
    float* part = my_parts + (first_seg ? 0 : PART);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float li[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = l_run[nb][e];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        l_run[nb][e] = l;
        li[e] = whole ? inverse_sum(p, h, nb * 8 + 2 * j + e, rows, m_run[nb][e], l) * v_pow : v_pow;
      }
#pragma unroll
      for (int x = 0; x < NOT; ++x) {
        const float4 v = make_float4(o[nb][x][0] * li[0], o[nb][x][1] * li[1], o[nb][x][2] * li[0], o[nb][x][3] * li[1]);
        if (whole) {
          emit_pair<N>(p, s, h, nb * 8 + 2 * j, rows, r, x, v.x, v.z);
          emit_pair<N>(p, s, h, nb * 8 + 2 * j + 1, rows, r, x, v.y, v.w);
        } else {
          reinterpret_cast<float4*>(part)[(nb * NOT + x) * 32 + lane] = v;
        }
      }
      if (!whole && r == 0) {
        float* ml = part + NB * NOT * 128 + nb * 16 + 2 * j;
        ml[0] = m_run[nb][0]; ml[1] = m_run[nb][1]; ml[8] = l_run[nb][0]; ml[9] = l_run[nb][1];
      }
    }
    first_seg = false;
    ++u;
  }
  __syncthreads();

  // ---- units cut between this CTA's warps -----------------------------------------------------------------------------------------
  // (every warp's first segment left its part in slot 0, a later one that is cut, the stretch's last, in slot 1)
  const float* cta_parts = p.parts + (size_t)blockIdx.x * NW * 2 * PART;
  float* out_parts = p.parts + ((size_t)gridDim.x * NW + blockIdx.x) * 2 * PART;
  for (int v = u_first; c0 < c1 && v < n_units; ++v) {
    const int b0 = __ldg(p.base + v), b1 = __ldg(p.base + v + 1);
    if (b0 >= c1) break;
    const int wa = warp_of(b0, total, n_warps), wb = warp_of(b1 - 1, total, n_warps);
    if (wa == wb) continue;
    const int la = max(wa - k * NW, 0), lb = min(wb - k * NW, NW - 1);
    const int first_slot = b0 > stretch_begin(k * NW + la, total, n_warps) ? 1 : 0;
    auto part_of = [&](int x) { return cta_parts + ((la + x) * 2 + (x == 0 ? first_slot : 0)) * PART; };
    const bool done = wa >= k * NW && wb < (k + 1) * NW;
    for (int idx = threadIdx.x; idx < NB * NOT * 32; idx += THREADS) {
      float4 x; float2 m, l;
      merge_parts<N, NB>(idx, lb - la + 1, part_of, x, m, l);
      if (done) emit_merged<N, NB>(p, seq_of(p, v), h, idx, x, m, l);
      else {
        float* dst = out_parts + (b0 > c0 ? PART : 0);
        reinterpret_cast<float4*>(dst)[idx] = x;
        const int nb = idx / (NOT * 32), i_ = (idx - nb * NOT * 32) >> 5;
        if (i_ == 0 && (idx & 31) < 4) {
          float* ml = dst + NB * NOT * 128 + nb * 16 + 2 * (idx & 3);
          ml[0] = m.x; ml[1] = m.y; ml[8] = l.x; ml[9] = l.y;
        }
      }
    }
  }
  // ---- units cut between CTAs: where those are a cluster, its CTAs share them out -------------------------------------------------
  if (p.fused) {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
    constexpr int PER = NB * NOT * 32;
    const int n_cuts = p.hdr[5];
    const float* all = p.parts + ((size_t)gridDim.x * NW + (size_t)h * p.ctas) * 2 * PART;
    for (int y = k * THREADS + threadIdx.x; y < n_cuts * PER; y += p.ctas * THREADS) {
      const int4 c = __ldg(p.cuts + y / PER);
      const int idx = y % PER;
      auto part_of = [&](int x) { return all + ((size_t)(c.y + x) * 2 + (x == 0 ? c.w : 0)) * PART; };
      float4 x; float2 m, l;
      merge_parts<N, NB>(idx, c.z - c.y + 1, part_of, x, m, l);
      emit_merged<N, NB>(p, seq_of(p, c.x), h, idx, x, m, l);
    }
  }
}

// Units cut between CTAs, where those are no cluster: blockIdx.x = the cut, blockIdx.y = KV head, blockIdx.z = 64 of the part's quadruples.
template <int N, int NB>
__global__ void __launch_bounds__(64) paged_merge_kernel(const DecodeParams p) {
  constexpr int NW = NB == 1 ? kDecWarps : kDecWarpsWide, PART = part_floats<N, NB>();
  // (the plan was there before the kernel ahead of this one)
  const bool mine = (int)blockIdx.x < p.hdr[5];
  const int4 c = __ldg(p.cuts + (mine ? blockIdx.x : 0));
  const Seq s = seq_of(p, mine ? c.x : 0);
  grid_dep_wait();
  if (!mine) return;
  const int h = blockIdx.y, grid = p.ctas * (int)gridDim.y;
  const float* base = p.parts + ((size_t)grid * NW + (size_t)h * p.ctas) * 2 * PART;
  auto part_of = [&](int x) { return base + ((size_t)(c.y + x) * 2 + (x == 0 ? c.w : 0)) * PART; };
  const int idx = blockIdx.z * 64 + threadIdx.x;
  float4 x; float2 m, l;
  merge_parts<N, NB>(idx, c.z - c.y + 1, part_of, x, m, l);
  emit_merged<N, NB>(p, s, h, idx, x, m, l);
}

struct DecodeKernels { const void* decode; const void* merge; };
DecodeKernels decode_kernels_128(int ib, int rb, int nb, bool outl);
DecodeKernels decode_kernels_64(int ib, int rb, int nb, bool outl);

// Field widths that have kernels of their own.
inline bool compiled_fields(int ib, int rb) { return (ib == 10 && rb == 3) || (ib == 12 && rb == 4) || (ib == 13 && rb == 6); }
template <int N, int NB, bool OUTL>
const void* pick_decode(int ib, int rb) {
  if (ib == 10 && rb == 3) return (const void*)&paged_decode_kernel<N, 10, 3, NB, OUTL>;
  if (ib == 12 && rb == 4) return (const void*)&paged_decode_kernel<N, 12, 4, NB, OUTL>;
  if (ib == 13 && rb == 6) return (const void*)&paged_decode_kernel<N, 13, 6, NB, OUTL>;
  return (const void*)&paged_decode_kernel<N, 0, 0, NB, OUTL>;
}
template <int N>
DecodeKernels pick_kernels(int ib, int rb, int nb, bool outl) {
  if (nb == 1) return {outl ? pick_decode<N, 1, true>(ib, rb) : pick_decode<N, 1, false>(ib, rb), (const void*)&paged_merge_kernel<N, 1>};
  if (nb == 4) return {outl ? pick_decode<N, 4, true>(ib, rb) : pick_decode<N, 4, false>(ib, rb), (const void*)&paged_merge_kernel<N, 4>};
  return {outl ? pick_decode<N, 2, true>(ib, rb) : pick_decode<N, 2, false>(ib, rb), (const void*)&paged_merge_kernel<N, 2>};
}

}  // namespace paged
}  // namespace hqmq
