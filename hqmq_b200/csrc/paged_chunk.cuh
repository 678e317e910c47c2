// Prompt chunks of a ragged batch over pages: the pages are decoded once into operand tiles, and the attention of attn_prefill.cu runs
// over those with its units from a list.  Part of attn_prefill.cu.
#pragma once
#include <math.h>

#include <atomic>

#include "paged.cuh"

namespace hqmq {
namespace attn {
namespace {

struct PagedExpandParams {
  hqmq_packed K, V;
  const uint16_t* tblK; const uint16_t* tblV;
  const int4* seqs; const int* tabs; const int4* img;      // sequences with images: {sequence, first tile, tiles, image tile}
  int n_img, ib, table_rows, Hkv, h0, per, img_tiles, page_bits;
  float qscale, kmant, vscale;             // softmax scale * log2 e as a power of two and what K's operands are multiplied by, in [1, 2)
  unsigned char* kimg; unsigned char* vimg;
  float* kmul; float* vmul;
  uint32_t* status; uint32_t epoch;
};

// grid (stretches of the image tiles, heads of the group, 2), as prefill_expand_kernel: eight warps, a warp the 16 tokens of a block of
// a tile.  A 128-token tile lies in one page or two neighbouring entries of the table; a block lies in one.
// IB, RB: index and radius bits of a field (0: any, at run time).
template <int N, int IB, int RB>
__global__ void __launch_bounds__(256, 4) paged_expand_kernel(const PagedExpandParams e) {
  constexpr uint32_t TB = (uint32_t)pf_tile_bytes(4 * N);
  extern __shared__ __align__(16) unsigned char smem_raw[];
  uint2* tbl = reinterpret_cast<uint2*>(smem_raw);
  __shared__ float s_big[8];
  __shared__ uint16_t s_list[8][16 * N];
  __shared__ __align__(8) uint64_t s_bar;
  grid_dep_launch();
  const bool is_v = blockIdx.z != 0;
  const hqmq_packed& pk = is_v ? e.V : e.K;
  const int h = e.h0 + blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint2* src = reinterpret_cast<const uint2*>(is_v ? e.tblV : e.tblK) + (int64_t)h * e.table_rows;
  const uint32_t bar = smem_u32(&s_bar), tbytes = (uint32_t)e.table_rows * 8u;
  const bool bulk = ((reinterpret_cast<uintptr_t>(src) | tbytes) & 15u) == 0;
  if (bulk) {
    if (threadIdx.x == 0) {
      mbar_init(bar, 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      mbar_expect_tx(bar, tbytes);
      bulk_g2s(smem_u32(tbl), src, tbytes, bar);
    }
  } else {
    for (int i = threadIdx.x; i < e.table_rows; i += 256) tbl[i] = src[i];
  }
  const bool outl = pk.flags != nullptr;
  constexpr int TPW = 32 / N, NF = 16 / TPW;
  const int half = N == 32 ? 0 : lane >> 4, c = N == 32 ? lane : lane & 15;
  const int ib = IB ? IB : e.ib, cb = IB ? IB + RB : e.ib + pk.radius_bits, row_words = IB ? (N * (IB + RB) + 31) / 32 : pk.row_bytes >> 2;
  const int bit = c * cb, sh = bit & 31, w0 = bit >> 5, w1 = sh + cb > 32 ? 1 : 0;
  const uint32_t imask = (1u << ib) - 1u, fmask = (1u << cb) - 1u;
  const uint32_t* codes = reinterpret_cast<const uint32_t*>(pk.codes) + w0;
  const uint32_t last_row = (uint32_t)e.table_rows - 1u;      // (a field that no encoder writes reads the last codeword)
  const int pt_mask = (1 << e.page_bits) - 1;

  int seq = -1, tab = 0, kv = 0, at = 0, first = 0, tiles = 0, img0 = 0;      // the sequence at hand; `at` its place in the list
  uint32_t f[NF], myflag, run;
  int64_t ph = 0;
  float rs;
  auto fetch = [&](int tile) {                 // tile of the sequence
    const int tb = tile * kPfTok + warp * 16;
    rs = 0.f; myflag = 0u; run = 0u;
#pragma unroll
    for (int k = 0; k < NF; ++k) f[k] = 0u;
    if (tb >= kv) return;
    ph = (int64_t)__ldg(e.tabs + tab + (tb >> e.page_bits)) * e.Hkv + h;
    const int64_t row = (ph << e.page_bits) + (tb & pt_mask);
    if (lane < 16 && tb + lane < kv) {
      rs = bits16_to_float(__ldg(reinterpret_cast<const uint16_t*>(pk.rs) + row + lane), pk.scale_dtype);
      if (outl) myflag = __ldg(pk.flags + row + lane);
    }
    if (outl) run = __ldg(pk.out_off + ph * ((pt_mask + 1) / HQMQ_OUT_BLOCK + 1) + (tb & pt_mask) / HQMQ_OUT_BLOCK);
    const uint32_t* r0 = codes + (row + half) * row_words;
#pragma unroll
    for (int k = 0; k < NF; ++k) {
      if (tb + k * TPW + half < kv) {
        const uint32_t* r = r0 + k * TPW * row_words;
        if constexpr (IB + RB == 16) f[k] = __ldg(r) >> sh;          // (two fields a word: none straddles)
        else f[k] = __funnelshift_r(__ldg(r), __ldg(r + w1), sh);
      }
    }
  };
  const int i0 = blockIdx.x * e.per, i1 = min(e.img_tiles, i0 + e.per);
  bool have_table = false;
  float mul = 0.f, inv = 0.f;
  for (int i = i0; i < i1; ++i) {
    if (seq < 0 || i >= img0 + tiles) {
      // ---- another sequence: its place, the largest scale of its keys in range -------------------------------------------------
      while (at + 1 < e.n_img && __ldg(&e.img[at + 1].w) <= i) ++at;
      const int4 im = __ldg(e.img + at), s4 = __ldg(e.seqs + im.x);
      seq = im.x; first = im.y; tiles = im.z; img0 = im.w; kv = s4.x; tab = s4.w;
      fetch(first + i - img0);
      float big = 0.f;
      const int t_first = first * kPfTok, t_end = min(kv, (first + tiles) * kPfTok);
#pragma unroll 4
      for (int t = t_first + threadIdx.x * 8; t < t_end; t += 256 * 8) {
        const int64_t row = (((int64_t)__ldg(e.tabs + tab + (t >> e.page_bits)) * e.Hkv + h) << e.page_bits) + (t & pt_mask);
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(pk.rs) + row));
        const uint32_t w4[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const float y = bits16_to_float((uint16_t)(w4[x >> 1] >> (16 * (x & 1))), pk.scale_dtype);
          // (an infinite scale is its own key's: relative to it the others would be zeros, for queries that do not see it, too)
          if (t + x < t_end && fabsf(y) < INFINITY) big = fmaxf(big, fabsf(y));
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
      __syncthreads();                         // (the table's barrier word is initialised; nobody reads the last sequence's)
      if (lane == 0) s_big[warp] = big;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < 8; ++w) big = fmaxf(big, s_big[w]);
      pf_scale_of(big, mul, inv);
      if (i == img0 && threadIdx.x == 0) (is_v ? e.vmul : e.kmul)[seq * e.Hkv + h] = is_v ? inv : inv * e.qscale;
      if (bulk && !have_table) {
        uint32_t spins = 0;
        while (!mbar_try_wait(bar, 0)) {
          if (++spins > kWaitLimit) { *e.status = e.epoch; break; }
        }
      }
      have_table = true;
    }
    unsigned char* dst = (is_v ? e.vimg : e.kimg) + ((int64_t)blockIdx.y * e.img_tiles + i) * TB;
    // (The scores' factor is a power of two, so that a product with it is exact: score - maximum is 0 for the largest however large it is.  With
    // a factor of any value inside the fused multiply-add, scores from 2^26 on were ahead of their rounded maximum by so much that their
    // exponentials were infinite; rounding the products of such tiles first took 267 us for 4 x 8k, 500 queries, against 258.)
    const float to_op = is_v ? mul : mul * e.kmant, myfac = rs * e.vscale * to_op;
    const unsigned char* vals = outl ? reinterpret_cast<const unsigned char*>(pk.out_vals) + ph * pk.out_cap * 8 : nullptr;
    const uint32_t cap = outl ? (uint32_t)pk.out_cap : 0u;
    auto payload_of = [&](uint32_t slot) {
      if (slot >= cap) return make_uint2(0u, 0u);
      return __ldg(reinterpret_cast<const uint2*>(vals + (int64_t)slot * 8));
    };
    uint32_t n_ent = 0u;
    const uint32_t run0 = run;
    uint2 ent = make_uint2(0u, 0u);
    if (outl) {
      uint32_t incl = __popc(myflag);
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) { const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += y; }
      n_ent = __shfl_sync(0xffffffffu, incl, 15);
      if (n_ent) {
        if (lane < n_ent) ent = payload_of(run0 + lane);
        uint32_t pos = incl - __popc(myflag);
        for (uint32_t w = myflag; w; w &= w - 1u) s_list[warp][pos++] = (uint16_t)(lane * 32 + __ffs(w) - 1);
      }
    }
    unsigned char* kd = dst + (c >> 4) * 16384 + (c & 1) * 8;
#pragma unroll
    for (int k = 0; k < NF; ++k) {
      const int tl = warp * 16 + k * TPW + half;
      const float fac = __shfl_sync(0xffffffffu, myfac, k * TPW + half) * (float)((f[k] & fmask) >> ib);
      const uint2 cw = tbl[min(f[k] & imask, last_row)];
      const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&cw.x)), d = __half22float2(*reinterpret_cast<const __half2*>(&cw.y));
      *reinterpret_cast<uint2*>(kd + tl * 128 + ((((c & 15) >> 1) ^ (tl & 7)) << 4)) = make_uint2(pack_half2(a.x * fac, a.y * fac), pack_half2(d.x * fac, d.y * fac));
    }
    if (i + 1 < i1 && i + 1 < img0 + tiles) fetch(first + i + 1 - img0);
    if (n_ent) {
      __syncwarp();
      for (uint32_t x = lane; x < n_ent; x += 32) {
        if (x != lane) ent = payload_of(run0 + x);
        const uint32_t p_ = s_list[warp][x];
        const int tl = warp * 16 + (int)(p_ >> 5), cc = (int)(p_ & 31u);
        const float2 a = pair16_to_float2(ent.x, pk.out_dtype), d = pair16_to_float2(ent.y, pk.out_dtype);
        *reinterpret_cast<uint2*>(dst + (cc >> 4) * 16384 + tl * 128 + ((((cc & 15) >> 1) ^ (tl & 7)) << 4) + (cc & 1) * 8) =
            make_uint2(pack_half2(a.x * to_op, a.y * to_op), pack_half2(d.x * to_op, d.y * to_op));
      }
      __syncwarp();
    }
  }
}

template <int N>
const void* pick_expand(int ib, int rb) {
  if (ib == 10 && rb == 3) return (const void*)&paged_expand_kernel<N, 10, 3>;
  if (ib == 12 && rb == 4) return (const void*)&paged_expand_kernel<N, 12, 4>;
  if (ib == 13 && rb == 6) return (const void*)&paged_expand_kernel<N, 13, 6>;
  return (const void*)&paged_expand_kernel<N, 0, 0>;
}

struct ChunkPlaces { size_t mul, img, part, bytes; };
ChunkPlaces chunk_places(const hqmq_paged_plan& p) {
  ChunkPlaces c;
  c.mul = 16;
  c.img = (16 + (size_t)p.n_seqs * p.H_kv * 8 + 255) & ~(size_t)255;
  c.part = c.img + (size_t)2 * p.ch_heads * p.ch_img_tiles * pf_tile_bytes(p.d);
  c.bytes = c.part + (p.ch_whole ? 0 : (size_t)p.ch_ctas * 2 * 256 * (p.d + 2) * sizeof(float));
  return c;
}
std::atomic<uint32_t> chunk_epoch{0x3a9ed000u};

}  // namespace
}  // namespace attn

namespace paged {

size_t chunk_workspace(const hqmq_paged_attn_args* a) { return a->plan.ch_units ? chunk_places(a->plan).bytes : 0; }

int chunk_launch(const hqmq_paged_attn_args* a, void* workspace, cudaStream_t st) {
  const hqmq_paged_plan& pl = a->plan;
  const ChunkPlaces at = chunk_places(pl);
  unsigned char* ws = reinterpret_cast<unsigned char*>(workspace);
  PrefillParams p;
  memset(&p, 0, sizeof(p));
  p.Q = a->Q; p.q_dtype = a->q_dtype; p.qs_t = a->q_stride[0]; p.qs_h = a->q_stride[1];
  p.O = a->O; p.o_dtype = a->o_dtype; p.os_t = a->o_stride[0]; p.os_h = a->o_stride[1];
  auto vec = [](const void* ptr, const int64_t* s, int dt) { return dt != HQMQ_F32 && ((uintptr_t)ptr & 15) == 0 && s[0] % 8 == 0 && s[1] % 8 == 0; };
  auto near = [](int64_t x) { return x > -((int64_t)1 << 26) && x < ((int64_t)1 << 26); };
  p.q_vec = vec(a->Q, a->q_stride, a->q_dtype) && near(p.qs_h) && near(p.qs_t);
  p.o_vec = vec(a->O, a->o_stride, a->o_dtype);
  p.Hkv = pl.H_kv; p.G = pl.H_q / pl.H_kv; p.window = pl.window;
  p.P = 128 / p.G; p.streams = pl.ch_streams; p.units_m = pl.ch_units;
  p.total = (int64_t)pl.ch_tiles * pl.ch_heads;
  p.L = pl.ch_whole ? 0 : (p.total + pl.ch_ctas - 1) / pl.ch_ctas;
  p.units_all = pl.ch_units * pl.ch_heads;
  p.img_tiles = pl.ch_img_tiles;
  const int4* d = reinterpret_cast<const int4*>(a->plan_data);
  p.units = d + pl.ch_unit / 4; p.order = a->plan_data + pl.ch_order; p.starts = d + pl.ch_start / 4;
  p.sinks = a->sinks;
  if (a->softcap > 0.f) { p.cap_log2 = a->softcap * 1.4426950408889634f; p.cap_in = 1.f / p.cap_log2; }
  p.status = reinterpret_cast<uint32_t*>(ws);
  p.epoch = chunk_epoch.fetch_add(1u, std::memory_order_relaxed) + 1u;
  float* mul = reinterpret_cast<float*>(ws + at.mul);
  p.kmul = mul; p.vmul = mul + (size_t)pl.n_seqs * pl.H_kv;
  p.part = reinterpret_cast<float*>(ws + at.part);
  PagedExpandParams e;
  memset(&e, 0, sizeof(e));
  e.K = a->K; e.V = a->V; e.tblK = a->table_K; e.tblV = a->table_V;
  e.seqs = d + pl.seqs / 4; e.tabs = a->plan_data + pl.tabs; e.img = d + pl.ch_img / 4;
  e.n_img = pl.ch_seqs; e.ib = idx_bits_for(a->K.S); e.table_rows = 24 * a->K.S; e.Hkv = pl.H_kv; e.img_tiles = pl.ch_img_tiles;
  while ((1 << e.page_bits) < pl.page_tokens) ++e.page_bits;
  int exponent;
  e.kmant = 2.f * frexpf(a->softmax_scale * 1.4426950408889634f, &exponent);
  e.qscale = ldexpf(1.f, exponent - 1); e.vscale = 1.f / (float)a->r_qmax;
  e.kmul = mul; e.vmul = mul + (size_t)pl.n_seqs * pl.H_kv;
  e.status = p.status; e.epoch = p.epoch;
  e.kimg = ws + at.img; e.vimg = e.kimg + (size_t)pl.ch_heads * pl.ch_img_tiles * pf_tile_bytes(pl.d);
  p.kimg = e.kimg; p.vimg = e.vimg;
  const bool cap = a->softcap > 0.f, wide = pl.d == 128;
  const void* ek = wide ? pick_expand<32>(e.ib, a->K.radius_bits) : pick_expand<16>(e.ib, a->K.radius_bits);
  const void* ak = wide ? (cap ? (const void*)&prefill_attn_kernel<128, 2> : (const void*)&prefill_attn_kernel<128, 1>)
                        : (cap ? (const void*)&prefill_attn_kernel<64, 2> : (const void*)&prefill_attn_kernel<64, 1>);
  const void* mk = wide ? (const void*)&prefill_merge_kernel<128, 1> : (const void*)&prefill_merge_kernel<64, 1>;
  const size_t esmem = (size_t)e.table_rows * 8;
  HQMQ_CHECK_CUDA(raise_smem_limit(ek, esmem));
  HQMQ_CHECK_CUDA(raise_smem_limit(ak, pf_smem_bytes(pl.d)));
  const int64_t per = ((int64_t)pl.ch_img_tiles * pl.ch_heads * 2 + 6 * kPfMaxCtas - 1) / (6 * kPfMaxCtas);
  e.per = per < 1 ? 1 : (int)per;
  for (int h0 = 0; h0 < pl.H_kv; h0 += pl.ch_heads) {
    e.h0 = p.h0 = h0;
    void* ea[] = {&e};
    HQMQ_CHECK_CUDA(cudaLaunchKernel(ek, dim3((pl.ch_img_tiles + e.per - 1) / e.per, pl.ch_heads, 2), dim3(256), ea, esmem, st));
    void* pa[] = {&p};
    HQMQ_CHECK_CUDA(launch_dependent(ak, dim3(pl.ch_ctas), kPfThreads, pa, pf_smem_bytes(pl.d), st));
    if (!pl.ch_whole && pl.ch_ctas > 1) HQMQ_CHECK_CUDA(launch_dependent(mk, dim3(pl.ch_ctas - 1, 4 * p.streams), 256, pa, 0, st));
  }
  return HQMQ_OK;
}

}  // namespace paged
}  // namespace hqmq
