// A 16-token tile of a paged cache on its way into shared memory and out of it as tensor-core operands.
//
// Every warp has a ring of three stages of its own, filled with 16-byte asynchronous copies by all of its lanes: while tile i is
// computed, the rows, scales, flag words and block offsets of tile i + 2 are on their way, and the flagged chunks' values of tile
// i + 1, whose place in the side buffer the tile's offsets say.  Tiles lie inside a page (pages hold 64 tokens or more), so a tile
// is contiguous whatever the table says.
#pragma once
#include "paged.cuh"

namespace hqmq {
namespace paged {

constexpr int kPayK = 64, kPayV = 32;      // values of flagged chunks staged per tile (those of a tile with more go through global memory)
constexpr int kTileStages = 3;
constexpr size_t kPastPay = 16;            // (a lane without a flagged chunk reads the place behind a stage's last value)

// Rows of IB + RB bits per chunk; IB = 0: any width, at run time.
template <int N, int IB, int RB>
__host__ __device__ constexpr int row_bytes_of() { return (N * (IB + RB) + 31) / 32 * 4; }

// Where the parts of a stage lie.  Values of flagged chunks, 8 bytes each: K's, then V's; K's alone have 16, where a value is kept in two halves.
struct TileLayout { int v, rsk, rsv, flk, flv, off, pay, bytes; };
__host__ __device__ constexpr TileLayout tile_layout(int row, bool hasv, bool outl) {
  TileLayout l{};
  int at = kTile * row;
  l.v = at; at += hasv ? kTile * row : 0;
  l.rsk = at; at += kTile * 2;              // (V's follow K's: the two are read as one array of 32)
  l.rsv = at; at += hasv ? kTile * 2 : 0;
  l.flk = at; at += outl ? kTile * 4 : 0;
  l.flv = at; at += outl && hasv ? kTile * 4 : 0;
  l.off = at; at += outl ? 32 : 0;          // K's entries before the tile and behind it; V's; page
  l.pay = at; at += outl ? (hasv ? kPayK * 8 + kPayV * 8 : kPayK * 16) : 0;
  l.bytes = (at + 15) & ~15;
  return l;
}

// What the copies need to know of a pool; page_bits = log2(tokens of a page).
struct PoolView {
  hqmq_packed K, V;
  int Hkv, page_bits;
};

// A unit as a warp takes it up: its first row, its tiles' stretch of the flat sequence, where its tiles begin, the sequence.
struct Taken { int row0, b0, b1, lo; Seq s; };
__device__ __forceinline__ Taken take_unit(const int4* units, const int4* seqs, const int* base, int u) {
  const int4 un = __ldg(units + u), sq = __ldg(seqs + un.x);
  return Taken{un.y, __ldg(base + u), __ldg(base + u + 1), un.z, Seq{sq.x, sq.y, sq.z, sq.w}};
}
// ... the first one, from the warp's record (f0: the stretch's begin): no load waits for another
__device__ __forceinline__ Taken take_first(const int* record, int f0) {
  const int4 a = __ldg(reinterpret_cast<const int4*>(record)), b = __ldg(reinterpret_cast<const int4*>(record) + 1);
  const int4 c = __ldg(reinterpret_cast<const int4*>(record) + 2), sq = __ldg(reinterpret_cast<const int4*>(record) + 3);
  return Taken{b.w, c.x, c.y, a.w - (f0 - c.x), Seq{sq.x, sq.y, sq.z, sq.w}};
}

// The tiles of a warp's stretch, in order.  The page of a tile is loaded a tile ahead: it is what the copies' addresses wait for.
struct TileIter {
  int u, tile, hi, tab, left, page;
  // from a warp's record; returns the stretch
  __device__ __forceinline__ int2 init(const int* record) {
    const int4 a = __ldg(reinterpret_cast<const int4*>(record)), b = __ldg(reinterpret_cast<const int4*>(record) + 1);
    u = a.z; tile = a.w; hi = b.x; tab = b.y; page = b.z; left = a.y - a.x;
    return make_int2(a.x, a.y);
  }
  __device__ __forceinline__ void unit(const int4* units, const int4* seqs, int skip) {
    const int4 un = __ldg(units + u);
    tile = un.z + skip; hi = un.w;
    tab = __ldg(&seqs[un.x].w);
  }
  __device__ __forceinline__ void find_page(const int* tabs, int page_bits) { page = __ldg(tabs + tab + ((tile * kTile) >> page_bits)); }
  __device__ __forceinline__ void next(const int4* units, const int4* seqs, const int* tabs, int page_bits) {
    if (--left <= 0) return;
    if (++tile == hi) { ++u; unit(units, seqs, 0); }
    find_page(tabs, page_bits);
  }
};

// A lane's share of the copies of a tile: its 16 bytes of the code rows, and one piece of the scales, flag words or offsets.
template <bool HASV, bool OUTL>
struct Stager {
  const unsigned char* k; const unsigned char* v; const unsigned char* small; const uint32_t* off;
  uint32_t small_mul, small_dst, off_dst;      // bytes per row of the small piece (0: none), places in the stage
  __device__ __forceinline__ void init(const PoolView& p, const TileLayout& l, int lane) {
    k = p.K.codes + 16 * lane;
    v = HASV ? p.V.codes + 16 * lane : nullptr;
    small = nullptr; small_mul = small_dst = 0u; off = nullptr; off_dst = 0u;
    auto piece = [&](const void* base, int i, int mul, int dst) {
      if (base) { small = reinterpret_cast<const unsigned char*>(base) + 16 * i; small_mul = mul; small_dst = dst + 16 * i; }
    };
    if (lane < 2) piece(p.K.rs, lane, 2, l.rsk);
    else if (HASV && lane < 4) piece(p.V.rs, lane - 2, 2, l.rsv);
    else if (OUTL && lane >= 4 && lane < 8) piece(p.K.flags, lane - 4, 4, l.flk);
    else if (OUTL && HASV && lane >= 8 && lane < 12) piece(p.V.flags, lane - 8, 4, l.flv);
    if constexpr (OUTL) {
      if (lane >= 12 && lane < 14 && p.K.flags) { off = p.K.out_off + (lane - 12); off_dst = l.off + (lane - 12) * 4; }
      if (HASV && lane >= 14 && lane < 16 && p.V.flags) { off = p.V.out_off + (lane - 14); off_dst = l.off + (lane - 12) * 4; }
    }
  }
  template <int ROWC>
  __device__ __forceinline__ void tile(const PoolView& p, const TileLayout& l, int row_bytes, uint32_t sb, unsigned char* sp, int h, int page,
                                       int tile, int lane) const {
    const int in_page = (tile * kTile) & ((1 << p.page_bits) - 1), ph = page * p.Hkv + h;
    const int64_t row = ((int64_t)ph << p.page_bits) + in_page;
    const unsigned char* ks = k + row * row_bytes;
    const unsigned char* vs = HASV ? v + row * row_bytes : nullptr;
    // (16 rows of row_bytes are row_bytes pieces of 16 bytes)
    if constexpr (ROWC != 0) {
#pragma unroll
      for (int c = 0; c < (ROWC + 31) / 32; ++c) {
        if (32 * c + 32 <= ROWC || lane < ROWC - 32 * c) {
          cp_async16(sb + 16 * lane + 512 * c, ks + 512 * c);
          if constexpr (HASV) cp_async16(sb + l.v + 16 * lane + 512 * c, vs + 512 * c);
        }
      }
    } else {
      for (int c = 0; c * 32 + lane < row_bytes; ++c) {
        cp_async16(sb + 16 * lane + 512 * c, ks + 512 * c);
        if constexpr (HASV) cp_async16(sb + l.v + 16 * lane + 512 * c, vs + 512 * c);
      }
    }
    if (small_mul) cp_async16(sb + small_dst, small + row * small_mul);
    if constexpr (OUTL) {
      if (off_dst) cp_async4(sb + off_dst, off + (int64_t)ph * ((1 << p.page_bits) / HQMQ_OUT_BLOCK + 1) + in_page / HQMQ_OUT_BLOCK);
      if (lane == 16) *reinterpret_cast<int*>(sp + l.off + 16) = ph;
    }
  }
};

// The values of a staged tile's flagged chunks, as many as there is room for (an entry the side buffer had no room for reads as 0).  A
// lane copies up to two of K's and one of V's: no loop.
template <bool HASV>
__device__ __forceinline__ void stage_values(const PoolView& p, const TileLayout& l, uint32_t sb, unsigned char* sp, int lane) {
  const uint4 o = *reinterpret_cast<const uint4*>(sp + l.off);       // entries before the tile and behind it: K's, V's
  const int ph = *reinterpret_cast<const int*>(sp + l.off + 16);
  auto copy = [&](const hqmq_packed& x, uint32_t from, uint32_t end, int to, bool twice) {
    const uint32_t at = from + lane, room = min(end, (uint32_t)x.out_cap);
    const unsigned char* v = reinterpret_cast<const unsigned char*>(x.out_vals) + ((int64_t)ph * x.out_cap + at) * 8;
    if (at < room) cp_async8(sb + l.pay + to + 8 * lane, v);
    if (twice && at + 32 < room) cp_async8(sb + l.pay + to + 256 + 8 * lane, v + 256);
    if (end > (uint32_t)x.out_cap) {           // (hardly ever: a side buffer that overflowed)
      if (at >= room) *reinterpret_cast<uint2*>(sp + l.pay + to + 8 * lane) = make_uint2(0u, 0u);
      if (twice && at + 32 >= room) *reinterpret_cast<uint2*>(sp + l.pay + to + 256 + 8 * lane) = make_uint2(0u, 0u);
    }
  };
  if (p.K.flags && o.y != o.x) copy(p.K, o.x, o.y, 0, true);
  if (HASV && p.V.flags && o.w != o.z) copy(p.V, o.z, o.w, kPayK * 8, false);
}

// Two 16-bit values times f as two fp16 ones.
__device__ __forceinline__ uint32_t scaled_pair(uint32_t v, float f, bool bf16) {
  float2 x;
  if (bf16) x = make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  else x = __half22float2(*reinterpret_cast<const __half2*>(&v));
  return pack_half2(x.x * f, x.y * f);
}
__device__ __forceinline__ float4 values_of(uint2 v, int dtype) {
  float2 a, b;
  if (dtype == HQMQ_BF16) {
    a = make_float2(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u));
    b = make_float2(__uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
  } else {
    a = __half22float2(*reinterpret_cast<const __half2*>(&v.x));
    b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
  }
  return make_float4(a.x, a.y, b.x, b.y);
}

// Sum over the lanes before this one in its half of the warp, of counts up to 32: by their bits, of which two hardly ever do not do.
__device__ __forceinline__ uint32_t counts_before(uint32_t own, int lane) {
  const uint32_t earlier = ((1u << lane) - 1u) & (lane < 16 ? 0xffffu : 0xffff0000u);
  uint32_t n = __popc(__ballot_sync(0xffffffffu, own & 1u) & earlier) + 2u * __popc(__ballot_sync(0xffffffffu, own & 2u) & earlier);
  if (__any_sync(0xffffffffu, own > 3u)) {
#pragma unroll
    for (int b = 2; b < 6; ++b) n += (uint32_t)__popc(__ballot_sync(0xffffffffu, own & (1u << b)) & earlier) << b;
  }
  return n;
}

// The codeword and radius of field `c` of a row of `cb`-bit fields (sign-folded index, the sign in the radius).
__device__ __forceinline__ void cut_any(const uint32_t* row, int c, int ib, int cb, uint32_t& idx, __half2& rr) {
  const uint32_t v = row_field(row, c, cb);
  const __half2 r2 = radius_half2(v >> ib);
  idx = (v & ((1u << ib) - 1u)) >> 1;
  const uint32_t ru = *reinterpret_cast<const uint32_t*>(&r2) ^ ((0u - (v & 1u)) & 0x80008000u);
  rr = *reinterpret_cast<const __half2*>(&ru);
}

// One head's table, sign-folded and replicated: entry i of the even codewords `reps` times in a row.
template <int THREADS>
__device__ __forceinline__ void load_table(unsigned char* tbl, const uint16_t* src16, int h, int rows, int rep_log2) {
  const uint2* src = reinterpret_cast<const uint2*>(src16) + (int64_t)h * rows;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rows_f = rows >> 1;
  for (int i0 = warp * 32; i0 < rows_f; i0 += THREADS) {
    uint2 e = make_uint2(0u, 0u);
    if (i0 + lane < rows_f) e = __ldg(src + 2 * (i0 + lane));
    uint2* d = reinterpret_cast<uint2*>(tbl) + ((size_t)i0 << rep_log2);
    for (int k = 0; k < 1 << rep_log2; ++k) {
      const int s = k * 32 + lane, from = s >> rep_log2;
      const uint2 v = make_uint2(__shfl_sync(0xffffffffu, e.x, from), __shfl_sync(0xffffffffu, e.y, from));
      if (i0 + from < rows_f) d[s] = v;
    }
  }
}

// ---- the queries of a unit: rows as columns of the product ----------------------------------------------------------------------
struct QueryView { const void* Q; int dtype, vec; int64_t st_t, st_h; int G; };

// Row `row` (query * G + head) of a unit, this lane's dims [4 NKS j, 4 NKS (j + 1)), in fp16 after division by a power of two that
// brings the row's largest value to [1, 2); returns that power.  A power per row: rows are other heads and tokens, and one that is far
// larger, or infinite, is no reason for the others to lose their bits.  A row that is not there is zeros.
template <int NKS>
__device__ __forceinline__ float load_query(uint32_t (*qb)[2], const QueryView& q, int q_off, int h, int row, int rows, int j) {
  float f[4 * NKS];
  const int qi = row / q.G, g = row - qi * q.G;
  const bool real = row < rows;
  const int64_t o = (int64_t)(q_off + qi) * q.st_t + (int64_t)(h * q.G + g) * q.st_h + 4 * NKS * j;
#pragma unroll
  for (int i = 0; i < 4 * NKS; ++i) f[i] = 0.f;
  if (real) {
    if (q.vec) {
#pragma unroll
      for (int i = 0; i < 4 * NKS; i += 8) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(q.Q) + o + i));
        const float4 a = values_of(make_uint2(v.x, v.y), q.dtype), b = values_of(make_uint2(v.z, v.w), q.dtype);
        f[i] = a.x; f[i + 1] = a.y; f[i + 2] = a.z; f[i + 3] = a.w;
        f[i + 4] = b.x; f[i + 5] = b.y; f[i + 6] = b.z; f[i + 7] = b.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4 * NKS; ++i) f[i] = load_float(q.Q, o + i, q.dtype);
    }
  }
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 4 * NKS; ++i) m = fmaxf(m, fabsf(f[i]));
  m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
  int e = (int)(__float_as_uint(m) >> 23) - 127;               // (subnormal: -127; infinite: 128)
  e = min(126, max(-126, e));
  const float div = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) {
    qb[ks][0] = pack_half2(f[4 * ks] * div, f[4 * ks + 1] * div);
    qb[ks][1] = pack_half2(f[4 * ks + 2] * div, f[4 * ks + 3] * div);
  }
  return __uint_as_float((uint32_t)(127 + e) << 23);
}

// A key's scale as its score is multiplied by: an infinite one is no number (the key's values are infinite of either sign, so a score is
// none; times an infinity it could be minus infinity, a weight of zero).
__device__ __forceinline__ float key_scale(float x) { return fmaf(x, 0.f, x); }

// tanh(x): for |x| <= 1/2 as x times a cubic in x^2 through its values at the Chebyshev nodes of [0, 1/4] (within 5e-7 of the value,
// however small: a cap far above the scores leaves them as they are), beyond as 1 - 2 / (e^2x + 1).
__device__ __forceinline__ float tanh_of(float x) {
  const float q = x * x;
  const float near = x * fmaf(q, fmaf(q, fmaf(q, -0.0443927385f, 0.131899402f), -0.333262831f), 0.999999464f);
  const float far = 1.f - __fdividef(2.f, fast_exp2(2.885390081777927f * x) + 1.f);
  return q <= 0.25f ? near : far;
}

}  // namespace paged
}  // namespace hqmq
