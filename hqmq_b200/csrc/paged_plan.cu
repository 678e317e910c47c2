// Plans of calls over a paged cache: host code.  A plan is one array of 32-bit words that the caller copies to the device.
#include <algorithm>

#include "paged.cuh"

namespace hqmq {
namespace paged {

// Sequences of up to 32 rows, which is what the decode kernel holds, take that; the others decode their cache once into operand tiles
// (attn_prefill.cu).  Below 32 rows the tiles pay for one short sequence only (8 KV heads of 128, G 4, decode / tiles in us: 1 x 2048 tokens, 16
// rows 17 / 25, 32 rows 28 / 25; 1 x 8192 23 / 37, 33 / 37; 8 x 8192 50 / 164, 82 / 166; 8 x 65536 269 / 1299, 400 / 1303).
bool chunked(int q, int G) { return q * G > 32; }

int check_plan(const hqmq_paged_plan& p) {
  if (p.struct_size != sizeof(hqmq_paged_plan)) return HQMQ_ERR_ARG;
  if ((int64_t)p.n_pages * p.H_kv > 0x7fffffff) return HQMQ_ERR_SHAPE;
  if (p.n_seqs < 1 || p.n_seqs > (1 << 20) || p.n_pages < 1 || p.H_kv < 1 || p.H_kv > 1024 || p.window < 0) return HQMQ_ERR_SHAPE;
  if (p.page_tokens < HQMQ_T_ALIGN || (p.page_tokens & (p.page_tokens - 1)) || p.page_tokens > kMaxPage) return HQMQ_ERR_SHAPE;
  if (p.d != 64 && p.d != 128) return HQMQ_ERR_UNSUPPORTED;
  if (p.H_q != 0) {
    if (p.H_q < 0 || p.H_q % p.H_kv) return HQMQ_ERR_SHAPE;
    if (p.H_q / p.H_kv > 16) return HQMQ_ERR_UNSUPPORTED;
  }
  return HQMQ_OK;
}

int check_pool(const hqmq_packed& k, const hqmq_paged_plan& p) {
  int rc = check_packed(k, false);
  if (rc) return rc;
  if (k.B != p.n_pages || k.H != p.H_kv || k.T_cap != p.page_tokens || k.n_chunks * 4 != p.d) return HQMQ_ERR_SHAPE;
  if (!is_half_dtype(k.scale_dtype) || (k.flags && !is_half_dtype(k.out_dtype))) return HQMQ_ERR_UNSUPPORTED;
  if (k.flags && ((uintptr_t)k.out_off & 3)) return HQMQ_ERR_ALIGN;
  if (24 * k.S > kMaxCodewords || k.ofrag) return HQMQ_ERR_UNSUPPORTED;
  return HQMQ_OK;
}

namespace {
inline int up4(int64_t x) { return (int)((x + 3) & ~(int64_t)3); }
inline int blocks_of(int n, int b) { return (n + b - 1) / b; }


void chunk_unit(const hqmq_paged_plan& p, int kv, int q, int m, int& lo, int& n) {
  const int P = 128 / (p.H_q / p.H_kv), per = p.ch_streams * P;
  const int i0 = m * per, i1 = std::min(i0 + per, q);
  int beg, end;
  unit_keys(kv, q, 1, p.window, i0, i1, beg, end);
  lo = beg / 128;
  n = std::max(1, blocks_of(end, 128) - lo);
}
}  // namespace
}  // namespace paged
}  // namespace hqmq

using namespace hqmq;
using namespace hqmq::paged;

extern "C" int hqmq_paged_plan_size(hqmq_paged_plan* plan, const int32_t* kv_lens, const int32_t* q_lens) {
  if (!plan || !kv_lens || !q_lens) return HQMQ_ERR_ARG;
  int rc = check_plan(*plan);
  if (rc) return rc;
  hqmq_paged_plan& p = *plan;
  const hqmq_paged_plan had = p;
  if (p.tab_room < 0 || p.tab_room > (1 << 24) || (p.renew && !p.tab_room)) return HQMQ_ERR_SHAPE;
  const int G = p.H_q ? p.H_q / p.H_kv : 1;
  int64_t total_q = 0, n_tab = 0, dec_tiles = 0, ms_tiles = 0, ms_groups = 0, ms_units = 0;
  int dec_units = 0, dec_rows = 0, ch_seqs = 0, most_q = 0, most_rows = 0, all_q = 0;
  for (int s = 0; s < p.n_seqs; ++s) {
    if (kv_lens[s] < 0 || q_lens[s] < 0 || q_lens[s] > kv_lens[s] || kv_lens[s] > (1 << 30)) return HQMQ_ERR_SHAPE;
    total_q += q_lens[s];
    all_q = std::max(all_q, q_lens[s]);
    n_tab += blocks_of(kv_lens[s], p.page_tokens);
    if (!p.H_q || !q_lens[s]) continue;
    if (q_lens[s] > (1 << 26)) return HQMQ_ERR_SHAPE;
    most_rows = std::max(most_rows, q_lens[s] * G);
    if (chunked(q_lens[s], G)) { ++ch_seqs; most_q = std::max(most_q, q_lens[s]); continue; }
    int beg, end;
    unit_keys(kv_lens[s], q_lens[s], G, p.window, 0, q_lens[s] * G, beg, end);
    dec_tiles += blocks_of(end, 16) - beg / 16;
    dec_rows = std::max(dec_rows, q_lens[s] * G);
    ++dec_units;
  }
  if (total_q > (1 << 30) || n_tab > (1 << 28) || dec_tiles > (1 << 29)) return HQMQ_ERR_SHAPE;
  p.total_q = (int)total_q; p.most_q = all_q; p.n_tab = (int)n_tab;
  p.dec_units = dec_units; p.dec_rows = dec_rows > 16 ? 32 : dec_rows > 8 ? 16 : 8; p.dec_tiles = (int)dec_tiles;
  // CTAs per head: one per SM in all, no more than leave every warp two tiles; or one, while the CTAs of all heads fit as clusters (whose
  // parts need no second kernel)
  const int most = std::max(1, HQMQ_PAGED_MAX_CTAS / p.H_kv);
  auto ctas = [&](int64_t tiles, int warps) { return (int)std::max<int64_t>(1, std::min<int64_t>(most, (tiles + 2 * warps - 1) / (2 * warps))); };
  const int W_ = dec_warps(p.dec_rows);
  // Of a plan with room, by the tiles that the room holds: the lengths that it is first made with do not bound those it will serve.  (A unit's
  // tiles are its sequence's at most, and with a window the window's, the new tokens' and one cut at either end.)
  const auto room_of = [&](int64_t units, int queries) {
    const int64_t held = (int64_t)p.tab_room * (p.page_tokens / 16);
    return p.window > 0 ? std::min(held, units * (((int64_t)p.window + queries) / 16 + 2)) : held;
  };
  const int64_t dec_most = p.tab_room && dec_units ? std::max(dec_tiles, room_of(dec_units, (dec_rows + G - 1) / G)) : dec_tiles;
  p.dec_ctas = ctas(dec_most, W_);
  const int single = (int)std::min<int64_t>(1 << 20, (dec_most + W_ - 1) / W_);
  if (single >= 1 && as_cluster(single, p.H_kv)) p.dec_ctas = single;
  // chunks
  p.ch_seqs = ch_seqs;
  const int P = 128 / G;
  p.ch_streams = most_q > P ? 2 : 1;
  int64_t ch_units = 0, ch_tiles = 0, img = 0;
  p.ms_rows = most_rows > 8 ? kMassRowsWide : 8;
  for (int s = 0; s < p.n_seqs; ++s) ms_groups += blocks_of(kv_lens[s], mass_group(p.ms_rows));
  for (int s = 0; s < p.n_seqs; ++s) {
    if (!p.H_q || !q_lens[s]) continue;
    const int rows = q_lens[s] * G;
    for (int r = 0; r < rows; r += p.ms_rows, ++ms_units) {
      int beg, end;
      unit_keys(kv_lens[s], q_lens[s], G, p.window, r, std::min(rows, r + p.ms_rows), beg, end);
      ms_tiles += blocks_of(end, 16) - beg / 16;
    }
    if (!chunked(q_lens[s], G)) continue;
    const int um = blocks_of(q_lens[s], p.ch_streams * P);
    int first = 0, last = 0;
    for (int m = 0; m < um; ++m) {
      int lo, n;
      chunk_unit(p, kv_lens[s], q_lens[s], m, lo, n);
      if (m == 0) first = lo;
      last = std::max(last, lo + n);
      ch_tiles += n;
    }
    ch_units += um;
    img += last - first;
  }
  if (ch_tiles > (1 << 26)) return HQMQ_ERR_SHAPE;
  // (a prompt whose weights nobody could hold is no reason to refuse its attention)
  const int64_t ms_blocks = blocks_of(most_rows, p.ms_rows), ms_held = ms_blocks * p.tab_room * (p.page_tokens / 16);
  p.no_mass = std::max(ms_tiles, ms_held) > (1 << 29);
  if (p.no_mass) ms_tiles = ms_units = ms_groups = 0;
  p.ch_units = (int)ch_units; p.ch_tiles = (int)ch_tiles; p.ch_img_tiles = (int)img;
  // the operand images of as many heads at a time as half a gigabyte holds, a divisor of the heads
  p.ch_heads = p.H_kv;
  while (p.ch_heads > 1 && (int64_t)p.ch_heads * img * 2 * p.d * 256 > ((int64_t)512 << 20)) {
    do --p.ch_heads; while (p.H_kv % p.ch_heads);
  }
  // whole units per CTA or equal pieces (costs in tiles as in prefill_plan): the longest hand, dealt out to and fro
  p.ch_whole = 0; p.ch_ctas = 0;
  if (ch_units) {
    const int64_t n_units = ch_units * p.ch_heads, total = ch_tiles * p.ch_heads, L = (total + HQMQ_PAGED_MAX_CTAS - 1) / HQMQ_PAGED_MAX_CTAS;
    const int grid_w = (int)std::min<int64_t>(n_units, HQMQ_PAGED_MAX_CTAS);
    // (an upper bound of the longest hand without the sorted list: the mean and the longest unit)
    int longest = 0;
    for (int s = 0; s < p.n_seqs; ++s) {
      if (!q_lens[s] || !chunked(q_lens[s], G)) continue;
      const int um = blocks_of(q_lens[s], p.ch_streams * P);
      for (int m = 0; m < um; ++m) { int lo, n; chunk_unit(p, kv_lens[s], q_lens[s], m, lo, n); longest = std::max(longest, n); }
    }
    const int64_t hands = (n_units + grid_w - 1) / grid_w;
    const int64_t whole = hands == 1 ? longest + 2 : total / grid_w + longest / 2 + 2 * hands;
    const int64_t cut = L + 2 * (hands + 1) + 2 + 6;
    p.ch_whole = whole <= cut;
    p.ch_ctas = p.ch_whole ? grid_w : (int)((total + L - 1) / L);
  }
  p.ms_units = (int)ms_units; p.ms_tiles = (int)ms_tiles; p.ms_groups = p.H_q ? (int)ms_groups : 0;
  int64_t ms_most = ms_tiles;
  p.ms_tile_room = p.ms_tiles; p.ms_group_room = p.ms_groups;
  if (p.tab_room) {
    if (n_tab > p.tab_room) return HQMQ_ERR_CAPACITY;
    // (every unit walks its sequence's tiles at most; a sequence has that many units)
    const int64_t tiles = p.no_mass ? 0 : ms_held;
    p.ms_tile_room = (int)tiles;
    if (ms_units) ms_most = std::max(ms_tiles, std::min(tiles, ms_blocks * room_of(ms_units, (p.ms_rows + G - 1) / G)));
    p.ms_group_room = p.H_q && !p.no_mass ? (int)((int64_t)p.tab_room * p.page_tokens / mass_group(p.ms_rows) + p.n_seqs) : 0;
  }
  p.ms_ctas = (int)std::max<int64_t>(1, std::min<int64_t>(most, (ms_most + kMassWarps - 1) / kMassWarps));
  if (p.renew) {
    if (ch_units || had.ch_units) return HQMQ_ERR_UNSUPPORTED;
    if (had.dec_units != p.dec_units || had.dec_rows != p.dec_rows || had.ms_units != p.ms_units || had.no_mass != p.no_mass || had.ms_rows != p.ms_rows ||
        had.total_q != p.total_q || had.most_q != p.most_q) return HQMQ_ERR_SHAPE;
    p.dec_ctas = had.dec_ctas; p.ms_ctas = had.ms_ctas;
  }
  int64_t at = 16;
  auto take = [&](int32_t& where, int64_t words) { where = (int32_t)at; at += up4(words); };
  take(p.seqs, 4 * (int64_t)p.n_seqs);
  take(p.dec_unit, 4 * (int64_t)p.dec_units);
  take(p.dec_base, (int64_t)p.dec_units + 1);
  take(p.dec_warp, kWarpRecord * (int64_t)p.dec_ctas * dec_warps(p.dec_rows));
  take(p.dec_cut, 4 * (int64_t)p.dec_ctas);
  take(p.ch_unit, 8 * ch_units);
  take(p.ch_order, p.ch_whole ? ch_units : 0);
  take(p.ch_start, p.ch_whole ? 0 : 4 * (int64_t)p.ch_ctas);
  take(p.ch_img, 4 * (int64_t)ch_seqs);
  take(p.ms_unit, 4 * ms_units);
  take(p.ms_base, ms_units + 1);
  take(p.ms_warp, kWarpRecord * (int64_t)p.ms_ctas * kMassWarps);
  take(p.ms_group, 4 * (int64_t)p.ms_group_room);
  take(p.tabs, p.tab_room ? p.tab_room : n_tab);
  if (at > (1 << 30)) return HQMQ_ERR_SHAPE;
  p.words = (int32_t)at;
  return HQMQ_OK;
}

extern "C" int hqmq_paged_plan_fill(const hqmq_paged_plan* plan, const int32_t* kv_lens, const int32_t* q_lens, const int32_t* tables,
                                    int64_t table_stride, int32_t* out) {
  if (!plan || !kv_lens || !q_lens || !tables || !out) return HQMQ_ERR_ARG;
  int rc = check_plan(*plan);
  if (rc) return rc;
  const hqmq_paged_plan& p = *plan;
  const int G = p.H_q ? p.H_q / p.H_kv : 1;
  std::fill(out, out + p.words, 0);
  out[0] = p.dec_units; out[1] = p.dec_tiles; out[2] = p.ms_units; out[3] = p.ms_tiles; out[4] = p.ms_groups;
  int q_off = 0, tab = 0, du = 0, dt = 0, cu = 0, cs = 0, img = 0, mu = 0, mt = 0, mg = 0;
  for (int s = 0; s < p.n_seqs; ++s) {
    const int kv = kv_lens[s], q = q_lens[s], pages = blocks_of(kv, p.page_tokens);
    int32_t* sq = out + p.seqs + 4 * s;
    sq[0] = kv; sq[1] = q; sq[2] = q_off; sq[3] = tab;
    for (int i = 0; i < pages; ++i) {
      const int32_t page = tables[s * table_stride + i];
      if (page < 0 || page >= p.n_pages) return HQMQ_ERR_SHAPE;
      out[p.tabs + tab + i] = page;
    }
    const int my_mu = mu;
    if (p.H_q && q) {
      const int rows = q * G;
      for (int r = 0; r < rows && !p.no_mass; r += p.ms_rows, ++mu) {
        int beg, end;
        unit_keys(kv, q, G, p.window, r, std::min(rows, r + p.ms_rows), beg, end);
        int32_t* u = out + p.ms_unit + 4 * mu;
        u[0] = s; u[1] = r; u[2] = beg / 16; u[3] = blocks_of(end, 16);
        out[p.ms_base + mu] = mt;
        mt += u[3] - u[2];
      }
      if (!chunked(q, G)) {
        int beg, end;
        unit_keys(kv, q, G, p.window, 0, rows, beg, end);
        int32_t* u = out + p.dec_unit + 4 * du;
        u[0] = s; u[1] = 0; u[2] = beg / 16; u[3] = blocks_of(end, 16);
        out[p.dec_base + du] = dt;
        dt += u[3] - u[2];
        ++du;
      } else {
        const int um = blocks_of(q, p.ch_streams * (128 / G));
        int first = 0, last = 0;
        for (int m = 0; m < um; ++m, ++cu) {
          int lo, n;
          chunk_unit(p, kv, q, m, lo, n);
          if (m == 0) first = lo;
          last = std::max(last, lo + n);
          int32_t* u = out + p.ch_unit + 8 * cu;
          u[0] = s; u[1] = m; u[2] = lo; u[3] = n; u[4] = kv; u[5] = q; u[6] = q_off; u[7] = img - first;
        }
        int32_t* ci = out + p.ch_img + 4 * cs++;
        ci[0] = s; ci[1] = first; ci[2] = last - first; ci[3] = img;
        img += last - first;
      }
    }
    if (p.H_q && !p.no_mass)
      for (int t = 0; t < kv; t += mass_group(p.ms_rows)) {
        int32_t* g = out + p.ms_group + 4 * mg++;
        g[0] = s; g[1] = t; g[2] = my_mu; g[3] = mu;
      }
    q_off += q; tab += pages;
  }
  // flat sequences: what every warp's stretch begins with; units cut between CTAs
  auto stretches = [&](int units, int total, int ctas, int warps, int unit_at, int base_at, int warp_at) {
    const int n = ctas * warps;
    out[base_at + units] = total;
    int u = 0;
    for (int w = 0; w < n; ++w) {
      const int f0 = stretch_begin(w, total, n), f1 = stretch_begin(w + 1, total, n);
      while (u + 1 < units && out[base_at + u + 1] <= f0) ++u;
      const int32_t* un = out + unit_at + 4 * u;
      const int32_t* sq = out + p.seqs + 4 * un[0];
      const int tile = f0 < total ? un[2] + f0 - out[base_at + u] : un[2];
      int32_t* r = out + warp_at + kWarpRecord * w;
      r[0] = f0; r[1] = f1; r[2] = u; r[3] = tile;
      r[4] = un[3]; r[5] = sq[3]; r[6] = out[p.tabs + sq[3] + tile * 16 / p.page_tokens]; r[7] = un[1];
      r[8] = out[base_at + u]; r[9] = out[base_at + u + 1];
      for (int i = 0; i < 4; ++i) r[12 + i] = sq[i];
    }
  };
  if (p.dec_units) {
    const int W = dec_warps(p.dec_rows), n = p.dec_ctas * W;
    stretches(p.dec_units, p.dec_tiles, p.dec_ctas, W, p.dec_unit, p.dec_base, p.dec_warp);
    int cuts = 0;
    for (int u = 0; u < p.dec_units; ++u) {
      const int b0 = out[p.dec_base + u], b1 = out[p.dec_base + u + 1];
      const int k0 = warp_of(b0, p.dec_tiles, n) / W, k1 = warp_of(b1 - 1, p.dec_tiles, n) / W;
      if (k0 == k1) continue;
      int32_t* c = out + p.dec_cut + 4 * cuts++;
      c[0] = u; c[1] = k0; c[2] = k1; c[3] = b0 > stretch_begin(k0 * W, p.dec_tiles, n) ? 1 : 0;    // slot of the first part
    }
    out[5] = cuts;
  }
  if (p.ms_units) stretches(p.ms_units, p.ms_tiles, p.ms_ctas, kMassWarps, p.ms_unit, p.ms_base, p.ms_warp);
  if (p.ch_units) {
    const int32_t* un = out + p.ch_unit;
    if (p.ch_whole) {
      int32_t* o = out + p.ch_order;
      for (int i = 0; i < p.ch_units; ++i) o[i] = i;
      std::sort(o, o + p.ch_units, [un](int32_t a, int32_t b) { return un[8 * a + 3] != un[8 * b + 3] ? un[8 * a + 3] > un[8 * b + 3] : a < b; });
    } else {
      const int64_t total = (int64_t)p.ch_tiles * p.ch_heads, L = (total + p.ch_ctas - 1) / p.ch_ctas;
      int64_t at = 0;
      int m = 0, h = 0;
      for (int c = 0; c < p.ch_ctas; ++c) {
        const int64_t pos = std::min<int64_t>(c * L, total - 1);
        while (pos - at >= un[8 * m + 3]) {
          at += un[8 * m + 3];
          if (++m == p.ch_units) { m = 0; ++h; }
        }
        int32_t* st = out + p.ch_start + 4 * c;
        st[0] = h; st[1] = m; st[2] = (int32_t)(pos - at); st[3] = 0;
      }
    }
  }
  return HQMQ_OK;
}
