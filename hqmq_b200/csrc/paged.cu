// Attention and attention weights over a paged cache: host entry points.  Storing and evicting: paged_move.cu; prompt chunks: attn_prefill.cu.
#include <string.h>

#include <algorithm>

#include "attn_prefill.cuh"
#include "paged_decode.cuh"
#include "paged_mass.cuh"

namespace hqmq {
namespace paged {
namespace {

constexpr size_t kSmemMax = 232448;          // 227 KB
constexpr float kLog2e = 1.4426950408889634f;

int log2_of(int x) { int b = 0; while ((1 << b) < x) ++b; return b; }
size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

int check_args(const hqmq_paged_attn_args* a, bool mass) {
  if (!a || a->struct_size != sizeof(hqmq_paged_attn_args)) return HQMQ_ERR_ARG;
  int rc = check_plan(a->plan);
  if (rc) return rc;
  const hqmq_paged_plan& p = a->plan;
  if (p.H_q < 1 || p.words < 16) return HQMQ_ERR_ARG;
  if ((rc = check_pool(a->K, p)) != 0) return rc;
  if (!a->plan_data || !a->table_K || (p.total_q > 0 && !a->Q)) return HQMQ_ERR_ARG;
  if (!is_float_dtype(a->q_dtype)) return HQMQ_ERR_DTYPE;
  if (((uintptr_t)a->plan_data & 15) || ((uintptr_t)a->table_K & 7)) return HQMQ_ERR_ALIGN;
  if (a->r_qmax != (1 << a->K.radius_bits) - 1) return HQMQ_ERR_SHAPE;
  if (!(a->softcap >= 0.f) || a->softcap > 1e4f || (a->softcap > 0.f && a->softcap < 1e-3f)) return HQMQ_ERR_ARG;
  if (!(a->softmax_scale > 0.f && a->softmax_scale < INFINITY)) return HQMQ_ERR_ARG;
  if (mass) {
    if (!is_half_dtype(a->q_dtype)) return HQMQ_ERR_UNSUPPORTED;
    if (p.no_mass) return HQMQ_ERR_CAPACITY;
    return a->mass ? HQMQ_OK : HQMQ_ERR_ARG;
  }
  if ((rc = check_pool(a->V, p)) != 0) return rc;
  if (a->V.S != a->K.S || a->V.radius_bits != a->K.radius_bits || a->V.scale_dtype != a->K.scale_dtype ||
      (a->K.flags && a->V.flags && a->K.out_dtype != a->V.out_dtype)) return HQMQ_ERR_UNSUPPORTED;
  if (!a->table_V || (p.total_q > 0 && !a->O)) return HQMQ_ERR_ARG;
  if (!is_float_dtype(a->o_dtype)) return HQMQ_ERR_DTYPE;
  if ((uintptr_t)a->table_V & 7) return HQMQ_ERR_ALIGN;
  return HQMQ_OK;
}

QueryView query_view(const hqmq_paged_attn_args* a) {
  QueryView q;
  q.Q = a->Q; q.dtype = a->q_dtype; q.st_t = a->q_stride[0]; q.st_h = a->q_stride[1]; q.G = a->plan.H_q / a->plan.H_kv;
  q.vec = is_half_dtype(a->q_dtype) && ((uintptr_t)a->Q & 15) == 0 && a->q_stride[0] % 8 == 0 && a->q_stride[1] % 8 == 0;
  return q;
}
PoolView pool_view(const hqmq_paged_attn_args* a) {
  PoolView v;
  v.K = a->K; v.V = a->V; v.Hkv = a->plan.H_kv; v.page_bits = log2_of(a->plan.page_tokens);
  return v;
}

cudaError_t launch(const void* k, dim3 grid, int threads, void** args, size_t smem, cudaStream_t st, bool dependent, int cluster = 1) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at;
  if (cluster > 1) {
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = cluster; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
    dependent = true;
  } else {
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  if (dependent) { cfg.attrs = &at; cfg.numAttrs = 1; }          // (never both)
  return cudaLaunchKernelExC(&cfg, k, args);
}

size_t part_bytes(const hqmq_paged_plan& p) {
  const int nb = p.dec_rows / 8;
  return (size_t)nb * (p.d / 16 * 128 + 16) * 4;
}
size_t decode_parts(const hqmq_paged_plan& p) { return up256((size_t)p.dec_ctas * p.H_kv * (dec_warps(p.dec_rows) + 1) * 2 * part_bytes(p)); }
size_t decode_workspace(const hqmq_paged_attn_args* a) {
  const hqmq_paged_plan& p = a->plan;
  if (!p.dec_units) return 0;
  const size_t wide = a->K.flags || a->V.flags ? (size_t)p.dec_ctas * p.H_kv * dec_warps(p.dec_rows) * 32 * (p.d / 4) * 8 : 0;
  return decode_parts(p) + wide;
}

int decode_launch(const hqmq_paged_attn_args* a, void* ws, cudaStream_t st) {
  const hqmq_paged_plan& pl = a->plan;
  DecodeParams p;
  memset(&p, 0, sizeof(p));
  p.pool = pool_view(a);
  p.q = query_view(a);
  p.O = a->O; p.o_dtype = a->o_dtype; p.os_t = a->o_stride[0]; p.os_h = a->o_stride[1];
  p.o_vec = is_half_dtype(a->o_dtype) && ((uintptr_t)a->O & 3) == 0 && a->o_stride[0] % 2 == 0 && a->o_stride[1] % 2 == 0;
  p.tblK = a->table_K; p.tblV = a->table_V; p.sinks = a->sinks;
  p.table_rows = 24 * a->K.S; p.ib = idx_bits_for(a->K.S); p.row_bytes = a->K.row_bytes;
  p.window = pl.window; p.sdt = a->K.scale_dtype; p.pay_bf16 = (a->K.flags ? a->K : a->V).out_dtype == HQMQ_BF16;
  p.qmaxf = (float)a->r_qmax; p.vfac = 1.f / (float)a->r_qmax;
  p.kfac = a->softmax_scale * kLog2e / (float)a->r_qmax;
  if (a->softcap > 0.f) { p.cap_log2 = a->softcap * kLog2e; p.kfac *= 1.f / p.cap_log2; }
  const int4* d = reinterpret_cast<const int4*>(a->plan_data);
  p.hdr = a->plan_data;
  p.seqs = d + pl.seqs / 4; p.units = d + pl.dec_unit / 4; p.cuts = d + pl.dec_cut / 4;
  p.base = a->plan_data + pl.dec_base; p.warps = a->plan_data + pl.dec_warp; p.tabs = a->plan_data + pl.tabs;
  p.ctas = pl.dec_ctas;
  p.parts = reinterpret_cast<float*>(ws);
  p.wide = reinterpret_cast<uint2*>(reinterpret_cast<unsigned char*>(ws) + decode_parts(pl));
  const bool outl = a->K.flags || a->V.flags;
  const int nb = pl.dec_rows / 8, warps = dec_warps(pl.dec_rows);
  const size_t rings = (size_t)warps * kTileStages * tile_layout(p.row_bytes, true, outl).bytes + kPastPay + (nb > 2 ? (size_t)warps * nb * pl.d * 16 : 0), table = (size_t)(p.table_rows >> 1) * 8;
  // (the tables with every warp's own entries behind the codebook, if it has some; a field that no encoder writes may index up to 2^ib / 2
  // entries: what that reaches lies in the block's shared memory, too)
  const size_t any = (size_t)4 << p.ib;
  size_t tk = table, tv = table;
  const int room = (int)((any - table) / 8) / warps;           // (any >= table: an index has the bits of the codebook)
  if (outl && has_ext(p.ib) && compiled_fields(p.ib, a->K.radius_bits) && room >= kExtLeast) {
    p.ext_k = std::min(room, kPayK); p.ext_v = std::min(room, kPayV);
    tk += (size_t)warps * p.ext_k * 8; tv += (size_t)warps * p.ext_v * 8;
  }
  auto need = [&](int rk, int rv) { return std::max(rings + (tk << rk) + (tv << rv), std::max(any << rk, (tk << rk) + (any << rv))); };
  auto fits = [&](int rk, int rv) { return rk <= 4 && rv <= 4 && need(rk, rv) <= kSmemMax; };
  if (p.ext_k && !fits(0, 0)) { p.ext_k = p.ext_v = 0; tk = tv = table; }
  if (!fits(0, 0)) return HQMQ_ERR_UNSUPPORTED;
  // (replicas of the tables against bank conflicts, K first)
  for (bool more = true; more;) {
    more = false;
    if (fits(p.repk + 1, p.repv) && p.repk <= p.repv) { ++p.repk; more = true; }
    else if (fits(p.repk, p.repv + 1) && p.repv < p.repk) { ++p.repv; more = true; }
  }
  const size_t smem = need(p.repk, p.repv);
  const DecodeKernels k = pl.d == 128 ? decode_kernels_128(p.ib, a->K.radius_bits, nb, outl) : decode_kernels_64(p.ib, a->K.radius_bits, nb, outl);
  HQMQ_CHECK_CUDA(raise_smem_limit(k.decode, smem));
  void* args[] = {&p};
  p.fused = p.ctas > 1 && as_cluster(p.ctas, pl.H_kv);
  HQMQ_CHECK_CUDA(launch(k.decode, dim3(p.ctas * pl.H_kv), warps * 32, args, smem, st, false, p.fused ? p.ctas : 1));
  if (p.ctas > 1 && !p.fused) HQMQ_CHECK_CUDA(launch(k.merge, dim3(p.ctas - 1, pl.H_kv, nb * pl.d / 16 * 32 / 64), 64, args, 0, st, true));
  return HQMQ_OK;
}

struct MassPlaces { size_t parts, cta, stats, wide, scores, bytes; };
MassPlaces mass_places(const hqmq_paged_attn_args* a) {
  const hqmq_paged_plan& p = a->plan;
  MassPlaces m;
  const size_t r = p.ms_rows, ctas = (size_t)p.ms_ctas * p.H_kv;
  m.parts = 0;
  m.cta = up256(ctas * kMassWarps * 2 * r * 8);
  m.stats = m.cta + up256(ctas * 2 * r * 8);
  m.wide = m.stats + up256((size_t)p.H_kv * p.ms_units * r * 8);
  m.scores = m.wide + (a->K.flags ? up256(ctas * kMassWarps * 16 * (p.d / 4) * 16) : 0);
  m.bytes = m.scores + (size_t)p.H_kv * p.ms_tile_room * kTile * r * 4 + 256;
  return m;
}

}  // namespace
}  // namespace paged
}  // namespace hqmq

using namespace hqmq;
using namespace hqmq::paged;

extern "C" size_t hqmq_paged_attn_workspace_bytes(const hqmq_paged_attn_args* args) {
  if (check_args(args, false)) return 0;
  return up256(decode_workspace(args)) + chunk_workspace(args) + 256;
}

extern "C" int hqmq_paged_attn(const hqmq_paged_attn_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_args(args, false);
  if (rc) return rc;
  if (!workspace || workspace_bytes < hqmq_paged_attn_workspace_bytes(args)) return HQMQ_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return HQMQ_ERR_ALIGN;
  if (args->plan.dec_units) {
    const int e = decode_launch(args, workspace, (cudaStream_t)stream);
    if (e) return e;
  }
  if (args->plan.ch_units) return chunk_launch(args, reinterpret_cast<unsigned char*>(workspace) + up256(decode_workspace(args)), (cudaStream_t)stream);
  return HQMQ_OK;
}

extern "C" size_t hqmq_paged_mass_workspace_bytes(const hqmq_paged_attn_args* args) {
  if (check_args(args, true)) return 0;
  return mass_places(args).bytes;
}

extern "C" int hqmq_paged_mass(const hqmq_paged_attn_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_args(a, true);
  if (rc) return rc;
  const hqmq_paged_plan& pl = a->plan;
  const MassPlaces m = mass_places(a);
  if (!workspace || workspace_bytes < m.bytes) return HQMQ_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return HQMQ_ERR_ALIGN;
  cudaStream_t st = (cudaStream_t)stream;
  unsigned char* ws = reinterpret_cast<unsigned char*>(workspace);
  MassParams p;
  memset(&p, 0, sizeof(p));
  p.pool = pool_view(a);
  memset(&p.pool.V, 0, sizeof(p.pool.V));
  p.q = query_view(a);
  p.tblK = a->table_K; p.sinks = a->sinks;
  p.table_rows = 24 * a->K.S; p.ib = idx_bits_for(a->K.S); p.row_bytes = a->K.row_bytes;
  p.window = pl.window; p.sdt = a->K.scale_dtype; p.qmaxf = (float)a->r_qmax;
  p.kfac = a->softmax_scale * kLog2e / (float)a->r_qmax;
  if (a->softcap > 0.f) { p.cap = a->softcap * kLog2e; p.cap_in = 1.f / p.cap; }
  const int4* d = reinterpret_cast<const int4*>(a->plan_data);
  p.hdr = a->plan_data;
  p.seqs = d + pl.seqs / 4; p.units = d + pl.ms_unit / 4; p.groups = d + pl.ms_group / 4;
  p.base = a->plan_data + pl.ms_base; p.warps = a->plan_data + pl.ms_warp; p.tabs = a->plan_data + pl.tabs;
  p.ctas = pl.ms_ctas;
  p.parts = reinterpret_cast<float2*>(ws + m.parts); p.cta_parts = reinterpret_cast<float2*>(ws + m.cta);
  p.stats = reinterpret_cast<float2*>(ws + m.stats); p.scores = reinterpret_cast<float*>(ws + m.scores);
  p.wide = reinterpret_cast<uint4*>(ws + m.wide);
  p.prior = a->prior; p.mass = a->mass; p.decay = a->decay;
  if (pl.ms_group_room == 0) return HQMQ_OK;
  const bool outl = a->K.flags != nullptr;
  const int nb = pl.ms_rows / 8;
  void* args[] = {&p};
  if (pl.ms_units) {
    const size_t rings = (size_t)kMassWarps * kTileStages * tile_layout(p.row_bytes, false, outl).bytes + kPastPay + (nb > 1 ? (size_t)kMassWarps * nb * pl.d * 16 : 0), table = (size_t)(p.table_rows >> 1) * 8;
    auto need = [&](int rk) { return std::max(rings + (table << rk), ((size_t)4 << p.ib) << rk); };
    if (need(0) > kSmemMax) return HQMQ_ERR_UNSUPPORTED;
    while (p.repk < 4 && need(p.repk + 1) <= kSmemMax) ++p.repk;
    const void* k = pl.d == 128 ? scores_kernel_128(p.ib, a->K.radius_bits, nb, outl) : scores_kernel_64(p.ib, a->K.radius_bits, nb, outl);
    const size_t smem = need(p.repk);
    HQMQ_CHECK_CUDA(raise_smem_limit(k, smem));
    HQMQ_CHECK_CUDA(launch(k, dim3(p.ctas * pl.H_kv), kMassWarps * 32, args, smem, st, false));
  }
  const void* sum = nb == 1 ? (const void*)&paged_mass_kernel<1> : (const void*)&paged_mass_kernel<4>;
  HQMQ_CHECK_CUDA(launch(sum, dim3(pl.ms_group_room, pl.H_kv), 256, args, 0, st, pl.ms_units != 0));
  return HQMQ_OK;
}
