// Attention of drafted nodes over a request's cached positions: the plan's sizes, the join, the entry point and
// the kernels of the 16-bit caches.
#include "dsv_attn.h"

namespace dsv {

template void launch_attn<DSV_BF16, DSV_BF16>(const AttnParams&, const AttnShape&, unsigned, hipStream_t);
template void launch_attn<DSV_F16, DSV_F16>(const AttnParams&, const AttnShape&, unsigned, hipStream_t);
extern template void launch_attn<DSV_BF16, DSV_E4M3>(const AttnParams&, const AttnShape&, unsigned, hipStream_t);
extern template void launch_attn<DSV_F16, DSV_E4M3>(const AttnParams&, const AttnShape&, unsigned, hipStream_t);
extern template void launch_attn<DSV_BF16, DSV_I8>(const AttnParams&, const AttnShape&, unsigned, hipStream_t);
extern template void launch_attn<DSV_F16, DSV_I8>(const AttnParams&, const AttnShape&, unsigned, hipStream_t);

// The pieces of a request's row joined, a wave a row: references, then sums in the pieces' order.
template <int XT, int DP>
__global__ __launch_bounds__(AT_THREADS) void k_attn_join(AttnParams P) {
  const dsv_tree_attention_args& a = P.a;
  const dsv_kv_cache& c = a.cache;
  constexpr int PER = DP / WAVE;
  const int lane = threadIdx.x & (WAVE - 1);
  const int per = c.heads * a.T * P.G;
  const int64_t i = (int64_t)blockIdx.x * AT_WAVES + threadIdx.x / WAVE;
  const int b = (int)(i / per);
  if (b >= a.bs) return;
  const int in = (int)(i - (int64_t)b * per), h = in / (a.T * P.G), r = in - h * (a.T * P.G);
  const Request req = request_of(a, b);
  if (r >= req.nodes * P.G) return;
  const int chunk = plan_chunk(P, lane), pieces = pieces_of(tiles_of(req), chunk);
  if (pieces < 2) return;
  const int first = items_before(P, chunk, b, lane);
  const int64_t rows = (int64_t)a.T * P.G, step = c.heads * rows;
  const int64_t at = ((int64_t)first * c.heads + h) * rows + r;
  float top = AT_LOW;
  for (int k = lane; k < pieces; k += WAVE) top = fmaxf(top, P.part_ml[at + k * step].x);
  top = wave_max_f32(top);
  float sum[PER], lt = 0.f;
#pragma unroll
  for (int u = 0; u < PER; ++u) sum[u] = 0.f;
  const int d = lane * PER;
#pragma unroll 4
  for (int k = 0; k < pieces; ++k) {
    const float2 ml = P.part_ml[at + k * step];
    const float f = __builtin_amdgcn_exp2f(ml.x - top);
    lt = fmaf(ml.y, f, lt);
    const float* po = P.part_o + (at + k * step) * c.dim + (d < c.dim ? d : 0);
#pragma unroll
    for (int u = 0; u < PER; ++u) sum[u] = fmaf(po[u], f, sum[u]);
  }
  const int node = r / P.G, qh = h * P.G + r - node * P.G;
  const int64_t row = row_of(a, b, node);
  if (row < 0) return;
  const float inv = lt == 0.f ? 0.f : 1.f / lt;
  if (d < c.dim) {
    uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + row * a.out_row_stride + qh * a.out_head_stride + d;
#pragma unroll
    for (int u = 0; u < PER; ++u) out[u] = (uint16_t)pack_act<XT>(sum[u] * inv, 0.f);
  }
  if (lane == 0 && a.lse) a.lse[row * a.q_heads + qh] = lt == 0.f ? -INFINITY : (top + log2f(lt)) * 0.693147180559945309f;
}

static int attn_target(int heads, int RB) {
  const int t = (1024 + heads * RB - 1) / (heads * RB);
  return t < 1 ? 1 : t;
}

static AttnShape attn_shape(int T, int G) {
  const int tiles = (T * G + 15) / 16;
  AttnShape s;
  s.staged = tiles > 1;
  s.R = tiles > 4 ? 2 : 1;
  const int groups = (tiles + s.R - 1) / s.R;
  s.WR = !s.staged ? 1 : (groups > 2 ? 4 : 2);  // (a staged tile has two steps for waves of the same rows)
  s.RB = (groups + s.WR - 1) / s.WR;
  return s;
}

}  // namespace dsv

using namespace dsv;

extern "C" int64_t dsv_tree_attention_workspace_bytes(int32_t bs, int32_t T, int32_t heads, int32_t q_heads,
                                                      int32_t dim) {
  if (bs < 1 || T < 1 || heads < 1 || q_heads < heads || dim < 1) return 0;
  const AttnShape s = attn_shape(T, q_heads / heads);
  const int64_t rows = ((int64_t)attn_target(heads, s.RB) + bs) * q_heads * T;
  return rows * (dim * (int64_t)sizeof(float) + (int64_t)sizeof(float2));
}

extern "C" int dsv_tree_attention(const dsv_tree_attention_args* args, dsv_stream_t stream_) {
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  if (!args) DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_attention: no arguments");
  const dsv_tree_attention_args& a = *args;
  const int rc = check_cache("dsv_tree_attention", &a.cache);
  if (rc != DSV_OK) return rc;
  if (a.dtype != DSV_BF16 && a.dtype != DSV_F16)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_attention: unknown activation type %d", a.dtype);
  const bool quant = a.cache.dtype == DSV_E4M3 || a.cache.dtype == DSV_I8;
  if (!quant && a.cache.dtype != a.dtype)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_attention: queries and an unquantised cache must be of one type");
  if (a.bs < 1 || a.T < 1 || a.T > AT_NODES || a.rows < 0 || (!a.row_offsets && a.rows != (int64_t)a.bs * a.T))
    DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_attention: invalid layout (bs %d, T %d, rows %lld)", a.bs, a.T, (long long)a.rows);
  if (a.q_heads < 1 || a.q_heads % a.cache.heads || a.q_heads > 65535)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_attention: %d query heads over %d cache heads", a.q_heads, a.cache.heads);
  if (a.rows == 0) return DSV_OK;
  if (!a.q || !a.out || !a.prefix_lens || !a.page_table || a.page_cols < 1 || a.page_cols > 0x7fffffc0)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_attention: q, out, prefix_lens and a page table are required");
  if ((uintptr_t)a.q % 16 || (uintptr_t)a.out % 16 || a.q_row_stride % 8 || a.q_head_stride % 8 ||
      a.out_row_stride % 8 || a.out_head_stride % 8)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_attention: rows of q and out must start on 16-byte boundaries");
  if (!(a.scale >= -3.4e38f && a.scale <= 3.4e38f)) DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_attention: scale must be finite");
  const int64_t esize = quant ? 1 : 2;
  if (a.cache.k_slot_stride * esize > 0x7fffffff || a.cache.v_slot_stride * esize > 0x7fffffff)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_attention: slots are too far apart");
  AttnParams P;
  P.a = a;
  P.G = a.q_heads / a.cache.heads;
  const AttnShape s = attn_shape(a.T, P.G);
  P.WR = s.WR;
  P.RB = s.RB;
  P.target = attn_target(a.cache.heads, s.RB);
  P.least = 2;
  P.joined = a.page_cols > (int64_t)P.least * AT_TILE;
  const int64_t items = (int64_t)P.target + a.bs, blocks = (items + 7) / 8 * 8 * a.cache.heads * s.RB;
  const int64_t rows = (int64_t)a.bs * a.T * a.q_heads;
  if (blocks > 0x7fffffffll || rows / AT_WAVES >= 0x7fffffffll)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_attention: too many nodes for one call");
  const int64_t need = dsv_tree_attention_workspace_bytes(a.bs, a.T, a.cache.heads, a.q_heads, a.cache.dim);
  if (!a.workspace || (uintptr_t)a.workspace % 16)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_attention: a 16-byte-aligned workspace is required");
  if (a.workspace_bytes < need)
    DSV_FAIL(DSV_ERR_WORKSPACE, "dsv_tree_attention: workspace %lld < %lld", (long long)a.workspace_bytes, (long long)need);
  P.num_slots = (uint32_t)(a.cache.num_slots < 0x7fffffff ? a.cache.num_slots : 0x7fffffff);
  P.k_step = (uint32_t)(a.cache.k_slot_stride * esize);
  P.v_step = (uint32_t)(a.cache.v_slot_stride * esize);
  P.part_o = reinterpret_cast<float*>(a.workspace);
  P.part_ml = reinterpret_cast<float2*>(P.part_o + items * a.q_heads * a.T * a.cache.dim);
  const bool bf = a.dtype == DSV_BF16;
  if (a.cache.dtype == DSV_E4M3)
    bf ? launch_attn<DSV_BF16, DSV_E4M3>(P, s, (unsigned)blocks, stream) : launch_attn<DSV_F16, DSV_E4M3>(P, s, (unsigned)blocks, stream);
  else if (a.cache.dtype == DSV_I8)
    bf ? launch_attn<DSV_BF16, DSV_I8>(P, s, (unsigned)blocks, stream) : launch_attn<DSV_F16, DSV_I8>(P, s, (unsigned)blocks, stream);
  else
    bf ? launch_attn<DSV_BF16, DSV_BF16>(P, s, (unsigned)blocks, stream) : launch_attn<DSV_F16, DSV_F16>(P, s, (unsigned)blocks, stream);
  DSV_CHECK_LAUNCH("k_attn");
  if (P.joined) {
    const dim3 grid((unsigned)((rows + AT_WAVES - 1) / AT_WAVES));
    auto join = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(AT_THREADS), 0, stream, P); };
    if (a.cache.dim <= 64)
      bf ? join(k_attn_join<DSV_BF16, 64>) : join(k_attn_join<DSV_F16, 64>);
    else if (a.cache.dim <= 128)
      bf ? join(k_attn_join<DSV_BF16, 128>) : join(k_attn_join<DSV_F16, 128>);
    else
      bf ? join(k_attn_join<DSV_BF16, 256>) : join(k_attn_join<DSV_F16, 256>);
    DSV_CHECK_LAUNCH("k_attn_join");
  }
  return DSV_OK;
}
