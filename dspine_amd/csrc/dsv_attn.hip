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

constexpr int AJ_THREADS = 256, AJ_PARTS = 4;

// The parts of a request joined: 8 elements of a row a thread, the parts in their order.  Bound by latency (the plan's
// lengths, then the parts: 5.1 us after one request's few parts, 7 to 8 us for most batches) and, for many rows, by the
// sums' bytes (14.3 us for 16 requests of 512 rows a head).  A launch of its own: a last workgroup that joins would need
// counters that somebody clears.
template <int XT, int DP>
__global__ __launch_bounds__(AJ_THREADS) void k_attn_join(AttnParams P) {
  const dsv_tree_attention_args& a = P.a;
  const dsv_kv_cache& c = a.cache;
  constexpr int PER = DP / 8, ROWS = AJ_THREADS / PER;
  const int lane = threadIdx.x & (WAVE - 1);
  const int rows = a.T * (int)P.G.d, blocks = (rows + ROWS - 1) / ROWS;
  const int b = (int)(blockIdx.x / (c.heads * blocks)), in = (int)(blockIdx.x - (int64_t)b * c.heads * blocks);
  const int h = in / blocks, r = (in - h * blocks) * ROWS + (int)threadIdx.x / PER, d = (int)threadIdx.x % PER * 8;
  const Plan plan = plan_of(P, lane);
  const Request req = request_in(P, plan, b);
  const int tiles = tiles_of(req);
  if ((in - h * blocks) * ROWS >= req.nodes * (int)P.G.d) return;
  const int before = tiles_before(P, plan, b, lane);
  const int i0 = plan.range_of(before), i1 = plan.range_of(before + tiles - 1);
  if (i0 == i1 || r >= req.nodes * (int)P.G.d || d >= c.dim) return;
  const int node = (int)P.G.div((uint32_t)r), qh = h * (int)P.G.d + r - node * (int)P.G.d;
  const int64_t row = row_of(a, b, node);
  if (row < 0) return;
  // the request's part of range i: the last of its range where that begins before it
  auto part = [&](int i) {
    return ((int64_t)(2 * i + (i == i0 && plan.start(i) < before ? 1 : 0)) * c.heads + h) * rows + r;
  };
  float top = AT_LOW, ref = 0.f, lt = 0.f, sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int i = i0; i <= i1; i += AJ_PARTS) {  // (the references and the sums of a few parts are asked for at once)
    float4 ml[AJ_PARTS];
    f32x4 x[AJ_PARTS][2];
#pragma unroll
    for (int j = 0; j < AJ_PARTS; ++j) {
      const int64_t at = part(i + j <= i1 ? i + j : i1);
      ml[j] = P.part_ml[at];
      x[j][0] = *reinterpret_cast<const f32x4*>(P.part_o + at * c.dim + d);
      x[j][1] = *reinterpret_cast<const f32x4*>(P.part_o + at * c.dim + d + 4);
    }
    const float old = top;
#pragma unroll
    for (int j = 0; j < AJ_PARTS; ++j) top = fmaxf(top, ml[j].x);  // (the last part again, where there are fewer)
    // (the weighted values' reference is kept relative to the scores': the difference is small where both are large)
    const float old_ref = ref + (old - top);
    ref = old_ref;
#pragma unroll
    for (int j = 0; j < AJ_PARTS; ++j) ref = fmaxf(ref, ml[j].x - top + ml[j].z);
    const float keep = __builtin_amdgcn_exp2f(old_ref - ref);
    lt *= __builtin_amdgcn_exp2f(old - top);
#pragma unroll
    for (int u = 0; u < 8; ++u) sum[u] *= keep;
#pragma unroll
    for (int j = 0; j < AJ_PARTS; ++j) {
      if (i + j > i1) break;
      const float f = __builtin_amdgcn_exp2f(ml[j].x - top + ml[j].z - ref);
      lt = fmaf(ml[j].y, __builtin_amdgcn_exp2f(ml[j].x - top), lt);
#pragma unroll
      for (int u = 0; u < 8; ++u) sum[u] = fmaf(x[j][u / 4][u & 3], f, sum[u]);
    }
  }
  // (two steps: either factor alone may leave float32 where the product does not)
  const float inv = lt == 0.f ? 0.f : 1.f / lt, up = __builtin_amdgcn_exp2f(ref);
#pragma unroll
  for (int u = 0; u < 8; ++u) sum[u] = sum[u] * inv * up;
  uint4 v;
  v.x = pack_act<XT>(sum[0], sum[1]);
  v.y = pack_act<XT>(sum[2], sum[3]);
  v.z = pack_act<XT>(sum[4], sum[5]);
  v.w = pack_act<XT>(sum[6], sum[7]);
  *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + row * a.out_row_stride + qh * a.out_head_stride + d) = v;
  if (d == 0 && a.lse) a.lse[row * a.q_heads + qh] = lt == 0.f ? -INFINITY : (top + log2f(lt)) * 0.693147180559945309f;
}

// The forms by rows a cache head (times are of captured calls replayed over three inputs in turn, 8 cache heads of dim 128;
// both sides of each line on one build and one card):
//   up to 16: direct.  8 x 1 node, 16k to 64k positions, int8: 183 us, 204 staged; 64 x 4 nodes, 1k to 8k, bf16: 253 and 249.
//   17 to 32: staged, two waves for the same rows.  32 rows, 1 x 640 positions: 18.1 us, 19.7 with one wave for them
//     and two that only bring; 16 x 2k to 8k: 87 and 90.
//   up to 128: staged, a wave for each 16.  With 32 a wave: 309 us for 278 (68 rows), 44.6 for 40.6 (100 rows).
//   more: staged, 32 a wave (half the LDS reads a product).  With 16: 559 us for 437 (512 rows, e4m3), 179 for 157
//     (132 rows, bf16).  Dims above 128 have no registers for it.
static AttnShape attn_shape(int T, int G, int dim) {
  const int tiles = (T * G + 15) / 16;
  AttnShape s;
  s.form = tiles == 1 ? AT_DIRECT : (tiles == 2 ? AT_PAIRS : AT_ROWS);
  s.R = tiles > AT_MOST && dim <= 128 ? 2 : 1;
  const int groups = (tiles + s.R - 1) / s.R;
  s.WR = groups < AT_MOST ? groups : AT_MOST;
  s.RB = (groups + s.WR - 1) / s.WR;
  s.waves = s.R == 2 ? AT_MOST : (s.WR > AT_WAVES ? s.WR : AT_WAVES);  // (those without rows bring positions)
  return s;
}

// Ranges at most: as many as workgroups run at once (or a few times as many where the heads and row blocks leave too
// many of those idle otherwise).
static int attn_ranges(const AttnShape& s, int heads, int dim) {
  const int lds = s.form == AT_DIRECT ? (dim > 128 ? 2 : 4) : (dim > 128 ? 1 : (dim > 64 ? 2 : 4)) / s.R;
  int per = 4 * attn_occupancy(s.form, s.R, dim) / s.waves;  // workgroups a CU
  per = per > lds ? lds : per;
  per = per < 1 ? 1 : per;
  const int64_t slots = 256 * per, hb = (int64_t)heads * s.RB;
  int64_t best = 1;
  double use = 0.0;
  for (int k = 1; k <= 4; ++k) {
    const int64_t n = k * slots / hb;
    const double u = (double)(n * hb) / (double)(k * slots);
    if (n > 0 && u > use + 0.05) use = u, best = n;
  }
  return (int)best;
}

}  // namespace dsv

using namespace dsv;

extern "C" int64_t dsv_tree_attention_workspace_bytes(int32_t bs, int32_t T, int32_t heads, int32_t q_heads,
                                                      int32_t dim) {
  if (bs < 1 || T < 1 || heads < 1 || q_heads < heads || dim < 1) return 0;
  const AttnShape s = attn_shape(T, q_heads / heads, dim);
  const int64_t rows = 2 * (int64_t)attn_ranges(s, heads, dim) * q_heads * T;
  return rows * (dim * (int64_t)sizeof(float) + (int64_t)sizeof(float4));
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
  // (times log2 e and the int8 codes' 512 it has to stay within float32)
  if (!(a.scale >= -0x1p100f && a.scale <= 0x1p100f))
    DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_attention: scale must be finite, at most 2^100");
  const int64_t esize = quant ? 1 : 2;
  if (a.cache.k_slot_stride * esize > 0x7fffffff || a.cache.v_slot_stride * esize > 0x7fffffff)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_attention: slots are too far apart");
  AttnParams P;
  P.a = a;
  const int G = a.q_heads / a.cache.heads;
  P.G = fast_div((uint32_t)G);
  const AttnShape s = attn_shape(a.T, G, a.cache.dim);
  P.WR = s.WR;
  P.RB = s.RB;
  P.most = attn_ranges(s, a.cache.heads, a.cache.dim);
  // A part of a request costs its start and its sums, so a range has a few tiles at least (twice and half of these, replayed
  // as above: 18.5 and 19.3 us for 17.2 direct, 1 x 640; 44.0 and 43.9 for 38.3 staged, 13 x 23 nodes; 41.6 and 40.5 for
  // 40.6, 4 x 25 nodes).
  P.least = fast_div(s.form == AT_ROWS ? 4 : 2);
  const int64_t blocks = (P.most + 7) / 8 * 8 * (int64_t)a.cache.heads * s.RB;
  const int64_t wide = a.cache.dim <= 64 ? 64 : (a.cache.dim <= 128 ? 128 : 256), per = AJ_THREADS / (wide / 8);
  const int64_t joins = (a.T * (int64_t)G + per - 1) / per * a.cache.heads * a.bs;
  const int64_t tiles = ((a.page_cols + AT_TILE - 1) / AT_TILE + 1) * a.bs;  // at most
  if (blocks > 0x7fffffffll || joins > 0x7fffffffll || tiles > 0x7fffff00ll)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_attention: too many nodes or positions for one call");
  const int64_t need = dsv_tree_attention_workspace_bytes(a.bs, a.T, a.cache.heads, a.q_heads, a.cache.dim);
  if (!a.workspace || (uintptr_t)a.workspace % 16)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_attention: a 16-byte-aligned workspace is required");
  if (a.workspace_bytes < need)
    DSV_FAIL(DSV_ERR_WORKSPACE, "dsv_tree_attention: workspace %lld < %lld", (long long)a.workspace_bytes, (long long)need);
  P.num_slots = (uint32_t)(a.cache.num_slots < 0x7fffffff ? a.cache.num_slots : 0x7fffffff);
  P.k_step = (uint32_t)(a.cache.k_slot_stride * esize);
  P.v_step = (uint32_t)(a.cache.v_slot_stride * esize);
  P.part_o = reinterpret_cast<float*>(a.workspace);
  P.part_ml = reinterpret_cast<float4*>(P.part_o + 2 * (int64_t)P.most * a.q_heads * a.T * a.cache.dim);
  const bool bf = a.dtype == DSV_BF16;
  if (a.cache.dtype == DSV_E4M3)
    bf ? launch_attn<DSV_BF16, DSV_E4M3>(P, s, (unsigned)blocks, stream) : launch_attn<DSV_F16, DSV_E4M3>(P, s, (unsigned)blocks, stream);
  else if (a.cache.dtype == DSV_I8)
    bf ? launch_attn<DSV_BF16, DSV_I8>(P, s, (unsigned)blocks, stream) : launch_attn<DSV_F16, DSV_I8>(P, s, (unsigned)blocks, stream);
  else
    bf ? launch_attn<DSV_BF16, DSV_BF16>(P, s, (unsigned)blocks, stream) : launch_attn<DSV_F16, DSV_F16>(P, s, (unsigned)blocks, stream);
  DSV_CHECK_LAUNCH("k_attn");
  if (P.most > 1) {
    auto join = [&](auto kern) { hipLaunchKernelGGL(kern, dim3((unsigned)joins), dim3(AJ_THREADS), 0, stream, P); };
    if (wide == 64)
      bf ? join(k_attn_join<DSV_BF16, 64>) : join(k_attn_join<DSV_F16, 64>);
    else if (wide == 128)
      bf ? join(k_attn_join<DSV_BF16, 128>) : join(k_attn_join<DSV_F16, 128>);
    else
      bf ? join(k_attn_join<DSV_BF16, 256>) : join(k_attn_join<DSV_F16, 256>);
    DSV_CHECK_LAUNCH("k_attn_join");
  }
  return DSV_OK;
}
