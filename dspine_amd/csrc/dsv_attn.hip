// Attention of drafted nodes over a request's cached positions for gfx950.
#include "dsv_cache.h"
#include "dsv_common.h"

namespace dsv {

constexpr int AT_THREADS = 256;
constexpr int AT_NODES = 64;

struct AttnParams {
  dsv_tree_attention_args a;
};

// The request's nodes, its context and its positions (context and window) that the page table has.
struct Request {
  int nodes;
  int64_t prefix, total;
};
__device__ __forceinline__ Request request_of(const dsv_tree_attention_args& a, int64_t b) {
  Request r;
  int n = a.verify_lens ? a.verify_lens[b] : a.T;
  r.nodes = n < 0 ? 0 : (n > a.T ? a.T : n);
  const int pre = a.prefix_lens[b];
  r.prefix = pre < 0 ? 0 : pre;
  r.total = r.prefix + r.nodes < a.page_cols ? r.prefix + r.nodes : a.page_cols;
  return r;
}

template <int CT>
__device__ __forceinline__ float cache_value(const void* base, int64_t at) {
  if constexpr (CT == DSV_E4M3) {
    float f[4];
    unpack_codes<CT>(reinterpret_cast<const uint8_t*>(base)[at], f);
    return f[0];
  } else if constexpr (CT == DSV_I8) {
    return (float)reinterpret_cast<const int8_t*>(base)[at];
  } else {
    return act_to_f32<CT>(reinterpret_cast<const uint16_t*>(base)[at]);
  }
}

// A workgroup per (node, query head): a position a thread for the scores, then a channel a thread for the sum
// over the positions, with the running maximum and sum of the softmax.
template <int XT, int CT>
__global__ __launch_bounds__(AT_THREADS) void k_attn(AttnParams P) {
  const dsv_tree_attention_args& a = P.a;
  const dsv_kv_cache& c = a.cache;
  constexpr bool QUANT = CT == DSV_E4M3 || CT == DSV_I8;
  __shared__ float s_q[256], s_p[AT_THREADS], s_red[AT_THREADS / WAVE];
  __shared__ int64_t s_slot[AT_THREADS];
  const int tid = threadIdx.x;
  const int64_t b = blockIdx.x / a.T;
  const int node = (int)(blockIdx.x - b * a.T), qh = blockIdx.y, h = qh / (a.q_heads / c.heads);
  const Request r = request_of(a, b);
  if (node >= r.nodes) return;
  const int64_t row = a.row_offsets ? load_index(a.row_offsets, a.row_offsets_i64, b) + node : b * a.T + node;
  if (row < 0 || row >= a.rows) return;
  if (tid < c.dim)
    s_q[tid] = act_to_f32<XT>(
        reinterpret_cast<const uint16_t*>(a.q)[row * a.q_row_stride + qh * a.q_head_stride + tid]);
  const uint64_t mask = a.masks ? (uint64_t)a.masks[b * a.T + node] : (node >= 63 ? ~0ull : (2ull << node) - 1ull);
  float m = -INFINITY, sum = 0.f, acc = 0.f;
  for (int64_t p0 = 0; p0 < r.total; p0 += AT_THREADS) {
    const int64_t p = p0 + tid;
    int64_t slot = -1;
    if (p < r.total && (p < r.prefix || ((mask >> (p - r.prefix)) & 1))) slot = a.page_table[b * a.page_stride + p];
    if (slot >= c.num_slots) slot = -1;
    __syncthreads();
    float s = -INFINITY;
    if (slot >= 0) {
      const int64_t at = slot * c.k_slot_stride + h * c.k_head_stride;
      float dot = 0.f;
      for (int d = 0; d < c.dim; ++d) dot = fmaf(s_q[d], cache_value<CT>(c.k, at + d), dot);
      if constexpr (QUANT) dot *= c.k_scale[slot * c.ks_slot_stride + h * c.ks_head_stride];
      s = dot * a.scale;
    }
    float top = wave_max_f32(s);
    if ((tid & (WAVE - 1)) == 0) s_red[tid / WAVE] = top;
    __syncthreads();
    for (int i = 0; i < AT_THREADS / WAVE; ++i) top = fmaxf(top, s_red[i]);
    const float next = fmaxf(m, top);
    const float ref = next == -INFINITY ? 0.f : next;
    const float keep = __expf(m - ref);
    const float e = slot >= 0 ? __expf(s - ref) : 0.f;
    m = next;
    s_p[tid] = e;
    s_slot[tid] = slot;
    sum *= keep;
    acc *= keep;
    const float part = block_sum<AT_THREADS / WAVE>(e, s_red);
    sum += part;
    if (tid < c.dim) {
      const int64_t left = r.total - p0 < AT_THREADS ? r.total - p0 : AT_THREADS;
      for (int i = 0; i < (int)left; ++i) {
        const int64_t at = s_slot[i];
        if (at < 0) continue;
        float w = s_p[i];
        if constexpr (QUANT) w *= c.v_scale[at * c.vs_slot_stride + h * c.vs_head_stride];
        acc = fmaf(w, cache_value<CT>(c.v, at * c.v_slot_stride + h * c.v_head_stride + tid), acc);
      }
    }
  }
  if (tid < c.dim) {
    const float o = sum == 0.f ? 0.f : acc / sum;
    reinterpret_cast<uint16_t*>(a.out)[row * a.out_row_stride + qh * a.out_head_stride + tid] =
        (uint16_t)pack_act<XT>(o, 0.f);
  }
  if (tid == 0 && a.lse) a.lse[row * a.q_heads + qh] = sum == 0.f ? -INFINITY : m + logf(sum);
}

}  // namespace dsv

using namespace dsv;

extern "C" int64_t dsv_tree_attention_workspace_bytes(int32_t bs, int32_t T, int32_t heads, int32_t q_heads,
                                                      int32_t dim) {
  return bs > 0 && T > 0 && heads > 0 && q_heads > 0 && dim > 0 ? 16 : 0;
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
  if (!a.q || !a.out || !a.prefix_lens || !a.page_table || a.page_cols < 1)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_attention: q, out, prefix_lens and a page table are required");
  if ((uintptr_t)a.q % 16 || (uintptr_t)a.out % 16 || a.q_row_stride % 8 || a.q_head_stride % 8 ||
      a.out_row_stride % 8 || a.out_head_stride % 8)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_attention: rows of q and out must start on 16-byte boundaries");
  if (!(a.scale >= -3.4e38f && a.scale <= 3.4e38f)) DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_attention: scale must be finite");
  if ((int64_t)a.bs * a.T > 0x7fffffffll) DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_attention: too many nodes for one call");
  AttnParams P;
  P.a = a;
  const dim3 grid((unsigned)(a.bs * a.T), (unsigned)a.q_heads);
  auto launch = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(AT_THREADS), 0, stream, P); };
  const bool bf = a.dtype == DSV_BF16;
  if (a.cache.dtype == DSV_E4M3)
    bf ? launch(k_attn<DSV_BF16, DSV_E4M3>) : launch(k_attn<DSV_F16, DSV_E4M3>);
  else if (a.cache.dtype == DSV_I8)
    bf ? launch(k_attn<DSV_BF16, DSV_I8>) : launch(k_attn<DSV_F16, DSV_I8>);
  else
    bf ? launch(k_attn<DSV_BF16, DSV_BF16>) : launch(k_attn<DSV_F16, DSV_F16>);
  DSV_CHECK_LAUNCH("k_attn");
  return DSV_OK;
}
