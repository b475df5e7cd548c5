// The KV cache's write and read for gfx950: new keys and values into cache slots (quantised to 8 bits
// with a scale for each (token, head) where the cache is), and slots gathered back to activations.
#include "dsv_cache.h"
#include "dsv_common.h"

namespace dsv {

// A row (one token's, one head's keys or values) is held by a group of G lanes, 16 values a lane where the cache holds
// codes (16 bytes of them), else 8: the row's largest magnitude is then a reduction inside the group, and every access
// to the cache is 16 bytes.  A group takes KV_ROWS rows, all loaded before the first is used.  Keys and values are two
// halves of the grid, so that the tensor's address and strides are scalars.
constexpr int KV_THREADS = 256;
constexpr int KV_ROWS = 2;

// Keys or values: the cache's tensor, its scales, and the activations (read by the write, written by the read).
struct KvSide {
  void* base;
  float* scale;
  void* x;
  int64_t slot_stride, head_stride, scale_slot, scale_head, row_stride, x_head;
};
struct KvParams {
  KvSide side[2];
  const void* slots;
  int32_t slots_i64;
  int dim, G;
  uint32_t rows;  // n * heads
  FastDiv heads;
  int64_t num_slots;
};

template <int CT>
constexpr int kv_lane() {
  return CT == DSV_E4M3 || CT == DSV_I8 ? 16 : 8;
}

// One of a lane group's rows.  Heads run fastest, so that neighbouring groups touch neighbouring memory on both sides.
struct KvRow {
  uint32_t token, head;
  int64_t slot;  // (one outside the cache, or of no row: -1)
  bool live;
};
__device__ __forceinline__ KvRow kv_row(const KvParams& P, int u) {
  const uint32_t groups = KV_THREADS / P.G;
  const uint32_t r = (blockIdx.x * KV_ROWS + u) * groups + threadIdx.x / P.G;
  KvRow w;
  w.live = r < P.rows;
  w.token = P.heads.div(w.live ? r : 0);
  w.head = (w.live ? r : 0) - w.token * P.heads.d;
  w.slot = load_index(P.slots, P.slots_i64, w.token);
  if (!w.live || w.slot < 0 || w.slot >= P.num_slots) w.slot = -1;
  return w;
}

// Codes of a quantised row: a = the row's largest magnitude, scale = a * (1 / top), code = rne(x * ((1 / a) * top)).
// The magnitudes are compared as the type's own 15 bits, which order like the values and keep a NaN or an infinity
// on top.  Bound by memory: each activation is read once, each code and scale written once (16384 tokens of 8 heads of
// 128 into int8: 22.9 us, 4.5 TB/s; 8 values a lane and one row a group: 34 us).  A few tokens: 3.2 us, latency.
template <int XT, int CT>
__global__ __launch_bounds__(KV_THREADS) void k_kv_write(KvParams P) {
  constexpr int EL = kv_lane<CT>(), V = EL / 8;
  const KvSide& S = P.side[blockIdx.y];
  const int l = threadIdx.x & (P.G - 1);
  const bool in = l * EL < P.dim;
  KvRow row[KV_ROWS];
  uint4 x[KV_ROWS][V];
#pragma unroll
  for (int u = 0; u < KV_ROWS; ++u) {
    row[u] = kv_row(P, u);
    const uint16_t* from = reinterpret_cast<const uint16_t*>(S.x) + row[u].token * S.row_stride + row[u].head * S.x_head + l * EL;
#pragma unroll
    for (int i = 0; i < V; ++i)
      x[u][i] = in && row[u].live ? reinterpret_cast<const uint4*>(from)[i] : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int u = 0; u < KV_ROWS; ++u) {
    const int64_t at = row[u].slot * S.slot_stride + row[u].head * S.head_stride + l * EL;
    if constexpr (CT == XT) {
      if (in && row[u].slot >= 0) *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(S.base) + at) = x[u][0];
    } else {
      uint32_t w[EL / 2];
#pragma unroll
      for (int i = 0; i < V; ++i)
        w[4 * i] = x[u][i].x, w[4 * i + 1] = x[u][i].y, w[4 * i + 2] = x[u][i].z, w[4 * i + 3] = x[u][i].w;
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < EL / 2; ++i) {
        const uint32_t lo = w[i] & 0x7fffu, hi = (w[i] >> 16) & 0x7fffu;
        top = lo > top ? lo : top;
        top = hi > top ? hi : top;
      }
      for (int o = P.G / 2; o; o /= 2) {
        const uint32_t t = (uint32_t)__shfl_xor((int)top, o, WAVE);
        top = t > top ? t : top;
      }
      const float most = CT == DSV_E4M3 ? 448.f : 127.f;
      const float a = act_to_f32<XT>(top);
      const bool finite = top < (XT == DSV_BF16 ? 0x7f80u : 0x7c00u);
      const bool live = finite && a >= KV_TINY;
      const float inverse = live ? (1.f / a) * most : 0.f;
      const float scale = live ? a * (1.f / most) : (finite ? 0.f : __uint_as_float(0x7fc00000u));
      if (in && row[u].slot >= 0) {
        uint32_t code[EL / 4];
#pragma unroll
        for (int i = 0; i < EL / 4; ++i) {
          float f[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float y = act_to_f32<XT>((w[2 * i + k / 2] >> (16 * (k & 1))) & 0xffffu);
            f[k] = live ? y * inverse : 0.f;
          }
          code[i] = CT == DSV_E4M3 ? pack_e4m3(f[0], f[1], f[2], f[3]) : pack_i8(f[0], f[1], f[2], f[3]);
        }
        *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(S.base) + at) = make_uint4(code[0], code[1], code[2], code[3]);
        if (l == 0) S.scale[row[u].slot * S.scale_slot + row[u].head * S.scale_head] = scale;
      }
    }
  }
}

// The values of the slots' rows, code * scale in float32, rounded once to the output's type.  Bound by memory (50000
// slots of 8 heads of 128, int8 to bf16: 69 us, 4.5 TB/s; 8 values a lane and one row a group: 109 us).
template <int CT, int XT>
__global__ __launch_bounds__(KV_THREADS) void k_kv_read(KvParams P) {
  constexpr bool QUANT = CT == DSV_E4M3 || CT == DSV_I8;
  constexpr int EL = kv_lane<CT>();
  const KvSide& S = P.side[blockIdx.y];
  const int l = threadIdx.x & (P.G - 1);
  if (l * EL >= P.dim) return;
  KvRow row[KV_ROWS];
  uint4 x[KV_ROWS];
  float scale[KV_ROWS];
#pragma unroll
  for (int u = 0; u < KV_ROWS; ++u) row[u] = kv_row(P, u);
#pragma unroll
  for (int u = 0; u < KV_ROWS; ++u) {
    const bool has = row[u].slot >= 0;
    const int64_t slot = has ? row[u].slot : 0;
    const int64_t at = slot * S.slot_stride + row[u].head * S.head_stride + l * EL;
    if constexpr (QUANT) {
      scale[u] = S.scale[slot * S.scale_slot + row[u].head * S.scale_head];
      x[u] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(S.base) + at);
    } else {
      x[u] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(S.base) + at);
    }
  }
#pragma unroll
  for (int u = 0; u < KV_ROWS; ++u) {
    if (!row[u].live) continue;
    const uint32_t w[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
    float f[EL];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (QUANT) {
        unpack_codes<CT>(w[i], f + 4 * i);
#pragma unroll
        for (int k = 0; k < 4; ++k) f[4 * i + k] *= scale[u];
      } else {
        f[2 * i] = act_to_f32<CT>(w[i] & 0xffffu);
        f[2 * i + 1] = act_to_f32<CT>(w[i] >> 16);
      }
    }
    if (row[u].slot < 0)
#pragma unroll
      for (int i = 0; i < EL; ++i) f[i] = 0.f;
    const int64_t o = row[u].token * S.row_stride + row[u].head * S.x_head + l * EL;
    if constexpr (XT == DSV_F32) {
      float4* out = reinterpret_cast<float4*>(reinterpret_cast<float*>(S.x) + o);
#pragma unroll
      for (int i = 0; i < EL / 4; ++i) out[i] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
    } else {
      uint4* out = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(S.x) + o);
#pragma unroll
      for (int i = 0; i < EL / 8; ++i)
        out[i] = make_uint4(pack_act<XT>(f[8 * i], f[8 * i + 1]), pack_act<XT>(f[8 * i + 2], f[8 * i + 3]),
                            pack_act<XT>(f[8 * i + 4], f[8 * i + 5]), pack_act<XT>(f[8 * i + 6], f[8 * i + 7]));
    }
  }
}

// The launch's parameters; false (with the error set) where the call is too large.
static int kv_params(const char* what, const dsv_kv_cache& c, int64_t n, void* k, void* v, const int64_t (&x_strides)[4],
                     const void* slots, int32_t slots_i64, KvParams& P, dim3& grid) {
  P.side[0] = KvSide{c.k, c.k_scale, k, c.k_slot_stride, c.k_head_stride, c.ks_slot_stride, c.ks_head_stride,
                     x_strides[0], x_strides[1]};
  P.side[1] = KvSide{c.v, c.v_scale, v, c.v_slot_stride, c.v_head_stride, c.vs_slot_stride, c.vs_head_stride,
                     x_strides[2], x_strides[3]};
  P.slots = slots;
  P.slots_i64 = slots_i64;
  P.dim = c.dim;
  P.num_slots = c.num_slots;
  const int lane = c.dtype == DSV_E4M3 || c.dtype == DSV_I8 ? 16 : 8;
  P.G = 1;  // lanes of a row: a power of two
  while (P.G * lane < c.dim) P.G *= 2;
  const int64_t rows = n * c.heads, per = (int64_t)KV_THREADS / P.G * KV_ROWS;
  if (n > 0x7fffffffll || rows > 0x7fffffffll - per)
    DSV_FAIL(DSV_ERR_INVALID, "%s: %lld tokens of %d heads are too many for one call", what, (long long)n, c.heads);
  P.rows = (uint32_t)rows;
  P.heads = fast_div((uint32_t)c.heads);
  grid = dim3((unsigned)((rows + per - 1) / per), 2);
  return DSV_OK;
}

}  // namespace dsv

using namespace dsv;

int dsv::check_cache(const char* what, const dsv_kv_cache* c) {
  if (!c || !c->k || !c->v) DSV_FAIL(DSV_ERR_INVALID, "%s: the cache's k and v are required", what);
  if (c->dtype != DSV_BF16 && c->dtype != DSV_F16 && c->dtype != DSV_E4M3 && c->dtype != DSV_I8)
    DSV_FAIL(DSV_ERR_INVALID, "%s: unknown cache type %d", what, c->dtype);
  if (c->heads < 1 || c->heads > 65535 || c->num_slots < 1 || c->dim < 16 || c->dim > 256 || c->dim % 16)
    DSV_FAIL(DSV_ERR_INVALID, "%s: a cache needs slots, heads and a dim that is a multiple of 16 up to 256 (got %lld, %d, %d)",
             what, (long long)c->num_slots, c->heads, c->dim);
  const bool quant = c->dtype == DSV_E4M3 || c->dtype == DSV_I8;
  if (quant != (c->k_scale != nullptr) || quant != (c->v_scale != nullptr))
    DSV_FAIL(DSV_ERR_INVALID, "%s: scales belong to quantised caches, both of them", what);
  const int64_t esize = quant ? 1 : 2;
  const int64_t strides[4] = {c->k_slot_stride, c->k_head_stride, c->v_slot_stride, c->v_head_stride};
  for (int i = 0; i < 4; ++i)
    if (strides[i] < 0 || strides[i] * esize % 16)
      DSV_FAIL(DSV_ERR_INVALID, "%s: cache rows must start on 16-byte boundaries", what);
  if ((uintptr_t)c->k % 16 || (uintptr_t)c->v % 16)
    DSV_FAIL(DSV_ERR_INVALID, "%s: cache rows must start on 16-byte boundaries", what);
  return DSV_OK;
}

extern "C" int dsv_kv_write(const dsv_kv_cache* cache, const void* k, const void* v, int32_t dtype, int64_t n,
                            int64_t k_row_stride, int64_t k_head_stride, int64_t v_row_stride, int64_t v_head_stride,
                            const void* slots, int32_t slots_i64, dsv_stream_t stream_) {
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  const int rc = check_cache("dsv_kv_write", cache);
  if (rc != DSV_OK) return rc;
  if (dtype != DSV_BF16 && dtype != DSV_F16) DSV_FAIL(DSV_ERR_INVALID, "dsv_kv_write: unknown activation type %d", dtype);
  if ((cache->dtype == DSV_BF16 || cache->dtype == DSV_F16) && cache->dtype != dtype)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_kv_write: an unquantised cache holds its own type only");
  if (n < 0) DSV_FAIL(DSV_ERR_INVALID, "dsv_kv_write: n %lld", (long long)n);
  if (n == 0) return DSV_OK;
  if (!k || !v || !slots) DSV_FAIL(DSV_ERR_INVALID, "dsv_kv_write: null pointer");
  if ((uintptr_t)k % 16 || (uintptr_t)v % 16 || k_row_stride % 8 || k_head_stride % 8 || v_row_stride % 8 ||
      v_head_stride % 8)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_kv_write: rows of k and v must start on 16-byte boundaries");
  KvParams P;
  dim3 grid;
  const int bad = kv_params("dsv_kv_write", *cache, n, const_cast<void*>(k), const_cast<void*>(v),
                            {k_row_stride, k_head_stride, v_row_stride, v_head_stride}, slots, slots_i64, P, grid);
  if (bad != DSV_OK) return bad;
  const bool bf = dtype == DSV_BF16;
  auto launch = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(KV_THREADS), 0, stream, P); };
  if (cache->dtype == DSV_E4M3)
    bf ? launch(k_kv_write<DSV_BF16, DSV_E4M3>) : launch(k_kv_write<DSV_F16, DSV_E4M3>);
  else if (cache->dtype == DSV_I8)
    bf ? launch(k_kv_write<DSV_BF16, DSV_I8>) : launch(k_kv_write<DSV_F16, DSV_I8>);
  else
    launch(k_kv_write<DSV_BF16, DSV_BF16>);  // (a copy of 16-bit values, whichever type)
  DSV_CHECK_LAUNCH("k_kv_write");
  return DSV_OK;
}

extern "C" int dsv_kv_read(const dsv_kv_cache* cache, void* k, void* v, int32_t dtype, int64_t n, const void* slots,
                           int32_t slots_i64, dsv_stream_t stream_) {
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  const int rc = check_cache("dsv_kv_read", cache);
  if (rc != DSV_OK) return rc;
  if (dtype != DSV_F32 && dtype != DSV_BF16 && dtype != DSV_F16)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_kv_read: unknown output type %d", dtype);
  if (n < 0) DSV_FAIL(DSV_ERR_INVALID, "dsv_kv_read: n %lld", (long long)n);
  if (n == 0) return DSV_OK;
  if (!k || !v || !slots || (uintptr_t)k % 16 || (uintptr_t)v % 16)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_kv_read: slots and 16-byte-aligned k and v are required");
  KvParams P;
  dim3 grid;
  const int64_t token = (int64_t)cache->heads * cache->dim;
  const int bad = kv_params("dsv_kv_read", *cache, n, k, v, {token, cache->dim, token, cache->dim}, slots, slots_i64, P, grid);
  if (bad != DSV_OK) return bad;
  auto launch = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(KV_THREADS), 0, stream, P); };
  auto to = [&](auto ct) {
    constexpr int CT = decltype(ct)::value;
    if (dtype == DSV_F32)
      launch(k_kv_read<CT, DSV_F32>);
    else if (dtype == DSV_BF16)
      launch(k_kv_read<CT, DSV_BF16>);
    else
      launch(k_kv_read<CT, DSV_F16>);
  };
  if (cache->dtype == DSV_BF16)
    to(Int<DSV_BF16>{});
  else if (cache->dtype == DSV_F16)
    to(Int<DSV_F16>{});
  else if (cache->dtype == DSV_E4M3)
    to(Int<DSV_E4M3>{});
  else
    to(Int<DSV_I8>{});
  DSV_CHECK_LAUNCH("k_kv_read");
  return DSV_OK;
}
