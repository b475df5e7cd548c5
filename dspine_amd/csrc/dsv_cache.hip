// The KV cache's write and read for gfx950: new keys and values into cache slots (quantised to 8 bits
// with a scale for each (token, head) where the cache is), and slots gathered back to activations.
#include "dsv_cache.h"
#include "dsv_common.h"

namespace dsv {

// A row (one token's, one head's keys or values) is held by a group of G lanes, 8 values a lane: the row's
// largest magnitude is then a reduction inside the group, and every access is 16 bytes (codes: 8).
constexpr int KV_THREADS = 256;

struct KvParams {
  dsv_kv_cache c;
  void* x[2];  // keys, values: read by the write, written by the read
  int64_t row_stride[2], head_stride[2];
  const void* slots;
  int32_t slots_i64;
  int64_t n;
};

// The row of this lane group: its token, whether it is a key's or a value's, its head.  Heads run fastest, so
// that neighbouring groups touch neighbouring memory on both sides.
__device__ __forceinline__ bool kv_row(const KvParams& P, int G, int64_t& token, int& which, int& head, int64_t& slot) {
  const int64_t r = (int64_t)blockIdx.x * (KV_THREADS / G) + threadIdx.x / G;
  const int per = 2 * P.c.heads;
  token = r / per;
  const int in = (int)(r - token * per);
  which = in >= P.c.heads;
  head = in - (which ? P.c.heads : 0);
  if (token >= P.n) return false;
  slot = load_index(P.slots, P.slots_i64, token);
  return true;
}

// Codes of a quantised row: a = the row's largest magnitude, scale = a * (1 / top), code = rne(x * ((1 / a) * top)).
// The magnitudes are compared as the type's own 15 bits, which order like the values and keep a NaN or an infinity
// on top.  Bound by memory: each activation is read once, each code and scale written once.
template <int XT, int CT>
__global__ __launch_bounds__(KV_THREADS) void k_kv_write(KvParams P, int G) {
  int64_t token, slot;
  int which, head;
  if (!kv_row(P, G, token, which, head, slot)) return;
  if (slot < 0 || slot >= P.c.num_slots) return;
  const int l = threadIdx.x & (G - 1);
  const bool in = l * 8 < P.c.dim;
  const uint16_t* x = reinterpret_cast<const uint16_t*>(P.x[which]) + token * P.row_stride[which] +
                      head * P.head_stride[which] + l * 8;
  uint4 v = make_uint4(0, 0, 0, 0);
  if (in) v = *reinterpret_cast<const uint4*>(x);
  const int64_t at = slot * (which ? P.c.v_slot_stride : P.c.k_slot_stride) +
                     head * (which ? P.c.v_head_stride : P.c.k_head_stride) + l * 8;
  void* base = which ? P.c.v : P.c.k;
  if constexpr (CT == XT) {
    if (in) *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(base) + at) = v;
  } else {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = w[i] & 0x7fffu, hi = (w[i] >> 16) & 0x7fffu;
      top = lo > top ? lo : top;
      top = hi > top ? hi : top;
    }
    for (int o = G / 2; o; o /= 2) {
      const uint32_t t = (uint32_t)__shfl_xor((int)top, o, WAVE);
      top = t > top ? t : top;
    }
    const float most = CT == DSV_E4M3 ? 448.f : 127.f;
    const float a = act_to_f32<XT>(top);
    const bool finite = top < (XT == DSV_BF16 ? 0x7f80u : 0x7c00u);
    const bool live = finite && a >= KV_TINY;
    const float inverse = live ? (1.f / a) * most : 0.f;
    const float scale = live ? a * (1.f / most) : (finite ? 0.f : __uint_as_float(0x7fc00000u));
    if (in) {
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = act_to_f32<XT>((w[i / 2] >> (16 * (i & 1))) & 0xffffu);
        f[i] = live ? y * inverse : 0.f;
      }
      uint2 code;
      if constexpr (CT == DSV_E4M3) {
        code.x = pack_e4m3(f[0], f[1], f[2], f[3]);
        code.y = pack_e4m3(f[4], f[5], f[6], f[7]);
      } else {
        code.x = pack_i8(f[0], f[1], f[2], f[3]);
        code.y = pack_i8(f[4], f[5], f[6], f[7]);
      }
      *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(base) + at) = code;
    }
    if (l == 0) {
      float* s = which ? P.c.v_scale : P.c.k_scale;
      s[slot * (which ? P.c.vs_slot_stride : P.c.ks_slot_stride) + head * (which ? P.c.vs_head_stride : P.c.ks_head_stride)] =
          scale;
    }
  }
}

// The values of the slots' rows, code * scale in float32, rounded once to the output's type.
template <int CT, int XT>
__global__ __launch_bounds__(KV_THREADS) void k_kv_read(KvParams P, int G) {
  int64_t token, slot;
  int which, head;
  if (!kv_row(P, G, token, which, head, slot)) return;
  const int l = threadIdx.x & (G - 1);
  if (l * 8 >= P.c.dim) return;
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = 0.f;
  if (slot >= 0 && slot < P.c.num_slots) {
    const int64_t at = slot * (which ? P.c.v_slot_stride : P.c.k_slot_stride) +
                       head * (which ? P.c.v_head_stride : P.c.k_head_stride) + l * 8;
    const void* base = which ? P.c.v : P.c.k;
    if constexpr (CT == DSV_E4M3 || CT == DSV_I8) {
      const float* s = which ? P.c.v_scale : P.c.k_scale;
      const float scale = s[slot * (which ? P.c.vs_slot_stride : P.c.ks_slot_stride) +
                            head * (which ? P.c.vs_head_stride : P.c.ks_head_stride)];
      const uint2 code = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(base) + at);
      unpack_codes<CT>(code.x, f);
      unpack_codes<CT>(code.y, f + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] *= scale;
    } else {
      const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(base) + at);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = act_to_f32<CT>((w[i / 2] >> (16 * (i & 1))) & 0xffffu);
    }
  }
  const int64_t o = (token * P.c.heads + head) * P.c.dim + l * 8;
  if constexpr (XT == DSV_F32) {
    float* out = reinterpret_cast<float*>(P.x[which]) + o;
    *reinterpret_cast<float4*>(out) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(out + 4) = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    uint4 v;
    v.x = pack_act<XT>(f[0], f[1]);
    v.y = pack_act<XT>(f[2], f[3]);
    v.z = pack_act<XT>(f[4], f[5]);
    v.w = pack_act<XT>(f[6], f[7]);
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(P.x[which]) + o) = v;
  }
}

// lanes of a row: 8 values each, a power of two
static int lanes_of(int dim) {
  int g = 8;
  while (g * 8 < dim) g *= 2;
  return g;
}

static int kv_blocks(const char* what, const dsv_kv_cache& c, int64_t n, int G, unsigned* blocks) {
  const int64_t per = KV_THREADS / G;
  if (n > (((int64_t)1 << 31) - 1) * per / (2 * (int64_t)c.heads))
    DSV_FAIL(DSV_ERR_INVALID, "%s: %lld tokens of %d heads are too many for one call", what, (long long)n, c.heads);
  *blocks = (unsigned)((n * 2 * c.heads + per - 1) / per);
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
  P.c = *cache;
  P.x[0] = const_cast<void*>(k);
  P.x[1] = const_cast<void*>(v);
  P.row_stride[0] = k_row_stride;
  P.row_stride[1] = v_row_stride;
  P.head_stride[0] = k_head_stride;
  P.head_stride[1] = v_head_stride;
  P.slots = slots;
  P.slots_i64 = slots_i64;
  P.n = n;
  const int G = lanes_of(cache->dim);
  unsigned blocks;
  const int bad = kv_blocks("dsv_kv_write", *cache, n, G, &blocks);
  if (bad != DSV_OK) return bad;
  const bool bf = dtype == DSV_BF16;
  auto launch = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(blocks), dim3(KV_THREADS), 0, stream, P, G); };
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
  P.c = *cache;
  P.x[0] = k;
  P.x[1] = v;
  P.row_stride[0] = P.row_stride[1] = (int64_t)cache->heads * cache->dim;
  P.head_stride[0] = P.head_stride[1] = cache->dim;
  P.slots = slots;
  P.slots_i64 = slots_i64;
  P.n = n;
  const int G = lanes_of(cache->dim);
  unsigned blocks;
  const int bad = kv_blocks("dsv_kv_read", *cache, n, G, &blocks);
  if (bad != DSV_OK) return bad;
  auto launch = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(blocks), dim3(KV_THREADS), 0, stream, P, G); };
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
