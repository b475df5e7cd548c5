// Attention of drafted nodes over a request's cached positions for gfx950.
//
// For request b, cache head h and the query rows r = (node, query head of h's group), with s = scale * q.k:
// out = sum_p e^(s_p - m) v_p / sum_p e^(s_p - m), in one pass over the positions with a reference m of the softmax
// that moves up where a score exceeds it by more than a few powers of two (the weights are then at most 2^LIM, and the
// partial sums are rescaled; most steps only compare).
//
// The matrix cores take keys as they lie in memory: S^T = K Q^T with the positions on the rows of the tile, so that a
// lane holds, for one query row, the weights of the four (twice: eight) positions that the second product
// O^T = V^T P^T wants from it: no weight moves between lanes.  Keys go from memory to the operand registers; values
// too, as 16-byte pieces of whole rows whose 16-bit elements a v_perm each puts in the positions' order.  Nothing is
// staged in LDS, the waves run free of each other, and each holds all its rows' sums in registers.
//
// The positions of a batch are cut into about `target` equal pieces (a rule on the lengths, which only the device
// knows: every workgroup computes the same plan from them); pieces of a request are joined by k_attn_join.
#include "dsv_cache.h"
#include "dsv_common.h"

namespace dsv {

constexpr int AT_THREADS = 256;
constexpr int AT_WAVES = AT_THREADS / WAVE;
constexpr int AT_NODES = 64;
constexpr int AT_TILE = 32;  // positions of a step
constexpr float AT_LOW = -3e38f;

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef __bf16 bhalf8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct AttnParams {
  dsv_tree_attention_args a;
  int G, WR, RB;       // query heads a cache head; waves over the rows, row blocks of a request
  int target;          // pieces aimed at
  int least;           // tiles of a piece at least
  int joined;          // whether a request may have several pieces
  uint32_t num_slots, k_step, v_step;  // slots; bytes from slot to slot
  float* part_o;       // [item][head][row][dim]
  float2* part_ml;     // [item][head][row]: reference, sum
};

// The request's nodes, its context and its positions (context and window) that the page table has.
struct Request {
  int nodes;
  int prefix, total;  // within the table
};
__device__ __forceinline__ Request request_of(const dsv_tree_attention_args& a, int64_t b) {
  Request r;
  int n = a.verify_lens ? a.verify_lens[b] : a.T;
  r.nodes = n < 0 ? 0 : (n > a.T ? a.T : n);
  const int pre = a.prefix_lens[b];
  const int64_t from = pre < 0 ? 0 : pre, to = from + r.nodes;
  r.prefix = (int)(from < a.page_cols ? from : a.page_cols);
  r.total = (int)(to < a.page_cols ? to : a.page_cols);
  return r;
}
__device__ __forceinline__ int tiles_of(const Request& r) {
  const int t = (r.total + AT_TILE - 1) / AT_TILE;
  return r.nodes == 0 ? 0 : (t < 1 ? 1 : t);
}

// The plan, computed by every wave from the batch's lengths: tiles of a piece.
__device__ __forceinline__ int plan_chunk(const AttnParams& P, int lane) {
  int64_t sum = 0;
  for (int b = lane; b < P.a.bs; b += WAVE) sum += tiles_of(request_of(P.a, b));
  sum = wave_sum(sum);
  const int64_t c = (sum + P.target - 1) / P.target;
  return (int)(c < P.least ? P.least : c);
}
__device__ __forceinline__ int pieces_of(int tiles, int chunk) { return (tiles + chunk - 1) / chunk; }

// Pieces of the requests before b.
__device__ __forceinline__ int items_before(const AttnParams& P, int chunk, int b, int lane) {
  int sum = 0;
  for (int i = lane; i < b; i += WAVE) sum += pieces_of(tiles_of(request_of(P.a, i)), chunk);
  return wave_sum(sum);
}
// The request and the piece of a work item; false past the last.
__device__ __forceinline__ bool item_at(const AttnParams& P, int chunk, int item, int lane, int& b, int& piece) {
  int before = 0;
  for (int b0 = 0; b0 < P.a.bs; b0 += WAVE) {
    const int i = b0 + lane;
    const int n = i < P.a.bs ? pieces_of(tiles_of(request_of(P.a, i)), chunk) : 0;
    const int end = before + wave_incl_scan(n);
    const uint64_t past = __ballot(end > item);
    if (past) {
      const int l = __ffsll((unsigned long long)past) - 1;
      b = b0 + l;
      piece = item - (readlane_at(end, l) - readlane_at(n, l));
      return true;
    }
    before = readlane<WAVE - 1>(end);
  }
  return false;
}

template <int XT>
__device__ __forceinline__ f32x4 mfma(const uint32_t (&x)[4], const uint32_t (&y)[4], f32x4 c) {
  const uint4 a = make_uint4(x[0], x[1], x[2], x[3]), b = make_uint4(y[0], y[1], y[2], y[3]);
  if constexpr (XT == DSV_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bhalf8, a), __builtin_bit_cast(bhalf8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// N 32-bit words from memory (16-byte loads where there are that many).
template <int N>
__device__ __forceinline__ void load_words(const void* p, uint32_t (&w)[N]) {
  if constexpr (N >= 4) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[i];
      w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
    }
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// int8 codes as float16: a byte of code + 128 is the float16 (code + 128) * 2^-24; times 2^15 less 1/4 that is
// code / 512, exact.  (Two instructions for two codes.)
constexpr float I8_UNIT = 512.f;
__device__ __forceinline__ uint32_t i8_pair(uint32_t bytes) {
  const half2v up = {(_Float16)32768.f, (_Float16)32768.f}, off = {(_Float16)-0.25f, (_Float16)-0.25f};
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(half2v, bytes), up, off));
}
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t w, bool hi, bool bf) {
  if (bf)
    return __builtin_bit_cast(uint32_t, hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true)
                                           : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false));
  return __builtin_bit_cast(uint32_t, hi ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true)
                                         : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
}

// Eight keys' elements of the products' type (8-bit codes: two words) -- exact in either type.
template <int XT, int CT>
__device__ __forceinline__ void key_operand(const uint32_t* w, uint32_t (&o)[4]) {
  if constexpr (CT == DSV_E4M3) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = e4m3_pair(w[i / 2], i & 1, XT == DSV_BF16);
  } else if constexpr (CT == DSV_I8 && XT == DSV_F16) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      o[i] = i8_pair(__builtin_amdgcn_perm(0u, w[i / 2] ^ 0x80808080u, i & 1 ? 0x0c030c02u : 0x0c010c00u));
  } else if constexpr (CT == DSV_I8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t x = w[i / 2] >> (16 * (i & 1));
      const float lo = (float)(int8_t)x, hi = (float)(int8_t)(x >> 8);
      o[i] = __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = w[i];
  }
}

// Element e of eight positions' value words (wv[j]: position j's elements) in the positions' order.
template <int CT, int W>
__device__ __forceinline__ void value_operand(const uint32_t (&wv)[8][W], int e, uint32_t (&o)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (CT == DSV_I8) {
      const uint32_t sel = 0x0c040c00u + (uint32_t)(e & 3) * 0x00010001u;
      o[i] = i8_pair(__builtin_amdgcn_perm(wv[2 * i + 1][e / 4], wv[2 * i][e / 4], sel));
    } else if constexpr (CT == DSV_E4M3) {
      const uint32_t lo = e4m3_pair(wv[2 * i][e / 4], (e & 2) != 0, false);
      const uint32_t hi = e4m3_pair(wv[2 * i + 1][e / 4], (e & 2) != 0, false);
      o[i] = __builtin_amdgcn_perm(hi, lo, e & 1 ? 0x07060302u : 0x05040100u);
    } else {
      o[i] = __builtin_amdgcn_perm(wv[2 * i + 1][e / 2], wv[2 * i][e / 2], e & 1 ? 0x07060302u : 0x05040100u);
    }
  }
}

__device__ __forceinline__ float across_groups_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, WAVE));
  return fmaxf(v, __shfl_xor(v, 32, WAVE));
}
__device__ __forceinline__ float across_groups_sum(float v) {
  v += __shfl_xor(v, 16, WAVE);
  return v + __shfl_xor(v, 32, WAVE);
}

// The row of q of a request's node, or -1 where it lies outside.
__device__ __forceinline__ int64_t row_of(const dsv_tree_attention_args& a, int64_t b, int node) {
  const int64_t r = (a.row_offsets ? load_index(a.row_offsets, a.row_offsets_i64, b) : b * a.T) + node;
  return r >= 0 && r < a.rows ? r : -1;
}
__device__ __forceinline__ uint64_t mask_of(const dsv_tree_attention_args& a, int64_t b, int node) {
  if (a.masks) return (uint64_t)a.masks[b * a.T + node];
  return node >= 63 ? ~0ull : (2ull << node) - 1ull;
}

template <int XT, int CT, int DP, int R, int OCC>
__global__ __launch_bounds__(AT_THREADS, OCC) void k_attn(AttnParams P) {
  const dsv_tree_attention_args& a = P.a;
  const dsv_kv_cache& c = a.cache;
  constexpr bool QUANT = CT == DSV_E4M3 || CT == DSV_I8;
  constexpr int PT = CT == DSV_BF16 ? DSV_BF16 : DSV_F16;  // the weights' type
  // float16 weights are held 2^11 higher, so that what their range loses lies below 2^-35 of the row's largest
  constexpr float SHIFT = PT == DSV_F16 ? 11.f : 0.f, LIM = PT == DSV_F16 ? 4.f : 8.f;
  constexpr int ESZ = QUANT ? 1 : 2;
  constexpr int EPL = DP / 16;            // value elements a lane loads of a position
  constexpr int VW = EPL * ESZ / 4;       // words of them
  constexpr int NK = DP / 32;             // key products of a tile
  constexpr int KL = DP * ESZ / 64;       // 16-byte key loads a lane of a position
  constexpr int OS = DP + 4;              // row stride of the sums in LDS
  __shared__ float s_o[AT_WAVES][16][OS];
  __shared__ float s_m[AT_WAVES][16 * R], s_l[AT_WAVES][16 * R];

  const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
  const int m = lane & 15, g = lane >> 4;
  // Items round the XCDs, a request's heads and row blocks on one: they share its page table rows, scales and keys in
  // that XCD's L2.
  const int HB = c.heads * P.RB;
  const int inner = (int)((blockIdx.x / 8) % HB), item = (int)((blockIdx.x / 8) / HB) * 8 + (int)(blockIdx.x % 8);
  const int h = inner / P.RB, rb = inner - h * P.RB;
  const int chunk = plan_chunk(P, lane);
  int b, piece;
  if (!item_at(P, chunk, item, lane, b, piece)) return;
  b = __builtin_amdgcn_readfirstlane(b);
  piece = __builtin_amdgcn_readfirstlane(piece);
  const Request req = request_of(a, b);
  const int n_rows = req.nodes * P.G, tiles = tiles_of(req), pieces = pieces_of(tiles, chunk);
  const int WR = P.WR, WK = AT_WAVES / WR, wr = wave / WK, wk = wave - wr * WK;
  const int block0 = rb * 16 * R * WR;
  if (block0 >= n_rows) return;
  const int row0 = block0 + wr * 16 * R;

  // queries, in the order of the keys' elements
  uint32_t qf[R][NK][4];
#pragma unroll
  for (int rt = 0; rt < R; ++rt) {
    const int r = row0 + rt * 16 + m;
    const int64_t row = r < n_rows ? row_of(a, b, r / P.G) : -1;
    const uint16_t* q = reinterpret_cast<const uint16_t*>(a.q) + (row < 0 ? 0 : row) * a.q_row_stride +
                        (int64_t)(h * P.G + r % P.G) * a.q_head_stride;
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) {
      const int d = QUANT ? (kk / 2) * 64 + g * 16 + (kk & 1) * 8 : kk * 32 + g * 8;
      uint32_t w[4] = {0, 0, 0, 0};
      if (row >= 0 && d < c.dim) load_words<4>(q + d, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) qf[rt][kk][i] = w[i];
    }
  }

  const int32_t* table = a.page_table + (int64_t)b * a.page_stride;
  const uint8_t* kbase = reinterpret_cast<const uint8_t*>(c.k) + (int64_t)h * c.k_head_stride * ESZ + g * 16;
  const bool v_in = m * EPL < c.dim;  // (else the lane repeats the row's first piece: its sums are not stored)
  const uint8_t* vbase = reinterpret_cast<const uint8_t*>(c.v) + (int64_t)h * c.v_head_stride * ESZ + (v_in ? m * EPL * ESZ : 0);
  const float* ksc = QUANT ? c.k_scale + (int64_t)h * c.ks_head_stride : nullptr;
  const float* vsc = QUANT ? c.v_scale + (int64_t)h * c.vs_head_stride : nullptr;
  const float c0 = a.scale * 1.44269504088896340736f * (CT == DSV_I8 && XT == DSV_F16 ? I8_UNIT : 1.f);
  const int clear = req.prefix;  // positions before it are seen by every row

  f32x4 o[R][EPL];
  float mref[R], l[R];
  float vref = 0.f, vinv = 0.f;
#pragma unroll
  for (int rt = 0; rt < R; ++rt) {
    mref[rt] = AT_LOW;
    l[rt] = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) o[rt][e] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const int t0 = (int)((int64_t)tiles * piece / pieces), t1 = (int)((int64_t)tiles * (piece + 1) / pieces);
  const int last = req.total - 1;
  // a tile's slots: of the key rows m and 16 + m, and of this lane's eight positions g * 4 + j, 16 + g * 4 + j
  auto load_slots = [&](int t, uint32_t (&ks)[2], uint32_t (&vs)[8]) {
    const int base = t * AT_TILE;
    if (base + AT_TILE <= req.total) {
#pragma unroll
      for (int i = 0; i < 2; ++i) ks[i] = (uint32_t)table[base + i * 16 + m];
#pragma unroll
      for (int j = 0; j < 8; ++j) vs[j] = (uint32_t)table[base + (j / 4) * 16 + g * 4 + (j & 3)];
    } else {
      auto at = [&](int p) { return p <= last ? (uint32_t)table[p] : ~0u; };
#pragma unroll
      for (int i = 0; i < 2; ++i) ks[i] = at(base + i * 16 + m);
#pragma unroll
      for (int j = 0; j < 8; ++j) vs[j] = at(base + (j / 4) * 16 + g * 4 + (j & 3));
    }
  };
  auto load_keys = [&](const uint32_t (&ks)[2], uint32_t (&kw)[2][KL][4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t s = ks[i] < P.num_slots ? ks[i] : 0u;
      const uint8_t* p = kbase + (uint64_t)s * P.k_step;
#pragma unroll
      for (int u = 0; u < KL; ++u)
        if (u * 64 < c.dim * ESZ) {
          // (past the row's end: its first piece, replaced by zeros before it is used)
          load_words<4>(p + (u * 64 + g * 16 < c.dim * ESZ ? u * 64 : -(g * 16)), kw[i][u]);
        }
    }
  };
  auto load_scales = [&](const uint32_t (&vs)[8], float (&kf)[8], float (&vf)[8]) {
    if constexpr (QUANT) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t s = vs[j] < P.num_slots ? vs[j] : 0u;
        kf[j] = ksc[(int64_t)s * c.ks_slot_stride];
        vf[j] = vsc[(int64_t)s * c.vs_slot_stride];
      }
    }
  };

  uint32_t ks0[2], vs0[8], ks1[2], vs1[8];
  uint32_t kw[2][KL][4];
  float kf[8], vf[8];
  int t = t0 + wk;
  if (row0 >= n_rows) t = t1;
  if (t < t1) {
    load_slots(t, ks0, vs0);
    load_keys(ks0, kw);
    load_scales(vs0, kf, vf);
    if (t + WK < t1) load_slots(t + WK, ks1, vs1);
  }
  for (; t < t1; t += WK) {
    const int base = t * AT_TILE;
    const bool whole = base + AT_TILE <= clear && !__any(ks0[0] >= P.num_slots || ks0[1] >= P.num_slots);
    uint32_t wv[8][VW];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t s = vs0[j] < P.num_slots ? vs0[j] : 0u;
      load_words<VW>(vbase + (uint64_t)s * P.v_step, wv[j]);
    }
    // scores
    f32x4 s[R][2];
#pragma unroll
    for (int rt = 0; rt < R; ++rt)
#pragma unroll
      for (int i = 0; i < 2; ++i) s[rt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) {
      if (kk * 32 < c.dim || QUANT) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t ko[4];
          if constexpr (QUANT) {
            if ((kk / 2) * 64 < c.dim) {
              key_operand<XT, CT>(&kw[i][kk / 2][(kk & 1) * 2], ko);
              if ((kk / 2) * 64 + 64 > c.dim)
#pragma unroll
                for (int u = 0; u < 4; ++u) ko[u] = (kk / 2) * 64 + g * 16 < c.dim ? ko[u] : 0u;
#pragma unroll
              for (int rt = 0; rt < R; ++rt) s[rt][i] = mfma<XT>(ko, qf[rt][kk], s[rt][i]);
            }
          } else {
            key_operand<XT, CT>(kw[i][kk], ko);
            if (kk * 32 + 32 > c.dim)
#pragma unroll
              for (int u = 0; u < 4; ++u) ko[u] = kk * 32 + g * 8 < c.dim ? ko[u] : 0u;
#pragma unroll
            for (int rt = 0; rt < R; ++rt) s[rt][i] = mfma<XT>(ko, qf[rt][kk], s[rt][i]);
          }
        }
      }
    }
    // the positions' factors: of a score (base 2), of a weight
    float cs[8], vn[8];
    if constexpr (QUANT) {
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        cs[j] = kf[j] * c0;
        const float v = fabsf(vf[j]);
        top = fmaxf(top, v < INFINITY ? v : 0.f);
      }
      if (__any(top > vref)) {
        // value scales are taken relative to a power of two at or above the largest so far
        top = across_groups_max(wave_max_f32(top));
        int ex;
        (void)frexpf(top, &ex);
        ex = ex > 120 ? 120 : (ex < -120 ? -120 : ex);
        const float next = ldexpf(1.f, ex);
        if (next > vref) {
          const float keep = vref / next;
#pragma unroll
          for (int rt = 0; rt < R; ++rt)
#pragma unroll
            for (int e = 0; e < EPL; ++e) o[rt][e] *= keep;
          vref = next;
          vinv = 1.f / next;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) vn[j] = vf[j] * vinv;
    }
    uint32_t seen[R];  // bit j: the row sees this lane's position j
    uint32_t here = 0xffu;
    if (!whole) {
      here = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) here |= (vs0[j] < P.num_slots ? 1u : 0u) << j;
#pragma unroll
      for (int rt = 0; rt < R; ++rt) {
        const int r = row0 + rt * 16 + m;
        const uint64_t mask = r < n_rows ? mask_of(a, b, r / P.G) : 0ull;
        uint32_t bits = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int p = base + (j / 4) * 16 + g * 4 + (j & 3) - req.prefix;
          const bool sees = p < 0 || (p < 64 && ((mask >> (p & 63)) & 1));
          bits |= (sees ? 1u : 0u) << j;
        }
        seen[rt] = bits & here;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!((seen[rt] >> j) & 1)) s[rt][j / 4][j & 3] = -INFINITY;
      }
    }
    // the next tile's keys and scales, and the slots of the one after it
    if (t + WK < t1) {
#pragma unroll
      for (int i = 0; i < 2; ++i) ks0[i] = ks1[i];
#pragma unroll
      for (int j = 0; j < 8; ++j) vs0[j] = vs1[j];
      load_keys(ks0, kw);
      load_scales(vs0, kf, vf);
      if (t + 2 * WK < t1) load_slots(t + 2 * WK, ks1, vs1);
    }
    // weights
    float x[R][8];
    float over = AT_LOW;
#pragma unroll
    for (int rt = 0; rt < R; ++rt) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        // (a masked score stays -inf whatever its position's scale)
        float f = QUANT ? cs[j] : c0;
        if (QUANT && !whole) f = (seen[rt] >> j) & 1 ? f : 1.f;
        if (!QUANT && !whole) f = (seen[rt] >> j) & 1 ? f : 1.f;
        s[rt][j / 4][j & 3] *= f;
        x[rt][j] = s[rt][j / 4][j & 3] - mref[rt];
        over = fmaxf(over, x[rt][j]);
      }
    }
    if (__any(over > SHIFT + LIM)) {
#pragma unroll
      for (int rt = 0; rt < R; ++rt) {
        float top = AT_LOW;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, s[rt][j / 4][j & 3]);
        top = across_groups_max(top);
        const float next = fmaxf(mref[rt], top - SHIFT);
        const float keep = __builtin_amdgcn_exp2f(mref[rt] - next);
        mref[rt] = next;
        l[rt] *= keep;
#pragma unroll
        for (int e = 0; e < EPL; ++e) o[rt][e] *= keep;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[rt][j] = s[rt][j / 4][j & 3] - next;
      }
    }
    uint32_t pf[R][4];
#pragma unroll
    for (int rt = 0; rt < R; ++rt) {
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float p = __builtin_amdgcn_exp2f(x[rt][j]);
        l[rt] += p;
        w[j] = p;
        if constexpr (QUANT) {
          w[j] = p * vn[j];
          if (!whole) w[j] = (seen[rt] >> j) & 1 ? w[j] : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) pf[rt][i] = pack_act<PT>(w[2 * i], w[2 * i + 1]);
    }
    // sums
    if (!whole) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (!((here >> j) & 1))
#pragma unroll
          for (int u = 0; u < VW; ++u) wv[j][u] = 0u;
    }
    if constexpr (CT == DSV_I8)
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int u = 0; u < VW; ++u) wv[j][u] ^= 0x80808080u;
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      uint32_t vo[4];
      value_operand<CT, VW>(wv, e, vo);
      if (CT != DSV_I8 && !whole) {
        // A value that is not finite reaches only the rows that see it: it leaves the product (0 * NaN is NaN), and three
        // products of indicators say which rows get an infinity or a NaN.
        constexpr uint32_t INF = PT == DSV_BF16 ? 0x7f80u : 0x7c00u, ONE = PT == DSV_BF16 ? 0x3f80u : 0x3c00u;
        bool odd = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) odd |= (vo[i] & INF) == INF || ((vo[i] >> 16) & INF) == INF;
        if (__any(odd)) {
          uint32_t kind[3][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            kind[0][i] = kind[1][i] = kind[2][i] = 0u;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const uint32_t v = (vo[i] >> (16 * u)) & 0xffffu;
              if ((v & INF) == INF) {
                kind[(v & 0x7fffu) != INF ? 2 : (v >> 15)][i] |= ONE << (16 * u);
                vo[i] &= u ? 0x0000ffffu : 0xffff0000u;
              }
            }
          }
#pragma unroll
          for (int rt = 0; rt < R; ++rt) {
            uint32_t sf[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              sf[i] = ((seen[rt] >> (2 * i)) & 1 ? ONE : 0u) | ((seen[rt] >> (2 * i + 1)) & 1 ? ONE << 16 : 0u);
            const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
            const f32x4 up = mfma<PT>(kind[0], sf, zero), down = mfma<PT>(kind[1], sf, zero),
                        nan = mfma<PT>(kind[2], sf, zero);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              if (up[r] > 0.f) o[rt][e][r] += INFINITY;
              if (down[r] > 0.f) o[rt][e][r] -= INFINITY;
              if (nan[r] > 0.f) o[rt][e][r] = NAN;
            }
          }
        }
      }
#pragma unroll
      for (int rt = 0; rt < R; ++rt) o[rt][e] = mfma<PT>(vo, pf[rt], o[rt][e]);
    }
  }

  // The waves of the same rows join: their references, then the sums of one row tile after another through LDS.
#pragma unroll
  for (int rt = 0; rt < R; ++rt) {
    l[rt] = across_groups_sum(l[rt]);
    if (g == 0) {
      s_m[wave][rt * 16 + m] = mref[rt];
      s_l[wave][rt * 16 + m] = l[rt];
    }
  }
  __syncthreads();
  const float unit = QUANT ? vref * (CT == DSV_I8 ? I8_UNIT : 1.f) : 1.f;
#pragma unroll
  for (int rt = 0; rt < R; ++rt) {
    float top = AT_LOW;
    for (int k = 0; k < WK; ++k) top = fmaxf(top, s_m[wr * WK + k][rt * 16 + m]);
    const float f = __builtin_amdgcn_exp2f(mref[rt] - top) * unit;
    if (rt) __syncthreads();
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int e = 0; e < EPL; e += 4)
        *reinterpret_cast<float4*>(&s_o[wave][m][(g * 4 + r) * EPL + e]) =
            make_float4(o[rt][e][r] * f, o[rt][e + 1][r] * f, o[rt][e + 2][r] * f, o[rt][e + 3][r] * f);
    __syncthreads();
    for (int i = tid - wr * WK * WAVE; i < 16 * DP / 8; i += WK * WAVE) {
      const int rr = i / (DP / 8), d = i % (DP / 8) * 8, r = row0 + rt * 16 + rr;
      if (r >= n_rows || d >= c.dim) continue;
      float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      float mt = AT_LOW, lt = 0.f;
      for (int k = 0; k < WK; ++k) mt = fmaxf(mt, s_m[wr * WK + k][rt * 16 + rr]);
      for (int k = 0; k < WK; ++k) {
        lt += s_l[wr * WK + k][rt * 16 + rr] * __builtin_amdgcn_exp2f(s_m[wr * WK + k][rt * 16 + rr] - mt);
#pragma unroll
        for (int u = 0; u < 8; ++u) sum[u] += s_o[wr * WK + k][rr][d + u];
      }
      if (pieces > 1) {
        const int64_t at = ((int64_t)item * c.heads + h) * (a.T * P.G) + r;
        float* po = P.part_o + at * c.dim + d;
        *reinterpret_cast<float4*>(po) = make_float4(sum[0], sum[1], sum[2], sum[3]);
        *reinterpret_cast<float4*>(po + 4) = make_float4(sum[4], sum[5], sum[6], sum[7]);
        if (d == 0) P.part_ml[at] = make_float2(mt, lt);
      } else {
        const int node = r / P.G, qh = h * P.G + r - node * P.G;
        const int64_t row = row_of(a, b, node);
        if (row < 0) continue;
        const float inv = lt == 0.f ? 0.f : 1.f / lt;
        uint4 v;
        v.x = pack_act<XT>(sum[0] * inv, sum[1] * inv);
        v.y = pack_act<XT>(sum[2] * inv, sum[3] * inv);
        v.z = pack_act<XT>(sum[4] * inv, sum[5] * inv);
        v.w = pack_act<XT>(sum[6] * inv, sum[7] * inv);
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + row * a.out_row_stride + qh * a.out_head_stride + d) = v;
        if (d == 0 && a.lse) a.lse[row * a.q_heads + qh] = lt == 0.f ? -INFINITY : (mt + log2f(lt)) * 0.693147180559945309f;
      }
    }
  }
}

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
  const int t = (2048 + heads * RB - 1) / (heads * RB);
  return t < 1 ? 1 : t;
}

// Row tiles a wave, waves over the rows and row blocks of T nodes with G query heads each.
struct AttnShape {
  int R, WR, RB;
};
static AttnShape attn_shape(int T, int G, int dim) {
  const int rows = T * G, tiles = (rows + 15) / 16;
  AttnShape s;
  const int most = dim > 128 ? 2 : 4;
  s.R = tiles <= 1 ? 1 : (tiles <= 2 ? 2 : most);
  const int groups = (tiles + s.R - 1) / s.R;
  s.WR = groups >= 3 ? 4 : groups;
  s.RB = (groups + s.WR - 1) / s.WR;
  return s;
}

}  // namespace dsv

using namespace dsv;

extern "C" int64_t dsv_tree_attention_workspace_bytes(int32_t bs, int32_t T, int32_t heads, int32_t q_heads,
                                                      int32_t dim) {
  if (bs < 1 || T < 1 || heads < 1 || q_heads < heads || dim < 1) return 0;
  const AttnShape s = attn_shape(T, q_heads / heads, dim);
  const int64_t rows = ((int64_t)attn_target(heads, s.RB) + bs) * q_heads * T;
  return rows * (dim * (int64_t)sizeof(float) + (int64_t)sizeof(float2));
}

template <int XT, int CT>
static void launch_attn(const AttnParams& P, const AttnShape& s, unsigned blocks, hipStream_t stream) {
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(blocks), dim3(AT_THREADS), 0, stream, P); };
  const int D = P.a.cache.dim;
  if (D <= 64)
    s.R == 1 ? go(k_attn<XT, CT, 64, 1, 2>) : s.R == 2 ? go(k_attn<XT, CT, 64, 2, 2>) : go(k_attn<XT, CT, 64, 4, 1>);
  else if (D <= 128)
    s.R == 1 ? go(k_attn<XT, CT, 128, 1, 2>) : s.R == 2 ? go(k_attn<XT, CT, 128, 2, 2>) : go(k_attn<XT, CT, 128, 4, 1>);
  else
    s.R == 1 ? go(k_attn<XT, CT, 256, 1, 1>) : go(k_attn<XT, CT, 256, 2, 1>);
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
  const AttnShape s = attn_shape(a.T, P.G, a.cache.dim);
  P.WR = s.WR;
  P.RB = s.RB;
  P.target = attn_target(a.cache.heads, s.RB);
  P.least = 4;
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
