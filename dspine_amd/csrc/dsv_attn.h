// Attention of drafted nodes over a request's cached positions for gfx950.
//
// For request b, cache head h and the query rows r = (node, query head of h's group), with s = scale * q.k:
// out = sum_p e^(s_p - m) v_p / sum_p e^(s_p - m), in one pass over the positions with a reference m of the softmax
// that moves up where a score exceeds it by more than a few powers of two (the weights are then at most 2^LIM, and the
// partial sums are rescaled; most steps only compare).  With value scales the weighted values have a reference of their
// own, the largest weight times scale: a scale counts by the weight of its position.
//
// The matrix cores take keys as they lie in memory: S^T = K Q^T with the positions on the rows of the tile, so that a
// lane holds, for one query row, the weights of the four (twice: eight) positions that the second product
// O^T = V^T P^T wants from it: no weight moves between lanes.  Values come as 16-byte pieces of whole rows, whose
// elements a v_perm each puts in the positions' order.  Two forms of one kernel:
//   direct   (few rows) every wave loads the operands of its own positions from memory to registers; the waves run free
//            of each other and join at the end
//   staged   the workgroup's waves share their positions and split the rows: each wave brings a quarter of a tile
//            of 64 positions from memory, converts it to the operands' 16-bit layout once and puts it into LDS (two
//            buffers), from where every wave reads whole operands without bank conflicts
//
// The tiles of all requests, one request after the other, are cut into `ranges` equal ranges, as many as workgroups run
// at once, so that all end together; a range may hold the end of a request, whole requests and the beginning of one.
// Only the device knows the lengths: every wave computes the same plan from them.  A request within one range is
// finished there; the parts of the others are left as sums and joined by k_attn_join.
//
// Measured in kernel traces of replayed graphs, the attention and the join, us, a few percent more than a call takes in a row of
// eager ones (8 cache heads, dim 128; the card copies at 4.7 to 5.3 TB/s and multiplies at 1.37 PF):
//   64 requests, 17 nodes, 4 query heads a cache head, bf16, 1k to 8k positions   270 + 7.6   4.4 TB/s: memory
//   8 requests, 1 node, int8, 16k to 64k positions                                178 + 5.4   3.7 TB/s: memory, and 8 to 16 bits
//   16 requests, 64 nodes, 8 query heads a cache head, e4m3, 4k to 12k            432 + 14.7  0.60 PF: a wave's own chain of LDS
//       reads, products, exponentials and products (matrix pipe busy 25 % of the time, VALU 40 %)
//   4 requests, 25 nodes, bf16, 1.5k to 4.7k                                      28 + 6.0    1.6 TB/s: latency (the plan, the
//       first loads, the outputs and the second launch take longer than a workgroup's six tiles)
//   1 request, 1 node, bf16, 640                                                  9.0 + 4.0   latency
//
// BLOCKS: the same over a list of blocks for each (request, cache head).  The positions are numbered as they are read, so only
// the way to a slot differs: a group of 16 positions lies in one block, and its list entry is asked for a step (a tile, where
// tiles are staged) before its slots.
//   64 requests, up to 17 nodes, 4 query heads a cache head, bf16, 64 blocks of 64  275 + 7.8  (263 a call in a row of eager
//       ones, 4.2 TB/s): memory, 256 bytes at a time
//   1 request, 1 node, 32 blocks of 64                                              9.4 + 5.7  latency
//   16 requests, 1 node, 8192 positions in blocks of 16, 64, 128, both launches: bf16 130 to 135, int8 101 to 104 (277 MB, 2.7 TB/s);
//       with heads as the caches' outer dimension, where a slot's scales no longer lie beside other heads', 123 and 95.  What keeps
//       the 8-bit ones from the rate of whole contexts is not known.
#pragma once
#include "dsv_cache.h"
#include "dsv_common.h"

namespace dsv {

constexpr int AT_WAVES = 4;   // waves of a direct workgroup, and those that bring a staged tile
constexpr int AT_MOST = 8;    // waves of a staged workgroup at most
constexpr int AT_NODES = 64;
constexpr int AT_STEP = 32;  // positions of a step: two tiles of the first product, one of the second
constexpr int AT_TILE = 64;  // positions of a plan's unit, and of a staged tile
constexpr float AT_LOW = -3e38f;

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef __bf16 bhalf8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct AttnParams {
  dsv_tree_attention_args a;
  FastDiv G;           // query heads a cache head
  int WR, RB;          // groups of rows a workgroup, row blocks of a request
  int most;            // ranges at most
  FastDiv least;       // tiles of a range at least (a batch of fewer is one range); not for BLOCKS
  uint32_t num_slots, k_step, v_step;  // slots; bytes from slot to slot
  float* part_o;       // [2 * range + (the range's last request, not its first)][head][row][dim]
  float4* part_ml;     // the same of [row]: the scores' reference, the weights' sum, the weighted values' reference less the first
  // (attention over selected blocks)
  const int32_t* blocks;  // [request][cache head][count]
  int count, shift;       // blocks of 2^shift positions
};

// The request's nodes, its context and its positions (context and window) that the page table has.  BLOCKS: its positions
// are numbered as they are read, those of the selected blocks, then those of the unfinished block and the window.
struct Request {
  int nodes;
  int prefix, total;  // within the table
};
// (so far from the largest int that a window behind it stays below)
__device__ __forceinline__ int context_of(const dsv_tree_attention_args& a, int64_t b) {
  const int pre = a.prefix_lens[b];
  return pre < 0 ? 0 : (pre > 0x7fffff00 ? 0x7fffff00 : pre);
}
// A request's finished blocks, and how many entries of its lists are read.
struct Finished {
  int full, read;
};
__device__ __forceinline__ Finished finished_of(const AttnParams& P, int64_t b) {
  Finished f;
  f.full = context_of(P.a, b) >> P.shift;
  f.read = f.full < P.count ? f.full : P.count;
  return f;
}
template <bool BLOCKS>
__device__ __forceinline__ Request request_of(const AttnParams& P, int64_t b) {
  const dsv_tree_attention_args& a = P.a;
  Request r;
  int n = a.verify_lens ? a.verify_lens[b] : a.T;
  r.nodes = n < 0 ? 0 : (n > a.T ? a.T : n);
  if constexpr (BLOCKS) {
    r.prefix = (finished_of(P, b).read << P.shift) + (context_of(a, b) & ((1 << P.shift) - 1));
    r.total = r.prefix + r.nodes;
    return r;
  }
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

// The plan, computed by every wave from the batch's lengths: the first `more` ranges are `size` + 1 tiles, the others
// `size`.  Up to 64 requests are read once, a request a lane, and looked up among the lanes; larger batches are read
// again where they are asked for.
struct Plan {
  int total, ranges, size, more;
  bool small;    // up to 64 requests
  Request mine;  // this lane's, of a small batch
  int tiles;     // its tiles
  __device__ __forceinline__ int start(int i) const { return i * size + (i < more ? i : more); }
  // the range that holds a tile
  __device__ __forceinline__ int range_of(int tile) const {
    const int wide = more * (size + 1);
    return tile < wide ? (int)((uint32_t)tile / (uint32_t)(size + 1))
                       : more + (int)((uint32_t)(tile - wide) / (uint32_t)(size < 1 ? 1 : size));
  }
};
template <bool BLOCKS>
__device__ __forceinline__ Plan plan_of(const AttnParams& P, int lane) {
  Plan p;
  p.small = P.a.bs <= WAVE;
  p.tiles = 0;
  p.mine = Request{0, 0, 0};
  int sum = 0;
  if (p.small) {
    if (lane < P.a.bs) {
      p.mine = request_of<BLOCKS>(P, lane);
      p.tiles = tiles_of(p.mine);
    }
    sum = p.tiles;
  } else {
    for (int b = lane; b < P.a.bs; b += WAVE) sum += tiles_of(request_of<BLOCKS>(P, b));
  }
  p.total = wave_sum(sum);
  int r;
  if constexpr (BLOCKS) {
    // About 16 parts of a request at most: a part costs the join 0.2 us, a tile more in a range 1 to 2 us, and a range that
    // holds two requests 4 us, so short lists get a tile a range.  Replayed, 8 cache heads, against two tiles a range (four
    // where tiles are staged): 1 node, 2 x 5 tiles 12.3 us for 16.5, 1 x 129 22.1 for 27.3, 1 x 257 27.0 for 34.6; 17 nodes, group 4,
    // 4 x 5 tiles 17.3 for 25.3, 2 x 17 22.0 for 25.4; 40 nodes, group 8, 2 x 17 30.4 for 37.8, 1 x 17 29.5 for 27.9.
    const uint32_t least = ((uint32_t)p.total / (uint32_t)P.a.bs + 8) / 16;
    r = (int)(least < 2 ? (uint32_t)p.total : ((uint32_t)p.total + least - 1) / least);
  } else {
    r = (int)P.least.div((uint32_t)p.total + P.least.d - 1);
  }
  p.ranges = r < 1 ? 1 : (r > P.most ? P.most : r);
  p.size = (int)((uint32_t)p.total / (uint32_t)p.ranges);
  p.more = p.total - p.size * p.ranges;
  return p;
}
// Request b (the same in every lane).
template <bool BLOCKS>
__device__ __forceinline__ Request request_in(const AttnParams& P, const Plan& p, int b) {
  if (!p.small) return request_of<BLOCKS>(P, b);
  return Request{readlane_at(p.mine.nodes, b), readlane_at(p.mine.prefix, b), readlane_at(p.mine.total, b)};
}
// Tiles of the requests before b.
template <bool BLOCKS>
__device__ __forceinline__ int tiles_before(const AttnParams& P, const Plan& p, int b, int lane) {
  int sum = 0;
  if (p.small)
    sum = lane < b ? p.tiles : 0;
  else
    for (int i = lane; i < b; i += WAVE) sum += tiles_of(request_of<BLOCKS>(P, i));
  return wave_sum(sum);
}
// The request of a tile (tile < total) and the tiles before it; -1 if there is none (lengths that change under the call).
template <bool BLOCKS>
__device__ __forceinline__ int request_at(const AttnParams& P, const Plan& p, int tile, int lane, int& before) {
  before = 0;
  for (int b0 = 0; b0 < P.a.bs; b0 += WAVE) {
    const int i = b0 + lane;
    const int n = p.small ? p.tiles : (i < P.a.bs ? tiles_of(request_of<BLOCKS>(P, i)) : 0);
    const int end = before + wave_incl_scan(n);
    const uint64_t past = __ballot(end > tile);
    if (past) {
      const int l = __ffsll((unsigned long long)past) - 1;
      before = readlane_at(end, l) - readlane_at(n, l);
      return b0 + l;
    }
    before = readlane<WAVE - 1>(end);
  }
  return -1;
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

// Element e of N positions' value words (wv[j]: position j's elements) in the positions' order.
template <int CT, int N, int W>
__device__ __forceinline__ void value_operand(const uint32_t (&wv)[N][W], int e, uint32_t (&o)[N / 2]) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    if constexpr (CT == DSV_I8) {
      const uint32_t sel = 0x0c040c00u + (uint32_t)(e & 3) * 0x00010001u;
      o[i] = i8_pair(__builtin_amdgcn_perm(wv[2 * i + 1][e / 4] ^ 0x80808080u, wv[2 * i][e / 4] ^ 0x80808080u, sel));
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

// An element of the cache's rows.
template <int CT>
__device__ __forceinline__ float cache_value(const void* row, int i) {
  if constexpr (CT == DSV_E4M3) {
    float f[4];
    unpack_codes<CT>(reinterpret_cast<const uint8_t*>(row)[i], f);
    return f[0];
  } else if constexpr (CT == DSV_I8) {
    return (float)reinterpret_cast<const int8_t*>(row)[i];
  } else {
    return act_to_f32<CT>(reinterpret_cast<const uint16_t*>(row)[i]);
  }
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

// FORM: direct, or staged with a wave (AT_ROWS) or two (AT_PAIRS) for a group of rows.
enum { AT_DIRECT = 0, AT_PAIRS = 1, AT_ROWS = 2 };
// Tiles a turn: two row tiles a wave leave one workgroup of eight waves a CU, and LDS for four staged tiles: its first four
// waves bring one tile and the others the next, so that all do the same work between two barriers.
constexpr int AT_TILES(int FORM, int R) { return FORM == 2 && R == 2 ? 2 : 1; }
constexpr int AT_DEPTH(int R, int DP) { return R == 1 && DP <= 128 ? 2 : 1; }

template <int XT, int CT, int DP, bool FULL, int R, int FORM, int WAVES, int OCC, bool BLOCKS>
__global__ __launch_bounds__(WAVES * WAVE, OCC) void k_attn(AttnParams P) {
  const dsv_tree_attention_args& a = P.a;
  const dsv_kv_cache& c = a.cache;
  const int dim = FULL ? DP : c.dim;  // (a constant for the common sizes: no test of it in the loop)
  constexpr bool QUANT = CT == DSV_E4M3 || CT == DSV_I8, STAGED = FORM != AT_DIRECT;
  constexpr int WK = FORM == AT_DIRECT ? AT_WAVES : (FORM == AT_PAIRS ? 2 : 1);  // waves of the same rows
  // The weights' type in the second product: the values' own for 16-bit caches, float16 for the 8-bit codes (exact in it).  A
  // weight (times its value scale) is rounded to it once, by 2^-9 (bfloat16) or 2^-12 at most.  The errors are random: over n
  // positions of like weight they leave 1 / sqrt(n) of that.  Measured against float64, the output's own rounding included:
  // bfloat16 caches 1.7e-3 to 2.3e-3 (with float32 weights 1.7e-3), 8-bit ones 1.7e-3 (1.7e-3), float16 ones 2.5e-4
  // (2.1e-4).  That is at most what the output's rounding to bfloat16 adds anyway.  Keeping the low half takes a second product of
  // every value: 64 x 17 nodes of 4 heads 299 us for 277 (over selected blocks 300 for 293), 16 x 64 of 8 over blocks 423 for
  // 336, single nodes 130 for 129.  Sums, references, partial outputs and the join are float32.
  constexpr int PT = CT == DSV_BF16 ? DSV_BF16 : DSV_F16;
  // float16 weights are held 2^11 higher, so that what their range loses lies below 2^-35 of the row's largest
  constexpr float SHIFT = PT == DSV_F16 ? 11.f : 0.f, LIM = PT == DSV_F16 ? 4.f : 8.f;
  constexpr int ESZ = QUANT ? 1 : 2;
  constexpr int EPL = DP / 16;            // value elements a lane loads of a position
  constexpr int VW = EPL * ESZ / 4;       // words of them
  constexpr int NK = DP / 32;             // key products of a step
  constexpr int KL = DP * ESZ / 64;       // 16-byte key loads a lane of a position
  constexpr int OS = DP + 4;              // row stride of the sums in LDS
  constexpr int SET_ASIDE = STAGED ? AT_TILE : AT_STEP;
  constexpr int FRAGS = 4 * NK + 2 * EPL;  // operands of a staged tile: keys, then values, 16 bytes a lane each (values as
                                           // two halves of 8, so that their writes find all banks)
  constexpr int NT = AT_TILES(FORM, R);
  constexpr size_t SUMS = sizeof(float) * WAVES * 16 * OS, TILES = STAGED ? sizeof(uint4) * 2 * NT * FRAGS * WAVE : 0;
  __shared__ __attribute__((aligned(16))) unsigned char s_mem[SUMS > TILES ? SUMS : TILES];
  __shared__ float s_m[WAVES][16 * R], s_l[WAVES][16 * R], s_r[WAVES][16 * R];
  __shared__ uint64_t s_mask[WAVES][16 * R];  // of the wave's rows
  __shared__ int s_odd;
  float(*const s_o)[16][OS] = reinterpret_cast<float(*)[16][OS]>(s_mem);

  const int tid = threadIdx.x, lane = tid & (WAVE - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / WAVE);  // (and all that follows from it: scalar)
  const int m = lane & 15, g = lane >> 4;
  // Ranges round the XCDs, a range's heads and row blocks on one: they share its page table rows, scales and keys in
  // that XCD's L2.
  const int HB = c.heads * P.RB;
  const int inner = (int)((blockIdx.x / 8) % HB), range = (int)((blockIdx.x / 8) / HB) * 8 + (int)(blockIdx.x % 8);
  const int h = inner / P.RB, rb = inner - h * P.RB;
  const Plan plan = plan_of<BLOCKS>(P, lane);
  if (range >= plan.ranges || plan.total == 0) return;
  const int wr = wave / WK, wk = wave - wr * WK;
  const int block0 = rb * 16 * R * P.WR, row0 = block0 + wr * 16 * R;
  int tile = plan.start(range), before;
  const int stop = plan.start(range + 1);
  int b = __builtin_amdgcn_readfirstlane(request_at<BLOCKS>(P, plan, tile, lane, before));
  // the range's requests, one after the other
  for (bool first = true; tile < stop && b >= 0 && b < a.bs; first = false) {
  const Request req = request_in<BLOCKS>(P, plan, b);
  const int n_rows = req.nodes * (int)P.G.d, tiles = tiles_of(req);
  const int t0 = tile - before, t1 = stop - before < tiles ? stop - before : tiles;
  const int request = b;
  before += tiles;
  tile += t1 - t0;
  ++b;
  if (block0 >= n_rows || t0 == t1) continue;
  __syncthreads();  // (the sums of the request before have been read)
  if (tid == 0) s_odd = 0;
  __syncthreads();

  // Queries, in the order of the keys' elements.  They are waited for here, before the loops: a wait inside would be one
  // for every load in flight.
  uint32_t qf[R][NK][4];
  auto load_queries = [&]() {
#pragma unroll
    for (int rt = 0; rt < R; ++rt) {
      const int r = row0 + rt * 16 + m, node = (int)P.G.div((uint32_t)r), head = h * (int)P.G.d + r - node * (int)P.G.d;
      const int64_t row = r < n_rows ? row_of(a, request, node) : -1;
      const uint16_t* q = reinterpret_cast<const uint16_t*>(a.q) + (row < 0 ? 0 : row * a.q_row_stride + head * a.q_head_stride);
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) {
        const int d = QUANT ? (kk / 2) * 64 + g * 16 + (kk & 1) * 8 : kk * 32 + g * 8;
        uint32_t w[4] = {0, 0, 0, 0};
        if (row >= 0 && d < dim) load_words<4>(q + d, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) qf[rt][kk][i] = w[i];
      }
      if (g == 0) s_mask[wave][rt * 16 + m] = r < n_rows ? mask_of(a, request, node) : 0ull;
    }
#pragma unroll
    for (int rt = 0; rt < R; ++rt)
#pragma unroll
      for (int kk = 0; kk < NK; ++kk)
#pragma unroll
        for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(qf[rt][kk][i]));
  };

  const int32_t* table = a.page_table + (int64_t)request * a.page_stride;
  const uint8_t* kbase = reinterpret_cast<const uint8_t*>(c.k) + (int64_t)h * c.k_head_stride * ESZ + g * 16;
  const bool v_in = m * EPL < dim;  // (else the lane repeats the row's first piece: its sums are not stored)
  const uint8_t* vhead = reinterpret_cast<const uint8_t*>(c.v) + (int64_t)h * c.v_head_stride * ESZ;
  const uint8_t* vbase = vhead + (v_in ? m * EPL * ESZ : 0);
  const float* ksc = QUANT ? c.k_scale + (int64_t)h * c.ks_head_stride : nullptr;
  const float* vsc = QUANT ? c.v_scale + (int64_t)h * c.vs_head_stride : nullptr;
  const float c0 = a.scale * 1.44269504088896340736f * (CT == DSV_I8 && XT == DSV_F16 ? I8_UNIT : 1.f);
  const int clear = req.prefix;  // positions before it are seen by every row

  f32x4 o[R][EPL];
  float mref[R], l[R];
  // With value scales the row has two references, both powers of two that only move up: m of its scores, 2^4 at most below
  // any, for the sum l of the weights, and `mref` of weight times scale, for the float16 operands: those of the positions that
  // count lie within [2^10, 2^15] at their largest, whatever scales positions without weight have.  A score is taken against
  // mref, and the difference vlog = mref - m goes back into l.  -120 <= vlog, so that the weights stay within float32, and
  // vlog <= 117 for any finite scale: weights down to 2^-32 of the row's largest are then float32 numbers, subnormal ones
  // at the far end, and count in l.
  float vlog[R];
  bool fresh = true;  // some row has no reference yet
#pragma unroll
  for (int rt = 0; rt < R; ++rt) {
    mref[rt] = AT_LOW;
    l[rt] = 0.f;
    vlog[rt] = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) o[rt][e] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const int last = req.total - 1;
  auto good = [&](uint32_t slot) { return slot < P.num_slots; };
  // BLOCKS: where a group of 16 positions, numbered as they are read, begins in the request, or -1 where its entry names no
  // finished block.  The list is read through the scalar cache: the group is the same in every lane.
  const Finished done = BLOCKS ? finished_of(P, request) : Finished{0, 0};
  const auto* const list = reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(
      reinterpret_cast<uintptr_t>(P.blocks + (BLOCKS ? ((int64_t)request * c.heads + h) * P.count : 0)));
  auto entry = [&](int v) {
    const int e = v >> P.shift;
    return list[e < P.count ? e : P.count - 1];
  };
  auto group_of = [&](int v, int id) {
    if (v >> P.shift >= done.read) return ((done.full - done.read) << P.shift) + v;
    return (uint32_t)id < (uint32_t)done.full ? (id << P.shift) + (v & ((1 << P.shift) - 1)) : -1;
  };
  auto group = [&](int v) { return group_of(v, entry(v)); };
  // the slot of position i of the group that begins at `from`
  auto slot_in = [&](int from, int i) {
    return from >= 0 && (int64_t)from + i < a.page_cols ? (uint32_t)table[from + i] : ~0u;
  };
  // those of its positions g * 4 .. g * 4 + 3
  auto four_slots = [&](int from, uint32_t* vs) {
    if (from >= 0 && (int64_t)from + 16 <= a.page_cols) {
      uint4 v;
      __builtin_memcpy(&v, table + from + g * 4, 16);
      vs[0] = v.x, vs[1] = v.y, vs[2] = v.z, vs[3] = v.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) vs[j] = slot_in(from, g * 4 + j);
    }
  };
  // the slots of 32 positions from `base`: of the key rows m and 16 + m, and of this lane's eight positions
  // g * 4 + j, 16 + g * 4 + j (j < 4); the others' entries are not touched
  auto key_slots = [&](int base, uint32_t& k0, uint32_t& k1) {
    if constexpr (BLOCKS) {
      k0 = base + m <= last ? slot_in(group(base), m) : ~0u;
      k1 = base + 16 + m <= last ? slot_in(group(base + 16), m) : ~0u;
    } else if (base + AT_STEP <= req.total) {
      k0 = (uint32_t)table[base + m];
      k1 = (uint32_t)table[base + 16 + m];
    } else {
      k0 = base + m <= last ? (uint32_t)table[base + m] : ~0u;
      k1 = base + 16 + m <= last ? (uint32_t)table[base + 16 + m] : ~0u;
    }
  };
  auto value_slots = [&](auto whole_, int base, uint32_t (&vs)[8]) {
    if constexpr (BLOCKS) {
      four_slots(group(base), vs);
      four_slots(group(base + 16), vs + 4);
#pragma unroll
      for (int j = 0; j < 8; ++j) vs[j] = base + (j / 4) * 16 + g * 4 + (j & 3) <= last ? vs[j] : ~0u;
    } else if (decltype(whole_)::value || base + AT_STEP <= req.total) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint4 v;
        __builtin_memcpy(&v, table + base + i * 16 + g * 4, 16);
        vs[4 * i] = v.x, vs[4 * i + 1] = v.y, vs[4 * i + 2] = v.z, vs[4 * i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int p = base + (j / 4) * 16 + g * 4 + (j & 3);
        vs[j] = p <= last ? (uint32_t)table[p] : ~0u;
      }
    }
  };
  auto load_key = [&](uint32_t slot, uint32_t (&kw)[KL][4]) {
    const uint8_t* p = kbase + (uint64_t)(good(slot) ? slot : 0u) * P.k_step;
#pragma unroll
    for (int u = 0; u < KL; ++u)
      if (u * 64 < dim * ESZ)  // (past the row's end: its first piece, replaced by zeros before it is used)
        load_words<4>(p + (u * 64 + g * 16 < dim * ESZ ? u * 64 : -(g * 16)), kw[u]);
  };
  auto load_value = [&](uint32_t slot, uint32_t (&wv)[VW]) {
    load_words<VW>(vbase + (uint64_t)(good(slot) ? slot : 0u) * P.v_step, wv);
  };
  // the operand of key product kk
  auto key_frag = [&](const uint32_t (&kw)[KL][4], int kk, uint32_t (&ko)[4]) {
    const int from = QUANT ? (kk / 2) * 64 : kk * 32, width = QUANT ? 64 : 32;  // elements of the loads behind it
    if (from >= dim) {
#pragma unroll
      for (int u = 0; u < 4; ++u) ko[u] = 0u;
      return;
    }
    key_operand<XT, CT>(&kw[QUANT ? kk / 2 : kk][QUANT ? (kk & 1) * 2 : 0], ko);
    if (from + width > dim)
#pragma unroll
      for (int u = 0; u < 4; ++u) ko[u] = from + g * (width / 4) < dim ? ko[u] : 0u;
  };
  // Values of positions that hold nothing (bits of `here` unset) become zeros, and so do values that are not finite
  // where not every row sees them (0 * NaN is NaN in the product): the rows that do get them at the end.
  auto clear_values = [&](uint32_t here, bool aside, auto& wv) {
    constexpr int N = sizeof(wv) / sizeof(wv[0]);
    constexpr uint32_t INF = CT == DSV_BF16 ? 0x7f80u : 0x7c00u;
    bool odd = false;
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int u = 0; u < VW; ++u) {
        uint32_t w = (here >> j) & 1 ? wv[j][u] : 0u;
        if constexpr (CT != DSV_I8) {
          if (aside) {
            uint32_t bad;
            if constexpr (CT == DSV_E4M3)
              bad = ((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu;
            else
              bad = ((w & 0x7fffu) >= INF ? 0xffffu : 0u) | (((w >> 16) & 0x7fffu) >= INF ? 0xffff0000u : 0u);
            odd |= bad != 0;
            w &= ~bad;
          }
        }
        wv[j][u] = w;
      }
    if (odd) s_odd = 1;
  };
  // A step: scores of 32 positions' keys, weights, weighted values.  WHOLE: every row sees every position that holds
  // anything (`full`: all do; bit j of here_(): this lane's position j does).  cs: the positions' factors of a score
  // (base 2), vs: their value scales.  `next` runs when the keys have been used, `after` when the
  // values' operand e has.
  auto step = [&](auto whole_, int base, bool full, auto here_, const auto& cs, const auto& vs, auto key, auto value,
                  auto next, auto after) {
    constexpr bool WHOLE = decltype(whole_)::value;
    constexpr int GRP = R == 2 ? 4 : 1;  // operands asked for together (one, with two row tiles: 5 % slower)
    f32x4 s[R][2];
#pragma unroll
    for (int rt = 0; rt < R; ++rt)
#pragma unroll
      for (int i = 0; i < 2; ++i) s[rt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n0 = 0; n0 < 2 * NK; n0 += GRP) {
      uint32_t ko[GRP][4];
#pragma unroll
      for (int n = 0; n < GRP; ++n) key((n0 + n) & 1, (n0 + n) / 2, ko[n]);
#pragma unroll
      for (int n = 0; n < GRP; ++n)
#pragma unroll
        for (int rt = 0; rt < R; ++rt) s[rt][(n0 + n) & 1] = mfma<XT>(ko[n], qf[rt][(n0 + n) / 2], s[rt][(n0 + n) & 1]);
    }
    next();
    uint32_t seen[R];  // bit j: the row sees this lane's position j
    if constexpr (!WHOLE) {
      const uint32_t here = here_();
#pragma unroll
      for (int rt = 0; rt < R; ++rt) {
        const uint64_t mask = s_mask[wave][rt * 16 + m];
        uint32_t bits = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int p = base + (j / 4) * 16 + g * 4 + (j & 3) - req.prefix;
          const bool sees = p < 0 || (p < 64 && ((mask >> (p & 63)) & 1));
          bits |= (sees ? 1u : 0u) << j;
        }
        seen[rt] = bits & here;
      }
    }
    // The largest value scale of the lane's positions, as a power of two: with the lane's largest score it bounds weight times
    // scale from above, so most steps need no more to know that their operands stay within float16.
    float lift = -INFINITY;
    if constexpr (QUANT) {
      float v = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) v = fmaxf(v, fabsf(vs[j]));
      lift = __builtin_amdgcn_logf(v);
    }
    // scores against the rows' references
    float over = AT_LOW;
#pragma unroll
    for (int rt = 0; rt < R; ++rt) {
      const float ref = mref[rt] == AT_LOW ? 0.f : mref[rt];
      float top = AT_LOW;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float x = fmaf(s[rt][j / 4][j & 3], QUANT ? cs[j] : c0, -ref);
        if (!WHOLE && !((seen[rt] >> j) & 1)) x = -INFINITY;
        s[rt][j / 4][j & 3] = x;
        top = fmaxf(top, x);
      }
      over = fmaxf(over, QUANT ? top + fmaxf(vlog[rt] + SHIFT, lift) : top);
    }
    if (WHOLE && !full) {
      asm volatile("");  // (a branch: the selects are for bad slots only)
      const uint32_t here = here_();
      over = AT_LOW;
#pragma unroll
      for (int rt = 0; rt < R; ++rt) {
        float top = AT_LOW;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (!((here >> j) & 1)) s[rt][j / 4][j & 3] = -INFINITY;
          top = fmaxf(top, s[rt][j / 4][j & 3]);
        }
        over = fmaxf(over, QUANT ? top + fmaxf(vlog[rt] + SHIFT, lift) : top);
      }
    }
    if (fresh || __any(over > SHIFT + LIM)) {
      bool none = false;
#pragma unroll
      for (int rt = 0; rt < R; ++rt) {
        float top = AT_LOW;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, s[rt][j / 4][j & 3]);
        top = across_groups_max(top);
        const bool unset = mref[rt] == AT_LOW;
        // The reference moves up (or anywhere from none).  Where it is so large that float32 rounds it, the step's own scores still
        // move by what was meant: nothing leaves float16's range.
        float move;
        if constexpr (QUANT) {
          // the scores' reference relative to the present one of the weighted values, then the new one of those relative to it
          const bool any = top != AT_LOW;
          const float old = unset ? 0.f : -vlog[rt], low = !any ? old : (unset ? ceilf(top) : fmaxf(old, ceilf(top)));
          float high = -INFINITY;  // weight times scale
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float v = fabsf(vs[j]);
            high = fmaxf(high, s[rt][j / 4][j & 3] - low + (v < INFINITY ? __builtin_amdgcn_logf(v) : -INFINITY));
          }
          high = across_groups_max(high);
          const float up = any ? fmaxf(fmaxf(ceilf(high) - SHIFT, -120.f), unset ? -120.f : -low) : -low;
#pragma unroll
          for (int j = 0; j < 8; ++j) s[rt][j / 4][j & 3] = s[rt][j / 4][j & 3] - low - up;
          l[rt] *= unset ? 0.f : __builtin_amdgcn_exp2f(old - low);
          vlog[rt] = up;
          move = low + up;
        } else {
          move = top - SHIFT;
          if (top - move > SHIFT + LIM) move = top;
          if (top == AT_LOW || (!unset && move < 0.f)) move = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) s[rt][j / 4][j & 3] -= move;
        }
        if (top != AT_LOW || !unset) mref[rt] = (unset ? 0.f : mref[rt]) + move;
        none |= mref[rt] == AT_LOW;
        const float keep = unset ? 0.f : __builtin_amdgcn_exp2f(-move);
        if constexpr (!QUANT) l[rt] *= keep;
#pragma unroll
        for (int e = 0; e < EPL; ++e) o[rt][e] *= keep;
      }
      fresh = __any(none);
    }
    uint32_t pf[R][4];
#pragma unroll
    for (int rt = 0; rt < R; ++rt) {
      float sum = QUANT ? 0.f : l[rt];
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        float w[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          w[u] = __builtin_amdgcn_exp2f(s[rt][j / 4][(j + u) & 3]);
          sum += w[u];
          if constexpr (QUANT) {
            w[u] *= vs[j + u];
            if (!WHOLE && !((seen[rt] >> (j + u)) & 1)) w[u] = 0.f;
          }
        }
        pf[rt][j / 2] = pack_act<PT>(w[0], w[1]);
      }
      l[rt] = QUANT ? fmaf(sum, __builtin_amdgcn_exp2f(vlog[rt]), l[rt]) : sum;
    }
#pragma unroll
    for (int e0 = 0; e0 < EPL; e0 += GRP) {
      uint32_t vo[GRP][4];
#pragma unroll
      for (int e = 0; e < GRP; ++e) value(e0 + e, vo[e]);
#pragma unroll
      for (int e = 0; e < GRP; ++e) {
#pragma unroll
        for (int rt = 0; rt < R; ++rt) o[rt][e0 + e] = mfma<PT>(vo[e], pf[rt], o[rt][e0 + e]);
        after(e0 + e);
      }
    }
  };

  if constexpr (!STAGED) {
    // The scales of a step's 32 positions: lane (m, g) loads the key's (g < 2) or the value's of position
    // (g & 1) * 16 + m (zero where it holds nothing), and a lane's eight come back through LDS: 16 loads and their
    // addresses a lane were most of the step's instructions.
    __shared__ float s_scale[AT_WAVES][2][AT_STEP];
    auto load_scale = [&](uint32_t k0, uint32_t k1) {
      const uint32_t slot = g & 1 ? k1 : k0;
      if constexpr (!QUANT) return 0.f;
      const int64_t s = good(slot) ? slot : 0u;
      const float f = g < 2 ? ksc[s * c.ks_slot_stride] : vsc[s * c.vs_slot_stride];
      return good(slot) ? f : 0.f;
    };
    auto spread_scales = [&](float scale, float (&kf)[8], float (&vf)[8]) {
      if constexpr (QUANT) {
        s_scale[wave][g >> 1][(g & 1) * 16 + m] = g < 2 ? scale * c0 : scale;
        __builtin_amdgcn_wave_barrier();  // (the wave's own memory, in order)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float4 k4 = *reinterpret_cast<const float4*>(&s_scale[wave][0][i * 16 + g * 4]);
          const float4 v4 = *reinterpret_cast<const float4*>(&s_scale[wave][1][i * 16 + g * 4]);
          kf[4 * i] = k4.x, kf[4 * i + 1] = k4.y, kf[4 * i + 2] = k4.z, kf[4 * i + 3] = k4.w;
          vf[4 * i] = v4.x, vf[4 * i + 1] = v4.y, vf[4 * i + 2] = v4.z, vf[4 * i + 3] = v4.w;
        }
        __builtin_amdgcn_wave_barrier();
      }
    };
    auto holds = [&](const uint32_t (&vs)[8]) {
      uint32_t here = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) here |= (good(vs[j]) ? 1u : 0u) << j;
      return here;
    };
    load_queries();
    // steps of this wave: every WK-th
    int t = t0 * (AT_TILE / AT_STEP) + wk;
    int end = t1 * (AT_TILE / AT_STEP);
    const int some = (req.total + AT_STEP - 1) / AT_STEP;
    end = end < some ? end : some;
    if (row0 >= n_rows) t = end;
    // Those in the context: the next step's keys, values and scales are loaded when this one's scores are done, the slots
    // two steps ahead.
    const int whole = clear / AT_STEP < end ? clear / AT_STEP : end;
    if (t < whole) {
      uint32_t ks0[2], vs0[8], ks1[2], vs1[8], here0, here1, kw[2][KL][4], wv0[8][VW], wv1[8][VW];
      float scale;
      // (BLOCKS: the entries of a step's groups are asked for a step before its slots)
      int entries[2] = {0, 0}, entries_at = 0;
      auto ask_entries = [&](int i) {
        if constexpr (BLOCKS) {
          entries_at = (i < whole ? i : t) * AT_STEP;
          entries[0] = entry(entries_at);
          entries[1] = entry(entries_at + 16);
        }
      };
      auto slots = [&](int i, uint32_t (&ks)[2], uint32_t (&vs)[8]) {
        if constexpr (BLOCKS) {
          const int from0 = group_of(entries_at, entries[0]), from1 = group_of(entries_at + 16, entries[1]);
          ks[0] = slot_in(from0, m);
          ks[1] = slot_in(from1, m);
          four_slots(from0, vs);
          four_slots(from1, vs + 4);
          return;
        }
        ks[0] = (uint32_t)table[i * AT_STEP + m];
        ks[1] = (uint32_t)table[i * AT_STEP + 16 + m];
        value_slots(Int<1>{}, i * AT_STEP, vs);
      };
      auto load = [&](const uint32_t (&ks)[2], const uint32_t (&vs)[8], uint32_t (&wv)[8][VW], uint32_t& here) {
        load_key(ks[0], kw[0]);
        load_key(ks[1], kw[1]);
        scale = load_scale(ks[0], ks[1]);
        here = holds(vs);
#pragma unroll
        for (int j = 0; j < 8; ++j) load_value(vs[j], wv[j]);
      };
      // (the slots of the step after the next are asked for before the next one's data: a wait for them, loads being
      // counted in order, is none for that data)
      auto go = [&](uint32_t (&wv)[8][VW], uint32_t here, uint32_t (&then)[8][VW], uint32_t& then_here, uint32_t (&ks)[2],
                    uint32_t (&slot)[8], uint32_t (&then_ks)[2], uint32_t (&then_slot)[8]) {
        float cs[8], vs[8];
        spread_scales(scale, cs, vs);
        const bool full = !__any(here != 0xffu);
        step(Int<1>{}, t * AT_STEP, full, [&]() { return here; }, cs, vs,
             [&](int i, int kk, uint32_t (&ko)[4]) { key_frag(kw[i], kk, ko); },
             [&](int e, uint32_t (&vo)[4]) { value_operand<CT>(wv, e, vo); },
             [&]() {
               slots(t + 2 * WK < whole ? t + 2 * WK : t, then_ks, then_slot);
               ask_entries(t + 3 * WK);
               __builtin_amdgcn_sched_barrier(0);
               load(ks, slot, then, then_here);
               __builtin_amdgcn_sched_barrier(0);
               if (!full) clear_values(here, false, wv);
             },
             [](int) {});
        t += WK;
      };
      ask_entries(t);
      slots(t, ks0, vs0);
      ask_entries(t + WK);
      slots(t + WK < whole ? t + WK : t, ks1, vs1);
      ask_entries(t + 2 * WK);
      load(ks0, vs0, wv0, here0);
      while (true) {
        go(wv0, here0, wv1, here1, ks1, vs1, ks0, vs0);
        if (t >= whole) break;
        go(wv1, here1, wv0, here0, ks0, vs0, ks1, vs1);
        if (t >= whole) break;
      }
    }
    // The window's.
    for (; t < end; t += WK) {
      uint32_t ks[2], slot[8], kw[2][KL][4], wv[8][VW];
      float cs[8], vs[8];
      const int base = t * AT_STEP;
      key_slots(base, ks[0], ks[1]);
      value_slots(Int<0>{}, base, slot);
      load_key(ks[0], kw[0]);
      load_key(ks[1], kw[1]);
      spread_scales(load_scale(ks[0], ks[1]), cs, vs);
#pragma unroll
      for (int j = 0; j < 8; ++j) load_value(slot[j], wv[j]);
      const uint32_t here = holds(slot);
      clear_values(here, true, wv);
      step(Int<0>{}, base, false, [&]() { return here; }, cs, vs,
           [&](int i, int kk, uint32_t (&ko)[4]) { key_frag(kw[i], kk, ko); },
           [&](int e, uint32_t (&vo)[4]) { value_operand<CT>(wv, e, vo); }, [] {}, [](int) {});
    }
  } else {
    uint4(*const s_frag)[FRAGS][WAVE] = reinterpret_cast<uint4(*)[FRAGS][WAVE]>(s_mem);
    __shared__ float s_scale[2 * NT][2][AT_TILE];
    __shared__ uint32_t s_here[2 * NT][AT_WAVES];
    // Each of the first waves brings 16 positions: lane (m, g) pieces of the key of position m, and of the values of
    // g * 4 .. g * 4 + 3.  The loads run DEPTH tiles ahead of the one that is put away (in two sets of registers where
    // there are that many).
    constexpr int DEPTH = AT_DEPTH(R, DP);
    struct Brought {
      uint32_t kw[KL][4], wv[4][VW];
      uint32_t kslot, vslot[4];  // of the next tile to be loaded
      int entry;                 // BLOCKS: of the piece of the tile whose slots are asked for next
      uint32_t have;             // bits of the 16 positions
      float scale;
    };
    Brought sets[DEPTH];
    const bool brings = wave < AT_WAVES * NT;
    const int piece = wave % AT_WAVES, ahead = NT > 1 ? wave / AT_WAVES : 0;  // what of a turn's which tile
    auto fetch_entry = [&](Brought& f, int t) {
      if constexpr (BLOCKS) f.entry = entry(t * AT_TILE + piece * 16);
    };
    auto fetch_slots = [&](Brought& f, int t) {
      if (t >= t1) return;
      const int base = t * AT_TILE + piece * 16;
      if constexpr (BLOCKS) {
        const int from = group_of(base, f.entry);
        f.kslot = base + m <= last ? slot_in(from, m) : ~0u;
        four_slots(from, f.vslot);
        if (base + 16 > req.total)
#pragma unroll
          for (int j = 0; j < 4; ++j) f.vslot[j] = base + g * 4 + j <= last ? f.vslot[j] : ~0u;
        fetch_entry(f, t + NT * DEPTH);
        return;
      }
      if (base + 16 <= req.total) {
        f.kslot = (uint32_t)table[base + m];
        uint4 v;
        __builtin_memcpy(&v, table + base + g * 4, 16);
        f.vslot[0] = v.x, f.vslot[1] = v.y, f.vslot[2] = v.z, f.vslot[3] = v.w;
      } else {
        f.kslot = base + m <= last ? (uint32_t)table[base + m] : ~0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) f.vslot[j] = base + g * 4 + j <= last ? (uint32_t)table[base + g * 4 + j] : ~0u;
      }
    };
    auto fetch = [&](Brought& f) {
      load_key(f.kslot, f.kw);
#pragma unroll
      for (int j = 0; j < 4; ++j) load_value(f.vslot[j], f.wv[j]);
      f.have = (uint32_t)__ballot(good(f.kslot)) & 0xffffu;
      if constexpr (QUANT) {
        const int64_t s = good(f.kslot) ? f.kslot : 0u;
        if (g < 2) f.scale = g == 0 ? ksc[s * c.ks_slot_stride] : vsc[s * c.vs_slot_stride];
        if (!good(f.kslot)) f.scale = 0.f;
      }
    };
    auto put = [&](Brought& f, int t, int to_buf) {
      const int at = to_buf * NT + ahead;
      uint4(*const to)[WAVE] = s_frag[at];
      const bool aside = t * AT_TILE + SET_ASIDE > clear;
      if (aside || f.have != 0xffffu) clear_values(f.have >> (g * 4), aside, f.wv);
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) {
        uint32_t ko[4];
        key_frag(f.kw, kk, ko);
        to[piece * NK + kk][lane] = make_uint4(ko[0], ko[1], ko[2], ko[3]);
      }
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        uint32_t vo[2];
        value_operand<CT>(f.wv, e, vo);
        reinterpret_cast<uint2*>(to[4 * NK + (piece / 2) * EPL + e])[(piece & 1) * WAVE + lane] = make_uint2(vo[0], vo[1]);
      }
      if constexpr (QUANT)
        if (g < 2) s_scale[at][g][piece * 16 + m] = g == 0 ? f.scale * c0 : f.scale;
      if (lane == 0) s_here[at][piece] = f.have;
    };
    int buf = 0;
    // the loads of tile t and the slots of the set's next one
    auto ask = [&](Brought& f, int t) {
      if (t < t1) {
        fetch(f);
        fetch_slots(f, t + NT * DEPTH);
      }
    };
    if (brings) {
      fetch_entry(sets[0], t0 + ahead);
      if constexpr (DEPTH > 1) fetch_entry(sets[1], t0 + 1);
      fetch_slots(sets[0], t0 + ahead);
      if constexpr (DEPTH > 1) fetch_slots(sets[1], t0 + 1);
      ask(sets[0], t0 + ahead);
      if constexpr (DEPTH > 1) ask(sets[1], t0 + 1);
    }
    load_queries();
    if (brings && t0 + ahead < t1) {
      put(sets[0], t0 + ahead, 0);
      ask(sets[0], t0 + ahead + NT * DEPTH);
    }
    static_assert(NT == 1 || DEPTH == 1, "one set a wave");
    // A turn: the next tile (or two) into the other buffer, the loads of the one after it, the products of this one.  A step's keys
    // are read from LDS while the step before it multiplies (the first step's while the next tile is put away), its values
    // while its weights are computed, into the same registers: read where they are used, the reads' latencies were most
    // of a turn.
    constexpr bool AHEAD = R == 1 && DP <= 128;  // (with more rows the registers are not there, nor are the reads most of a step)
    uint4 fr[EPL];
    static_assert(2 * NK == EPL, "a step has as many key operands as value operands");
    auto read_key = [&](int cur, int blk, int n) { fr[n] = s_frag[cur][blk * 2 * NK + n][lane]; };
    auto read_value = [&](int cur, int blk, int e) {
      const uint2* v = reinterpret_cast<const uint2*>(s_frag[cur][4 * NK + blk * EPL + e]);
      const uint2 lo = v[lane], hi = v[WAVE + lane];
      fr[e] = make_uint4(lo.x, lo.y, hi.x, hi.y);
    };
    auto turn = [&](auto whole_, Brought& next, int t) {
      __syncthreads();
      const bool works = row0 < n_rows;
      if constexpr (AHEAD) {
        if (works)
#pragma unroll
          for (int n = 0; n < EPL; ++n) read_key(buf, wk, n);
        __builtin_amdgcn_sched_barrier(0);
      }
      const int own = t + NT + ahead;
      if (brings && own < t1) {
        put(next, own, buf ^ 1);
        ask(next, own + NT * DEPTH);
      }
      if (works) {
        auto one = [&](int cur, int tile, int blk, auto more_) {
          constexpr bool more = decltype(more_)::value;
          float cs[8], vs[8];
          if constexpr (QUANT) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float4 k4 = *reinterpret_cast<const float4*>(&s_scale[cur][0][blk * AT_STEP + i * 16 + g * 4]);
              const float4 v4 = *reinterpret_cast<const float4*>(&s_scale[cur][1][blk * AT_STEP + i * 16 + g * 4]);
              cs[4 * i] = k4.x, cs[4 * i + 1] = k4.y, cs[4 * i + 2] = k4.z, cs[4 * i + 3] = k4.w;
              vs[4 * i] = v4.x, vs[4 * i + 1] = v4.y, vs[4 * i + 2] = v4.z, vs[4 * i + 3] = v4.w;
            }
          }
          const uint32_t h0 = __builtin_amdgcn_readfirstlane(s_here[cur][2 * blk]);
          const uint32_t h1 = __builtin_amdgcn_readfirstlane(s_here[cur][2 * blk + 1]);
          step(whole_, tile * AT_TILE + blk * AT_STEP, (h0 & h1) == 0xffffu,
               [&]() { return ((h0 >> (g * 4)) & 0xfu) | (((h1 >> (g * 4)) & 0xfu) << 4); }, cs, vs,
               [&](int i, int kk, uint32_t (&ko)[4]) {
                 if constexpr (!AHEAD) read_key(cur, blk, i * NK + kk);
                 const uint4 v = fr[i * NK + kk];
                 ko[0] = v.x, ko[1] = v.y, ko[2] = v.z, ko[3] = v.w;
               },
               [&](int e, uint32_t (&vo)[4]) {
                 if constexpr (!AHEAD) read_value(cur, blk, e);
                 const uint4 v = fr[e];
                 vo[0] = v.x, vo[1] = v.y, vo[2] = v.z, vo[3] = v.w;
               },
               [&]() {
                 if constexpr (AHEAD) {
                   __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                   for (int e = 0; e < EPL; ++e) read_value(cur, blk, e);
                   __builtin_amdgcn_sched_barrier(0);
                 }
               },
               [&](int e) {
                 if constexpr (AHEAD && more) {
                   read_key(cur, blk + 1, e);
                   __builtin_amdgcn_sched_barrier(0);
                 }
               });
        };
#pragma unroll 1
        for (int i = 0; i < NT && t + i < t1; ++i) {
          one(buf * NT + i, t + i, wk, Int<WK == 1>{});
          if constexpr (WK == 1) one(buf * NT + i, t + i, 1, Int<0>{});
        }
      }
      buf ^= 1;
    };
    const int whole = clear / AT_TILE < t1 ? clear / AT_TILE : t1;
    int t = t0;
    if constexpr (DEPTH == 1) {
      for (; t + NT <= whole; t += NT) turn(Int<1>{}, sets[0], t);
      for (; t < t1; t += NT) turn(Int<0>{}, sets[0], t);
    } else {
      // (turn t puts away the set of t + 1 - t0)
      for (; t + 1 < whole; t += 2) {
        turn(Int<1>{}, sets[1], t);
        turn(Int<1>{}, sets[0], t + 1);
      }
      for (; t < t1; t += 2) {
        turn(Int<0>{}, sets[1], t);
        if (t + 1 < t1) turn(Int<0>{}, sets[0], t + 1);
      }
    }
  }

  // The waves of the same rows join: their references, then the sums of one row tile after another through LDS.
#pragma unroll
  for (int rt = 0; rt < R; ++rt) {
    l[rt] = across_groups_sum(l[rt]);
    if (g == 0) {
      s_m[wave][rt * 16 + m] = QUANT && mref[rt] != AT_LOW ? mref[rt] - vlog[rt] : mref[rt];
      s_r[wave][rt * 16 + m] = vlog[rt];
      s_l[wave][rt * 16 + m] = l[rt];
    }
  }
  __syncthreads();
  constexpr float unit = CT == DSV_I8 ? I8_UNIT : 1.f;
  // the waves' common reference of the weighted values, relative to that of the scores, `top`
  auto lifted = [&](int wr, int r, float top) {
    float ref = AT_LOW;
    for (int k = 0; k < WK; ++k) ref = fmaxf(ref, s_m[wr * WK + k][r] - top + s_r[wr * WK + k][r]);
    return ref;
  };
  // the positions whose values were set aside where they are not finite
  const int aside0 = clear / SET_ASIDE * SET_ASIDE > t0 * AT_TILE ? clear / SET_ASIDE * SET_ASIDE : t0 * AT_TILE;
  const int aside1 = t1 * AT_TILE < req.total ? t1 * AT_TILE : req.total;
#pragma unroll
  for (int rt = 0; rt < R; ++rt) {
    float top = AT_LOW;
    for (int k = 0; k < WK; ++k) top = fmaxf(top, s_m[wr * WK + k][rt * 16 + m]);
    float less = s_m[wave][rt * 16 + m] - top;
    if constexpr (QUANT) less = less + vlog[rt] - lifted(wr, rt * 16 + m, top);
    const float f = __builtin_amdgcn_exp2f(less) * unit;
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
      if (r >= n_rows || d >= dim) continue;
      float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      float mt = AT_LOW, lt = 0.f;
      for (int k = 0; k < WK; ++k) mt = fmaxf(mt, s_m[wr * WK + k][rt * 16 + rr]);
      const float ref = QUANT ? lifted(wr, rt * 16 + rr, mt) : 0.f;
      for (int k = 0; k < WK; ++k) {
        lt += s_l[wr * WK + k][rt * 16 + rr] * __builtin_amdgcn_exp2f(s_m[wr * WK + k][rt * 16 + rr] - mt);
#pragma unroll
        for (int u = 0; u < 8; ++u) sum[u] += s_o[wr * WK + k][rr][d + u];
      }
      const int node = (int)P.G.div((uint32_t)r), qh = h * (int)P.G.d + r - node * (int)P.G.d;
      if (CT != DSV_I8 && s_odd) {
        const uint64_t mask = mask_of(a, request, node);
        for (int p = aside0; p < aside1; ++p) {
          const uint32_t slot = BLOCKS ? slot_in(group(p & ~15), p & 15) : (uint32_t)table[p];
          const int j = p - req.prefix;
          if (!good(slot) || !(j < 0 || (j < 64 && ((mask >> (j & 63)) & 1)))) continue;
          const uint8_t* v = vhead + (uint64_t)slot * P.v_step + d * ESZ;
          for (int u = 0; u < 8; ++u) {
            const float x = cache_value<CT>(v, u);
            if (!(fabsf(x) < INFINITY)) sum[u] += x;
          }
        }
      }
      if (t1 - t0 < tiles) {
        // (its first part is its range's last request's, unless it begins the range; the others begin theirs)
        const int64_t at = ((int64_t)(2 * range + (first ? 0 : 1)) * c.heads + h) * (a.T * (int)P.G.d) + r;
        float* po = P.part_o + at * dim + d;
        *reinterpret_cast<float4*>(po) = make_float4(sum[0], sum[1], sum[2], sum[3]);
        *reinterpret_cast<float4*>(po + 4) = make_float4(sum[4], sum[5], sum[6], sum[7]);
        if (d == 0) P.part_ml[at] = make_float4(mt, lt, ref, 0.f);
      } else {
        const int64_t row = row_of(a, request, node);
        if (row < 0) continue;
        const float inv = lt == 0.f ? 0.f : 1.f / lt;
        if constexpr (QUANT) {  // (two steps: either factor alone may leave float32 where the product does not)
          const float up = __builtin_amdgcn_exp2f(ref);
#pragma unroll
          for (int u = 0; u < 8; ++u) sum[u] = sum[u] * inv * up;
        } else {
#pragma unroll
          for (int u = 0; u < 8; ++u) sum[u] *= inv;
        }
        uint4 v;
        v.x = pack_act<XT>(sum[0], sum[1]);
        v.y = pack_act<XT>(sum[2], sum[3]);
        v.z = pack_act<XT>(sum[4], sum[5]);
        v.w = pack_act<XT>(sum[6], sum[7]);
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + row * a.out_row_stride + qh * a.out_head_stride + d) = v;
        if (d == 0 && a.lse) a.lse[row * a.q_heads + qh] = lt == 0.f ? -INFINITY : (mt + log2f(lt)) * 0.693147180559945309f;
      }
    }
  }
  }
}

// How the rows of a request (T nodes of G query heads) are split: row tiles a wave, waves (or pairs) a workgroup, row
// blocks.
struct AttnShape {
  int form, R, WR, RB;
  int waves;  // of a workgroup
};
// Waves a SIMD that the registers are for: 256 of them each, 512 where the sums of a wide dim need more.  Vector registers that
// are spilled, over whole contexts and over blocks: two row tiles of dim 128 none and 2 (16-bit caches), 8 to 10 and 14 to 16 (8-bit
// ones), of dims 80 to 112 10 and 16, 16 to 24 and 24 to 27; the direct form of 16-bit caches 7 and 13 at dims 80 to 112, 3 and 5 at
// 256, up to 14 and 17 at 144 to 240 (which also keeps up to 469 scalar ones in vector lanes); one row tile a wave none and 2 at
// 80 to 112, 17 and 22 at 144 to 240 (8-bit caches up to 2 and 6).  No other form spills any.
constexpr int attn_occupancy(int form, int R, int dim) {
  return dim > 128 && form != AT_ROWS ? 1 : 2;
}

template <int XT, int CT, bool BLOCKS>
void launch_attn(const AttnParams& P, const AttnShape& s, unsigned blocks, hipStream_t stream) {
  auto go = [&](auto kern, int n) { hipLaunchKernelGGL(kern, dim3(blocks), dim3((unsigned)n * 64u), 0, stream, P); };
  const int D = P.a.cache.dim;
  auto width = [&](auto dp, auto full) {
    constexpr int DP = decltype(dp)::value;
    constexpr bool FULL = decltype(full)::value;
    if (s.form == AT_DIRECT)
      go(k_attn<XT, CT, DP, FULL, 1, AT_DIRECT, AT_WAVES, attn_occupancy(AT_DIRECT, 1, DP), BLOCKS>, s.waves);
    else if (s.form == AT_PAIRS)
      go(k_attn<XT, CT, DP, FULL, 1, AT_PAIRS, AT_WAVES, attn_occupancy(AT_PAIRS, 1, DP), BLOCKS>, s.waves);
    else if (s.R == 1)
      go(k_attn<XT, CT, DP, FULL, 1, AT_ROWS, AT_MOST, attn_occupancy(AT_ROWS, 1, DP), BLOCKS>, s.waves);
    else if constexpr (DP <= 128)
      go(k_attn<XT, CT, DP, FULL, 2, AT_ROWS, AT_MOST, attn_occupancy(AT_ROWS, 2, DP), BLOCKS>, s.waves);
  };
  if (D <= 64)
    D == 64 ? width(Int<64>{}, Int<1>{}) : width(Int<64>{}, Int<0>{});
  else if (D <= 128)
    D == 128 ? width(Int<128>{}, Int<1>{}) : width(Int<128>{}, Int<0>{});
  else
    D == 256 ? width(Int<256>{}, Int<1>{}) : width(Int<256>{}, Int<0>{});
}

}  // namespace dsv
