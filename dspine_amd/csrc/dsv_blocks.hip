// Blocks of a cache and what selects among them, for gfx950: the least and largest key elements of finished blocks, the
// bound of every block's attention scores that follows from them, and the best blocks of each (request, cache head).
#include "dsv_cache.h"
#include "dsv_common.h"

namespace dsv {

constexpr int BI_THREADS = 256;

struct IndexParams {
  dsv_block_index x;
  dsv_kv_cache c;
  const int32_t *page_table, *block_table, *from_lens, *to_lens;
  int64_t page_stride, page_cols, block_stride, block_cols;
  int bs, shift, most;  // block of 2^shift positions; blocks a request may have finished
};

// The least and largest of N elements over the lanes that differ in the bits from O down to G.  A step halves the elements
// that a lane is left with, as long as there are any to halve: 2 N exchanges in all in place of 2 N a step.
template <int N, int O, int G>
__device__ __forceinline__ void join_bounds(float* lo, float* hi, int lane) {
  if constexpr (O >= G) {
    if constexpr (N > 1) {
      const bool up = lane & O;
#pragma unroll
      for (int e = 0; e < N / 2; ++e) {
        const float l = __shfl_xor(up ? lo[e] : lo[e + N / 2], O, WAVE), h = __shfl_xor(up ? hi[e] : hi[e + N / 2], O, WAVE);
        lo[e] = __builtin_elementwise_minimum(up ? lo[e + N / 2] : lo[e], l);
        hi[e] = __builtin_elementwise_maximum(up ? hi[e + N / 2] : hi[e], h);
      }
      join_bounds<N / 2, O / 2, G>(lo, hi, lane);
    } else {
      lo[0] = __builtin_elementwise_minimum(lo[0], __shfl_xor(lo[0], O, WAVE));
      hi[0] = __builtin_elementwise_maximum(hi[0], __shfl_xor(hi[0], O, WAVE));
      join_bounds<1, O / 2, G>(lo, hi, lane);
    }
  }
}

// A finite bound past the index type's range as its largest number: infinite, a block of finite keys would have scores of
// no use, 0 * infinity among them.
template <int IT>
__device__ __forceinline__ float in_range(float v) {
  constexpr float TOP = IT == DSV_F16 ? 65504.f : 0x1.fep127f;
  return fabsf(v) < INFINITY ? fminf(fmaxf(v, -TOP), TOP) : v;
}

// Bounds of a finished block, a wave a (block, head): its lanes hold the block's slots, groups of G lanes take a position's
// row, 16 bytes a lane, BI_ROWS rows in flight together.  NaN counts as the least and the largest.  Bound by memory: the
// blocks of four prompts, 88 MB of e4m3 keys: 19.8 us in a kernel trace, 4.5 TB/s (a workgroup a block and head, two rows in
// flight: 57 us).  A round's few blocks: 5.1 us, latency.
constexpr int BI_ROWS = 8;
template <int CT, int IT, int G>
__global__ __launch_bounds__(BI_THREADS) void k_index_blocks(IndexParams P) {
  constexpr bool QUANT = CT == DSV_E4M3 || CT == DSV_I8;
  constexpr int EL = QUANT ? 16 : 8, GROUPS = WAVE / G;
  const dsv_kv_cache& c = P.c;
  const int lane = threadIdx.x & (WAVE - 1), l = lane & (G - 1), group = lane / G;
  const uint32_t unit = blockIdx.x * (BI_THREADS / WAVE) + __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const uint32_t at = unit / (uint32_t)c.heads, b = at / (uint32_t)P.most;
  const int h = (int)(unit - at * (uint32_t)c.heads);
  if (b >= (uint32_t)P.bs) return;
  const int from = P.from_lens[b], to = P.to_lens[b];
  const int64_t j = (int64_t)((from < 0 ? 0 : from) >> P.shift) + (at - b * (uint32_t)P.most);
  if (to < 0 || j >= to >> P.shift || j >= P.block_cols) return;
  const int32_t row = P.block_table[b * P.block_stride + j];
  const int B = 1 << P.shift;
  const int64_t p0 = j << P.shift;
  const int32_t* table = P.page_table + b * P.page_stride + p0;
  int32_t slots[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = k * WAVE + lane;
    slots[k] = i < B && p0 + i < P.page_cols ? table[i] : -1;
    if (slots[k] >= c.num_slots) slots[k] = -1;
  }
  if (row < 0 || row >= P.x.rows) return;
  const bool any = __any(slots[0] >= 0 || slots[1] >= 0);
  const bool in = l * EL < c.dim;
  const uint8_t* base = reinterpret_cast<const uint8_t*>(c.k) + (h * c.k_head_stride + (in ? l * EL : 0)) * (QUANT ? 1 : 2);
  float lo[EL], hi[EL];
#pragma unroll
  for (int e = 0; e < EL; ++e) lo[e] = INFINITY, hi[e] = -INFINITY;
  for (int i0 = 0; i0 < B; i0 += GROUPS * BI_ROWS) {
    uint4 x[BI_ROWS];
    float scale[BI_ROWS];
    bool has[BI_ROWS];
#pragma unroll
    for (int u = 0; u < BI_ROWS; ++u) {
      const int i = i0 + u * GROUPS + group;
      const int32_t slot = i < B ? __shfl(i < WAVE ? slots[0] : slots[1], i & (WAVE - 1), WAVE) : -1;
      has[u] = slot >= 0;
      const int64_t s = has[u] ? slot : 0;
      x[u] = *reinterpret_cast<const uint4*>(base + s * c.k_slot_stride * (QUANT ? 1 : 2));
      if constexpr (QUANT) scale[u] = c.k_scale[s * c.ks_slot_stride + h * c.ks_head_stride];
    }
#pragma unroll
    for (int u = 0; u < BI_ROWS; ++u) {
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
      if (has[u])
#pragma unroll
        for (int e = 0; e < EL; ++e) {
          lo[e] = __builtin_elementwise_minimum(lo[e], f[e]);
          hi[e] = __builtin_elementwise_maximum(hi[e], f[e]);
        }
    }
  }
  join_bounds<EL, WAVE / 2, G>(lo, hi, lane);
  // what is left of the lane's elements, and where: the highest lane bits chose the halves
  constexpr int STEPS = G == 32 ? 1 : (G == 16 ? 2 : (G == 8 ? 3 : 4)), HALVED = EL == 8 && STEPS > 3 ? 3 : STEPS;
  constexpr int LEFT = EL >> HALVED;
  int d = l * EL;
#pragma unroll
  for (int k = 0; k < HALVED; ++k) d += lane & (WAVE / 2 >> k) ? EL >> (k + 1) : 0;
  const bool first = (lane & (WAVE / (1 << HALVED) - 1) & ~(G - 1)) == 0;  // (of the lanes that hold the same)
  if (!in || !first) return;
  uint16_t* out = reinterpret_cast<uint16_t*>(P.x.bounds) + ((int64_t)row * c.heads + h) * 2 * c.dim + d;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float* const v = k ? hi : lo;
#pragma unroll
    for (int e = 0; e < LEFT; ++e) v[e] = in_range<IT>(v[e]);
    if constexpr (LEFT >= 2) {
#pragma unroll
      for (int e = 0; e < LEFT; e += 2)
        *reinterpret_cast<uint32_t*>(out + k * c.dim + e) = any ? pack_act<IT>(v[e], v[e + 1]) : 0u;
    } else {
      out[k * c.dim] = any ? (uint16_t)pack_act<IT>(v[0], 0.f) : (uint16_t)0;
    }
  }
}

// ---------------------------------------------------------------------------------------
// Scores: with q+ and q- a query's positive and negative elements, sum_d max(q lo, q hi) = q- . lo + q+ . hi where the bounds
// are finite, a product over 2 * dim elements of an index row as it lies in memory.  The matrix cores take 16 blocks as rows and 16 queries as
// columns; a block's score is the largest of its columns'.
// ---------------------------------------------------------------------------------------
constexpr int SB_WAVES = 4, SB_MANY = 8;  // waves of a workgroup, and where the queries take much LDS
constexpr int SB_STAGE = 60;  // pieces of 16 queries' 32 elements (1 KB) in LDS at most
constexpr int SB_STEPS = 8;   // steps of a workgroup at most, 16 blocks a wave each (32, with fewer steps: 43 us for 41)

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bhalf8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct ScoreParams {
  dsv_score_blocks_args a;
  FastDiv G;
  int shift, steps, chunks;  // steps of a workgroup, workgroups of a (request, head)
  int staged;                // query tiles in LDS at once
};

template <int IT>
__device__ __forceinline__ f32x4 mfma16(uint4 a, uint4 b, f32x4 c) {
  if constexpr (IT == DSV_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bhalf8, a), __builtin_bit_cast(bhalf8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// A pair's negative and positive elements, zeros in place of the others (a NaN stays in one of them).
__device__ __forceinline__ void split_signs(uint32_t w, uint32_t& negative, uint32_t& positive) {
  typedef short short2v __attribute__((ext_vector_type(2)));
  const uint32_t sign = __builtin_bit_cast(uint32_t, __builtin_bit_cast(short2v, w) >> 15);
  negative = w & sign;
  positive = w & ~sign;
}

// The largest sum by its definition, a row of queries at a time over the lanes' elements, for a block that the product gave
// NaN: with an infinite bound beside an element of the other sign it adds a 0 * infinity that is no term of the sum.
// NaN where no bound is infinite.
template <int IT>
__device__ __forceinline__ float defined_sum(const dsv_score_blocks_args& a, const FastDiv& G, int32_t block, int h, int64_t row0,
                                             int rows, int lane) {
  const dsv_block_index& x = a.index;
  const uint16_t* from = reinterpret_cast<const uint16_t*>(x.bounds) + ((int64_t)block * x.heads + h) * 2 * x.dim;
  const int d = lane * 4;  // (four elements a lane: up to 256)
  const bool in = d < x.dim;
  auto four = [&](const uint16_t* p, float (&f)[4]) {
    const uint2 w = in ? *reinterpret_cast<const uint2*>(p + d) : make_uint2(0, 0);
    f[0] = act_to_f32<IT>(w.x & 0xffffu), f[1] = act_to_f32<IT>(w.x >> 16);
    f[2] = act_to_f32<IT>(w.y & 0xffffu), f[3] = act_to_f32<IT>(w.y >> 16);
  };
  float lo[4], hi[4];
  four(from, lo);
  four(from + x.dim, hi);
  bool infinite = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) infinite |= fabsf(lo[e]) == INFINITY || fabsf(hi[e]) == INFINITY;
  if (!__any(infinite)) return NAN;
  float best = -INFINITY;
  for (int r = 0; r < rows; ++r) {
    const int node = (int)G.div((uint32_t)r), head = h * (int)G.d + r - node * (int)G.d;
    float q[4], sum = 0.f;
    four(reinterpret_cast<const uint16_t*>(a.q) + (row0 + node) * a.q_row_stride + head * a.q_head_stride, q);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum += __builtin_elementwise_maximum(q[e] * lo[e], q[e] * hi[e]);
    best = __builtin_elementwise_maximum(best, wave_sum(sum));
  }
  return best;
}

// A workgroup some steps of a (request, head)'s blocks, its queries as operands in LDS; a wave 16 blocks a step, their
// bounds in registers for all of the queries.  Bound by memory: 64 requests of 8k to 64k positions in blocks of 64, up to 17
// nodes, 154 MB read and written: 43.0 us in a kernel trace, 39.8 a call in a row of eager ones (3.6 and 3.9 TB/s).  Of 41 us in such
// a row, the next step's bounds loaded into a second set of registers first take 42; queries split by sign in LDS, twice the
// memory and half the workgroups a CU, 62.  Many rows are bound by operations, the split of the queries for each 16 blocks among
// them, and measured at 68 rows these say nothing of those.  One node over 32k: 5.0 us, latency.
// (Five waves a SIMD at dims 80 to 112: with the registers of four, 16 x 17 nodes of dim 96 take 19.0 us for 18.3.)
template <int IT, int NC, bool FULL, int WAVES>
__global__ __launch_bounds__(WAVES * WAVE, NC == 4 && !FULL ? 5 : 1) void k_score_blocks(ScoreParams P) {
  constexpr int SB_STEP = WAVES * 16;  // blocks of a step
  const dsv_score_blocks_args& a = P.a;
  const dsv_block_index& x = a.index;
  const int dim = FULL ? NC * 32 : x.dim;
  constexpr int AHEAD = 8;            // pieces of queries in flight
  extern __shared__ uint4 s_q[];      // [staged * NC][WAVE]
  __shared__ float s_best[SB_STEPS * SB_STEP];
  const int tid = threadIdx.x, lane = tid & (WAVE - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
  const int m = lane & 15, g = lane >> 4;
  // (the first chunks of all, then the second ones: neighbouring workgroups go to different XCDs, and chunk by chunk the XCDs
  // with the last ones of every request had least to do: 52 us for 43)
  const uint32_t bhs = (uint32_t)a.bs * (uint32_t)x.heads, bh = blockIdx.x % bhs;
  const int chunk = (int)(blockIdx.x / bhs);
  const int b = (int)(bh / (uint32_t)x.heads), h = (int)(bh - (uint32_t)b * x.heads);
  const int pre = a.prefix_lens[b];
  const int64_t full = pre < 0 ? 0 : pre >> P.shift;
  int n = a.verify_lens ? a.verify_lens[b] : a.T;
  n = n < 0 ? 0 : (n > a.T ? a.T : n);
  int64_t row0 = a.row_offsets ? load_index(a.row_offsets, a.row_offsets_i64, b) : (int64_t)b * a.T;
  // (nodes whose rows lie outside q are not there)
  const int skip = row0 < 0 ? (row0 > -(int64_t)n ? (int)-row0 : n) : 0;
  row0 += skip;
  n -= skip;
  if (n > 0 && a.rows - row0 < n) n = row0 < a.rows ? (int)(a.rows - row0) : 0;
  const int rows = n * (int)P.G.d, tiles = (rows + 15) / 16;
  const int64_t cols = a.block_cols, first = (int64_t)chunk * P.steps * SB_STEP;
  const int64_t past = first + P.steps * SB_STEP < cols ? first + P.steps * SB_STEP : cols;  // of the table
  const int64_t end = rows == 0 ? first : (past < full ? past : full);               // of the blocks that have a score
  float* const out = a.scores + (int64_t)bh * cols;
  const int32_t* const table = a.block_table + b * a.block_stride;
  for (int64_t i = (end > first ? end : first) + tid; i < past; i += WAVES * WAVE) out[i] = -INFINITY;
  if (end <= first) return;
  uint4 k[NC][2];
  bool there = false;
  // a step's bounds: lane (m, g) elements g * 8 .. of each 32 of block m's
  auto load = [&](int64_t j0) {
    const int64_t j = j0 + m;
    const int32_t row = j < end ? table[j] : -1;
    there = row >= 0 && row < x.rows;
    const uint4* from = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(x.bounds) +
                                                       ((int64_t)(there ? row : 0) * x.heads + h) * 2 * dim);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const bool in = FULL || c * 32 + g * 8 < dim;
      const int at = in ? c * 4 + g : 0;
      k[c][0] = from[at];
      k[c][1] = from[dim / 8 + at];
      if (!in) k[c][0] = k[c][1] = make_uint4(0, 0, 0, 0);
    }
  };
  for (int t0 = 0; t0 < tiles; t0 += P.staged) {
    const int here = tiles - t0 < P.staged ? tiles - t0 : P.staged;
    if (t0) __syncthreads();
    // (the first step's bounds are asked for behind the first queries)
    for (int i0 = wave; i0 < here * NC || i0 == wave; i0 += WAVES * AHEAD) {
      uint4 w[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int i = i0 + u * WAVES, t = i / NC, c = i - t * NC;
        int r = (t0 + t) * 16 + m;
        r = r < rows ? r : rows - 1;  // (a row again: the largest stays the largest)
        const int node = (int)P.G.div((uint32_t)r), head = h * (int)P.G.d + r - node * (int)P.G.d;
        const int d = c * 32 + g * 8;
        w[u] = make_uint4(0, 0, 0, 0);
        if (i < here * NC && (FULL || d < dim))
          w[u] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.q) + (row0 + node) * a.q_row_stride +
                                                 head * a.q_head_stride + d);
      }
      if (i0 == wave) load(first + wave * 16);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
        if (i0 + u * WAVES < here * NC) s_q[(i0 + u * WAVES) * WAVE + lane] = w[u];
    }
    __syncthreads();
    for (int step = 0; step < P.steps; ++step) {
      const int64_t j0 = first + step * SB_STEP + wave * 16;
      if (j0 >= end) break;
      f32x4 best = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      for (int rt = 0; rt < here; ++rt) {
        f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const uint4 q = s_q[(rt * NC + c) * WAVE + lane];
          uint4 low, high;
          split_signs(q.x, low.x, high.x);
          split_signs(q.y, low.y, high.y);
          split_signs(q.z, low.z, high.z);
          split_signs(q.w, low.w, high.w);
          s = mfma16<IT>(k[c][0], low, s);
          s = mfma16<IT>(k[c][1], high, s);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) best[r] = __builtin_elementwise_maximum(best[r], s[r]);
      }
      const bool has = __shfl((int)there, g * 4 + (m & 3), WAVE) != 0;  // (lane i knows block i)
      if (step + 1 < P.steps && j0 + SB_STEP < end) load(j0 + SB_STEP);
      // the 16 columns of a row lie in 16 neighbouring lanes; lane (r, g) keeps row g * 4 + r
      float mine = 0.f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float v = best[r];
        v = __builtin_elementwise_maximum(v, dpp<DPP_QUAD_XOR1>(v, v));
        v = __builtin_elementwise_maximum(v, dpp<DPP_QUAD_XOR2>(v, v));
        v = __builtin_elementwise_maximum(v, dpp<DPP_ROW_HALF_MIRROR>(v, v));
        v = __builtin_elementwise_maximum(v, dpp<DPP_ROW_MIRROR>(v, v));
        mine = m == r ? v : mine;
      }
      const int64_t j = j0 + g * 4 + m;
      const bool writes = m < 4 && j < end, final = t0 + here == tiles;
      const int at = (int)(j - first);
      if (writes && t0) mine = __builtin_elementwise_maximum(mine, s_best[at]);
      for (uint64_t odd = __ballot(writes && final && has && mine != mine); odd; odd &= odd - 1) {
        const int l = __ffsll((unsigned long long)odd) - 1;
        const float v = defined_sum<IT>(a, P.G, table[j0 + (l >> 4) * 4 + (l & 15)], h, row0, rows, lane);
        if (lane == l) mine = v;
      }
      if (writes) {
        if (final)
          out[j] = has ? mine * a.scale : -INFINITY;
        else
          s_best[at] = mine;  // (read by the same lane)
      }
    }
  }
}

// ---------------------------------------------------------------------------------------
// The best blocks.
// ---------------------------------------------------------------------------------------
struct SelectParams {
  const float* scores;
  const int32_t* prefix_lens;
  int32_t* blocks;
  int64_t cols;
  int heads, shift, count, first, last;
};

// A workgroup a (request, head), its scores in registers as keys that order like them.  The `need`-th largest key is
// found in 256 equal bins of the range that holds it, again within that bin until at most 64 keys are left, which one
// wave ranks by counting; equal keys count by their index, the lowest first.  The chosen ones are written in order.  Bound by
// latency: 8 heads of 500 blocks 6.2 us, 512 of up to 2000 7.7 us.
template <int NW, int PER>
__global__ __launch_bounds__(NW * WAVE) void k_select_blocks(SelectParams P) {
  constexpr int NT = NW * WAVE;
  __shared__ uint32_t s_hist[256], s_val[WAVE], s_red[2][NW], s_found[4];
  __shared__ int s_idx[WAVE], s_count[PER * NW + WAVE], s_n;
  const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
  const int64_t row = blockIdx.x;
  const float* scores = P.scores + row * P.cols;
  float score[PER];  // (asked for before it is known how many of them count)
#pragma unroll
  for (int i = 0; i < PER; ++i) score[i] = i * NT + tid < P.cols ? scores[i * NT + tid] : 0.f;
  const int pre = P.prefix_lens[row / P.heads];
  const int64_t full = pre < 0 ? 0 : pre >> P.shift;
  const int n = (int)(full < P.cols ? full : P.cols);
  int32_t* const out = P.blocks + row * P.count;
  if (n <= P.count) {
    for (int i = tid; i < P.count; i += NT) out[i] = i < n ? i : -1;
    return;
  }
  const int c0 = P.first, c1 = n - P.last;  // the candidates
  uint32_t key[PER];
  uint32_t lo = ~0u, hi = 0u;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int j = i * NT + tid;
    key[i] = 0;
    if (j >= c0 && j < c1) {
      const float v = score[i];
      key[i] = f32_key(v == v ? v : -INFINITY);
      lo = key[i] < lo ? key[i] : lo;
      hi = key[i] > hi ? key[i] : hi;
    }
  }
  uint32_t need = (uint32_t)(P.count - P.first - P.last), left = (uint32_t)(c1 - c0);
  // chosen: above `tkey`, or equal to it at an index up to `tidx`
  uint32_t tkey = ~0u;
  int tidx = -1;
  if (need) {
    lo = ~wave_max_u32(~lo);
    hi = wave_max_u32(hi);
    if (lane == 0) s_red[0][wave] = lo, s_red[1][wave] = hi;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      lo = s_red[0][w] < lo ? s_red[0][w] : lo;
      hi = s_red[1][w] > hi ? s_red[1][w] : hi;
    }
    bool ties = false;  // the values are now the indices, turned round, of the keys that equal tkey
    auto value = [&](int i) { return ties ? (key[i] == tkey ? ~(uint32_t)(i * NT + tid) : 0u) : key[i]; };
    while (true) {
      if (left == need) {  // all that is left
        if (ties)
          tidx = (int)~lo;
        else
          tkey = lo, tidx = 0x7fffffff;
        break;
      }
      if (left <= WAVE) {
        if (tid == 0) s_n = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const uint32_t v = value(i);
          if (v >= lo && v <= hi && v) {
            const int at = atomicAdd(&s_n, 1);
            if (at < WAVE) s_val[at] = v, s_idx[at] = i * NT + tid;
          }
        }
        __syncthreads();
        if (wave == 0) {
          const int held = s_n < WAVE ? s_n : WAVE;
          const uint32_t v = lane < held ? s_val[lane] : 0u;
          const int idx = lane < held ? s_idx[lane] : 0x7fffffff;
          uint32_t before = 0;
          for (int k = 0; k < held; ++k) {
            const uint32_t u = s_val[k];
            before += u > v || (u == v && s_idx[k] < idx);
          }
          if (lane < held && before == need - 1) s_found[0] = v, s_found[1] = (uint32_t)idx;
        }
        __syncthreads();
        if (!ties) tkey = s_found[0];
        tidx = (int)s_found[1];
        break;
      }
      if (lo == hi) {  // (more equal keys than a wave ranks)
        ties = true;
        tkey = lo;
        lo = ~(uint32_t)(n - 1);
        hi = ~0u;
      }
      const uint32_t range = hi - lo;
      const int bits = 32 - __builtin_clz(range), s = bits > 8 ? bits - 8 : 0;
      for (int i = tid; i < 256; i += NT) s_hist[i] = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const uint32_t v = value(i);
        if (v >= lo && v <= hi && v) atomicAdd(&s_hist[(v - lo) >> s], 1u);
      }
      __syncthreads();
      if (wave == 0) {  // from the top: lane l has the bins 255 - 4 l and the three below
        uint32_t bin[4], sum = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) bin[k] = s_hist[255 - 4 * lane - k], sum += bin[k];
        const uint32_t upto = wave_incl_scan(sum);
        uint32_t above = upto - sum;
        if (above < need && upto >= need) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (above < need && above + bin[k] >= need) s_found[0] = (uint32_t)(255 - 4 * lane - k), s_found[1] = above, s_found[2] = bin[k];
            above += bin[k];
          }
        }
      }
      __syncthreads();
      const uint32_t from = lo + (s_found[0] << s), most = from + ((1u << s) - 1u);
      need -= s_found[1];
      left = s_found[2];
      hi = most < hi && most >= from ? most : hi;
      lo = from;
      __syncthreads();  // (before s_found and s_hist are written again)
    }
  }
  uint32_t chosen = 0;  // bit i: this thread's index i
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int j = i * NT + tid;
    const bool yes = j < n && (j < c0 || j >= c1 || key[i] > tkey || (key[i] == tkey && j <= tidx));
    chosen |= (yes ? 1u : 0u) << i;
    const uint64_t all = __ballot(yes);
    if (lane == 0) s_count[i * NW + wave] = __popcll(all);
  }
  __syncthreads();
  if (wave == 0) {
    int before = 0;
    for (int k = 0; k < PER * NW; k += WAVE) {
      const int v = k + lane < PER * NW ? s_count[k + lane] : 0;
      const int upto = wave_incl_scan(v);
      if (k + lane < PER * NW) s_count[k + lane] = before + upto - v;
      before += readlane<WAVE - 1>(upto);
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const bool yes = (chosen >> i) & 1;
    const uint64_t all = __ballot(yes);
    if (yes) {
      const int at = s_count[i * NW + wave] + __popcll(all & ((1ull << lane) - 1));
      if (at < P.count) out[at] = i * NT + tid;
    }
  }
}

static int check_index(const char* what, const dsv_block_index& x) {
  if (!x.bounds || (uintptr_t)x.bounds % 16) DSV_FAIL(DSV_ERR_INVALID, "%s: the index's bounds are required, 16-byte aligned", what);
  if (x.dtype != DSV_BF16 && x.dtype != DSV_F16) DSV_FAIL(DSV_ERR_INVALID, "%s: unknown index type %d", what, x.dtype);
  if (x.heads < 1 || x.heads > 65535 || x.rows < 1 || x.dim < 16 || x.dim > 256 || x.dim % 16)
    DSV_FAIL(DSV_ERR_INVALID, "%s: an index needs rows, heads and a dim that is a multiple of 16 up to 256 (got %lld, %d, %d)",
             what, (long long)x.rows, x.heads, x.dim);
  if (x.block_size != 16 && x.block_size != 32 && x.block_size != 64 && x.block_size != 128)
    DSV_FAIL(DSV_ERR_INVALID, "%s: a block has 16, 32, 64 or 128 positions (got %d)", what, x.block_size);
  return DSV_OK;
}

}  // namespace dsv

using namespace dsv;

extern "C" int dsv_index_blocks(const dsv_block_index* index, const dsv_kv_cache* cache, const int32_t* page_table,
                                int64_t page_stride, int64_t page_cols, const int32_t* block_table, int64_t block_stride,
                                int64_t block_cols, const int32_t* from_lens, const int32_t* to_lens, int32_t bs,
                                int64_t longest, dsv_stream_t stream_) {
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  if (!index) DSV_FAIL(DSV_ERR_INVALID, "dsv_index_blocks: no index");
  int rc = check_index("dsv_index_blocks", *index);
  if (rc == DSV_OK) rc = check_cache("dsv_index_blocks", cache);
  if (rc != DSV_OK) return rc;
  if (index->heads != cache->heads || index->dim != cache->dim)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_index_blocks: the index and the cache must have the same heads and dim");
  if (bs < 0 || longest < 0) DSV_FAIL(DSV_ERR_INVALID, "dsv_index_blocks: invalid layout (bs %d, longest %lld)", bs, (long long)longest);
  if (bs == 0 || longest == 0) return DSV_OK;
  if (!page_table || !block_table || !from_lens || !to_lens || page_cols < 1 || block_cols < 1)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_index_blocks: tables and lengths are required");
  IndexParams P{*index, *cache, page_table, block_table, from_lens, to_lens, page_stride, page_cols, block_stride, block_cols, bs, 0, 0};
  P.shift = __builtin_ctz((unsigned)index->block_size);
  int64_t most = longest > 0x7fffffff ? 0x7fffffff : longest;
  most = (most + index->block_size - 1) >> P.shift;  // (a growth of n positions finishes ceil(n / size) blocks at most)
  if (most > block_cols) most = block_cols;
  const int64_t units = most * bs * cache->heads, grid = (units + BI_THREADS / WAVE - 1) / (BI_THREADS / WAVE);
  if (units > 0x7fffffffll) DSV_FAIL(DSV_ERR_INVALID, "dsv_index_blocks: too many blocks for one call");
  P.most = (int)most;
  const bool bf = index->dtype == DSV_BF16;
  auto to = [&](auto ct, auto g) {
    auto launch = [&](auto kern) { hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(BI_THREADS), 0, stream, P); };
    constexpr int CT = decltype(ct)::value, G = decltype(g)::value;
    bf ? launch(k_index_blocks<CT, DSV_BF16, G>) : launch(k_index_blocks<CT, DSV_F16, G>);
  };
  // (lanes of a row)
  auto width = [&](auto ct) {
    constexpr int CT = decltype(ct)::value, EL = CT == DSV_E4M3 || CT == DSV_I8 ? 16 : 8;
    const int lanes = (cache->dim + EL - 1) / EL;
    if constexpr (EL == 8)
      if (lanes > 16) return to(ct, Int<32>{});
    lanes > 8 ? to(ct, Int<16>{}) : (lanes > 4 ? to(ct, Int<8>{}) : to(ct, Int<4>{}));
  };
  if (cache->dtype == DSV_BF16)
    width(Int<DSV_BF16>{});
  else if (cache->dtype == DSV_F16)
    width(Int<DSV_F16>{});
  else if (cache->dtype == DSV_E4M3)
    width(Int<DSV_E4M3>{});
  else
    width(Int<DSV_I8>{});
  DSV_CHECK_LAUNCH("k_index_blocks");
  return DSV_OK;
}

extern "C" int dsv_score_blocks(const dsv_score_blocks_args* args, dsv_stream_t stream_) {
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  if (!args) DSV_FAIL(DSV_ERR_INVALID, "dsv_score_blocks: no arguments");
  const dsv_score_blocks_args& a = *args;
  const int rc = check_index("dsv_score_blocks", a.index);
  if (rc != DSV_OK) return rc;
  if (a.bs < 1 || a.T < 1 || a.T > 64 || a.rows < 0 || (!a.row_offsets && a.rows != (int64_t)a.bs * a.T))
    DSV_FAIL(DSV_ERR_INVALID, "dsv_score_blocks: invalid layout (bs %d, T %d, rows %lld)", a.bs, a.T, (long long)a.rows);
  if (a.q_heads < 1 || a.q_heads % a.index.heads || a.q_heads > 65535)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_score_blocks: %d query heads over %d index heads", a.q_heads, a.index.heads);
  if (!(a.scale > 0.f && a.scale <= 0x1p100f)) DSV_FAIL(DSV_ERR_INVALID, "dsv_score_blocks: scale must be positive, at most 2^100");
  if (!a.scores || !a.prefix_lens || !a.block_table || a.block_cols < 1 || a.block_cols > 0x7ffffff || (a.rows && !a.q))
    DSV_FAIL(DSV_ERR_INVALID, "dsv_score_blocks: q, scores, prefix_lens and a block table are required");
  if ((uintptr_t)a.q % 16 || a.q_row_stride % 8 || a.q_head_stride % 8)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_score_blocks: rows of q must start on 16-byte boundaries");
  ScoreParams P;
  P.a = a;
  P.G = fast_div((uint32_t)(a.q_heads / a.index.heads));
  P.shift = __builtin_ctz((unsigned)a.index.block_size);
  const int64_t bh = (int64_t)a.bs * a.index.heads;
  const int tiles = (a.T * (int)P.G.d + 15) / 16, pieces = a.index.dim <= 64 ? 2 : (a.index.dim <= 128 ? 4 : 8);
  P.staged = tiles < SB_STAGE / pieces ? tiles : SB_STAGE / pieces;
  // Waves of a workgroup, replayed, us, four and eight (16 requests, 32k positions at dim 128): queries of 16 KB (128 rows of dim 64,
  // 32 of 256) 20.0 and 19.4, 15.6 and 17.4; 20 KB (68 of 128) 16.6 and 17.0; 24 KB (96 of 128, 48 of 256) 17.3 and 17.1, 16.6 and 16.9;
  // 32 KB (256 of 64, 128 of 128, 64 of 256) 26.4 and 24.3, 18.6 and 17.8, 17.6 and 17.2; 56 to 60 KB (480, 240, 112) 44.0 and 32.9, 27.6
  // and 22.1, 20.6 and 19.2: eight where LDS holds few workgroups.
  const bool many = P.staged * pieces > 24;
  const int step = (many ? SB_MANY : SB_WAVES) * 16;
  const int64_t steps = (a.block_cols + step - 1) / step;
  const int64_t per = steps * bh / (many ? 2048 : 4096);  // (half and twice as many workgroups: 44 and 42 us for 41)
  P.steps = (int)(per < 1 ? 1 : (per > SB_STEPS ? SB_STEPS : per));
  P.chunks = (int)((steps + P.steps - 1) / P.steps);
  if (bh * P.chunks > 0x7fffffffll) DSV_FAIL(DSV_ERR_INVALID, "dsv_score_blocks: too many blocks for one call");
  auto launch = [&](auto few, auto more) {
    hipLaunchKernelGGL(many ? more : few, dim3((unsigned)(bh * P.chunks)), dim3((many ? SB_MANY : SB_WAVES) * WAVE),
                       (unsigned)(P.staged * pieces) * 1024u, stream, P);
  };
  auto type = [&](auto it) {
    constexpr int IT = decltype(it)::value;
    const int D = a.index.dim;
    auto width = [&](auto nc, auto full) {
      constexpr int NC = decltype(nc)::value;
      constexpr bool FULL = decltype(full)::value;
      launch(k_score_blocks<IT, NC, FULL, SB_WAVES>, k_score_blocks<IT, NC, FULL, SB_MANY>);
    };
    if (D <= 64)
      D == 64 ? width(Int<2>{}, Int<1>{}) : width(Int<2>{}, Int<0>{});
    else if (D <= 128)
      D == 128 ? width(Int<4>{}, Int<1>{}) : width(Int<4>{}, Int<0>{});
    else
      D == 256 ? width(Int<8>{}, Int<1>{}) : width(Int<8>{}, Int<0>{});
  };
  a.index.dtype == DSV_BF16 ? type(Int<DSV_BF16>{}) : type(Int<DSV_F16>{});
  DSV_CHECK_LAUNCH("k_score_blocks");
  return DSV_OK;
}

extern "C" int dsv_select_blocks(const float* scores, int32_t bs, int32_t heads, int64_t cols, const int32_t* prefix_lens,
                                 int32_t block_size, int32_t count, int32_t first, int32_t last, int32_t* blocks,
                                 dsv_stream_t stream_) {
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  if (bs < 1 || heads < 1 || heads > 65535 || cols < 1 || cols > 32768)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_select_blocks: 1 to 32768 blocks of a request are ranked (bs %d, heads %d, blocks %lld)", bs,
             heads, (long long)cols);
  if (block_size != 16 && block_size != 32 && block_size != 64 && block_size != 128)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_select_blocks: a block has 16, 32, 64 or 128 positions (got %d)", block_size);
  if (count < 1 || first < 0 || last < 0 || (int64_t)first + last > count)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_select_blocks: count %d has to hold the first %d and the last %d", count, first, last);
  if (!scores || !prefix_lens || !blocks) DSV_FAIL(DSV_ERR_INVALID, "dsv_select_blocks: null pointer");
  const int64_t rows = (int64_t)bs * heads;
  if (rows > 0x7fffffffll || rows * count > (1ll << 40)) DSV_FAIL(DSV_ERR_INVALID, "dsv_select_blocks: too many rows for one call");
  SelectParams P{scores, prefix_lens, blocks, cols, heads, __builtin_ctz((unsigned)block_size), count, first, last};
  auto launch = [&](auto kern, int waves) { hipLaunchKernelGGL(kern, dim3((unsigned)rows), dim3((unsigned)(waves * WAVE)), 0, stream, P); };
  if (cols <= 512)
    launch(k_select_blocks<1, 8>, 1);
  else if (cols <= 2048)
    launch(k_select_blocks<4, 8>, 4);
  else if (cols <= 8192)
    launch(k_select_blocks<16, 8>, 16);
  else
    launch(k_select_blocks<16, 32>, 16);
  DSV_CHECK_LAUNCH("k_select_blocks");
  return DSV_OK;
}
