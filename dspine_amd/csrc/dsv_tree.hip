// A drafted tree's masks, its greedy acceptance and the commit of an accepted path for gfx950.  A tree has at
// most 64 nodes: a node is a lane, a set of nodes a 64-bit mask.
#include "dsv_common.h"

namespace dsv {

constexpr int TREE_MAX = 64;

// The parent of the lane's node: -1 where it has none before it.
__device__ __forceinline__ int tree_parent(const int32_t* parents, int T, int i) {
  const int p = i > 0 && i < T ? parents[i] : -1;
  return p >= 0 && p < i ? p : -1;
}

// Node i and its ancestors as bits, by doubling: after s rounds a lane's mask covers its 2^s nearest ancestors
// and its link skips them.
__device__ __forceinline__ uint64_t tree_mask(int parent, int lane) {
  uint64_t m = 1ull << lane;
  int link = parent;
  for (int s = 1; s < TREE_MAX; s *= 2) {
    const uint64_t up = __shfl((unsigned long long)m, link < 0 ? lane : link, WAVE);
    const int next = __shfl(link, link < 0 ? lane : link, WAVE);
    if (link >= 0) {
      m |= up;
      link = next;
    }
  }
  return m;
}

__global__ __launch_bounds__(256) void k_tree_masks(const int32_t* parents, int bs, int T, int64_t* masks,
                                                    int32_t* depths) {
  const int64_t b = (int64_t)blockIdx.x * (256 / WAVE) + threadIdx.x / WAVE;
  const int lane = threadIdx.x & (WAVE - 1);
  if (b >= bs) return;
  const uint64_t m = tree_mask(tree_parent(parents + b * T, T, lane), lane);
  if (lane < T) {
    masks[b * T + lane] = (int64_t)m;
    if (depths) depths[b * T + lane] = __popcll(m) - 1;
  }
}

// The largest logit of a piece of a row as (value key, ~id): the maximum is the row's first argmax.  One pass over
// the logits, bound by memory: 16-byte vectors of the row's aligned part, TA_VECS in flight a thread; a thread keeps
// its best vector and looks into it at the end (with a key for every logit the pass ran at 1.5 TB/s).  Rows at or
// past their request's length are not read.  A NaN counts as -infinity wherever it lies.  64 requests of up to 17 rows of 151936
// bf16 logits (204 MB): 37.1 us, 5.5 TB/s.  (The greedy chain's chunk pass keeps statistics for its walk and reads every
// row of the window: with it 64 requests of 4 to 17 rows would take 59 us for 45 with this one, full windows 61 for 66.)
constexpr int TA_THREADS = 256;
constexpr int TA_VECS = 8;

template <int DT>
__host__ __device__ constexpr int ta_per() {
  return DT == DSV_BF16 ? 8 : 4;  // logits of a vector
}
template <int DT>
__host__ __device__ constexpr int64_t ta_piece() {
  return (int64_t)TA_THREADS * TA_VECS * ta_per<DT>();
}

// (quieted: the maximum of a number and a signalling NaN is a NaN, and the number lost; 37.1 us for 36.7 without)
template <int DT>
__device__ __forceinline__ float ta_value(const uint4& v, int i) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if constexpr (DT == DSV_BF16)
    return __builtin_canonicalizef(__uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16));
  else
    return __builtin_canonicalizef(__uint_as_float(w[i]));
}
__device__ __forceinline__ uint64_t ta_key(float x, uint32_t id) { return ((uint64_t)f32_key(x) << 32) | (uint32_t)~id; }

template <int DT>
__global__ __launch_bounds__(TA_THREADS) void k_tree_argmax(const void* logits, int64_t vocab, int64_t stride, int T,
                                                            const int32_t* lens, int C, uint64_t* best) {
  using elem = typename std::conditional<DT == DSV_BF16, uint16_t, uint32_t>::type;
  constexpr int PER = ta_per<DT>();
  __shared__ uint64_t s_best[TA_THREADS / WAVE];
  const int row = (int)(blockIdx.x / (unsigned)C), c = (int)(blockIdx.x - (unsigned)row * (unsigned)C);
  if (lens) {
    const int b = row / T, i = row - b * T;
    if (i > 0 && i >= lens[b]) return;
  }
  const elem* x = reinterpret_cast<const elem*>(logits) + row * stride;
  const int tid = threadIdx.x;
  // logits before the first 16-byte boundary, whole vectors, logits behind them
  int lead = (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(elem);
  lead = lead < vocab ? lead : (int)vocab;
  const int vecs = (int)((vocab - lead) / PER);
  const uint4* v = reinterpret_cast<const uint4*>(x + lead);
  uint4 got[TA_VECS];
  const int first = c * TA_THREADS * TA_VECS + tid;
#pragma unroll
  for (int u = 0; u < TA_VECS; ++u) {
    const int i = first + u * TA_THREADS;
    if (i < vecs) got[u] = v[i];
  }
  float top = -INFINITY;
  int at = -1;
  uint4 which = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int u = 0; u < TA_VECS; ++u) {
    const int i = first + u * TA_THREADS;
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < PER; ++k) m = fmaxf(m, ta_value<DT>(got[u], k));
    if (i < vecs && (m > top || at < 0)) {
      top = m;
      at = i;
      which = got[u];
    }
  }
  uint64_t key = 0;
  if (at >= 0) {
#pragma unroll
    for (int k = PER - 1; k >= 0; --k)  // (the first of equal ones is left)
      if (fmaxf(ta_value<DT>(which, k), -INFINITY) == top) key = ta_key(top, (uint32_t)(lead + at * PER + k));
  }
  if (c == 0) {  // the row's ends
    const int behind = (int)(vocab - lead) - vecs * PER;
    if (tid < lead + behind) {
      const int id = tid < lead ? tid : (int)vocab - behind + (tid - lead);
      const float y = fmaxf(__builtin_canonicalizef(DT == DSV_BF16 ? bf16_bits_to_f32(x[id]) : __uint_as_float(x[id])), -INFINITY);
      const uint64_t k = ta_key(y, (uint32_t)id);
      key = k > key ? k : key;
    }
  }
  key = block_max_u64<TA_THREADS / WAVE>(key, s_best);
  if (tid == 0) best[(int64_t)row * C + c] = key;
}

// The walk, without walking: node i fits when its token is its parent's argmax, no sibling before it carries the
// same token, and it lies within the request's length; it is on the path when it and all its ancestors fit.
// One workgroup a request: G lanes a row join the row's pieces, then one wave has a node a lane.  Bound by latency:
// 4.5 us.
constexpr int TW_THREADS = 1024;
__global__ __launch_bounds__(TW_THREADS) void k_tree_accept(const uint64_t* best, int C, int G, int T,
                                                            const int64_t* cand, const int32_t* parents,
                                                            const int32_t* lens, const int32_t* prefix,
                                                            int32_t* accept, int32_t* commit, int64_t* bonus,
                                                            int64_t* output, int32_t* new_seq, int32_t* path) {
  __shared__ int32_t s_top[TREE_MAX];
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, l = tid & (G - 1);
  int n = lens ? lens[b] : T;
  n = n < 1 ? 1 : (n > T ? T : n);
  for (int i = tid / G; i < n; i += blockDim.x / G) {
    uint64_t m = 0;
    for (int c = l; c < C; c += G) {
      const uint64_t k = best[(b * T + i) * C + c];
      m = k > m ? k : m;
    }
    for (int o = G / 2; o; o /= 2) {
      const uint64_t t = __shfl_xor((unsigned long long)m, o, WAVE);
      m = t > m ? t : m;
    }
    if (l == 0) s_top[i] = (int32_t) ~(uint32_t)m;
  }
  const int i = tid;
  const int64_t tok = i < T ? cand[b * T + i] : -1;
  const int par = i < TREE_MAX ? tree_parent(parents + b * T, T, i) : -1;
  __syncthreads();
  if (tid >= WAVE) return;
  bool fits = i == 0 || (i < n && par >= 0 && tok == (int64_t)s_top[par < 0 ? 0 : par]);
  for (int j = 1; j < n; ++j) {
    const int64_t t = readlane_at(tok, j);
    const int p = readlane_at(par, j);
    if (j < i && p == par && t == tok) fits = false;
  }
  const uint64_t ok = __ballot(fits);
  const uint64_t mine = tree_mask(par, i);
  const uint64_t on = __ballot((mine & ~ok) == 0 && (mine & 1ull));
  const int count = __popcll(on), last = 63 - __clzll((long long)on);
  const int64_t bon = s_top[last];
  // the path's nodes to the first lanes, the others behind them
  const uint64_t below = (1ull << i) - 1ull;
  const int place = (on >> i) & 1 ? __popcll(on & below) : count + __popcll(~on & below);
  const int node = __builtin_amdgcn_ds_permute(place * 4, i);
  const int after = __shfl(node, i + 1 < WAVE ? i + 1 : i, WAVE);
  const int64_t next = __shfl((long long)tok, after, WAVE);
  if (i < T) {
    path[b * T + i] = i < count ? node : -1;
    output[b * T + i] = i < count - 1 ? next : (i == count - 1 ? bon : 0);
  }
  if (i == 0) {
    accept[b] = count - 1;
    commit[b] = count;
    bonus[b] = bon;
    new_seq[b] = prefix[b] + count;
  }
}

__device__ __forceinline__ int64_t load_i(const void* p, int i64, int64_t i) {
  return i64 ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t) reinterpret_cast<const int32_t*>(p)[i];
}

// The commit of the accepted paths: one workgroup, requests in contiguous ranges a thread, a block scan places
// each request's freed slots (as the chain's commit does).  The path of a tree ascends, so its slots can be moved down inside
// the table one after the other; a caller's own order is left to the wave, an entry a lane, so that it is read whole before the
// first position is written (an array of the thread's own cost every call scratch memory: 8.9 us for 8.4 at 64 requests of
// 17 nodes; 8.1 where no order is kept).
constexpr int CT_THREADS = 1024;
__global__ __launch_bounds__(CT_THREADS) void k_commit_tree(int bs, int T, const int32_t* accept, const int32_t* path,
                                                            const int32_t* verify_lens, const void* prefix_lens,
                                                            int prefix_i64, const void* req_pool, int req_i64,
                                                            int32_t* req_to_token, int64_t rt_stride, int64_t rt_cols,
                                                            const int64_t* out_cache_loc, const int64_t* slot_offsets,
                                                            void* seq_lens, int seq_i64, int64_t* free_slots,
                                                            int32_t* free_count) {
  __shared__ int32_t sred[CT_THREADS / WAVE];
  const int tid = threadIdx.x;
  const int per = (bs + CT_THREADS - 1) / CT_THREADS;
  const int b0 = tid * per < bs ? tid * per : bs, b1 = b0 + per < bs ? b0 + per : bs;
  // the request's nodes n, its commit c (clamped into [1, n]), the nodes that are kept, and whether the path names them in
  // ascending order
  auto of = [&](int b, int& n, int& c, bool& rises) {
    n = verify_lens ? verify_lens[b] : T;
    n = n < 1 ? 1 : (n > T ? T : n);
    c = accept[b] + 1;
    c = c < 1 ? 1 : (c > n ? n : c);
    uint64_t kept = 0;
    rises = true;
    for (int i = 0; i < c; ++i) {
      const int node = path[(int64_t)b * T + i];
      const uint64_t bit = node >= 0 && node < n ? 1ull << node : 0ull;
      rises &= bit == 0 || kept < bit;  // (none at or past it so far)
      kept |= bit;
    }
    return kept;
  };
  int mine = 0;
  for (int b = b0; b < b1; ++b) {
    int n, c;
    bool rises;
    const uint64_t kept = of(b, n, c, rises);
    mine += n - __popcll(kept);
  }
  int total = 0;
  int at = block_excl_scan<CT_THREADS / WAVE>(mine, sred, &total);
  // a request's table row and window: node's slot, and a slot to the i-th of its new positions
  struct Window {
    int64_t row, pre, base, cols;
    int32_t* rt;
    const int64_t* loc;
    __device__ __forceinline__ int64_t slot_of(int node) const {
      if (loc) return loc[base + node];
      const int64_t pos = pre + node;
      return pos >= 0 && pos < cols ? (int64_t)rt[pos] : -1;
    }
    __device__ __forceinline__ void write(int i, int64_t slot) const {
      const int64_t pos = pre + i;
      if (pos >= 0 && pos < cols) rt[pos] = (int32_t)slot;
    }
  };
  auto window_of = [&](int b) {
    const int64_t row = load_i(req_pool, req_i64, b), pre = load_i(prefix_lens, prefix_i64, b);
    return Window{row, pre, slot_offsets ? slot_offsets[b] : (int64_t)b * T, rt_cols, req_to_token + row * rt_stride, out_cache_loc};
  };
  for (int step = 0; step < per; ++step) {
    const int b = b0 + step;
    int n = 0, c = 0;
    bool rises = true;
    if (b < b1) {
      const uint64_t kept = of(b, n, c, rises);
      const Window w = window_of(b);
      if (free_slots)  // (before the table changes: the slots may be read from it)
        for (int i = 0; i < n; ++i)
          if (!((kept >> i) & 1)) free_slots[at++] = w.slot_of(i);
      // kept nodes in ascending order: a position is written after every read at or before it
      int i = 0;
      if (rises)
        for (uint64_t left = kept; left; left &= left - 1, ++i) w.write(i, w.slot_of(__ffsll((unsigned long long)left) - 1));
      if (seq_lens) {
        const int64_t len = w.pre + __popcll(kept);
        if (seq_i64)
          reinterpret_cast<int64_t*>(seq_lens)[w.row] = len;
        else
          reinterpret_cast<int32_t*>(seq_lens)[w.row] = (int32_t)len;
      }
    }
    const int lane = tid & (WAVE - 1);
    for (uint64_t odd = __ballot(!rises); odd; odd &= odd - 1) {
      const int from = __ffsll((unsigned long long)odd) - 1, rb = readlane_at(b, from), rn = readlane_at(n, from),
                rc = readlane_at(c, from);
      const int node = lane < rc ? path[(int64_t)rb * T + lane] : -1;
      bool take = node >= 0 && node < rn;
      for (int j = 0; j < rc; ++j) {
        const int other = readlane_at(node, j);
        if (j < lane && other == node) take = false;
      }
      const Window w = window_of(rb);
      const uint64_t taken = __ballot(take);
      const int64_t slot = take ? w.slot_of(node) : 0;
      __builtin_amdgcn_wave_barrier();  // (every lane's slot has been asked for before any position is written)
      if (take) w.write(__popcll(taken & ((1ull << lane) - 1ull)), slot);
    }
  }
  if (tid == 0 && free_count) *free_count = total;
}

static int ta_chunks(int64_t vocab, int dtype) {
  const int64_t p = dtype == DSV_BF16 ? ta_piece<DSV_BF16>() : ta_piece<DSV_F32>();
  return (int)((vocab + p - 1) / p);
}

}  // namespace dsv

using namespace dsv;

extern "C" int dsv_tree_masks(const int32_t* parents, int32_t bs, int32_t T, int64_t* masks, int32_t* depths,
                              dsv_stream_t stream_) {
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  if (bs < 0 || T < 1 || T > TREE_MAX) DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_masks: invalid layout (bs %d, T %d)", bs, T);
  if (bs == 0) return DSV_OK;
  if (!parents || !masks) DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_masks: null pointer");
  hipLaunchKernelGGL(k_tree_masks, dim3((unsigned)((bs + 3) / 4)), dim3(256), 0, stream, parents, bs, T, masks, depths);
  DSV_CHECK_LAUNCH("k_tree_masks");
  return DSV_OK;
}

extern "C" int64_t dsv_tree_verify_workspace_bytes(int64_t rows, int64_t vocab) {
  // (the float32 pieces are the smaller ones)
  return rows > 0 && vocab > 0 ? rows * ta_chunks(vocab, DSV_F32) * (int64_t)sizeof(uint64_t) : 0;
}

extern "C" int dsv_tree_verify(const void* logits, int32_t dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                               int32_t bs, int32_t T, const int64_t* candidates, const int32_t* parents,
                               const int32_t* verify_lens, const int32_t* prefix_lens, int32_t* accept,
                               int32_t* commit, int64_t* bonus, int64_t* output, int32_t* new_seq, int32_t* path,
                               void* workspace, int64_t workspace_bytes, dsv_stream_t stream_) {
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  if (bs < 1 || T < 1 || T > TREE_MAX || rows != (int64_t)bs * T)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_verify: invalid layout (bs %d, T %d, rows %lld)", bs, T, (long long)rows);
  if (dtype != DSV_BF16 && dtype != DSV_F32) DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_verify: unknown logits type %d", dtype);
  if (vocab < 1 || vocab > (int64_t)1 << 30 || row_stride < vocab)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_verify: invalid vocab %lld or row stride %lld", (long long)vocab,
             (long long)row_stride);
  if (!logits || !candidates || !parents || !prefix_lens || !accept || !commit || !bonus || !output || !new_seq ||
      !path || !workspace)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_verify: required pointer is null");
  const int C = ta_chunks(vocab, dtype);
  if (rows * C > 0x7fffffffll) DSV_FAIL(DSV_ERR_INVALID, "dsv_tree_verify: too many rows for one call");
  if (workspace_bytes < rows * C * (int64_t)sizeof(uint64_t))
    DSV_FAIL(DSV_ERR_WORKSPACE, "dsv_tree_verify: workspace %lld < %lld", (long long)workspace_bytes,
             (long long)(rows * C * (int64_t)sizeof(uint64_t)));
  uint64_t* best = reinterpret_cast<uint64_t*>(workspace);
  auto argmax = dtype == DSV_BF16 ? k_tree_argmax<DSV_BF16> : k_tree_argmax<DSV_F32>;
  hipLaunchKernelGGL(argmax, dim3((unsigned)(rows * C)), dim3(TA_THREADS), 0, stream, logits, vocab, row_stride, T,
                     verify_lens, C, best);
  DSV_CHECK_LAUNCH("k_tree_argmax");
  int G = 1;  // lanes a row
  while (G < C && G < WAVE) G *= 2;
  int threads = T * G;
  threads = threads < WAVE ? WAVE : (threads > TW_THREADS ? TW_THREADS : (threads + WAVE - 1) / WAVE * WAVE);
  hipLaunchKernelGGL(k_tree_accept, dim3((unsigned)bs), dim3(threads), 0, stream, best, C, G, T, candidates, parents,
                     verify_lens, prefix_lens, accept, commit, bonus, output, new_seq, path);
  DSV_CHECK_LAUNCH("k_tree_accept");
  return DSV_OK;
}

extern "C" int dsv_commit_tree(int32_t bs, int32_t T, const int32_t* accept, const int32_t* path,
                               const int32_t* verify_lens, const void* prefix_lens, int32_t prefix_i64,
                               const void* req_pool_indices, int32_t req_pool_i64, int32_t* req_to_token,
                               int64_t rt_stride, int64_t rt_cols, const int64_t* out_cache_loc,
                               const int64_t* slot_offsets, void* seq_lens, int32_t seq_lens_i64, int64_t* free_slots,
                               int32_t* free_count, dsv_stream_t stream_) {
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  if (bs < 0 || T < 1 || T > TREE_MAX) DSV_FAIL(DSV_ERR_INVALID, "dsv_commit_tree: invalid layout (bs %d, T %d)", bs, T);
  if (bs > 0 && (!accept || !path || !prefix_lens || !req_pool_indices || !req_to_token || rt_cols < 1 ||
                 rt_stride < rt_cols))
    DSV_FAIL(DSV_ERR_INVALID, "dsv_commit_tree: accept, path, prefix_lens, req_pool_indices and req_to_token are required");
  hipLaunchKernelGGL(k_commit_tree, dim3(1), dim3(CT_THREADS), 0, stream, bs, T, accept, path, verify_lens,
                     prefix_lens, prefix_i64, req_pool_indices, req_pool_i64, req_to_token, rt_stride, rt_cols,
                     out_cache_loc, slot_offsets, seq_lens, seq_lens_i64, free_slots, free_count);
  DSV_CHECK_LAUNCH("k_commit_tree");
  return DSV_OK;
}
