// The life of a cache's pages around the rounds, for gfx950: requests forked from others whose slots they then share,
// requests that end, a fragmented pool compacted, rows of slots copied.  A page is a slot (page size 1); shared[slot] counts
// the requests beyond the first that hold it, so slots that nobody shares need no entry of their own.
#include "dsv_cache.h"
#include "dsv_common.h"

namespace dsv {

constexpr int RQ_THREADS = 256;
constexpr int RQ_CHUNK = RQ_THREADS * 16;  // slots of a workgroup that walks the pool

// The entries that a row of the table holds.
__device__ __forceinline__ int64_t held(const void* lens, int i64, int64_t row, int64_t cols) {
  const int64_t n = load_index(lens, i64, row);
  return n < 0 ? 0 : (n > cols ? cols : n);
}
__device__ __forceinline__ void set_len(void* lens, int i64, int64_t row, int64_t n) {
  if (i64)
    reinterpret_cast<int64_t*>(lens)[row] = n;
  else
    reinterpret_cast<int32_t*>(lens)[row] = (int32_t)n;
}

struct TableParams {
  int32_t* table;
  int64_t rows, stride, cols;
  void* lens;
  int lens_i64, rows_i64;
  const void* at;  // the rows of the call (a fork's parents)
  int64_t n, num_slots;
  int32_t* shared;
  int64_t chunks;
};

// A workgroup a (pair, 256 columns).  Pairs of one parent in a row count its slots together, the first for all.
__global__ __launch_bounds__(RQ_THREADS) void k_fork(TableParams P, const void* children) {
  const int64_t i = blockIdx.x / P.chunks, chunk = blockIdx.x - i * P.chunks;
  auto pair = [&](int64_t k, int64_t& parent, int64_t& child) {
    parent = load_index(P.at, P.rows_i64, k);
    child = load_index(children, P.rows_i64, k);
    return parent >= 0 && parent < P.rows && child >= 0 && child < P.rows && child != parent;
  };
  int64_t parent, child, other, unused;
  if (!pair(i, parent, child)) return;
  const int64_t len = held(P.lens, P.lens_i64, parent, P.cols), p = chunk * RQ_THREADS + threadIdx.x;
  if (p == 0) set_len(P.lens, P.lens_i64, child, len);
  if (chunk * RQ_THREADS >= len) return;
  int times = 1;
  if (i > 0 && pair(i - 1, other, unused) && other == parent)
    times = 0;
  else
    while (i + times < P.n && pair(i + times, other, unused) && other == parent) ++times;
  if (p >= len) return;
  const int32_t slot = P.table[parent * P.stride + p];
  P.table[child * P.stride + p] = slot;
  if (times && slot >= 0 && slot < P.num_slots) atomicAdd(&P.shared[slot], times);
}

// A workgroup a (row, 256 columns); a row named before is left out.
__global__ __launch_bounds__(RQ_THREADS) void k_release(TableParams P) {
  const int64_t i = blockIdx.x / P.chunks, chunk = blockIdx.x - i * P.chunks;
  const int64_t row = load_index(P.at, P.rows_i64, i);
  if (row < 0 || row >= P.rows) return;
  const int64_t len = held(P.lens, P.lens_i64, row, P.cols), p = chunk * RQ_THREADS + threadIdx.x;
  if (chunk * RQ_THREADS >= len) return;
  bool again = false;
  for (int64_t k = threadIdx.x; k < i; k += RQ_THREADS) again |= load_index(P.at, P.rows_i64, k) == row;
  if (__syncthreads_or(again) || p >= len) return;
  const int32_t slot = P.table[row * P.stride + p];
  if (slot >= 0 && slot < P.num_slots) atomicSub(&P.shared[slot], 1);
}

// Slots below zero in each chunk of the pool; the rows' lengths become zero.
__global__ __launch_bounds__(RQ_THREADS) void k_count_freed(TableParams P, int32_t* counts) {
  __shared__ int s_red[RQ_THREADS / WAVE];
  const int64_t first = (int64_t)blockIdx.x * RQ_CHUNK;
  int sum = 0;
#pragma unroll
  for (int k = 0; k < RQ_CHUNK / RQ_THREADS; ++k) {
    const int64_t s = first + k * RQ_THREADS + threadIdx.x;
    sum += s < P.num_slots && P.shared[s] < 0;
  }
  sum = block_sum<RQ_THREADS / WAVE>(sum, s_red);
  if (threadIdx.x == 0) counts[blockIdx.x] = sum;
  for (int64_t k = (int64_t)blockIdx.x * RQ_THREADS + threadIdx.x; k < P.n; k += (int64_t)gridDim.x * RQ_THREADS) {
    const int64_t row = load_index(P.at, P.rows_i64, k);
    if (row >= 0 && row < P.rows) set_len(P.lens, P.lens_i64, row, 0);
  }
}

// The sum of counts[0 .. n - 1].
__device__ __forceinline__ int sum_before(const int32_t* counts, int n, int* scratch) {
  int sum = 0;
  for (int k = threadIdx.x; k < n; k += RQ_THREADS) sum += counts[k];
  return block_sum<RQ_THREADS / WAVE>(sum, scratch);
}

// The freed slots in ascending order, their counts zero again.
__global__ __launch_bounds__(RQ_THREADS) void k_emit_freed(TableParams P, const int32_t* counts, int64_t* free_slots,
                                                           int64_t capacity, int32_t* free_count) {
  __shared__ int s_red[RQ_THREADS / WAVE];
  const int mine = counts[blockIdx.x];
  const bool final = blockIdx.x == gridDim.x - 1;
  if (mine == 0 && !final) return;
  int64_t before = sum_before(counts, (int)blockIdx.x, s_red);
  if (final && threadIdx.x == 0) *free_count = (int32_t)(before + mine);
  if (mine == 0) return;
  const int64_t s0 = (int64_t)blockIdx.x * RQ_CHUNK + threadIdx.x * 16;
  uint32_t freed = 0;
  for (int k = 0; k < 16; ++k) freed |= (s0 + k < P.num_slots && P.shared[s0 + k] < 0 ? 1u : 0u) << k;
  int64_t at = before + block_excl_scan<RQ_THREADS / WAVE>((int)__popc(freed), s_red, (int*)nullptr);
  for (int k = 0; k < 16; ++k) {
    if (!((freed >> k) & 1)) continue;
    P.shared[s0 + k] = 0;
    if (at < capacity) free_slots[at] = s0 + k;
    ++at;
  }
}

// ---------------------------------------------------------------------------------------
// Compaction.  used[slot] is a byte; U slots are used.  Used slots at or above U move, in ascending order, into the unused
// ones below U, in ascending order.
// ---------------------------------------------------------------------------------------
struct CompactParams {
  TableParams t;
  uint8_t* used;       // [pool rounded up to chunks]
  int32_t* counts;     // [pool / RQ_CHUNK]
  int32_t* place;      // [num_slots]: the rank of a slot that moves
  int64_t *src, *dst;  // the moves
  int32_t* out;        // [2]: used, moved
  int pool;            // chunks of the pool
};

__global__ __launch_bounds__(RQ_THREADS) void k_clear_used(CompactParams P) {
  const int64_t i = (int64_t)blockIdx.x * RQ_THREADS + threadIdx.x;  // (16 bytes a thread)
  reinterpret_cast<uint4*>(P.used)[i] = make_uint4(0, 0, 0, 0);
}

__global__ __launch_bounds__(RQ_THREADS) void k_mark_used(CompactParams P) {
  const int64_t i = blockIdx.x / P.t.chunks, chunk = blockIdx.x - i * P.t.chunks;
  const int64_t row = load_index(P.t.at, P.t.rows_i64, i);
  if (row < 0 || row >= P.t.rows) return;
  const int64_t p = chunk * RQ_THREADS + threadIdx.x;
  if (p >= held(P.t.lens, P.t.lens_i64, row, P.t.cols)) return;
  const int32_t slot = P.t.table[row * P.t.stride + p];
  if (slot >= 0 && slot < P.t.num_slots) P.used[slot] = 1;
}

// 16 slots' bytes as bits.
__device__ __forceinline__ uint32_t used_bits(const uint8_t* used, int64_t s0) {
  const uint4 v = *reinterpret_cast<const uint4*>(used + s0);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) bits |= ((w[i] * 0x01020408u) >> 24 & 0xfu) << (4 * i);  // (byte k's one to bit 24 + k)
  return bits;
}

__global__ __launch_bounds__(RQ_THREADS) void k_count_used(CompactParams P) {
  __shared__ int s_red[RQ_THREADS / WAVE];
  int n = __popc(used_bits(P.used, (int64_t)blockIdx.x * RQ_CHUNK + threadIdx.x * 16));
  n = block_sum<RQ_THREADS / WAVE>(n, s_red);
  if (threadIdx.x == 0) P.counts[blockIdx.x] = n;
}

__global__ __launch_bounds__(RQ_THREADS) void k_plan_moves(CompactParams P) {
  __shared__ int s_red[RQ_THREADS / WAVE];
  const int before = sum_before(P.counts, (int)blockIdx.x, s_red);
  const int U = sum_before(P.counts, P.pool, s_red);
  // the used slots below U: what moves is what is used above it
  const int edge = U / RQ_CHUNK < P.pool ? U / RQ_CHUNK : P.pool - 1;
  int low = sum_before(P.counts, edge, s_red);
  {
    const int64_t s0 = (int64_t)edge * RQ_CHUNK + threadIdx.x * 16;
    const int64_t take = U - s0;
    const uint32_t bits = used_bits(P.used, s0);
    const int n = take <= 0 ? 0 : __popc(take >= 16 ? bits : bits & ((1u << take) - 1u));
    low += block_sum<RQ_THREADS / WAVE>(n, s_red);
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) P.out[0] = U, P.out[1] = U - low;
  const int64_t s0 = (int64_t)blockIdx.x * RQ_CHUNK + threadIdx.x * 16;
  const uint32_t bits = used_bits(P.used, s0);
  int at = before + block_excl_scan<RQ_THREADS / WAVE>((int)__popc(bits), s_red, (int*)nullptr);  // used slots below s0
  for (int k = 0; k < 16; ++k) {
    const int64_t s = s0 + k;
    if ((bits >> k) & 1) {
      if (s >= U) P.src[at - low] = s, P.place[s] = at - low;
      ++at;
    } else if (s < U) {
      P.dst[s - at] = s;
    }
  }
}

// The rows' entries follow the moves, and so do the counts of holders (the grid's last rows).
__global__ __launch_bounds__(RQ_THREADS) void k_follow_moves(CompactParams P) {
  const int64_t i = blockIdx.x / P.t.chunks, chunk = blockIdx.x - i * P.t.chunks;
  const int64_t p = chunk * RQ_THREADS + threadIdx.x;
  const int32_t U = P.out[0], moved = P.out[1];
  if (i >= P.t.n) {  // (one row of workgroups more)
    if (P.t.shared)
      for (int64_t k = p; k < moved; k += P.t.chunks * RQ_THREADS) {
        const int64_t from = P.src[k];
        P.t.shared[P.dst[k]] = P.t.shared[from];
        P.t.shared[from] = 0;
      }
    return;
  }
  const int64_t row = load_index(P.t.at, P.t.rows_i64, i);
  if (moved == 0 || row < 0 || row >= P.t.rows || p >= held(P.t.lens, P.t.lens_i64, row, P.t.cols)) return;
  int32_t* entry = P.t.table + row * P.t.stride + p;
  const int32_t slot = *entry;
  if (slot < U || slot >= P.t.num_slots) return;
  const int32_t rank = P.place[slot];
  if (rank >= 0 && rank < moved) *entry = (int32_t)P.dst[rank];
}

// ---------------------------------------------------------------------------------------
// Rows of slots to other slots, several tensors in one launch.
// ---------------------------------------------------------------------------------------
constexpr int CS_PARTS = 64, CS_ROWS = 4;

struct CopyPart {
  uint8_t* base;
  int64_t slot_stride, head_stride;  // bytes
  int32_t pieces, per;               // of a slot, of a head
  int32_t wide, G;                   // bytes of a piece (16 or 4), lanes of a slot
};
struct CopyParams {
  CopyPart part[CS_PARTS];
  const void *src, *dst;
  const int32_t* count;
  int64_t n, num_slots;
  int32_t src_i64, dst_i64;
};

// Groups of G lanes take CS_ROWS moves at once, all loaded before the first is stored.
template <class V>
__device__ __forceinline__ void copy_rows(const CopyParams& P, const CopyPart& part, int64_t n) {
  const int l = threadIdx.x & (part.G - 1), groups = RQ_THREADS / part.G;
  for (int64_t i0 = (int64_t)blockIdx.x * groups * CS_ROWS + threadIdx.x / part.G; i0 < n;
       i0 += (int64_t)gridDim.x * groups * CS_ROWS) {
    int64_t from[CS_ROWS], to[CS_ROWS];
#pragma unroll
    for (int u = 0; u < CS_ROWS; ++u) {
      const int64_t i = i0 + u * groups;
      from[u] = i < n ? load_index(P.src, P.src_i64, i) : -1;
      to[u] = i < n ? load_index(P.dst, P.dst_i64, i) : -1;
      if (from[u] < 0 || from[u] >= P.num_slots || to[u] < 0 || to[u] >= P.num_slots) from[u] = to[u] = -1;
    }
    for (int k = l; k < part.pieces; k += part.G) {
      const int head = k / part.per;
      const int64_t at = head * part.head_stride + (int64_t)(k - head * part.per) * sizeof(V);
      V x[CS_ROWS];
#pragma unroll
      for (int u = 0; u < CS_ROWS; ++u)
        if (from[u] >= 0) x[u] = *reinterpret_cast<const V*>(part.base + from[u] * part.slot_stride + at);
#pragma unroll
      for (int u = 0; u < CS_ROWS; ++u)
        if (from[u] >= 0) *reinterpret_cast<V*>(part.base + to[u] * part.slot_stride + at) = x[u];
    }
  }
}

__global__ __launch_bounds__(RQ_THREADS) void k_copy_slots(CopyParams P) {
  const CopyPart& part = P.part[blockIdx.y];
  int64_t n = P.n;
  if (P.count) {
    const int32_t c = *P.count;
    n = c < 0 ? 0 : (c < n ? c : n);
  }
  if (part.wide == 16)
    copy_rows<uint4>(P, part, n);
  else
    copy_rows<uint32_t>(P, part, n);
}

static int launch_copy(const char* what, const dsv_slot_rows* rows, int32_t n_rows, const void* src, int32_t src_i64,
                       const void* dst, int32_t dst_i64, int64_t n, const int32_t* count, int64_t num_slots,
                       hipStream_t stream) {
  for (int32_t at = 0; at < n_rows; at += CS_PARTS) {
    CopyParams P;
    const int parts = n_rows - at < CS_PARTS ? n_rows - at : CS_PARTS;
    int64_t most = 1;
    for (int k = 0; k < parts; ++k) {
      const dsv_slot_rows& r = rows[at + k];
      CopyPart& p = P.part[k];
      p.base = reinterpret_cast<uint8_t*>(r.base);
      p.slot_stride = r.slot_stride;
      p.head_stride = r.head_stride;
      int64_t bytes = r.bytes, heads = r.heads;
      if (heads == 1 || r.head_stride == bytes) bytes *= heads, heads = 1, p.head_stride = 0;
      const bool wide = (uintptr_t)r.base % 16 == 0 && p.slot_stride % 16 == 0 && p.head_stride % 16 == 0 && bytes % 16 == 0;
      p.wide = wide ? 16 : 4;
      p.per = (int32_t)(bytes / p.wide);
      p.pieces = (int32_t)(p.per * heads);
      p.G = 1;
      while (p.G < p.pieces && p.G < RQ_THREADS) p.G *= 2;
      const int64_t groups = (n + (int64_t)RQ_THREADS / p.G * CS_ROWS - 1) / ((int64_t)RQ_THREADS / p.G * CS_ROWS);
      most = groups > most ? groups : most;
    }
    P.src = src;
    P.dst = dst;
    P.count = count;
    P.n = n;
    P.num_slots = num_slots;
    P.src_i64 = src_i64;
    P.dst_i64 = dst_i64;
    if (most > 1024) most = 1024;
    hipLaunchKernelGGL(k_copy_slots, dim3((unsigned)most, (unsigned)parts), dim3(RQ_THREADS), 0, stream, P);
    DSV_CHECK_LAUNCH(what);
  }
  return DSV_OK;
}

static int check_rows(const char* what, const dsv_slot_rows* rows, int32_t n_rows, int64_t num_slots) {
  if (n_rows < 0 || (n_rows && !rows) || num_slots < 1 || num_slots > 0x7fffffff)
    DSV_FAIL(DSV_ERR_INVALID, "%s: 1 to 2^31 - 1 slots and their rows are required", what);
  for (int32_t k = 0; k < n_rows; ++k) {
    const dsv_slot_rows& r = rows[k];
    if (!r.base || r.heads < 1 || r.bytes < 4 || r.bytes % 4 || (int64_t)r.heads * r.bytes > (1 << 24) || r.slot_stride < 0 ||
        r.head_stride < 0 || (uintptr_t)r.base % 4 || r.slot_stride % 4 || r.head_stride % 4)
      DSV_FAIL(DSV_ERR_INVALID, "%s: a slot's rows must be whole 4-byte words, up to 16 MiB a slot", what);
  }
  return DSV_OK;
}

static int check_table(const char* what, const int32_t* table, int64_t rows, int64_t stride, int64_t cols, const void* lens,
                       int64_t n, const void* at, int64_t num_slots) {
  if (n < 0 || n > 0x7fffffff) DSV_FAIL(DSV_ERR_INVALID, "%s: n %lld", what, (long long)n);
  if (rows < 1 || cols < 1 || stride < cols || !table || !lens || (n && !at))
    DSV_FAIL(DSV_ERR_INVALID, "%s: a request table, its lengths and rows are required", what);
  if (num_slots < 1 || num_slots > 0x7fffffff) DSV_FAIL(DSV_ERR_INVALID, "%s: 1 to 2^31 - 1 slots (got %lld)", what, (long long)num_slots);
  if (((cols + RQ_THREADS - 1) / RQ_THREADS) * (n + 1) > 0x7fffffffll)
    DSV_FAIL(DSV_ERR_INVALID, "%s: too many entries for one call", what);
  return DSV_OK;
}

static int64_t pool_chunks(int64_t num_slots) { return (num_slots + RQ_CHUNK - 1) / RQ_CHUNK; }

}  // namespace dsv

using namespace dsv;

extern "C" int dsv_copy_slots(const dsv_slot_rows* rows, int32_t n_rows, int64_t num_slots, const void* src, int32_t src_i64,
                              const void* dst, int32_t dst_i64, int64_t n, const int32_t* count, dsv_stream_t stream) {
  const int rc = check_rows("dsv_copy_slots", rows, n_rows, num_slots);
  if (rc != DSV_OK) return rc;
  if (n < 0 || n > 0x7fffffff) DSV_FAIL(DSV_ERR_INVALID, "dsv_copy_slots: n %lld", (long long)n);
  if (n == 0 || n_rows == 0) return DSV_OK;
  if (!src || !dst) DSV_FAIL(DSV_ERR_INVALID, "dsv_copy_slots: null pointer");
  return launch_copy("k_copy_slots", rows, n_rows, src, src_i64, dst, dst_i64, n, count, num_slots,
                     reinterpret_cast<hipStream_t>(stream));
}

extern "C" int dsv_fork_requests(int32_t* req_to_token, int64_t rows, int64_t rt_stride, int64_t rt_cols, void* seq_lens,
                                 int32_t seq_lens_i64, int32_t* shared, int64_t num_slots, const void* parents,
                                 const void* children, int32_t rows_i64, int64_t n, dsv_stream_t stream) {
  const int rc = check_table("dsv_fork_requests", req_to_token, rows, rt_stride, rt_cols, seq_lens, n, parents, num_slots);
  if (rc != DSV_OK) return rc;
  if (!shared || (n && !children)) DSV_FAIL(DSV_ERR_INVALID, "dsv_fork_requests: shared and children are required");
  if (n == 0) return DSV_OK;
  TableParams P{req_to_token, rows, rt_stride, rt_cols, seq_lens, seq_lens_i64, rows_i64, parents, n, num_slots, shared,
                (rt_cols + RQ_THREADS - 1) / RQ_THREADS};
  hipLaunchKernelGGL(k_fork, dim3((unsigned)(P.chunks * n)), dim3(RQ_THREADS), 0, reinterpret_cast<hipStream_t>(stream), P, children);
  DSV_CHECK_LAUNCH("k_fork");
  return DSV_OK;
}

extern "C" int64_t dsv_free_requests_workspace_bytes(int64_t num_slots) {
  return num_slots < 1 ? 0 : pool_chunks(num_slots) * (int64_t)sizeof(int32_t);
}

extern "C" int dsv_free_requests(int32_t* req_to_token, int64_t rows, int64_t rt_stride, int64_t rt_cols, void* seq_lens,
                                 int32_t seq_lens_i64, int32_t* shared, int64_t num_slots, const void* at, int32_t rows_i64,
                                 int64_t n, int64_t* free_slots, int64_t capacity, int32_t* free_count, void* workspace,
                                 int64_t workspace_bytes, dsv_stream_t stream_) {
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  const int rc = check_table("dsv_free_requests", req_to_token, rows, rt_stride, rt_cols, seq_lens, n, at, num_slots);
  if (rc != DSV_OK) return rc;
  if (!shared || !free_count || capacity < 0 || (capacity && !free_slots))
    DSV_FAIL(DSV_ERR_INVALID, "dsv_free_requests: shared, free_slots and free_count are required");
  if (!workspace || (uintptr_t)workspace % 16) DSV_FAIL(DSV_ERR_INVALID, "dsv_free_requests: a 16-byte-aligned workspace is required");
  const int64_t need = dsv_free_requests_workspace_bytes(num_slots);
  if (workspace_bytes < need)
    DSV_FAIL(DSV_ERR_WORKSPACE, "dsv_free_requests: workspace %lld < %lld", (long long)workspace_bytes, (long long)need);
  TableParams P{req_to_token, rows, rt_stride, rt_cols, seq_lens, seq_lens_i64, rows_i64, at, n, num_slots, shared,
                (rt_cols + RQ_THREADS - 1) / RQ_THREADS};
  int32_t* counts = reinterpret_cast<int32_t*>(workspace);
  if (n) {
    hipLaunchKernelGGL(k_release, dim3((unsigned)(P.chunks * n)), dim3(RQ_THREADS), 0, stream, P);
    DSV_CHECK_LAUNCH("k_release");
  }
  const dim3 pool((unsigned)pool_chunks(num_slots));
  hipLaunchKernelGGL(k_count_freed, pool, dim3(RQ_THREADS), 0, stream, P, counts);
  DSV_CHECK_LAUNCH("k_count_freed");
  hipLaunchKernelGGL(k_emit_freed, pool, dim3(RQ_THREADS), 0, stream, P, counts, free_slots, capacity, free_count);
  DSV_CHECK_LAUNCH("k_emit_freed");
  return DSV_OK;
}

extern "C" int64_t dsv_compact_requests_workspace_bytes(int64_t num_slots) {
  if (num_slots < 1) return 0;
  const int64_t pool = pool_chunks(num_slots);
  return pool * RQ_CHUNK * (int64_t)(1 + sizeof(int32_t)) + (pool * (int64_t)sizeof(int32_t) + 15) / 16 * 16;
}

extern "C" int dsv_compact_requests(int32_t* req_to_token, int64_t rows, int64_t rt_stride, int64_t rt_cols,
                                    const void* seq_lens, int32_t seq_lens_i64, int32_t* shared, int64_t num_slots,
                                    const void* at, int32_t rows_i64, int64_t n, const dsv_slot_rows* slot_rows,
                                    int32_t n_slot_rows, int64_t* src, int64_t* dst, int64_t capacity, int32_t* counts,
                                    void* workspace, int64_t workspace_bytes, dsv_stream_t stream_) {
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  int rc = check_table("dsv_compact_requests", req_to_token, rows, rt_stride, rt_cols, seq_lens, n, at, num_slots);
  if (rc == DSV_OK) rc = check_rows("dsv_compact_requests", slot_rows, n_slot_rows, num_slots);
  if (rc != DSV_OK) return rc;
  if (!counts || capacity < num_slots / 2 || (num_slots > 1 && (!src || !dst)))
    DSV_FAIL(DSV_ERR_INVALID, "dsv_compact_requests: counts and room for %lld moves are required", (long long)(num_slots / 2));
  if (!workspace || (uintptr_t)workspace % 16)
    DSV_FAIL(DSV_ERR_INVALID, "dsv_compact_requests: a 16-byte-aligned workspace is required");
  const int64_t need = dsv_compact_requests_workspace_bytes(num_slots);
  if (workspace_bytes < need)
    DSV_FAIL(DSV_ERR_WORKSPACE, "dsv_compact_requests: workspace %lld < %lld", (long long)workspace_bytes, (long long)need);
  const int64_t pool = pool_chunks(num_slots);
  CompactParams P;
  P.t = TableParams{req_to_token, rows, rt_stride, rt_cols, const_cast<void*>(seq_lens), seq_lens_i64, rows_i64, at, n, num_slots,
                    shared, (rt_cols + RQ_THREADS - 1) / RQ_THREADS};
  P.used = reinterpret_cast<uint8_t*>(workspace);
  P.place = reinterpret_cast<int32_t*>(P.used + pool * RQ_CHUNK);
  P.counts = P.place + pool * RQ_CHUNK;
  P.src = src;
  P.dst = dst;
  P.out = counts;
  P.pool = (int)pool;
  const dim3 over_pool((unsigned)pool), threads(RQ_THREADS);
  hipLaunchKernelGGL(k_clear_used, over_pool, threads, 0, stream, P);
  DSV_CHECK_LAUNCH("k_clear_used");
  if (n) {
    hipLaunchKernelGGL(k_mark_used, dim3((unsigned)(P.t.chunks * n)), threads, 0, stream, P);
    DSV_CHECK_LAUNCH("k_mark_used");
  }
  hipLaunchKernelGGL(k_count_used, over_pool, threads, 0, stream, P);
  DSV_CHECK_LAUNCH("k_count_used");
  hipLaunchKernelGGL(k_plan_moves, over_pool, threads, 0, stream, P);
  DSV_CHECK_LAUNCH("k_plan_moves");
  hipLaunchKernelGGL(k_follow_moves, dim3((unsigned)(P.t.chunks * (n + 1))), threads, 0, stream, P);
  DSV_CHECK_LAUNCH("k_follow_moves");
  if (n_slot_rows && num_slots > 1)
    return launch_copy("k_copy_slots", slot_rows, n_slot_rows, src, 1, dst, 1, num_slots / 2, counts + 1, num_slots, stream);
  return DSV_OK;
}
