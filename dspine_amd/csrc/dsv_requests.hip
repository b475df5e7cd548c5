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

// N indices at any places (`at(r)`; -1 where it is negative), and the clamped lengths of rows (0 for a row that is none): one test
// of the width for all of them.
template <int N, class At>
__device__ __forceinline__ void load_indices(const void* p, int i64, At at, int64_t (&out)[N]) {
  if (i64) {
#pragma unroll
    for (int r = 0; r < N; ++r) out[r] = at(r) < 0 ? -1 : reinterpret_cast<const int64_t*>(p)[at(r)];
  } else {
#pragma unroll
    for (int r = 0; r < N; ++r) out[r] = at(r) < 0 ? -1 : (int64_t) reinterpret_cast<const int32_t*>(p)[at(r)];
  }
}
template <int N>
__device__ __forceinline__ void load_lens(const void* lens, int i64, const int64_t (&row)[N], int64_t cols, int64_t (&len)[N]) {
  load_indices<N>(lens, i64, [&](int r) { return row[r]; }, len);
#pragma unroll
  for (int r = 0; r < N; ++r) len[r] = len[r] < 0 ? 0 : (len[r] > cols ? cols : len[r]);
}

// Samples of one prompt hold its slots at the same positions, so a thread takes its column's entries of RQ_ROWS rows and
// counts equal ones together: what bounds a fork or a release of long prompts is the touch of a scattered count for each
// slot (about 28 G/s; a plain read and write is as slow as the atomic, and neighbouring slots share their lines).  128 rows
// of 20000 positions, two of each prompt, slots in random order: 57 us a fork and 56 a release, 96 each with an atomic
// an entry; without the counts a fork is 17.  (Entries sorted by ranges of slots first, each range counted in LDS, was not tried.)
constexpr int RQ_ROWS = 8;
__device__ __forceinline__ void add_holders(const TableParams& P, int32_t (&slot)[RQ_ROWS], int sign) {
  int times[RQ_ROWS];
#pragma unroll
  for (int r = 0; r < RQ_ROWS; ++r) {
    times[r] = slot[r] >= 0 && slot[r] < P.num_slots;
#pragma unroll
    for (int k = 0; k < r; ++k) {
      const bool same = times[r] && times[k] && slot[k] == slot[r];
      times[k] += same;
      times[r] = same ? 0 : times[r];
    }
  }
#pragma unroll
  for (int r = 0; r < RQ_ROWS; ++r)
    if (times[r]) atomicAdd(&P.shared[slot[r]], sign * times[r]);
}

// A workgroup RQ_ROWS pairs' 256 columns.
__global__ __launch_bounds__(RQ_THREADS) void k_fork(TableParams P, const void* children) {
  const int64_t group = blockIdx.x / P.chunks, chunk = blockIdx.x - group * P.chunks;
  const int64_t p = chunk * RQ_THREADS + threadIdx.x;
  // (every load of a kind before the first of the next: a wait for each kind, not for each row)
  int32_t slot[RQ_ROWS];
  int64_t parent[RQ_ROWS], child[RQ_ROWS], len[RQ_ROWS];
  auto pair = [&](int r) { return group * RQ_ROWS + r < P.n ? group * RQ_ROWS + r : -1; };
  load_indices<RQ_ROWS>(P.at, P.rows_i64, pair, parent);
  load_indices<RQ_ROWS>(children, P.rows_i64, pair, child);
#pragma unroll
  for (int r = 0; r < RQ_ROWS; ++r)
    if (parent[r] >= P.rows || child[r] < 0 || child[r] >= P.rows || child[r] == parent[r]) parent[r] = -1;
  load_lens<RQ_ROWS>(P.lens, P.lens_i64, parent, P.cols, len);
#pragma unroll
  for (int r = 0; r < RQ_ROWS; ++r) slot[r] = p < len[r] ? P.table[parent[r] * P.stride + p] : -1;
#pragma unroll
  for (int r = 0; r < RQ_ROWS; ++r) {
    if (p == 0 && parent[r] >= 0) set_len(P.lens, P.lens_i64, child[r], len[r]);
    if (p < len[r]) P.table[child[r] * P.stride + p] = slot[r];
  }
  add_holders(P, slot, 1);
}

// The rows of a group that are named before, as bits (every thread of the workgroup).
__device__ __forceinline__ uint32_t named_before(const TableParams& P, int64_t first, uint32_t* scratch) {
  int64_t row[RQ_ROWS];
  load_indices<RQ_ROWS>(P.at, P.rows_i64, [&](int r) { return first + r < P.n ? first + r : -1; }, row);
  uint32_t again = 0;
#pragma unroll
  for (int r = 1; r < RQ_ROWS; ++r)
#pragma unroll
    for (int k = 0; k < r; ++k) again |= (row[k] == row[r] ? 1u : 0u) << r;
  uint32_t mine = 0;
  for (int64_t k = threadIdx.x; k < first; k += blockDim.x) {
    const int64_t other = load_index(P.at, P.rows_i64, k);
#pragma unroll
    for (int r = 0; r < RQ_ROWS; ++r) mine |= (other == row[r] ? 1u : 0u) << r;
  }
  if (first == 0) return again;
  if (threadIdx.x == 0) *scratch = 0;
  __syncthreads();
  if (mine) atomicOr(scratch, mine);
  __syncthreads();
  again |= *scratch;
  __syncthreads();
  return again;
}

// A column's entries of a group of rows, those named before left out.
__device__ __forceinline__ void release_column(const TableParams& P, int64_t first, uint32_t again, int64_t p) {
  int32_t slot[RQ_ROWS];
  int64_t row[RQ_ROWS], len[RQ_ROWS];
  load_indices<RQ_ROWS>(P.at, P.rows_i64, [&](int r) { return first + r < P.n && !((again >> r) & 1) ? first + r : -1; }, row);
#pragma unroll
  for (int r = 0; r < RQ_ROWS; ++r)
    if (row[r] >= P.rows) row[r] = -1;
  load_lens<RQ_ROWS>(P.lens, P.lens_i64, row, P.cols, len);
#pragma unroll
  for (int r = 0; r < RQ_ROWS; ++r) slot[r] = p < len[r] ? P.table[row[r] * P.stride + p] : -1;
  add_holders(P, slot, -1);
}

__global__ __launch_bounds__(RQ_THREADS) void k_release(TableParams P) {
  __shared__ uint32_t s_again;
  const int64_t group = blockIdx.x / P.chunks, chunk = blockIdx.x - group * P.chunks;
  const uint32_t again = named_before(P, group * RQ_ROWS, &s_again);
  release_column(P, group * RQ_ROWS, again, chunk * RQ_THREADS + threadIdx.x);
}

// Slots below zero in each chunk of the pool; the rows' lengths become zero.  (1.6 M slots: 5.8 us, and the list 7.1.)
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

// Rows of a small pool, all of it in one workgroup: a launch in place of three (2 rows of 750 columns: 3.7 us for 3.3 + 3.4 + 3.8
// and their gaps, and two launches less of the host's).  The rows and their lengths are read once, and the columns of all groups
// of RQ_ROWS rows are dealt to the threads in one row, so that many short rows wait for memory no longer than a few.
constexpr int RQ_WIDE = 1024, RQ_SMALL_SLOTS = 16 * RQ_WIDE;
struct SmallRows {
  int64_t row[RQ_WIDE];
  int32_t len[RQ_WIDE];
};
// What one workgroup takes: rows, columns of groups of rows, entries.  Replayed, us, and those of the launches in its place (whose
// host's time it saves):
//   an end      2 x 750 13.5 and 14.5, 4 x 1000 17.7 and 15.4, 8 x 1000 18.5 and 19.1, 16 x 500 18.7 and 18.9; not taken:
//               1 x 8000 23.1 and 15.0, 40 x 300 24.2 and 19.7, 75 x 320 29.1 and 20.0, 1000 x 8 40.7 and 17.4
//   compaction  2 x 750 11.0 and 13.9, 8 x 1000 13.9 and 14.9, 8 x 2000 8.5 and 10.5, 75 x 320 14.3 and 14.0, 1000 x 8 14.2 and
//               15.5, 1 x 8000 19.4 and 14.8
static bool few_rows(int64_t n, int64_t cols, int64_t rows, int64_t columns, int64_t entries) {
  return n <= rows && (n + RQ_ROWS - 1) / RQ_ROWS * cols <= columns && n * cols <= entries;
}
static bool few_to_free(int64_t n, int64_t cols) { return few_rows(n, cols, 64, 2 * RQ_WIDE, 8 * RQ_WIDE); }
static bool few_to_plan(int64_t n, int64_t cols) { return few_rows(n, cols, RQ_WIDE, 8 * RQ_WIDE, 24 * RQ_WIDE); }
__device__ __forceinline__ void read_rows(const TableParams& t, SmallRows& s) {
  const int i = (int)threadIdx.x;
  const int64_t row = i < t.n ? load_index(t.at, t.rows_i64, i) : -1;
  s.row[i] = row;
  s.len[i] = row < 0 || row >= t.rows ? 0 : (int32_t)held(t.lens, t.lens_i64, row, t.cols);
  __syncthreads();
}
// The entries of a column of a group of rows; false where there is none left for this thread.
__device__ __forceinline__ bool column_of(const TableParams& t, const SmallRows& s, uint32_t unit, int32_t (&slot)[RQ_ROWS]) {
  const uint32_t group = unit / (uint32_t)t.cols, p = unit - group * (uint32_t)t.cols, first = group * RQ_ROWS;
  if (first >= (uint32_t)t.n) return false;
#pragma unroll
  for (int r = 0; r < RQ_ROWS; ++r)
    slot[r] = (int32_t)p < s.len[first + r] ? t.table[s.row[first + r] * t.stride + p] : -1;
  return true;
}
// The holders that each slot loses are counted in LDS: with one workgroup's atomics on memory 2 rows of 750 columns take 8.8 us
// for 4.0, 8 of 1024 28.2 for 12.1.
__global__ __launch_bounds__(RQ_WIDE) void k_free_small(TableParams P, int64_t* free_slots, int64_t capacity, int32_t* free_count) {
  __shared__ int s_red[RQ_WIDE / WAVE];
  __shared__ SmallRows s_rows;
  __shared__ int32_t s_lost[RQ_SMALL_SLOTS];
  const int tid = threadIdx.x;
  for (int k = tid; k < P.num_slots; k += RQ_WIDE) s_lost[k] = 0;
  read_rows(P, s_rows);
  bool again = false;  // (a row that is named before counts once)
  for (int k = 0; k < tid && tid < P.n; ++k) again |= s_rows.row[k] == s_rows.row[tid];
  __syncthreads();
  if (again) s_rows.len[tid] = 0;
  __syncthreads();
  int32_t slot[RQ_ROWS];
  for (uint32_t unit = tid; column_of(P, s_rows, unit, slot); unit += RQ_WIDE)
#pragma unroll
    for (int r = 0; r < RQ_ROWS; ++r)
      if (slot[r] >= 0 && slot[r] < P.num_slots) atomicAdd(&s_lost[slot[r]], 1);
  __syncthreads();  // (and every length has been read)
  if (tid < P.n && s_rows.row[tid] >= 0 && s_rows.row[tid] < P.rows) set_len(P.lens, P.lens_i64, s_rows.row[tid], 0);
  const int per = (int)((P.num_slots + RQ_WIDE - 1) / RQ_WIDE), s0 = tid * per;
  uint32_t freed = 0;
  for (int k = 0; k < per && s0 + k < P.num_slots; ++k) {
    const int32_t lost = s_lost[s0 + k], was = P.shared[s0 + k], now = was - lost;
    if (now < 0) freed |= 1u << k;
    if (now < 0 || lost) P.shared[s0 + k] = now < 0 ? 0 : now;
  }
  int total;
  int64_t at = block_excl_scan<RQ_WIDE / WAVE>((int)__popc(freed), s_red, &total);
  if (tid == 0) *free_count = total;
  for (int k = 0; k < per; ++k) {
    if (!((freed >> k) & 1)) continue;
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

// The same for a small pool and few rows, in one workgroup, the used slots as bits in its LDS: a launch in place of four
// (7 rows of 2700 columns, 14000 slots: 11.2 us for 11 in all, and three launches less of the host's).
constexpr int RQ_BITS = 2 * 16 * RQ_WIDE;  // slots at most
__global__ __launch_bounds__(RQ_WIDE) void k_plan_small(CompactParams P) {
  __shared__ uint32_t s_bits[RQ_BITS / 32];
  __shared__ SmallRows s_rows;
  __shared__ int s_red[RQ_WIDE / WAVE];
  const TableParams& t = P.t;
  const int tid = threadIdx.x;
  static_assert(RQ_BITS / 32 == RQ_WIDE, "a word a thread");
  s_bits[tid] = 0;  // (a barrier follows, where the rows are read)
  read_rows(t, s_rows);
  int32_t slot[RQ_ROWS];
  for (uint32_t unit = tid; column_of(t, s_rows, unit, slot); unit += RQ_WIDE)
#pragma unroll
    for (int r = 0; r < RQ_ROWS; ++r)
      if (slot[r] >= 0 && slot[r] < t.num_slots) atomicOr(&s_bits[slot[r] / 32], 1u << (slot[r] % 32));
  __syncthreads();
  const uint32_t word = s_bits[tid];
  const int U = block_sum<RQ_WIDE / WAVE>((int)__popc(word), s_red);
  // the used slots below U: what moves is what is used above it
  const int take = U - tid * 32;
  const int low = block_sum<RQ_WIDE / WAVE>(take <= 0 ? 0 : (int)__popc(take >= 32 ? word : word & ((1u << take) - 1u)), s_red);
  if (tid == 0) P.out[0] = U, P.out[1] = U - low;
  int before = 0;
  for (int s0 = tid * 16; s0 - tid * 16 < t.num_slots; s0 += 16 * RQ_WIDE) {
    const uint32_t bits = (s_bits[s0 / 32] >> (s0 % 32)) & 0xffffu;
    int total;
    int at = before + block_excl_scan<RQ_WIDE / WAVE>((int)__popc(bits), s_red, &total);  // used slots below s0
    before += total;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int s = s0 + k;
      if ((bits >> k) & 1) {
        if (s >= U) P.src[at - low] = s, P.place[s] = at - low;
        ++at;
      } else if (s < U) {
        P.dst[s - at] = s;
      }
    }
  }
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
  int32_t parts;
};

typedef uint32_t uint32x4 __attribute__((ext_vector_type(4)));

// Groups of G lanes take CS_ROWS moves at once, all loaded before the first is stored.  Bound by memory: 45000 slots' rows of
// four layers, 1.6 GB read and written: 293 us, 5.5 TB/s (314 with loads and stores that the caches keep).
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
      const int head = part.per == part.pieces ? 0 : k / part.per;
      const int64_t at = head * part.head_stride + (int64_t)(k - head * part.per) * sizeof(V);
      V x[CS_ROWS];
#pragma unroll
      for (int u = 0; u < CS_ROWS; ++u)
        x[u] = __builtin_nontemporal_load(reinterpret_cast<const V*>(part.base + (from[u] < 0 ? 0 : from[u]) * part.slot_stride + at));
#pragma unroll
      for (int u = 0; u < CS_ROWS; ++u)
        if (from[u] >= 0) __builtin_nontemporal_store(x[u], reinterpret_cast<V*>(part.base + to[u] * part.slot_stride + at));
    }
  }
}

// The tensors' rows; after a plan the rows' entries and the counts of holders too, as two rows of workgroups more.
__global__ __launch_bounds__(RQ_THREADS) void k_copy_slots(CopyParams P, CompactParams M) {
  int64_t n = P.n;
  if (P.count) {
    const int32_t c = *P.count;
    n = c < 0 ? 0 : (c < n ? c : n);
  }
  if ((int)blockIdx.y < P.parts) {
    const CopyPart part = P.part[blockIdx.y];
    if (part.wide == 16)
      copy_rows<uint32x4>(P, part, n);
    else
      copy_rows<uint32_t>(P, part, n);
    return;
  }
  const TableParams& t = M.t;
  const int64_t step = (int64_t)gridDim.x * RQ_THREADS, first = (int64_t)blockIdx.x * RQ_THREADS + threadIdx.x;
  if (n == 0) return;
  if ((int)blockIdx.y == P.parts) {
    if (t.shared)
      for (int64_t k = first; k < n; k += step) {
        const int64_t from = M.src[k];
        t.shared[M.dst[k]] = t.shared[from];
        t.shared[from] = 0;
      }
    return;
  }
  const int32_t U = M.out[0];
  const int64_t units = t.n * t.chunks;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int64_t i = u / t.chunks, p = (u - i * t.chunks) * RQ_THREADS + threadIdx.x;
    const int64_t row = load_index(t.at, t.rows_i64, i);
    if (row < 0 || row >= t.rows || p >= held(t.lens, t.lens_i64, row, t.cols)) continue;
    int32_t* entry = t.table + row * t.stride + p;
    const int32_t slot = *entry;
    if (slot < U || slot >= t.num_slots) continue;
    const int32_t rank = M.place[slot];
    if (rank >= 0 && rank < n) *entry = (int32_t)M.dst[rank];
  }
}

static int launch_copy(const char* what, const dsv_slot_rows* rows, int32_t n_rows, const void* src, int32_t src_i64,
                       const void* dst, int32_t dst_i64, int64_t n, const int32_t* count, int64_t num_slots,
                       const CompactParams* follow, hipStream_t stream) {
  for (int32_t at = 0; at < n_rows || (follow && at == 0); at += CS_PARTS) {
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
    P.parts = parts;
    CompactParams M{};
    unsigned more = 0;
    if (follow && at == 0) {
      M = *follow;
      more = 2;
      const int64_t units = M.t.n * M.t.chunks;
      most = units > most ? units : most;
    }
    if (most > 4096) most = 4096;  // (1024: 320 us for 310)
    hipLaunchKernelGGL(k_copy_slots, dim3((unsigned)most, (unsigned)parts + more), dim3(RQ_THREADS), 0, stream, P, M);
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
  return launch_copy("k_copy_slots", rows, n_rows, src, src_i64, dst, dst_i64, n, count, num_slots, nullptr,
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
  hipLaunchKernelGGL(k_fork, dim3((unsigned)(P.chunks * ((n + RQ_ROWS - 1) / RQ_ROWS))), dim3(RQ_THREADS), 0,
                     reinterpret_cast<hipStream_t>(stream), P, children);
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
  if (num_slots <= RQ_SMALL_SLOTS && few_to_free(n, rt_cols)) {
    hipLaunchKernelGGL(k_free_small, dim3(1), dim3(RQ_WIDE), 0, stream, P, free_slots, capacity, free_count);
    DSV_CHECK_LAUNCH("k_free_small");
    return DSV_OK;
  }
  if (n) {
    hipLaunchKernelGGL(k_release, dim3((unsigned)(P.chunks * ((n + RQ_ROWS - 1) / RQ_ROWS))), dim3(RQ_THREADS), 0, stream, P);
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
  if (num_slots <= RQ_BITS && few_to_plan(n, rt_cols)) {
    hipLaunchKernelGGL(k_plan_small, dim3(1), dim3(RQ_WIDE), 0, stream, P);
    DSV_CHECK_LAUNCH("k_plan_small");
  } else {
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
  }
  return launch_copy("k_copy_slots", slot_rows, n_slot_rows, src, 1, dst, 1, num_slots / 2, counts + 1, num_slots, &P, stream);
}
