// Page tables of the paged 4-bit cache (include/tilemix_hip.h): tokens and pages for the
// sequences of a step, and pages back, without a word to the host.
//
// Both calls are bound by the launch and by a chain of dependent loads, not by bytes: every
// workgroup sums the whole batch's lengths for itself (prefix sums over at most 4096 sequences, kept
// in LDS) and then serves its share of the tokens or pages by a search in them, which is
// one launch.  The values that other workgroups read (seq_lens, free_count) are written by
// the last one to have read them, which a ticket finds.
#include "kv4_common.h"

#include <algorithm>

namespace tmx {

namespace {

constexpr int kMaxBatch = 4096;
constexpr int kThreads = 256;

struct TablesArgs {
  int32_t* table;
  int32_t* lens;
  int32_t* stack;
  int32_t* count;
  int32_t* ticket;
  const int32_t* change;
  int64_t* slots;
  int64_t* positions;
  int32_t* cu;
  int32_t* granted;
  int64_t s_table, tokens;
  int batch, columns, capacity;
  FastDiv by_page;
};

// The sum over the workgroup's threads before this one; `sums`: a place of its own for every scan of a kernel.
__device__ __forceinline__ uint32_t scan_before(uint32_t x, uint32_t* sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t sum = wave_scan(x);
  if (lane == 63) sums[wave] = sum;
  __syncthreads();
  uint32_t before = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)sum, 0x138, 0xf, 0xf, false);  // the lane before
  if (lane == 0) before = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 64 - 1; ++i)
    if (i < wave) before = __builtin_elementwise_add_sat(before, sums[i]);
  return before;
}

// The last entry i <= n - 1 of ascending first[] with first[i] <= x (first[0] <= x).
__device__ __forceinline__ int find(const int32_t* first, int n, int x) {
  int lo = 0, hi = n;  // first[lo] <= x, first[hi] > x or hi = n
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The load of `value` has come back.
__device__ __forceinline__ void arrived(int value) { asm volatile("" ::"v"(value)); }

// True in all threads of the workgroup that comes here last: seq_lens, free_count and the new lengths have been
// read by all then (before the barriers that every workgroup has passed: the lengths are in LDS, the count has arrived
// in each wave).  Nothing that the others wrote is read, so the count need not order it.
__device__ __forceinline__ bool last_workgroup(const TablesArgs& a) {
  __shared__ int last;
  if (gridDim.x == 1) return true;
  if (threadIdx.x == 0) {
    last = __hip_atomic_fetch_add(a.ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
    if (last) __hip_atomic_store(a.ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return last != 0;
}

__device__ __forceinline__ int clamp_int(int64_t x, int64_t lo, int64_t hi) {
  return (int)(x < lo ? lo : x > hi ? hi : x);
}

// LDS: cu [batch + 1], base [batch] (pages taken before; -1: nothing granted), old [batch] (tokens held)
// kTokens: consecutive tokens that a thread serves.
template <int kTokens>
__global__ void __launch_bounds__(kThreads) kv4_extend_kernel(const TablesArgs a) {
  extern __shared__ int32_t lds[];
  __shared__ uint32_t sums[2][kThreads / 64];
  int32_t* const cu = lds;
  int32_t* const base = cu + a.batch + 1;
  int32_t* const old = base + a.batch;
  const int page = a.by_page.d;
  const int64_t room = min((int64_t)a.columns * page, (int64_t)INT32_MAX - page);
  const int count = clamp_int(*a.count, 0, a.capacity);
  // Each thread has the same number of consecutive sequences.
  const int each = (a.batch + kThreads - 1) / kThreads, r0 = threadIdx.x * each, r1 = min(r0 + each, a.batch);
  uint32_t mine = 0;
  for (int r = r0; r < r1; ++r) {
    const int change = a.change[r];
    old[r] = clamp_int(a.lens[r], 0, room);
    base[r] = change;
    mine = __builtin_elementwise_add_sat(mine, (uint32_t)max(change, 0));
  }
  arrived(count);
  const uint32_t tokens_before = scan_before(mine, sums[0]);
  uint32_t at = tokens_before, pages = 0;
  for (int r = r0; r < r1; ++r) {
    const int change = base[r], held = old[r];
    cu[r] = (int)min((int64_t)at, a.tokens);
    at = __builtin_elementwise_add_sat(at, (uint32_t)max(change, 0));
    const bool fits = change >= 0 && at <= (uint32_t)a.tokens && (int64_t)held + change <= room;
    const int needs = fits ? fast_div(held + change + page - 1, a.by_page) - fast_div(held + page - 1, a.by_page) : -1;
    base[r] = needs;
    pages = __builtin_elementwise_add_sat(pages, (uint32_t)max(needs, 0));
  }
  if (r1 == a.batch && r0 < r1) cu[a.batch] = (int)min((int64_t)at, a.tokens);
  uint32_t first = scan_before(pages, sums[1]);
  for (int r = r0; r < r1; ++r) {
    const int needs = base[r];
    const uint32_t behind = __builtin_elementwise_add_sat(first, (uint32_t)max(needs, 0));
    base[r] = needs < 0 || (needs > 0 && behind > (uint32_t)count) ? -1 : needs == 0 ? 0 : (int)first;
    first = behind;
  }
  __syncthreads();
  const int end = cu[a.batch];
  // kTokens consecutive tokens a thread: one search for them, and their loads in flight together.
  const int64_t step = (int64_t)gridDim.x * kThreads * kTokens;
  for (int64_t t0 = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * kTokens; t0 < a.tokens; t0 += step) {
    const int32_t* from[kTokens];
    int32_t* enter[kTokens];
    int in_page[kTokens], place[kTokens];
    int r = t0 < end ? find(cu, a.batch, (int)t0) : 0;
#pragma unroll
    for (int k = 0; k < kTokens; ++k) {
      const int64_t t = t0 + k;
      from[k] = enter[k] = nullptr;
      place[k] = 0;
      if (t >= end) continue;
      while (t >= cu[r + 1]) ++r;
      if (base[r] < 0) continue;
      place[k] = old[r] + (int)t - cu[r];
      const int column = fast_div(place[k], a.by_page), have = fast_div(old[r] + page - 1, a.by_page);
      in_page[k] = place[k] - column * page;
      int32_t* const entry = a.table + r * a.s_table + column;
      from[k] = column < have ? entry : a.stack + (count - 1 - (base[r] + column - have));
      if (column >= have && in_page[k] == 0) enter[k] = entry;
    }
    int id[kTokens];
#pragma unroll
    for (int k = 0; k < kTokens; ++k) id[k] = from[k] != nullptr ? *from[k] : -1;
#pragma unroll
    for (int k = 0; k < kTokens; ++k) {
      if (t0 + k >= a.tokens) break;
      if (enter[k] != nullptr) *enter[k] = id[k];
      a.slots[t0 + k] = id[k] < 0 ? -1 : (int64_t)id[k] * page + in_page[k];
      a.positions[t0 + k] = place[k];
    }
  }
  if (blockIdx.x == 0) {
    for (int r = threadIdx.x; r <= a.batch; r += kThreads) {
      a.cu[r] = cu[r];
      if (r < a.batch) a.granted[r] = base[r] >= 0;
    }
  }
  if (last_workgroup(a)) {
    // what is granted are the first needs of the stack
    __shared__ int taken;
    if (threadIdx.x == 0) taken = 0;
    __syncthreads();
    for (int r = threadIdx.x; r < a.batch; r += kThreads) {
      if (base[r] < 0) {
        a.lens[r] = old[r];
        continue;
      }
      const int grown = old[r] + cu[r + 1] - cu[r];
      a.lens[r] = grown;
      const int needs = fast_div(grown + page - 1, a.by_page) - fast_div(old[r] + page - 1, a.by_page);
      if (needs > 0) atomicMax(&taken, base[r] + needs);
    }
    __syncthreads();
    if (threadIdx.x == 0) *a.count = count - taken;
  }
}

// LDS: base [batch + 1] (pages given back before), keep [batch] (tokens kept)
__global__ void __launch_bounds__(kThreads) kv4_truncate_kernel(const TablesArgs a) {
  extern __shared__ int32_t lds[];
  __shared__ uint32_t sums[kThreads / 64];
  int32_t* const base = lds;
  int32_t* const keep = base + a.batch + 1;
  const int page = a.by_page.d;
  const int64_t room = min((int64_t)a.columns * page, (int64_t)INT32_MAX - page);
  const int count = clamp_int(*a.count, 0, a.capacity);
  const int each = (a.batch + kThreads - 1) / kThreads, r0 = threadIdx.x * each, r1 = min(r0 + each, a.batch);
  uint32_t mine = 0;
  for (int r = r0; r < r1; ++r) {
    const int held = clamp_int(a.lens[r], 0, room), kept = clamp_int(a.change[r], 0, held);
    keep[r] = kept;
    base[r] = fast_div(held + page - 1, a.by_page) - fast_div(kept + page - 1, a.by_page);
    mine = __builtin_elementwise_add_sat(mine, (uint32_t)base[r]);
  }
  arrived(count);
  uint32_t first = scan_before(mine, sums);
  for (int r = r0; r < r1; ++r) {
    const int back = base[r];
    base[r] = (int)min(first, (uint32_t)INT32_MAX);
    first = __builtin_elementwise_add_sat(first, (uint32_t)back);
  }
  if (r1 == a.batch && r0 < r1) base[a.batch] = (int)min(first, (uint32_t)INT32_MAX);
  __syncthreads();
  const int total = base[a.batch];
  for (int64_t g = (int64_t)blockIdx.x * kThreads + threadIdx.x; g < total; g += (int64_t)gridDim.x * kThreads) {
    const int r = find(base, a.batch, (int)g);
    const int column = fast_div(keep[r] + page - 1, a.by_page) + (int)g - base[r];
    int32_t* const entry = a.table + r * a.s_table + column;
    const int64_t to = (int64_t)count + total - 1 - g;
    if (to < a.capacity) a.stack[to] = *entry;
    *entry = -1;
  }
  if (last_workgroup(a)) {
    for (int r = threadIdx.x; r < a.batch; r += kThreads) a.lens[r] = keep[r];
    if (threadIdx.x == 0) *a.count = clamp_int((int64_t)count + total, 0, a.capacity);
  }
}

}  // namespace

int launch_kv4_tables(const tilemix_kv4_tables_params& p, bool extend, hipStream_t stream) {
  const char* const what = extend ? "tilemix_kv4_extend" : "tilemix_kv4_truncate";
  if (p.batch < 0 || p.batch > kMaxBatch || p.table_columns < 0 || p.page_size <= 0 || p.page_size > (1 << 24) ||
      p.free_capacity < 0 || p.tokens < 0 || p.tokens > INT32_MAX) {
    set_error("%s: invalid sizes (batch %d, at most %d, table_columns %d, page_size %d, free pages %d, tokens %lld)",
              what, p.batch, kMaxBatch, p.table_columns, p.page_size, p.free_capacity, (long long)p.tokens);
    return TILEMIX_E_INVALID;
  }
  if (p.batch == 0) {
    if (!extend || p.tokens == 0) return TILEMIX_OK;
    set_error("%s: tokens without a sequence", what);
    return TILEMIX_E_INVALID;
  }
  if (p.seq_lens == nullptr || p.free_count == nullptr || p.ticket == nullptr || p.lens == nullptr ||
      (p.block_table == nullptr && p.table_columns > 0) || (p.free_pages == nullptr && p.free_capacity > 0) ||
      (extend && (p.cu_seqlens == nullptr || p.granted == nullptr ||
                  ((p.slots == nullptr || p.positions == nullptr) && p.tokens > 0)))) {
    set_error("%s: null pointer", what);
    return TILEMIX_E_INVALID;
  }
  TablesArgs a{};
  a.table = p.block_table;
  a.lens = p.seq_lens;
  a.stack = p.free_pages;
  a.count = p.free_count;
  a.ticket = p.ticket;
  a.change = p.lens;
  a.slots = p.slots;
  a.positions = p.positions;
  a.cu = p.cu_seqlens;
  a.granted = p.granted;
  a.s_table = p.stride_table;
  a.tokens = p.tokens;
  a.batch = p.batch;
  a.columns = p.table_columns;
  a.capacity = p.free_capacity;
  a.by_page = make_fast_div(p.page_size);
  if (extend) {
    // Four tokens a thread where that leaves enough workgroups: every one takes its turn at the ticket (300 sequences,
    // 97000 tokens: 13.0 us with one, 10.4 with four; 64 sequences and tokens: 3.4 and 4.6).
    const int each = p.tokens >= 16 * kThreads ? 4 : 1;
    const int64_t share = (int64_t)kThreads * each;
    const int64_t groups = std::min<int64_t>(std::max<int64_t>((p.tokens + share - 1) / share, 1), 256);
    const size_t bytes = (3 * (size_t)p.batch + 1) * sizeof(int32_t);
    const dim3 grid((unsigned)groups), block(kThreads);
    if (each == 4) hipLaunchKernelGGL(kv4_extend_kernel<4>, grid, block, bytes, stream, a);
    else hipLaunchKernelGGL(kv4_extend_kernel<1>, grid, block, bytes, stream, a);
  } else {
    // The pages that go back are known on the device only: at most all entries of the table.
    const int64_t entries = (int64_t)p.batch * p.table_columns;
    const int64_t groups = std::min<int64_t>(std::max<int64_t>((entries + kThreads - 1) / kThreads, 1), 64);
    const size_t bytes = (2 * (size_t)p.batch + 1) * sizeof(int32_t);
    hipLaunchKernelGGL(kv4_truncate_kernel, dim3((unsigned)groups), dim3(kThreads), bytes, stream, a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    set_error("%s: launch failed: %s", what, hipGetErrorString(e));
    return TILEMIX_E_LAUNCH;
  }
  return TILEMIX_OK;
}

}  // namespace tmx
