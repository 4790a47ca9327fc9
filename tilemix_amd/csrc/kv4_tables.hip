// Page tables of the paged 4-bit cache (include/tilemix_hip.h): tokens and pages for the
// sequences of a step, and pages back, without a word to the host.
//
// Both calls are bound by the launch and by a chain of dependent loads, not by bytes: every
// workgroup sums the whole batch's lengths for itself (two prefix sums over at most 4096 sequences,
// kept in LDS) and then serves its share of the tokens or pages by a search in them, which is
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

// Sum of x over the workgroup's threads before this one; total: over all of them.
__device__ __forceinline__ int64_t scan(int64_t x, int64_t* wave_sums, int64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t sum = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t other = __shfl_up(sum, off, 64);
    if (lane >= off) sum += other;
  }
  __syncthreads();  // the sums of the scan before are read
  if (lane == 63) wave_sums[wave] = sum;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) {
    if (i < wave) before += wave_sums[i];
    total += wave_sums[i];
  }
  return before + sum - x;
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

// True in all threads of the workgroup that comes here last; the others' loads are done by then.
__device__ __forceinline__ bool last_workgroup(const TablesArgs& a) {
  __shared__ int last;
  __syncthreads();
  if (threadIdx.x == 0) {
    last = 1;
    if (gridDim.x > 1) {
      last = __hip_atomic_fetch_add(a.ticket, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
      if (last) __hip_atomic_store(a.ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  __syncthreads();
  return last != 0;
}

__device__ __forceinline__ int clamp_int(int64_t x, int64_t lo, int64_t hi) {
  return (int)(x < lo ? lo : x > hi ? hi : x);
}

// LDS: cu [batch + 1], base [batch] (pages taken before; -1: nothing granted), old [batch] (tokens held)
__global__ void __launch_bounds__(kThreads) kv4_extend_kernel(const TablesArgs a) {
  extern __shared__ int32_t lds[];
  __shared__ int64_t wave_sums[kThreads / 64];
  int32_t* const cu = lds;
  int32_t* const base = cu + a.batch + 1;
  int32_t* const old = base + a.batch;
  const int page = a.by_page.d;
  const int64_t room = min((int64_t)a.columns * page, (int64_t)INT32_MAX - page);
  const int count = clamp_int(*a.count, 0, a.capacity);
  int64_t tokens_before = 0, pages_before = 0, taken = 0;
  for (int r0 = 0; r0 < a.batch; r0 += kThreads) {
    const int r = r0 + threadIdx.x;
    int64_t change = 0;
    int held = 0;
    if (r < a.batch) {
      change = a.change[r];
      held = clamp_int(a.lens[r], 0, room);
    }
    const bool wanted = r < a.batch && change >= 0;
    if (change < 0) change = 0;
    int64_t total;
    const int64_t start = tokens_before + scan(change, wave_sums, total), end = start + change;
    tokens_before += total;
    const bool fits = wanted && end <= a.tokens && held + change <= room;
    const int have = fast_div(held + page - 1, a.by_page);
    const int needs = fits ? fast_div((int)(held + change) + page - 1, a.by_page) - have : 0;
    const int64_t first = pages_before + scan(needs, wave_sums, total);
    pages_before += total;
    const bool ok = fits && (needs == 0 || first + needs <= count);
    if (r < a.batch) {
      cu[r] = clamp_int(start, 0, a.tokens);
      base[r] = ok ? (needs == 0 ? 0 : (int)first) : -1;
      old[r] = held;
      if (r == a.batch - 1) cu[a.batch] = clamp_int(end, 0, a.tokens);
      if (blockIdx.x == 0) {
        a.granted[r] = ok;
        a.cu[r] = clamp_int(start, 0, a.tokens);
        if (r == a.batch - 1) a.cu[a.batch] = clamp_int(end, 0, a.tokens);
      }
    }
    // what is granted ends where the needs first exceed the stack: the largest first + needs within it
    int64_t got = ok && needs > 0 ? first + needs : 0;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) got = max(got, (int64_t)__shfl_xor(got, off, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) wave_sums[threadIdx.x >> 6] = got;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) taken = max(taken, wave_sums[i]);
  }
  __syncthreads();
  const int end = cu[a.batch];
  for (int64_t t = (int64_t)blockIdx.x * kThreads + threadIdx.x; t < a.tokens; t += (int64_t)gridDim.x * kThreads) {
    int64_t slot = -1, position = 0;
    if (t < end) {
      const int r = find(cu, a.batch, (int)t);
      if (base[r] >= 0) {
        const int at = old[r] + (int)t - cu[r], column = fast_div(at, a.by_page);
        const int have = fast_div(old[r] + page - 1, a.by_page), in_page = at - column * page;
        int32_t* const entry = a.table + r * a.s_table + column;
        int id;
        if (column < have) {
          id = *entry;
        } else {
          id = a.stack[count - 1 - (base[r] + column - have)];
          if (in_page == 0) *entry = id;
        }
        position = at;
        slot = id < 0 ? -1 : (int64_t)id * page + in_page;
      }
    }
    a.slots[t] = slot;
    a.positions[t] = position;
  }
  if (last_workgroup(a)) {
    for (int r = threadIdx.x; r < a.batch; r += kThreads)
      a.lens[r] = base[r] < 0 ? old[r] : old[r] + (cu[r + 1] - cu[r]);
    if (threadIdx.x == 0) *a.count = count - (int)taken;
  }
}

// LDS: base [batch + 1] (pages given back before), keep [batch] (tokens kept)
__global__ void __launch_bounds__(kThreads) kv4_truncate_kernel(const TablesArgs a) {
  extern __shared__ int32_t lds[];
  __shared__ int64_t wave_sums[kThreads / 64];
  int32_t* const base = lds;
  int32_t* const keep = base + a.batch + 1;
  const int page = a.by_page.d;
  const int64_t room = min((int64_t)a.columns * page, (int64_t)INT32_MAX - page);
  const int count = clamp_int(*a.count, 0, a.capacity);
  int64_t before = 0;
  for (int r0 = 0; r0 < a.batch; r0 += kThreads) {
    const int r = r0 + threadIdx.x;
    int held = 0, kept = 0;
    if (r < a.batch) {
      held = clamp_int(a.lens[r], 0, room);
      kept = clamp_int(a.change[r], 0, held);
    }
    int64_t total;
    const int back = fast_div(held + page - 1, a.by_page) - fast_div(kept + page - 1, a.by_page);
    const int64_t first = before + scan(back, wave_sums, total);
    before += total;
    if (r < a.batch) {
      base[r] = clamp_int(first, 0, INT32_MAX);
      keep[r] = kept;
      if (r == a.batch - 1) base[a.batch] = clamp_int(first + back, 0, INT32_MAX);
    }
  }
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
    const int64_t groups = std::min<int64_t>(std::max<int64_t>((p.tokens + kThreads - 1) / kThreads, 1), 512);
    const size_t bytes = (3 * (size_t)p.batch + 1) * sizeof(int32_t);
    hipLaunchKernelGGL(kv4_extend_kernel, dim3((unsigned)groups), dim3(kThreads), bytes, stream, a);
  } else {
    // The pages that go back are known on the device only; most calls give back few.
    const int64_t groups = std::min<int64_t>(std::max<int64_t>(((int64_t)p.batch * p.table_columns) / 8192, 1), 64);
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
