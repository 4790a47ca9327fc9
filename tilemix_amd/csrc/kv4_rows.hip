// Rows of K and V into the paged 4-bit cache and back (format: include/tilemix_hip.h).
// Both are streaming kernels: at head_dim 128 a row is 256 bytes of values and 80 of codes
// and parameters.
#include "kv4_common.h"

#include <algorithm>
#include <type_traits>

namespace tmx {

bool kv4_pool_ok(const char* what, const void* kc, const void* kp, const void* vc, const void* vp, int pages,
                 int page_size, int heads, int head_dim, int dtype) {
  const uintptr_t codes = reinterpret_cast<uintptr_t>(kc) | reinterpret_cast<uintptr_t>(vc);
  const uintptr_t params = reinterpret_cast<uintptr_t>(kp) | reinterpret_cast<uintptr_t>(vp);
  if (kc == nullptr || kp == nullptr || vc == nullptr || vp == nullptr || (codes & 15) != 0 || (params & 3) != 0) {
    set_error("%s: null or misaligned cache pointer", what);
    return false;
  }
  if (pages <= 0 || page_size <= 0 || page_size % 16 != 0 || heads <= 0 || heads > 65535 || head_dim <= 0 ||
      head_dim > 128 || (dtype != 0 && dtype != 1) || (int64_t)pages * heads > INT32_MAX / page_size) {
    set_error("%s: invalid cache (pages %d, page_size %d, heads %d, head_dim %d, dtype %d)", what, pages, page_size,
              heads, head_dim, dtype);
    return false;
  }
  return true;
}

namespace {

struct RowsArgs {
  uint32_t* codes[2];   // K, V
  uint32_t* params[2];
  void* x[2];
  const int64_t* slots;
  const int32_t* table;
  const int32_t* cu;
  int64_t st[2], sh[2], s_table, tokens;
  int pages, heads, d, batch, columns, vec;
  FastDiv by_page;
};

// Thread = one word (eight channels) of the K and the V row of a token (load: of kPer tokens): 4 NG threads a
// row, so that a wave reads whole rows in 16-byte pieces and the four lanes of a group find its range among
// them.  A thread's loads are all in flight together, behind one look at the token's place.
// 16384 tokens of 8 heads x 128, 88 MB each way: load 16.4 us (5.4 TB/s, a large copy's rate; K and V by threads of
// their own 25), store 17.4 (5.1 TB/s; bound by its vector instructions: 20.9 with every value clamped and the codes
// shifted together in whole numbers, 33 with IEEE divisions).
template <int NG>
struct RowSplit {
  static constexpr int kWords = 4 * NG;
  static constexpr int kRows = 256 / kWords;  // at a time (NG = 3: the last four threads idle)
  static constexpr int kPer = 2;
};

// An fp32 result as such: its conversion to fp16 is a rounding of its own, which the compiler would fuse.
__device__ __forceinline__ float keep32(float x) {
  asm volatile("" : "+v"(x));
  return x;
}

__device__ __forceinline__ float quad_xor1(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0xb1, 0xf, 0xf, true));
}
__device__ __forceinline__ float quad_xor2(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x4e, 0xf, 0xf, true));
}

// Eight values; those behind `there` are copies of the first, which the group's range does not notice.
template <typename T>
__device__ __forceinline__ u32x4 read8(const T* x, int there, bool vec) {
  if (vec && there >= 8) return *reinterpret_cast<const u32x4*>(x);
  const uint16_t* const from = reinterpret_cast<const uint16_t*>(x);
  u32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t lo = from[2 * e < there ? 2 * e : 0], hi = from[2 * e + 1 < there ? 2 * e + 1 : 0];
    v[e] = lo | hi << 16;
  }
  return v;
}

// Smallest and largest of eight values, and all of them less a number in fp32, rounded once.  (NaNs are looked for
// elsewhere.)
struct Eight16 {
  f16x2 v[4];
  __device__ __forceinline__ Eight16(const u32x4& raw) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t pair = raw[e];
      v[e] = __builtin_bit_cast(f16x2, pair);
    }
  }
  __device__ __forceinline__ float least() const {
    const f16x2 x = __builtin_elementwise_min(__builtin_elementwise_min(v[0], v[1]), __builtin_elementwise_min(v[2], v[3]));
    return fminf((float)x[0], (float)x[1]);
  }
  __device__ __forceinline__ float most() const {
    const f16x2 x = __builtin_elementwise_max(__builtin_elementwise_max(v[0], v[1]), __builtin_elementwise_max(v[2], v[3]));
    return fmaxf((float)x[0], (float)x[1]);
  }
  __device__ __forceinline__ void cap() {
    const f16x2 top = {(f16)kKv4Limit, (f16)kKv4Limit};
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __builtin_elementwise_min(v[e], top);
  }
  __device__ __forceinline__ float less(int e, float m) const {
    const uint32_t pair = __builtin_bit_cast(uint32_t, v[e >> 1]);
    return e & 1 ? sub_hi(pair, -m) : sub_lo(pair, -m);
  }
};
struct EightBf16 {
  float v[8];
  __device__ __forceinline__ EightBf16(const u32x4& raw) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t pair = raw[e];
      v[2 * e] = __uint_as_float(pair << 16);
      v[2 * e + 1] = __uint_as_float(pair & 0xffff0000u);
    }
  }
  __device__ __forceinline__ float least() const {
    float x = v[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) x = fminf(x, v[e]);
    return x;
  }
  __device__ __forceinline__ float most() const {
    float x = v[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) x = fmaxf(x, v[e]);
    return x;
  }
  __device__ __forceinline__ void cap() {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = fminf(v[e], kKv4Limit);
  }
  __device__ __forceinline__ float less(int e, float m) const { return v[e] - m; }
};

// x / y as an IEEE division rounds it, from the correctly rounded reciprocal r of y: Markstein's correction of the
// quotient (no step underflows for the y >= 2^-24 and quotients below 2^18 here).
__device__ __forceinline__ float divide(float x, float y, float r) {
  const float q = x * r;
  return __builtin_fmaf(__builtin_fmaf(-q, y, x), r, q);
}

// The codes of a word of eight channels and, in every lane of the group, the group's parameters.  kPlain: there is
// neither a NaN nor anything beyond the limit among the wave's values.
template <typename T, bool kPlain>
__device__ __forceinline__ uint32_t quantise8(const u32x4& raw, bool present, bool nan, uint32_t& param) {
  constexpr bool kHalf = std::is_same<T, f16>::value;
  typename std::conditional<kHalf, Eight16, EightBf16>::type v(raw);
  // (the four lanes of a group are in or out together; a word behind the last channel has no say)
  float lo = present ? v.least() : __builtin_inff();
  float hi = present ? v.most() : -__builtin_inff();
  lo = fminf(lo, quad_xor1(lo));
  hi = fmaxf(hi, quad_xor1(hi));
  lo = fminf(lo, quad_xor2(lo));
  hi = fmaxf(hi, quad_xor2(hi));
  if (!kPlain) {
    lo = __builtin_amdgcn_fmed3f(lo, -kKv4Limit, kKv4Limit);
    hi = __builtin_amdgcn_fmed3f(hi, -kKv4Limit, kKv4Limit);
    v.cap();
  }
  f16 s = (f16)keep32(divide(hi - lo, 15.0f, 1.0f / 15.0f)), m = (f16)lo;
  if (!kPlain) {
    float bad = nan && present ? 1.0f : 0.0f;
    bad = fmaxf(bad, quad_xor1(bad));
    bad = fmaxf(bad, quad_xor2(bad));
    if (bad != 0.0f) {
      s = (f16)0.0f;
      m = (f16)__builtin_nanf("");
    }
  }
  param = (uint32_t)__builtin_bit_cast(uint16_t, s) | (uint32_t)__builtin_bit_cast(uint16_t, m) << 16;
  // 1 / s: a Newton step on the hardware reciprocal leaves 2^-22 of a last place before its rounding, and s has 11
  // bits: 1 / s is no nearer than 2^-12 of a last place to where two roundings meet.  So it is the right one.
  const float step = (float)s, least = (float)m, near = __builtin_amdgcn_rcpf(step);
  const float recip = __builtin_fmaf(__builtin_fmaf(-step, near, 1.0f), near, near);
  // A quotient becomes a byte, rounded to the nearest even number and 0 from below; even and odd channels make a word
  // of bytes each.  It is 15.5 or more only where s lost bits of the range: below the normal numbers of
  // fp16, or to a minimum that fp16 does not have.
  uint32_t even = 0, odd = 0;
  auto code = [&](int e, float q) {
    uint32_t& to = e & 1 ? odd : even;
    to = __builtin_amdgcn_cvt_pk_u8_f32(q, e >> 1, to);
  };
  if (kPlain && kHalf && __all(step >= 0x1p-14f || !present)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) code(e, divide(v.less(e, least), step, recip));
    return even | odd << 4;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    code(e, __builtin_amdgcn_fmed3f(divide(v.less(e, least), step, recip), 0.0f, 15.0f));
  return step > 0.0f ? even | odd << 4 : 0u;
}
template <typename T>
__device__ __forceinline__ uint32_t quantise8(const u32x4& raw, bool present, uint32_t& param) {
  constexpr bool kHalf = std::is_same<T, f16>::value;
  constexpr uint32_t kInf = kHalf ? 0x7c00u : 0x7f80u, kMost = kHalf ? 0x7bfcu : 0x477fu;  // kKv4Limit or next below
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  u16x2 size = {};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t pair = raw[e] & 0x7fff7fffu;
    size = __builtin_elementwise_max(size, __builtin_bit_cast(u16x2, pair));
  }
  const uint32_t largest = max((uint32_t)size[0], (uint32_t)size[1]);
  if (__all(largest <= kMost)) return quantise8<T, true>(raw, present, false, param);
  return quantise8<T, false>(raw, present, largest > kInf, param);
}

// (One token a thread: 21.4 us where two took 21.6 and four 24.5, before the last two steps above.)
template <int NG, typename T>
__global__ void __launch_bounds__(256) kv4_store_kernel(const RowsArgs a) {
  using S = RowSplit<NG>;
  const int r = threadIdx.x / S::kWords, w = threadIdx.x - r * S::kWords, h = blockIdx.y;
  const int64_t t = (int64_t)blockIdx.x * S::kRows + r;
  const int there = min(8, a.d - 8 * w);  // channels of this word
  if (r >= S::kRows || t >= a.tokens) return;
  const int64_t slot = a.slots[t];
  u32x4 raw[2];
#pragma unroll
  for (int z = 0; z < 2; ++z)  // (a word behind the last channel reads the row's first)
    raw[z] = read8(static_cast<const T*>(a.x[z]) + t * a.st[z] + h * a.sh[z] + (there > 0 ? 8 * w : 0),
                   there > 0 ? there : 8, a.vec);
  if (slot < 0 || slot >= (int64_t)a.pages * a.by_page.d) return;
  const int page = fast_div((int)slot, a.by_page), at = (int)slot - page * a.by_page.d;
  const int64_t row = ((int64_t)page * a.heads + h) * a.by_page.d + at;
#pragma unroll
  for (int z = 0; z < 2; ++z) {
    uint32_t param, word = quantise8<T>(raw[z], there > 0, param);
    if (there < 8) word &= there > 0 ? (1u << (4 * there)) - 1 : 0u;
    a.codes[z][row * S::kWords + w] = word;
    if ((w & 3) == 0) a.params[z][row * NG + (w >> 2)] = param;
  }
}

template <int NG, typename T>
__global__ void __launch_bounds__(256) kv4_load_kernel(const RowsArgs a) {
  using S = RowSplit<NG>;
  typedef T T8 __attribute__((ext_vector_type(8)));
  const int r = threadIdx.x / S::kWords, w = threadIdx.x - r * S::kWords, h = blockIdx.y;
  const int64_t first = (int64_t)blockIdx.x * (S::kRows * S::kPer);
  // The sequence that holds the workgroup's first row: entries 1 .. batch - 1 of cu at or before it.
  int b = 0;
  for (int i = 1 + (threadIdx.x & 63); i - (int)(threadIdx.x & 63) < a.batch; i += 64)
    b += __popcll(__ballot(i < a.batch && a.cu[i] <= first));
  const int64_t t0 = first + r;
  if (r >= S::kRows || t0 >= a.tokens) return;
  int64_t row[S::kPer];
#pragma unroll
  for (int k = 0; k < S::kPer; ++k) {
    const int64_t t = t0 + k * S::kRows;
    while (b + 1 < a.batch && a.cu[b + 1] <= t) ++b;
    row[k] = -1;
    if (t < a.tokens && a.cu[b] >= 0 && t >= a.cu[b] && t < a.cu[b + 1]) {
      const int at = (int)t - a.cu[b], column = fast_div(at, a.by_page);
      const int page = column < a.columns ? a.table[b * a.s_table + column] : -1;
      if (page >= 0 && page < a.pages) row[k] = ((int64_t)page * a.heads + h) * a.by_page.d + at - column * a.by_page.d;
    }
  }
  uint32_t word[S::kPer][2], param[S::kPer][2];
#pragma unroll
  for (int k = 0; k < S::kPer; ++k)
#pragma unroll
    for (int z = 0; z < 2; ++z) {  // (no row: the pool's first, for nothing)
      const int64_t from = max(row[k], (int64_t)0);
      word[k][z] = a.codes[z][from * S::kWords + w];
      param[k][z] = a.params[z][from * NG + (w >> 2)];
    }
  const int there = min(8, a.d - 8 * w);
#pragma unroll
  for (int k = 0; k < S::kPer; ++k) {
    const int64_t t = t0 + k * S::kRows;
    if (t >= a.tokens) continue;
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      const uint32_t p = row[k] >= 0 ? param[k][z] : 0u;
      const f16x2 sm = __builtin_bit_cast(f16x2, p), s = {sm[0], sm[0]}, m = {sm[1], sm[1]};
      f16x2 v[4];
      kv4_codes(word[k][z], v);
      T8 out;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = kv4_fma(v[i], s, m);
        out[i] = (T)(float)v[i][0];
        out[i + 4] = (T)(float)v[i][1];
      }
      T* x = static_cast<T*>(a.x[z]) + t * a.st[z] + h * a.sh[z] + 8 * w;
      if (a.vec && there == 8) {
        *reinterpret_cast<T8*>(x) = out;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < there) x[e] = out[e];
      }
    }
  }
}

template <int NG>
void launch_rows(const RowsArgs& a, bool store, bool bf, hipStream_t stream) {
  const int rows = RowSplit<NG>::kRows * (store ? 1 : RowSplit<NG>::kPer);
  const dim3 grid((unsigned)((a.tokens + rows - 1) / rows), a.heads), block(256);
  if (store && bf) hipLaunchKernelGGL((kv4_store_kernel<NG, bf16>), grid, block, 0, stream, a);
  else if (store) hipLaunchKernelGGL((kv4_store_kernel<NG, f16>), grid, block, 0, stream, a);
  else if (bf) hipLaunchKernelGGL((kv4_load_kernel<NG, bf16>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((kv4_load_kernel<NG, f16>), grid, block, 0, stream, a);
}

int run_rows(const char* what, const tilemix_kv4_rows_params& p, bool store, hipStream_t stream) {
  if (!kv4_pool_ok(what, p.k_codes, p.k_params, p.v_codes, p.v_params, p.pages, p.page_size, p.heads, p.head_dim,
                   p.dtype))
    return TILEMIX_E_INVALID;
  // The grid has at most 2^24 - 1 workgroups along x (HIP takes fewer than 2^32 threads); the fewest
  // rows of one are 16.
  if (p.tokens < 0 || p.tokens > (int64_t)16 * ((1 << 24) - 1)) {
    set_error("%s: %lld rows in one call", what, (long long)p.tokens);
    return TILEMIX_E_INVALID;
  }
  if (p.tokens == 0) return TILEMIX_OK;
  if (p.k == nullptr || p.v == nullptr || (store && p.slots == nullptr) ||
      (!store && (p.cu_seqlens == nullptr || p.batch <= 0 || p.table_columns < 0 ||
                  (p.block_table == nullptr && p.table_columns > 0)))) {
    set_error("%s: null pointer or no sequence", what);
    return TILEMIX_E_INVALID;
  }
  RowsArgs a{};
  void* const codes[2] = {p.k_codes, p.v_codes};
  void* const params[2] = {p.k_params, p.v_params};
  void* const x[2] = {p.k, p.v};
  const int64_t st[2] = {p.stride_k_token, p.stride_v_token}, sh[2] = {p.stride_k_head, p.stride_v_head};
  a.vec = 1;
  for (int i = 0; i < 2; ++i) {
    a.codes[i] = static_cast<uint32_t*>(codes[i]);
    a.params[i] = static_cast<uint32_t*>(params[i]);
    a.x[i] = x[i];
    a.st[i] = st[i];
    a.sh[i] = sh[i];
    if ((reinterpret_cast<uintptr_t>(x[i]) & 15) != 0 || ((st[i] | sh[i]) & 7) != 0) a.vec = 0;
  }
  a.slots = p.slots;
  a.table = p.block_table;
  a.cu = p.cu_seqlens;
  a.s_table = p.stride_table;
  a.tokens = p.tokens;
  a.pages = p.pages;
  a.heads = p.heads;
  a.d = p.head_dim;
  a.batch = p.batch;
  a.columns = p.table_columns;
  a.by_page = make_fast_div(p.page_size);
  switch ((p.head_dim + kKv4Group - 1) / kKv4Group) {
    case 1:
      launch_rows<1>(a, store, p.dtype == 1, stream);
      break;
    case 2:
      launch_rows<2>(a, store, p.dtype == 1, stream);
      break;
    case 3:
      launch_rows<3>(a, store, p.dtype == 1, stream);
      break;
    default:
      launch_rows<4>(a, store, p.dtype == 1, stream);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    set_error("%s: launch failed: %s", what, hipGetErrorString(e));
    return TILEMIX_E_LAUNCH;
  }
  return TILEMIX_OK;
}

}  // namespace

int launch_kv4_store(const tilemix_kv4_rows_params& p, hipStream_t stream) {
  return run_rows("tilemix_kv4_store", p, true, stream);
}
int launch_kv4_load(const tilemix_kv4_rows_params& p, hipStream_t stream) {
  return run_rows("tilemix_kv4_load", p, false, stream);
}

}  // namespace tmx
