// Shared pieces of the paged 4-bit KV cache (format: include/tilemix_hip.h).
#pragma once

#include "attn_common.h"

namespace tmx {

constexpr int kKv4Group = 32;          // channels that share a scale and a minimum
constexpr float kKv4Limit = 65408.0f;  // values are clamped here: 15 s + m < 65520 then rounds to a finite fp16

// (x & mask) | bits in one instruction (the compiler takes two, each with a literal: VOP3 has none).
__device__ __forceinline__ f16x2 kv4_and_or(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "s"(mask), "v"(bits));
  return __builtin_bit_cast(f16x2, r);
}

// The eight codes of a word as four pairs of fp16 whole numbers, channels (0, 4), (1, 5), (2, 6),
// (3, 7).  A code in the low four bits of fp16 1024 (one unit in the last place) reads 1024 + n, in the
// next four of 64 it reads 64 + n; the subtraction is exact.
__device__ __forceinline__ void kv4_codes(uint32_t w, f16x2 (&n)[4]) {
  const uint32_t lo = 0x000f000fu, hi = 0x00f000f0u, k1024 = 0x64006400u, k64 = 0x54005400u;
  const f16x2 m1024 = {(f16)-1024.0f, (f16)-1024.0f}, m64 = {(f16)-64.0f, (f16)-64.0f};
  const uint32_t u = w >> 8;
  n[0] = kv4_and_or(w, lo, k1024) + m1024;
  n[1] = kv4_and_or(w, hi, k64) + m64;
  n[2] = kv4_and_or(u, lo, k1024) + m1024;
  n[3] = kv4_and_or(u, hi, k64) + m64;
}

__device__ __forceinline__ f16x2 kv4_fma(f16x2 n, f16x2 s, f16x2 m) { return __builtin_elementwise_fma(n, s, m); }

// True where the scale or the minimum of a group is an infinity or a NaN.
__device__ __forceinline__ bool kv4_not_finite(uint32_t param) {
  return (param & 0x7c00u) == 0x7c00u || (param & 0x7c000000u) == 0x7c000000u;
}

// x + the values of the lanes before it in the wave (saturating, so that sums past 32 bits stay past every bound).
// Shifts within 16 lanes, then the last lane of a row to the rows behind it.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t add_shifted(uint32_t x) {
  return __builtin_elementwise_add_sat(
      x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  x = add_shifted<0x111, 0xf>(x);
  x = add_shifted<0x112, 0xf>(x);
  x = add_shifted<0x114, 0xf>(x);
  x = add_shifted<0x118, 0xf>(x);
  x = add_shifted<0x142, 0xa>(x);
  x = add_shifted<0x143, 0xc>(x);
  return x;
}

typedef __bf16 bf16;
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

// The checks that the entry points share; what: the entry point's name.
bool kv4_pool_ok(const char* what, const void* kc, const void* kp, const void* vc, const void* vp, int pages,
                 int page_size, int heads, int head_dim, int dtype);

}  // namespace tmx
