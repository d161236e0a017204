// paged_attn.hpp -- what the attention kernels of the paged cache share: operand forms of 16-bit and int8 keys and values, scores,
// visible keys, and values that are no numbers.
#pragma once

#include <type_traits>

#include "paged_device.hpp"

namespace ti {

struct PagedAttn {
  PagedCache c;
  PagedRows r;
  const void* q;
  void* out;
  const float* slopes;
  const int32_t* first;
  const int32_t* prefix;
  float* part_o;    // sums of parts of the keys (NULL: none), relative to 2^part_ml[..][0]: [row][head][split][D]; dealt: [head][deal + seqs][D]
  float* part_ml;   // [..][2]: reference, denominator
  int heads, G, ldq, ldo, window, splits, deal;
  float unit;       // of the denominators: int8 kPagedUnit, else 1
  float f, cap;     // weights are 2^(f s), or with a cap 2^(cap paged_capped(s, f))
};

constexpr float kPagedLog2e = 1.44269504088896341f;

// Weights are 2^(exponent - reference).  A column's reference moves (its sums with it) where an exponent passes it by kUp, to the exponent + kSet: fp16
// weights are at most 2^15 and the largest is at least 2^7, so that only what is 2^-21 of it loses bits; bf16 weights, whose range is fp32's, are at
// most 1, so that sums overflow only where the result does.
template <class M>
struct PagedRef {
  static constexpr bool H = std::is_same_v<M, f16>;
  static constexpr float kUp = H ? 15.0f : 0.0f, kSet = H ? -7.0f : 8.0f;
};
// int8: the denominators' terms (weight / vs), at most 2^115 for the least scale, are taken 2^-12 times, the result with them: 2^24 keys fit.
constexpr float kPagedUnit = 0x1p-12f;

// Matrix operands: int8 keys and values are multiplied as fp16, which holds them exactly.
template <class T, bool I8>
struct PagedMat {
  typedef std::conditional_t<I8, f16, T> M;
  typedef M V8 __attribute__((ext_vector_type(8)));
};
__device__ __forceinline__ f32x4 pmma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 pmma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// Two int8 as fp16: bytes (q, 0, q', 0) -> 1024 + 128 + q in both halves (the exponent's bits, the sign bit turned) - 1152.
__device__ __forceinline__ uint32_t i8_pair(uint32_t bytes) {
  const f16x2 h = __builtin_bit_cast(f16x2, bytes ^ 0x64806480u) + (f16x2){(f16)-1152.0f, (f16)-1152.0f};
  return __builtin_bit_cast(uint32_t, h);
}
// Bytes of x: 0 and 1 (hi: 2 and 3) as fp16.
template <bool HI>
__device__ __forceinline__ uint32_t i8_of(uint32_t x) {
  return i8_pair(__builtin_amdgcn_perm(0u, x, HI ? 0x0c030c02u : 0x0c010c00u));
}

// A score under a cap c, c tanh(x) = c - 2 c / (e^2x + 1): what 2 c log2 e (PagedAttn::cap) is multiplied with to an exponent of 2, without the
// first term, which all keys have.  f: 2 scale log2 e / c (int8: times the keys' scale).
__device__ __forceinline__ float paged_capped(float s, float f) { return __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(s * f)); }

// Keys that a row at token p sees: [lo, hi].
struct PagedSpan {
  int lo, hi;
};
__device__ __forceinline__ PagedSpan paged_span(const PagedAttn& a, const PagedSeq& s, int m, int p) {
  int lo = a.window > 0 ? p - a.window + 1 : 0, hi = p;
  if (a.first) lo = max(lo, a.first[m]);
  if (a.prefix) hi = max(hi, max(a.prefix[s.b], 0) - 1);
  return {max(lo, 0), min(hi, s.len - 1)};
}

// Values that are infinities or NaN, where not every column sees the keys (0 times them is NaN): they are counted by the columns that see
// them, and replaced by 0 for the products.
template <class M>
struct PagedOdd {
  static constexpr bool H = std::is_same_v<M, f16>;
  static constexpr uint32_t kExp = H ? 0x7c007c00u : 0x7f807f80u, kLow = H ? 0x04000400u : 0x00800080u, kMan = H ? 0x03ff03ffu : 0x007f007fu;
  static constexpr uint32_t kOne = H ? 0x3c00u : 0x3f80u;
  static constexpr int kBits = H ? 10 : 7;
  typedef M V8 __attribute__((ext_vector_type(8)));
  // bits 15 and 31: the elements of x that are no numbers
  static __device__ __forceinline__ uint32_t any(uint32_t x) { return ((x & kExp) + kLow) & 0x80008000u; }
  static __device__ __forceinline__ uint32_t finite(uint32_t x) { return x & ~((any(x) >> 15) * 0xffffu); }
  // 1 for the keys of a fragment that this lane's column sees (bit e: key e)
  static __device__ __forceinline__ V8 seen(uint32_t see) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (see >> 2 * i & 1) * kOne | (see >> (2 * i + 1) & 1) * (kOne << 16);
    return __builtin_bit_cast(V8, w);
  }
  // 1 in the places of +inf or NaN, of -inf or NaN
  static __device__ __forceinline__ u32x2 signs(uint32_t x) {
    const uint32_t n = any(x) >> 15, neg = x >> 15 & 0x00010001u, nan = ((x & kMan) + kMan) >> kBits & 0x00010001u;
    return (u32x2){(n & (~neg | nan)) * kOne, (n & (neg | nan)) * kOne};
  }
  // acc + what the fragment v's infinities and NaN come to
  static __device__ __forceinline__ f32x4 add(u32x4 v, V8 one, f32x4 acc) {
    u32x4 up, down;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32x2 n = signs(v[i]);
      up[i] = n[0];
      down[i] = n[1];
    }
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f}, n_up = pmma(__builtin_bit_cast(V8, up), one, zero), n_down = pmma(__builtin_bit_cast(V8, down), one, zero);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc[i] = n_up[i] > 0.0f ? acc[i] + INFINITY : acc[i];
      acc[i] = n_down[i] > 0.0f ? acc[i] - INFINITY : acc[i];
    }
    return acc;
  }
};

// The kernel of many rows (paged_prefill.hip): a launch of `tiles` tiles a kv-head, of 32 columns for each of `waves` (4, 8) waves.
int paged_block_run(const PagedAttn& a, const ti_paged_cache* c, int waves, long tiles, hipStream_t s);

}  // namespace ti
