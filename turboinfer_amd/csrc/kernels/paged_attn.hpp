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
  float f, cap;     // weights are 2^(f s), or with a cap 2^(cap paged_capped(s, f)); caps that are not near: 2^(cap tanh(fx s)) (paged_cap)
  float fx;         // scale / the cap, where it is not near
  int far;          // a cap that is not near (paged_cap_near)
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
// first term, which all keys have.  f: 2 scale log2 e / c (int8: times the keys' scale).  Its error goes with the cap, 2^-22 of it.
__device__ __forceinline__ float paged_capped(float s, float f) { return __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(s * f)); }
// So it serves caps of which that is less than a weight's rounding to 16 bits (2^-16 at 64), and with which f is a normal number (at 1 / 16 and a scale of
// 1 also times the keys' largest scale, 2^121).
static inline bool paged_cap_near(float cap, float scale) { return cap >= 0x1p-4f && cap <= 64.0f && fabsf(scale) >= 0x1p-100f; }

// Any other cap: exponents of 2 in place of the scores, C tanh(x), C = c log2 e (PagedAttn::cap), with errors that go with the score.
//   |x| <= 1/2: f s P(x^2), f = scale log2 e, P = tanh(x) / x within 2^-25 (minimax polynomial of 4 terms);
//   else: C - 2 C / (e^2x + 1), where the score is at least 0.46 of the cap.
// Where all of a wave's are small, and they are where a cap is meant to do nothing, only the first is computed.  In kernels of their own: us, 4000 rows of
// 32 heads on 8 of 128, cap 1000, this / paged_capped 194 / 188, int8 223 / 210, heads of 64 164 / 135; with this by a ballot in the kernels of near caps
// those took more registers, cap 30 197 instead of 189, slopes alone 180 instead of 174, int8 of 64 dims 205 instead of 176.
// sc: KT vectors of scores, E of them a block of keys; f, fx (x = fx s) by blocks.
constexpr float kPagedMost = 1e38f;   // of |fx|, so that 2 log2 e times it, times a score of 0, is 0
__device__ __forceinline__ float paged_tanh_ratio(float x) {
  const float u = x * x;
  return fmaf(u, fmaf(u, fmaf(u, fmaf(u, 0x1.1a7c0ep-6f, -0x1.b28c76p-5f), 0x1.10e9fcp-3f), -0x1.5554d6p-2f), 1.0f);
}
template <int E, int KT, class V>
__device__ __forceinline__ void paged_cap(float cap, V (&sc)[KT], const float* f, const float* fx) {
  constexpr int N = sizeof(V) / sizeof(float), B = N / E;
  float top = 0.0f, m[KT * B];
#pragma unroll
  for (int b = 0; b < KT * B; ++b) m[b] = fx[b] > kPagedMost ? kPagedMost : fx[b] < -kPagedMost ? -kPagedMost : fx[b];   // (NaN stays)
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, fabsf(sc[t][i] * m[t * B + i / E]));
#pragma unroll
  for (int b = 0; b < KT * B; ++b) asm volatile("" : "+v"(m[b]));   // (the products again, not 32 of them kept)
  if (__builtin_amdgcn_ballot_w64(top > 0.5f) == 0) {
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int i = 0; i < N; ++i) sc[t][i] *= f[t * B + i / E] * paged_tanh_ratio(sc[t][i] * m[t * B + i / E]);
  } else {
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int b = t * B + i / E;
        const float x = sc[t][i] * m[b], big = fmaf(2.0f * cap, paged_capped(x, 2.0f * kPagedLog2e), cap);
        float y = fabsf(x) > 0.5f ? big : sc[t][i] * f[b] * paged_tanh_ratio(x);
        asm volatile("" : "+v"(y), "+v"(m[b]));   // (a few at a time: registers)
        sc[t][i] = y;
      }
  }
}

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
