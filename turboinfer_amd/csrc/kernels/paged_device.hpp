// paged_device.hpp -- what the kernels of the paged cache share (paged_cache.hip, paged_attn.hip).
#pragma once

#include "elem.hpp"
#include "paged.hpp"

namespace ti {

typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

struct PagedCache {
  void* k;
  void* v;
  float* ks;
  float* vs;
  const int32_t* table;
  const int32_t* len;
  int table_ld, seqs;
  PagedShape s;
};

// Ragged rows: where the sequences' rows start (NULL: row b is sequence b's).
struct PagedRows {
  const int32_t* start;
  int rows;
};

// A sequence's rows: row0 .. row0 + n - 1 of the call, tokens pos0 ..; len: its keys, within the table.
struct PagedSeq {
  int b, row0, n, pos0, len;
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedCache& c, const PagedRows& r, int b, int from, int to, int len) {
  const int r0 = max(from, 0), r1 = min(to, r.rows), n = max(r1 - r0, 0), most = c.s.blocks * kPagedBlock;
  return {b, r0, n, (int)max((long)len - n, (long)INT32_MIN / 2), min(max(len, 0), most)};
}

// The last sequence whose first tile (row, ..: key(row_start[b], b), not falling) is at most i, by one wave: the number of b in 1 .. seqs - 1
// with key <= i.  Up to 64: one load of all that is asked of it, a lane each (10 rows of 4 prompts 7.3 -> 6.5 us).  More: 64 keys at a time part what is left in 65; an int8
// append of 4096 rows and sequences, and its read, 64 after 64 / so: 256 / 60 us.  Without starts: sequence i.
template <class Key>
__device__ __forceinline__ PagedSeq paged_find(const PagedCache& c, const PagedRows& r, long i, Key key) {
  if (!r.start) return paged_seq(c, r, (int)i, (int)i, (int)i + 1, c.len[i]);
  const int lane = threadIdx.x & 63;
  if (c.seqs <= 64) {
    const int j = min(lane, c.seqs - 1), from = r.start[j], to = r.start[j + 1], len = c.len[j];
    const int b = __popcll(__builtin_amdgcn_ballot_w64(lane > 0 && lane < c.seqs && key(from, j) <= i));
    return paged_seq(c, r, b, __builtin_amdgcn_readlane(from, b), __builtin_amdgcn_readlane(to, b), __builtin_amdgcn_readlane(len, b));
  }
  int b = 0, n = c.seqs;   // of b .. b + n - 1
  while (n > 1) {
    const int step = (n + 64) / 65, at = b + (lane + 1) * step;
    const int below = __popcll(__builtin_amdgcn_ballot_w64((lane + 1) * step < n && key(r.start[at], at) <= i));
    b += below * step;
    n = min(step, n - below * step);
  }
  b = __builtin_amdgcn_readfirstlane(b);
  return paged_seq(c, r, b, r.start[b], r.start[b + 1], c.len[b]);
}

// Values of a 16-bit type.
template <class T>
__device__ __forceinline__ u16x8 pack8(const float* v) {
  typedef T V __attribute__((ext_vector_type(8)));
  V o;
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = (T)v[e];
  return __builtin_bit_cast(u16x8, o);
}

// fn<D, T>(args ..) of the cache's sizes
#define TI_PAGED_FORM(c, fn, ...)                                                                                     \
  ((c)->dtype == TI_PAGED_F16                                                                                        \
       ? (c)->head_dim == 64 ? fn<64, f16>(__VA_ARGS__) : (c)->head_dim == 128 ? fn<128, f16>(__VA_ARGS__) : fn<256, f16>(__VA_ARGS__) \
       : (c)->head_dim == 64 ? fn<64, bf16>(__VA_ARGS__) : (c)->head_dim == 128 ? fn<128, bf16>(__VA_ARGS__) : fn<256, bf16>(__VA_ARGS__))

constexpr int kPagedRows = 1 << 23;   // of a call
}  // namespace ti

// Checks of a cache's description (TI_OK, or the error set), and its kernels' form.
extern "C++" int ti_paged_check(const ti_paged_cache* c, const char* who);
extern "C++" ti::PagedCache ti_paged_form(const ti_paged_cache* c);
