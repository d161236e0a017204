// paged_attn.hip -- attention over the paged cache: single tokens and few rows (ti_paged_decode, ti_paged_prefill; many rows:
// paged_prefill.hip).
//
// o = sum_j w_j v_j / sum_j w_j, w_j = 2^(score_j - m): one pass over the keys, the running reference m moved only where a weight
// would pass 2^15 (bf16: 1; PagedRef), the sums following by 2^(m - m').
//
// 16 columns -- (row, query head) pairs that share a kv-head -- are a tile; a workgroup's four waves take the tile's keys 32 at a
// time in turn, straight from HBM into registers:
//   S^T = K Q^T   16x16x32: lane (r = l & 15, g = l >> 4) loads key r of a block of 16; gets the scores of keys 4g .. of column r
//   O^T += V^T P^T 16x16x32 over two blocks: the lane's own 8 weights are its operand; values: the lane loads dims r D/16 .. of keys
//                 4g .. of both blocks (whole rows by 16 lanes), byte permutes make 8 keys of one dim of them.
// So a block's rows come in by whole cache lines, nothing goes through LDS but the waves' sums at the end, and every accumulator
// belongs to the lane's own column.  Blocks that the table does not have, and rows past the sequence's end, are read through
// buffer descriptors of their own size: they come in as zeros whatever memory holds, and are masked.
//
// int8: score (q . k) ks, ks a block's; weights are taken with the values' scale, 2^(score + log2 vs - m), so that fp16 weights stay
// near 1 whatever vs, times exact values; the denominator gets them times 1 / vs.  Queries are scaled to fp16 by a power of 2.
//
// A tile's keys are cut over workgroups, and joined by a second launch (4 - 6 us with its gap): in equal splits (grid z), or, long keys of single tokens,
// as runs of one list of all sequences' steps, so that long sequences keep no workgroup longer than another.
//
// Bound: HBM.  us and TB/s: 32 streams of 4k - 8k, 32 heads on 8 of 128, int8 87 / 4.6, f16 146 / 5.5; one of 128k int8 59 / 4.6; without any arithmetic 82, 145, 57.
// Loads of the next step stand in front of a step's products; loading keys behind theirs, values behind theirs needs no more registers, but int8 took 99.
#include <math.h>
#include <stdio.h>

#include "paged_attn.hpp"

namespace ti {

constexpr int kStreamWaves = 4, kStreamKeys = 32;   // keys a wave takes at a time

// Raw keys and values of 32 keys.
template <int D, bool I8>
struct StreamRaw {
  static constexpr int KW = D / (I8 ? 64 : 32), DV = D / 16, VD = DV * (I8 ? 1 : 2) / 4;   // loads a key tile; dims a lane; dwords a key
  u32x4 k[2][KW];
  uint32_t v[8][VD];
};

template <int VD>
__device__ __forceinline__ void load_dwords(__amdgpu_buffer_rsrc_t rs, int off, uint32_t* to) {
  if constexpr (VD == 1) {
    to[0] = __builtin_amdgcn_raw_buffer_load_b32(rs, off, 0, 0);
  } else if constexpr (VD == 2) {
    const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rs, off, 0, 0));
    to[0] = x[0];
    to[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < VD / 4; ++i) {
      const u32x4 x = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, off + 16 * i, 0, 0));
#pragma unroll
      for (int j = 0; j < 4; ++j) to[4 * i + j] = x[j];
    }
  }
}

template <int D>
struct StreamLds {
  float sums[kStreamWaves][16][D + 4], ml[2][kStreamWaves][16];
};

// One tile of a sequence over some of its keys: steps u0 .. u1 - 1 of 32, counted from the tile's first (u1 < 0: split u0's part of all).
// Sums go to part `at` of a row's head, or (a.splits 1) the result to `out`.
template <int D, class T, bool I8, bool FAR, bool AHEAD>   // FAR: a cap that is not near; AHEAD: the next step's loads stand in front of a step's products
__device__ __forceinline__ void stream_tile(const PagedAttn& a, StreamLds<D>& x_lds, const PagedSeq& s, long tile, int kvh, int u0, int u1, long slot) {
  typedef typename PagedMat<T, I8>::M M;
  typedef typename PagedMat<T, I8>::V8 V8;
  typedef StreamRaw<D, I8> Raw;
  constexpr int NK = D / 32, DV = Raw::DV, ES = I8 ? 1 : 2, NW = kStreamWaves;
  auto& sums = x_lds.sums;
  auto& ml = x_lds.ml;
  const int b = s.b;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int ci = (int)tile * 16 + r, row = ci / a.G, head = kvh * a.G + (ci - row * a.G), m = s.row0 + row, p = s.pos0 + row;
  const bool live = row < s.n && p >= 0 && p < a.c.s.blocks * kPagedBlock;
  PagedSpan span = {1, 0};
  if (live) span = paged_span(a, s, m, p);
  // the tile's keys: any column's, every column's
  const bool some = span.lo <= span.hi;
  int lo_any = some ? span.lo : INT32_MAX, hi_any = some ? span.hi : -1, lo_all = live ? span.lo : 0, hi_all = live ? span.hi : INT32_MAX;
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    lo_any = min(lo_any, __shfl_xor(lo_any, o, 64));
    hi_any = max(hi_any, __shfl_xor(hi_any, o, 64));
    lo_all = max(lo_all, __shfl_xor(lo_all, o, 64));
    hi_all = min(hi_all, __shfl_xor(hi_all, o, 64));
  }
  lo_any = __builtin_amdgcn_readfirstlane(lo_any);
  hi_any = __builtin_amdgcn_readfirstlane(hi_any);
  lo_all = __builtin_amdgcn_readfirstlane(lo_all);
  hi_all = __builtin_amdgcn_readfirstlane(hi_all);

  // queries: 16-bit keys' step c: dims 32 c + 8 g ..; int8: dims 64 (c / 2) + 16 g + 8 (c & 1) ..
  V8 qf[NK];
  float f = a.f, fx = a.fx;
  {
    const T* qr = (const T*)a.q + (size_t)m * a.ldq + (size_t)head * D;
    u16x8 raw[NK];
#pragma unroll
    for (int c = 0; c < NK; ++c) {
      raw[c] = (u16x8){};
      if (live) raw[c] = *(const u16x8*)(qr + (I8 ? 64 * (c >> 1) + 16 * g + 8 * (c & 1) : 32 * c + 8 * g));
    }
    if constexpr (std::is_same_v<M, T>) {
#pragma unroll
      for (int c = 0; c < NK; ++c) qf[c] = __builtin_bit_cast(V8, raw[c]);
    } else {   // bf16 queries as fp16: the column's largest brought to [1, 2), exactly; smaller ones by 2^-24 of it at worst
      uint32_t top = 0;
#pragma unroll
      for (int c = 0; c < NK; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, raw[c][e] & 0x7f80u);
      top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
      top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
      const int ex = (int)(top >> 7) - 127;   // (0, subnormal, infinite: as they are)
      const bool scaled = top != 0 && top != 0x7f80u;
      const float up = scaled ? ldexpf(1.0f, -ex) : 1.0f;
      if (scaled) {
        f = ldexpf(f, ex);
        fx = ldexpf(fx, ex);
      }
#pragma unroll
      for (int c = 0; c < NK; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) qf[c][e] = (M)(__builtin_bit_cast(float, (uint32_t)raw[c][e] << 16) * up);
    }
  }
  const float slope = a.slopes && live ? a.slopes[head] * kPagedLog2e : 0.0f;

  f32x4 o[DV];
#pragma unroll
  for (int t = 0; t < DV; ++t) o[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
  float mr = -INFINITY, lr = 0.0f;   // o, lr: relative to 2^mr

  const int step_lo = hi_any < 0 ? 0 : lo_any / kStreamKeys, n_steps = hi_any < 0 ? 0 : hi_any / kStreamKeys + 1 - step_lo;
  if (u1 < 0) {
    const int each = (n_steps + a.splits - 1) / a.splits;
    u0 *= each;
    u1 = u0 + each;
  }
  const int s0 = step_lo + u0, s1 = step_lo + min(u1, n_steps);
  {
    for (int at = s0 + wave; at < s1; at += 32 * NW) {
      // lane 2 i + t: block t of the wave's i-th step from here
      const int my = at + (lane >> 1) * NW, blk = 2 * my + (lane & 1);
      int id = -1;
      if (my < s1 && blk < a.c.s.blocks) id = paged_block(a.c.s, a.c.table[(size_t)b * a.c.table_ld + paged_column(a.c.s, blk)], kvh, blk);
      float ks = 1.0f, vs = 1.0f;
      if (I8 && id >= 0) {
        ks = a.c.ks[id];
        vs = a.c.vs[id];
        vs = vs < kPagedTiny ? kPagedTiny : vs;
      }
      const int n = min(32, (s1 - at + NW - 1) / NW);
      auto load = [&](int i, Raw& x) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int ib = i < n ? __builtin_amdgcn_readlane(id, 2 * (i & 31) + t) : -1;
          const int have = ib < 0 ? 0 : min(16, s.len - 16 * (2 * (at + i * NW) + t)) * D * ES;   // (bytes of the block that there are)
          const size_t off = (size_t)max(ib, 0) * (16 * D * ES);
          const auto krs = __builtin_amdgcn_make_buffer_rsrc((char*)a.c.k + off, 0, max(have, 0), 0x00020000);
          const auto vrs = __builtin_amdgcn_make_buffer_rsrc((char*)a.c.v + off, 0, max(have, 0), 0x00020000);
#pragma unroll
          for (int c = 0; c < Raw::KW; ++c)
            x.k[t][c] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(krs, r * D * ES + 64 * c + 16 * g, 0, 0));
#pragma unroll
          for (int e = 0; e < 4; ++e) load_dwords<Raw::VD>(vrs, ((4 * g + e) * D + r * DV) * ES, x.v[4 * t + e]);
        }
      };
      auto compute = [&](int i, Raw& x) {
        f32x4 sc[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          sc[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < NK; ++c) {
            u32x4 kw;
            if constexpr (I8) {
              const uint32_t w0 = x.k[t][c >> 1][2 * (c & 1)], w1 = x.k[t][c >> 1][2 * (c & 1) + 1];
              kw = (u32x4){i8_of<false>(w0), i8_of<true>(w0), i8_of<false>(w1), i8_of<true>(w1)};
            } else {
              kw = x.k[t][c];
            }
            sc[t] = pmma(__builtin_bit_cast(V8, kw), qf[c], sc[t]);
          }
        }
        const int key0 = (at + i * NW) * kStreamKeys;
        const int id0 = __builtin_amdgcn_readlane(id, 2 * i), id1 = __builtin_amdgcn_readlane(id, 2 * i + 1);
        const bool ragged = key0 < lo_all || key0 + kStreamKeys - 1 > hi_all || (id0 | id1) < 0;
        float vl[2] = {0.0f, 0.0f}, vi[2] = {1.0f, 1.0f};
        if constexpr (FAR) {
          float fk[2] = {f, f}, fxk[2] = {fx, fx};
          if constexpr (I8)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const float sk = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ks), 2 * i + t));
              fk[t] *= sk;
              fxk[t] *= sk;
            }
          paged_cap<4>(a.cap, sc, fk, fxk);
        }
        float mx = -INFINITY;
        uint32_t see = 255;
        if (ragged) {
          int lo = span.lo;
          asm volatile("" : "+v"(lo));   // (a branch, not selects: most steps skip it)
          see = 0;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int j = key0 + 16 * t + 4 * g + e;
              if (j >= lo && j <= span.hi && (t ? id1 : id0) >= 0) see |= 1u << (4 * t + e);
            }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          float ft = FAR ? 1.0f : f;
          if constexpr (I8) {
            if constexpr (!FAR) ft *= __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ks), 2 * i + t));
            const float sv = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, vs), 2 * i + t));
            vl[t] = __builtin_amdgcn_logf(sv);
            vi[t] = ragged && !(see >> 4 * t & 15) ? 0.0f : __builtin_amdgcn_rcpf(sv) * kPagedUnit;   // (0 of a block, whose scale may be NaN)
          }
          if (!FAR && a.cap != 0.0f) {
            asm volatile("" : "+v"(ft));
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[t][e] = paged_capped(sc[t][e], ft);
            ft = a.cap;
          }
          if (a.slopes) {
            float slope_ = slope;
            asm volatile("" : "+v"(slope_));
            const float base = fmaf(slope_, (float)(key0 + 16 * t + 4 * g - p), vl[t]);
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[t][e] = fmaf(sc[t][e], ft, fmaf(slope_, (float)e, base));
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[t][e] = I8 ? fmaf(sc[t][e], ft, vl[t]) : sc[t][e] * ft;
          }
          if (ragged) {
            uint32_t have = see;
            asm volatile("" : "+v"(have));
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!(have >> (4 * t + e) & 1)) sc[t][e] = -INFINITY;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) mx = fmaxf(mx, sc[t][e]);
        }
        mx = xor32_max(xor16_max(mx));
        typedef PagedRef<M> Ref;
        if (__builtin_amdgcn_ballot_w64(mx > mr + Ref::kUp) != 0) {
          const float mn = mx > mr + Ref::kUp ? mx + Ref::kSet : mr, alpha = mn == mr ? 1.0f : __builtin_amdgcn_exp2f(mr - mn);
          mr = mn;
          lr *= alpha;
#pragma unroll
          for (int t = 0; t < DV; ++t) o[t] *= alpha;
        }
        const float off = mr == -INFINITY ? 0.0f : mr;
        V8 pf;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          float l = 0.0f;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float w = __builtin_amdgcn_exp2f(sc[t][e] - off);
            l += w;
            pf[4 * t + e] = (M)w;
          }
          lr = fmaf(l, vi[t], lr);
        }
        // 8 keys of dims r DV + t: the values' operand
        auto frag = [&](int t) {
          u32x4 vw;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (I8) {
              const uint32_t sel = 0x0c000c00u | (uint32_t)(t & 3) | (uint32_t)(4 + (t & 3)) << 16;
              vw[e] = i8_pair(__builtin_amdgcn_perm(x.v[2 * e + 1][t >> 2], x.v[2 * e][t >> 2], sel));
            } else {
              vw[e] = __builtin_amdgcn_perm(x.v[2 * e + 1][t >> 1], x.v[2 * e][t >> 1], t & 1 ? 0x07060302u : 0x05040100u);
            }
          }
          return vw;
        };
        if constexpr (!I8)
          if (ragged) {
            typedef PagedOdd<M> Odd;
            uint32_t bad = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
              for (int w = 0; w < Raw::VD; ++w) bad |= Odd::any(x.v[e][w]);
            if (__builtin_amdgcn_ballot_w64(bad != 0) != 0) {
              const V8 one = Odd::seen(see);
#pragma unroll
              for (int t = 0; t < DV; ++t) o[t] = Odd::add(frag(t), one, o[t]);
#pragma unroll
              for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int w = 0; w < Raw::VD; ++w) x.v[e][w] = Odd::finite(x.v[e][w]);
            }
          }
#pragma unroll
        for (int t = 0; t < DV; ++t) o[t] = pmma(__builtin_bit_cast(V8, frag(t)), pf, o[t]);
      };
      if constexpr (AHEAD) {
        Raw x0, x1;
        load(0, x0);
        for (int i = 0; i < n; i += 2) {
          load(i + 1, x1);
          compute(i, x0);
          load(i + 2, x0);
          if (i + 1 < n) compute(i + 1, x1);
        }
      } else {
        Raw x0;
        for (int i = 0; i < n; ++i) {
          load(i, x0);
          compute(i, x0);
        }
      }
    }
  }
  lr += lane_xor<16>(lr);
  lr += lane_xor<32>(lr);
  // the waves' sums: dims (4 g + i) DV + t of column r
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int t = 0; t < DV; ++t) sums[wave][r][(4 * g + i) * DV + t] = o[t][i];
  if (g == 0) {
    ml[0][wave][r] = mr;
    ml[1][wave][r] = lr;
  }
  __syncthreads();
  const int col = threadIdx.x >> 4, part = threadIdx.x & 15;   // thread: dims part * DV .. of column col
  const int cj = (int)tile * 16 + col, row_c = cj / a.G, head_c = kvh * a.G + (cj - row_c * a.G), p_c = s.pos0 + row_c;
  if (row_c >= s.n || p_c < 0 || p_c >= a.c.s.blocks * kPagedBlock) return;
  float mm = -INFINITY, l = 0.0f, w[NW];
#pragma unroll
  for (int i = 0; i < NW; ++i) mm = fmaxf(mm, ml[0][i][col]);
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const float mi = ml[0][i][col];
    w[i] = mi == -INFINITY && ml[1][i][col] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(mi - mm);
    l += ml[1][i][col] * w[i];
  }
  float acc[DV];
#pragma unroll
  for (int d = 0; d < DV; ++d) {
    acc[d] = 0.0f;
#pragma unroll
    for (int i = 0; i < NW; ++i)
      if (w[i] != 0.0f) acc[d] += w[i] * sums[i][col][part * DV + d];
  }
  if (a.part_o) {
    const size_t at = a.deal ? (size_t)head_c * (a.deal + a.c.seqs) + slot : ((size_t)(s.row0 + row_c) * a.heads + head_c) * a.splits + slot;
    if (part == 0) *(float2*)(a.part_ml + 2 * at) = make_float2(mm, l);
    float* po = a.part_o + at * D + part * DV;
#pragma unroll
    for (int d = 0; d < DV; d += 4) *(f32x4*)(po + d) = (f32x4){acc[d], acc[d + 1], acc[d + 2], acc[d + 3]};
    return;
  }
  const float inv = a.unit / l;
  T* out = (T*)a.out + (size_t)(s.row0 + row_c) * a.ldo + (size_t)head_c * D + part * DV;
#pragma unroll
  for (int d = 0; d < DV; d += 4) {
    typedef T Q4 __attribute__((ext_vector_type(4)));
    Q4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (T)(l == 0.0f ? 0.0f : acc[d + e] * inv);
    *(Q4*)(out + d) = y;
  }
}

// Grid (tiles, kv-heads, splits).  Steps are few: more waves a CU instead of the next step's loads in flight (us, 46 x 30 - 84 keys, 32 heads on 32: dims of
// 128 18.6 -> 13.8, 256 52.6 -> 34.0, in int8 45.8 -> 25.0; 64 x 145 - 200 of 128 dims 42.6 -> 38.1).
template <int D, class T, bool I8, bool FAR>
__global__ __launch_bounds__(64 * kStreamWaves, D == 256 ? 2 : 3) void paged_stream_kernel(const PagedAttn a) {
  __shared__ StreamLds<D> lds;
  const int per_seq = (a.G + 15) >> 4;
  const PagedSeq s = paged_find(a.c, a.r, a.r.start ? (int)blockIdx.x : (int)blockIdx.x / per_seq,
                                [&](int start, int j) { return paged_tile0((long)start * a.G, j, 16); });
  const long tile = a.r.start ? blockIdx.x - paged_tile0((long)s.row0 * a.G, s.b, 16) : (int)blockIdx.x - s.b * per_seq;
  if (tile < 0 || tile * 16 >= (long)s.n * a.G) return;
  stream_tile<D, T, I8, FAR, false>(a, lds, s, tile, blockIdx.y, blockIdx.z, -1, blockIdx.z);
}

// Single tokens: steps of 32 keys that sequence b's row sees.
__device__ __forceinline__ int decode_steps(const PagedAttn& a, int b) {
  const int len = a.c.len[b], p = len - 1;
  if (p < 0 || p >= a.c.s.blocks * kPagedBlock) return 0;
  int lo = a.window > 0 ? max(p - a.window + 1, 0) : 0;
  if (a.first) lo = max(lo, a.first[b]);
  return lo > p ? 0 : p / kStreamKeys - lo / kStreamKeys + 1;
}
__device__ __forceinline__ long uniform(long v) {
  return (long)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}
// Sum over this lane and those in front of it.  (64 sequences of less than 2^26 steps, as paged_plan sees to: 32 bits unsigned.)
__device__ __forceinline__ unsigned wave_scan(unsigned v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}
// Steps of a run.  us, 1 / 2 / 4 / 8: one kv-head of 128 dims, int8, one stream of 12000 keys 19.6 / 15.3 / 14.5 / 13.8, two of 6500 16.2 / 14.3 / 13.1 / 17.3; f16, two of
// 12000 14.3 / 14.7 / 17.1 / 16.6, of 256 dims 22.1 / 22.0 / 25.8 / 25.8.
constexpr int kDealLeast = 2;
__device__ __forceinline__ long deal_run(const PagedAttn& a, long all) { return max((all + a.deal - 1) / a.deal, (long)kDealLeast); }

// The steps of all sequences are one list, cut into equal runs for the a.deal workgroups of a kv-head: grid (a.deal, kv-heads * tiles of 16
// query heads).  Part w + b of a head is workgroup w's of sequence b: each differs from the one in front by 1 in
// w or more in b.
template <int D, class T, bool I8, bool FAR>
__global__ __launch_bounds__(64 * kStreamWaves, D == 256 && !I8 ? 1 : 2) void paged_deal_kernel(const PagedAttn a) {
  __shared__ StreamLds<D> lds;
  const int lane = threadIdx.x & 63, w = blockIdx.x, per_seq = (a.G + 15) >> 4, kvh = blockIdx.y / per_seq, tile = blockIdx.y - kvh * per_seq;
  int mine = lane < a.c.seqs ? decode_steps(a, lane) : 0;
  unsigned sum = wave_scan(mine);
  long all = (unsigned)__builtin_amdgcn_readlane((int)sum, 63);
  for (int b0 = 64; b0 < a.c.seqs; b0 += 64)
    all += (unsigned)__builtin_amdgcn_readlane((int)wave_scan(b0 + lane < a.c.seqs ? decode_steps(a, b0 + lane) : 0), 63);
  const long per = uniform(deal_run(a, all)), from = w * per, to = from + per;
  if (from >= all) return;
  // the sequence that step `from` is in
  long base = 0;   // steps in front of b
  int b = 0, n = 0;
  for (int b0 = 0;;) {
    const unsigned long long past = __builtin_amdgcn_ballot_w64(base + sum > from);
    if (past) {
      const int l = __builtin_ctzll(past);
      b = b0 + l;
      n = __builtin_amdgcn_readlane(mine, l);
      base += (unsigned)__builtin_amdgcn_readlane((int)sum, l) - (unsigned)n;
      break;
    }
    base += (unsigned)__builtin_amdgcn_readlane((int)sum, 63);
    b0 += 64;
    if (b0 >= a.c.seqs) return;
    mine = b0 + lane < a.c.seqs ? decode_steps(a, b0 + lane) : 0;
    sum = wave_scan(mine);
  }
  base = uniform(base);
  for (; n > 0; n = b < a.c.seqs ? __builtin_amdgcn_readfirstlane(decode_steps(a, b)) : 0) {
    stream_tile<D, T, I8, FAR, !(D == 256 && I8)>(a, lds, paged_seq(a.c, a.r, b, b, b + 1, a.c.len[b]), tile, kvh, (int)(max(from, base) - base), (int)min((long)n, to - base), (long)w + b);
    base += n;
    if (base >= to) break;
    do ++b;
    while (b < a.c.seqs && __builtin_amdgcn_readfirstlane(decode_steps(a, b)) == 0);
    __syncthreads();
  }
}

// The parts of single tokens: a workgroup a (row, head), four waves in turn.
template <int D, class T>
__global__ __launch_bounds__(256) void deal_join_kernel(const PagedAttn a) {
  constexpr int E = D / 64;
  __shared__ float sums[4][D], ls[4];
  const int lane = threadIdx.x & 63, m = blockIdx.x, head = blockIdx.y, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = m, p = a.c.len[b] - 1;
  if (p < 0 || p >= a.c.s.blocks * kPagedBlock) return;
  long all = 0, before = 0;   // steps of all sequences, of those in front of b
  int own = 0;
  for (int b0 = 0; b0 < a.c.seqs; b0 += 64) {
    const int mine = b0 + lane < a.c.seqs ? decode_steps(a, b0 + lane) : 0;
    const unsigned sum = wave_scan(mine);
    if ((b ^ b0) < 64) {   // (b0 is a multiple of 64)
      own = __builtin_amdgcn_readlane(mine, b - b0);
      before = all + ((unsigned)__builtin_amdgcn_readlane((int)sum, b - b0) - (unsigned)own);
    }
    all += (unsigned)__builtin_amdgcn_readlane((int)sum, 63);
  }
  const long per = deal_run(a, all), w0 = before / per;
  const size_t at = (size_t)head * (a.deal + a.c.seqs) + w0 + b;
  const int n = own ? (int)((before + own - 1) / per - w0) + 1 : 0;
  float mm = -INFINITY;
  for (int i = lane; i < n; i += 64) mm = fmaxf(mm, a.part_ml[2 * (at + i)]);
  mm = wave_max(mm);
  float l = 0.0f, acc[E] = {};
  for (int i0 = wave * 16; i0 < n; i0 += 64) {   // 16 parts at a time
    float w = 0.0f;
    if (lane < 16 && i0 + lane < n) {
      const float2 x = *(const float2*)(a.part_ml + 2 * (at + i0 + lane));
      w = x.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(x.x - mm);
      l += x.y * w;
    }
    float x[16][E];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float* po = a.part_o + (at + min(i0 + j, n - 1)) * D + lane * E;
#pragma unroll
      for (int e = 0; e < E; ++e) x[j][e] = po[e];
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float wj = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), j));
      if (wj != 0.0f)   // (a part without keys holds no sums)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(wj, x[j][e], acc[e]);
    }
  }
  l = group_sum<64>(l);
#pragma unroll
  for (int e = 0; e < E; ++e) sums[wave][lane * E + e] = acc[e];
  if (lane == 0) ls[wave] = l;
  __syncthreads();
  if (threadIdx.x >= D) return;
  const int d = threadIdx.x;
  l = (ls[0] + ls[1]) + (ls[2] + ls[3]);
  const float o = (sums[0][d] + sums[1][d]) + (sums[2][d] + sums[3][d]);
  ((T*)a.out)[(size_t)m * a.ldo + (size_t)head * D + d] = (T)(l == 0.0f ? 0.0f : o * (a.unit / l));
}

// The splits of rows: D / 4 threads a (row, head), 1024 / D heads a workgroup.  Grid (rows, groups of heads).
template <int D, class T>
__global__ __launch_bounds__(256) void split_join_kernel(const PagedAttn a) {
  constexpr int NT = D / 4, NH = 256 / NT, U = 8;
  const int m = blockIdx.x, d = threadIdx.x % NT * 4, head = blockIdx.y * NH + threadIdx.x / NT;
  const PagedSeq s = paged_find(a.c, a.r, m, [](int start, int) { return (long)start; });
  const int p = s.pos0 + (m - s.row0);
  if (m < s.row0 || m >= s.row0 + s.n || p < 0 || p >= a.c.s.blocks * kPagedBlock || head >= a.heads) return;
  const size_t at = ((size_t)m * a.heads + head) * a.splits;
  const float2* ml = (const float2*)a.part_ml + at;
  const float* po = a.part_o + at * D + d;
  float mm = -INFINITY, l = 0.0f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = 0; i0 < a.splits; i0 += U) {   // (the sums so far follow the reference)
    float2 x[U];
    f32x4 y[U];
#pragma unroll
    for (int i = 0; i < U; ++i) x[i] = i0 + i < a.splits ? ml[i0 + i] : make_float2(-INFINITY, 0.0f);
#pragma unroll
    for (int i = 0; i < U; ++i) y[i] = *(const f32x4*)(po + (size_t)min(i0 + i, a.splits - 1) * D);
    float mn = mm;
#pragma unroll
    for (int i = 0; i < U; ++i) mn = fmaxf(mn, x[i].x);
    const float back = mm == mn ? 1.0f : __builtin_amdgcn_exp2f(mm - mn);
    mm = mn;
    l *= back;
    acc *= back;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const float w = x[i].y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(x[i].x - mm);   // (a split without keys holds no sums)
      l = fmaf(x[i].y, w, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = w != 0.0f ? fmaf(w, y[i][e], acc[e]) : acc[e];
    }
  }
  typedef T Q4 __attribute__((ext_vector_type(4)));
  Q4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = (T)(l == 0.0f ? 0.0f : acc[e] * (a.unit / l));
  *(Q4*)((T*)a.out + (size_t)m * a.ldo + (size_t)head * D + d) = y;
}

// A call's kernel and splits of its keys: enough workgroups for the CUs.
struct PagedPlan {
  int waves;          // of paged_prefill.hip's kernel (0: this file's)
  long tiles;
  int splits, most;   // most: splits of any length
  int deal;           // workgroups a kv-head and tile of query heads that share all keys (0: a workgroup a tile and split)
  long filled;        // workgroups with work, about
};
static PagedPlan paged_plan(const ti_paged_cache* c, const ti_paged_attn_args* p) {
  const int G = p->heads / c->kv_heads;
  const long columns = (long)p->rows * G, per_seq = columns / c->seqs;
  const bool i8 = c->kv_type == TI_KV_I8;
  long span = (long)c->table_ld * c->page;
  if (p->max_len > 0) span = std::min<long>(span, p->max_len);
  auto seen = [&](long rows) { return p->window > 0 && !p->prefix ? std::min(span, p->window + rows) : span; };   // by a tile of these rows

  // This file's kernels.  A split has a step of each wave at least, from 17 splits on two: us, one / two, a row behind 8k of 8 kv-heads 19.6 / 16.4,
  // 4 rows 25 / 20, one token of 5k 15.9 / 13.9 (1000 keys of 256 dims 12.8 / 14.6).  64 splits at most: a row behind 64k of one kv-head, 32 / 64 / 256
  // splits 31 / 26 / 43, int8 128k of 8 59 / 60 / 74.
  // Two workgroups a CU: us, 1024 / 768 / 512 in all, 64 streams of 700, 8 kv-heads of 128 41 / 41 / 36, of 256 86 / 86 / 77, int8 16 of 2000 of 256 39 / 41
  // / 33, 40 of 700 of 128 21 / 19 / 20.  Few keys in one split and launch: us, one / two or more, 16 streams of 500 of 128 10.5 / 13.5, one of 256 7.6 / 9.9,
  // of 500 9.5 / 10.0, of 768 11 - 12 / 9.8; of 64 dims, 768 8.6 / 9.8, 1024 9.8 / 9.9; of 256 dims, 256 11.5 / 12.6, 500 16 / 13.
  const long tiles = p->row_start ? paged_tiles(columns, c->seqs, 16) : (long)c->seqs * ((G + 15) / 16), units = std::max(1l, tiles * c->kv_heads);
  const long keys = seen(16), steps = (keys + kStreamKeys - 1) / kStreamKeys, most = std::min((512 + units - 1) / units, 64l);
  PagedPlan stream{0, tiles, (int)std::max(1l, std::min({keys * c->head_dim <= 65536 ? 1l : most, (steps + 3) / 4, std::max(16l, (steps + 7) / 8)})), (int)most, 0, 0};
  if (!p->row_start) {
    // Dealing pays where a tile's keys are many and uneven; it has every workgroup look through all lengths, and joins all.  us, splits / dealt, 8
    // kv-heads of 128: 16 streams of 1 - 4k 39 / 38, 1 - 8k 68 / 61, 1 - 16k 121 / 102; 4 of 2k 15 / 20, 1 - 32k 71 / 59; 64 of 1 - 2k 64 / 70, 1 - 4k 117 /
    // 107; 160 of 1 - 2k 134 / 150; 1024 of 1 - 680 373 / 654.  Of 256 dims, whose waves hold fewer loads, sooner: 16 of 500 - 1500 50 / 45, 48 of 1000 - 3000
    // 183 / 165, 160 of 2 heads 167 / 166.  Workgroups a CU: 1 (32 streams of 4k - 8k, f16 of 128 dims, 1 / 2 / 3: 146 / 151 / 151 us; 48 capped
    // of 256 dims 87 / 100 / 122), but 2 of int8 heads up to 128 dims, whose waves convert (64 of 64 dims 60 / 50 / 52, 64 x 700 37 / 32 / 39).
    // Rounded down: 52 heads, 4 / 5 workgroups each 164 / 229; from 257 heads on splits (300: 213 / 173, 250: 144 / 144).
    const long lists = c->kv_heads * (long)((G + 15) / 16);
    const int deal = (int)std::max(1l, (i8 && c->head_dim < 256 ? 512l : 256l) / lists);
    // (64 sequences of the longest table's 2^26 steps would pass the runs' sums: wave_scan)
    const bool sums = (long)c->table_ld * c->page <= (1l << 31) - kStreamKeys;
    const long bytes = 2l * c->seqs * c->kv_heads * keys * c->head_dim * (i8 ? 1 : 2), seqs = c->seqs;
    if (sums && lists <= 256 && (keys >= 6144 || bytes >= 192l << 20) &&
        keys >= (c->head_dim == 256 ? std::max(512l, 20 * seqs) : std::max(2048l, 48 * seqs))) stream.deal = deal;
    stream.most = std::max(stream.most, deal / c->seqs + 2);   // (its seqs + deal parts a head, as splits of seqs rows)
    return stream;
  }
  // From 32 columns a sequence on keys are shared in LDS.  us, stream / block: 16 sequences behind 2k, 8 rows of 32 heads on 8 52 / 39, 64 behind
  // 600, 16 rows 98 / 63; 32 behind 2k, 4 rows (16 columns) 70 / 70.  But the first steps of a block take 8 us and its splits' join 4: not a few tiles
  // of few keys.  32 heads on 8 of 128: a prompt of 16 rows 7 / 10, 64 behind 600 16 / 19, 100 behind 300 11 / 20, 600 18 / 20, 4 x 20 behind 1000 24 / 21,
  // on 32, 100 behind 600 22 / 20; int8 100 behind 600 18 / 23, 4 x 20 behind 1000 21 / 23; of 256 dims, 40 behind 600 23 / 32, 100 behind 300 38 / 34, int8
  // 29 / 37.
  const bool few = units <= 256;
  if (per_seq < 32 || (few && units * seen(per_seq / G) <= (c->head_dim == 256 ? 65536 : 131072) * (i8 ? 2 : 1))) return stream;
  // waves of a workgroup, workgroups that fill the CUs, least steps of a split (a prompt's own keys: half of them seen)
  auto form = [&](int waves, long want, long least) {
    const int cols = c->head_dim == 256 ? 128 : 32 * waves;
    const long full = (long)c->seqs * ((per_seq + cols - 1) / cols) * c->kv_heads;
    const long n = (seen(cols) - std::min(seen(cols), per_seq / G) / 2 + 63) / 64;
    const long most = std::max(1l, std::min(want / full, 64l)), splits = std::max(1l, std::min(most, n / least));
    return PagedPlan{waves, paged_tiles(columns, c->seqs, cols), (int)splits, (int)std::max<long>(most, few ? stream.most : 1), 0, full * splits};
  };
  if (c->head_dim == 256) return form(8, 256, 4);
  // Eight waves read each block of keys from L2 and convert it once for twice the columns, two workgroups of four hide each other's
  // waits: eight for long keys and enough columns, four where prompts are short, CUs would idle, or (heads of 64) three workgroups of four fit
  // a CU.  us, 8 / 4 waves, 32 heads on 8 of 128: 4000 rows 155 / 172, capped 205 / 214, 3 x 512 behind 4k 152 / 166, int8 173 / 192, 128 behind 32k int8
  // 105 / 109, 4 x 256 behind 2k 65 / 68, 1600 behind 1500 113 / 104; 2000 rows 69 / 62, 1000 36 / 35, 8 x 200 rows of 32 heads on 32 37 / 22, 64 x 64 rows
  // 50 / 36, 512 26 / 23 (64 workgroups of eight); heads of 64, 4000 rows 111 / 103, int8 126 / 117, 8 x 300 behind 3k 180 / 135, 2 x 512 behind 7.5k 123 / 131.
  // Least steps of four waves' splits, 8 / 4 / 2: 130 rows behind 600 34 / 24 / 22, 16 behind 600 26 / 21 / 15, 8 x 64 of 8 heads behind 2k 36 / 31 / 30.
  const PagedPlan narrow = form(4, 512, 2);
  if (c->head_dim == 64) return narrow;
  const PagedPlan wide = form(8, 256, 4);
  PagedPlan plan = per_seq >= 192 && span >= 2048 && wide.filled >= 192 ? wide : narrow;
  plan.most = std::max(wide.most, narrow.most);
  return plan;
}

template <int D, class T>
int launch_attn(PagedAttn a, const PagedPlan& plan, const ti_paged_cache* c, hipStream_t s) {
  const bool i8 = c->kv_type == TI_KV_I8;
  if (plan.waves) {
    if (const int rc = paged_block_run(a, c, plan.waves, plan.tiles, s)) return rc;
  } else if (plan.deal) {
    auto* fn = a.far ? i8 ? paged_deal_kernel<D, T, true, true> : paged_deal_kernel<D, T, false, true>
                     : i8 ? paged_deal_kernel<D, T, true, false> : paged_deal_kernel<D, T, false, false>;
    hipLaunchKernelGGL(fn, dim3(plan.deal, c->kv_heads * ((a.G + 15) / 16)),
                       dim3(64 * kStreamWaves), 0, s, a);
    TI_LAUNCH_CHECK("paged_deal_kernel");
  } else {
    auto* fn = a.far ? i8 ? paged_stream_kernel<D, T, true, true> : paged_stream_kernel<D, T, false, true>
                     : i8 ? paged_stream_kernel<D, T, true, false> : paged_stream_kernel<D, T, false, false>;
    hipLaunchKernelGGL(fn, dim3((unsigned)plan.tiles, c->kv_heads, plan.splits),
                       dim3(64 * kStreamWaves), 0, s, a);
    TI_LAUNCH_CHECK("paged_stream_kernel");
  }
  if (a.part_o) {
    constexpr int NH = 1024 / D;
    if (a.deal)
      hipLaunchKernelGGL((deal_join_kernel<D, T>), dim3(a.r.rows, a.heads), dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((split_join_kernel<D, T>), dim3(a.r.rows, (a.heads + NH - 1) / NH), dim3(256), 0, s, a);
    TI_LAUNCH_CHECK("join kernel");
  }
  return TI_OK;
}

// Parts of all rows and heads.
static size_t parts(const ti_paged_cache* c, const ti_paged_attn_args* p, const PagedPlan& plan) {
  return plan.deal ? (size_t)p->heads * (plan.deal + c->seqs) : plan.splits > 1 ? (size_t)p->rows * p->heads * plan.splits : 0;
}
static size_t part_bytes(const ti_paged_cache* c, size_t n) { return n * ((size_t)c->head_dim + 2) * sizeof(float); }

static int check_attn(const ti_paged_cache* c, const ti_paged_attn_args* p, const char* who) {
  if (const int rc = ti_paged_check(c, who)) return rc;
  if (!p) return ti_set_error(TI_ERR_ARG, "%s: null arguments", who);
  if (p->rows < 0 || p->rows > kPagedRows || p->heads < 1 || p->heads > 16384 || p->heads % c->kv_heads || p->max_len < 0 || p->window < 0)
    return ti_set_error(TI_ERR_ARG, "%s: bad sizes rows=%d heads=%d kv_heads=%d max_len=%d window=%d", who, p->rows, p->heads, c->kv_heads,
                        p->max_len, p->window);
  if (!p->row_start && p->rows != c->seqs) return ti_set_error(TI_ERR_ARG, "%s: %d rows of %d sequences without row_start", who, p->rows, c->seqs);
  if ((int64_t)p->rows * p->heads > INT32_MAX) return ti_set_error(TI_ERR_ARG, "%s: %d rows of %d heads in a call", who, p->rows, p->heads);
  if (!(p->softcap == 0.0f || (p->softcap >= 1e-20f && p->softcap <= 1e30f)) || !(fabsf(p->scale) <= 1e30f))
    return ti_set_error(TI_ERR_ARG, "%s: scale %g, softcap %g", who, (double)p->scale, (double)p->softcap);
  return TI_OK;
}

static bool far_cap(const ti_paged_attn_args* p) { return p->softcap > 0.0f && !paged_cap_near(p->softcap, p->scale); }

static int attend(const ti_paged_cache* c, const ti_paged_attn_args* p, ti_stream_t stream_, const char* who) {
  if (const int rc = check_attn(c, p, who)) return rc;
  const PagedPlan plan = paged_plan(c, p);
  if (plan.tiles > (1 << 23) || (int64_t)plan.tiles * plan.splits * c->kv_heads > INT32_MAX)
    return ti_set_error(TI_ERR_ARG, "%s: %d rows of %d sequences and %d heads in a call", who, p->rows, c->seqs, p->heads);
  const size_t n = parts(c, p, plan), need = part_bytes(c, n);
  if (need && (!p->workspace || p->workspace_bytes < (int64_t)need))
    return ti_set_error(TI_ERR_ARG, "%s: workspace of %ld bytes, %zu needed", who, (long)(p->workspace ? p->workspace_bytes : 0), need);
  if (!p->q || !p->out) return ti_set_error(TI_ERR_ARG, "%s: null pointer", who);
  const int64_t w = (int64_t)p->heads * c->head_dim;
  if (p->ldq < w || p->ldo < w || p->ldq % 8 || p->ldo % 8 || ((uintptr_t)p->q | (uintptr_t)p->out) % 16)
    return ti_set_error(TI_ERR_ARG, "%s: rows of pitch %d, %d for %ld values, or not 16-byte aligned", who, p->ldq, p->ldo, (long)w);
  if (((uintptr_t)p->row_start | (uintptr_t)p->slopes | (uintptr_t)p->first | (uintptr_t)p->prefix) % 4 || (uintptr_t)p->workspace % 16)
    return ti_set_error(TI_ERR_ARG, "%s: pointers are not aligned", who);
  if (p->rows == 0) return TI_OK;
  float* ws = (float*)p->workspace;
  const float cap = p->softcap;
  const bool far = far_cap(p), near = cap > 0.0f && !far;
  PagedAttn a = {ti_paged_form(c), {p->row_start, p->rows}, p->q, p->out, p->slopes, p->first, p->prefix, n ? ws : nullptr,
                 n ? ws + n * c->head_dim : nullptr, p->heads, p->heads / c->kv_heads, p->ldq, p->ldo, p->window, plan.splits, plan.deal,
                 c->kv_type == TI_KV_I8 ? kPagedUnit : 1.0f, near ? 2.0f * p->scale * kPagedLog2e / cap : p->scale * kPagedLog2e,
                 near ? 2.0f * cap * kPagedLog2e : cap * kPagedLog2e, 0.0f, far};
  if (far) a.fx = (float)std::clamp((double)p->scale / cap, -(double)kPagedMost, (double)kPagedMost);
  return TI_PAGED_FORM(c, launch_attn, a, plan, c, (hipStream_t)stream_);
}

}  // namespace ti

extern "C" size_t ti_paged_workspace_bytes(const ti_paged_cache* c, const ti_paged_attn_args* a) {
  if (ti::check_attn(c, a, "ti_paged_workspace_bytes")) return 0;
  ti_paged_attn_args any = *a;   // (of any length)
  any.max_len = any.window = 0;
  const ti::PagedPlan plan = ti::paged_plan(c, &any);
  return ti::part_bytes(c, (size_t)a->rows * a->heads * (plan.most > 1 ? plan.most : 0));
}

extern "C" int ti_paged_kernel_name(const ti_paged_cache* c, const ti_paged_attn_args* a, char* buf, int len) {
  if (!buf || len < 1) return ti_set_error(TI_ERR_ARG, "ti_paged_kernel_name: null buffer");
  if (const int rc = ti::check_attn(c, a, "ti_paged_kernel_name")) return rc;
  const ti::PagedPlan plan = ti::paged_plan(c, a);
  const char *kv = c->kv_type == TI_KV_I8 ? "int8" : "16 bits", *cap = ti::far_cap(a) ? "far cap" : a->softcap != 0.0f || a->slopes ? "shaped" : "plain";
  if (plan.waves)
    snprintf(buf, (size_t)len, "paged_block_kernel<%d,%d,%s,%s>, splits %d", c->head_dim, plan.waves, kv, cap, plan.splits);
  else if (plan.deal)
    snprintf(buf, (size_t)len, "paged_deal_kernel<%d,%s,%s>, runs %d", c->head_dim, kv, cap, plan.deal);
  else
    snprintf(buf, (size_t)len, "paged_stream_kernel<%d,%s,%s>, splits %d", c->head_dim, kv, cap, plan.splits);
  return TI_OK;
}

extern "C" int ti_paged_decode(const ti_paged_cache* c, const ti_paged_attn_args* a, ti_stream_t s) {
  if (a && a->row_start) return ti_set_error(TI_ERR_ARG, "ti_paged_decode: row_start (rows of several tokens: ti_paged_prefill)");
  return ti::attend(c, a, s, "ti_paged_decode");
}

extern "C" int ti_paged_prefill(const ti_paged_cache* c, const ti_paged_attn_args* a, ti_stream_t s) { return ti::attend(c, a, s, "ti_paged_prefill"); }
