// paged_prefill.hip -- attention of many rows over the paged cache (ti_paged_prefill).
//
// A workgroup holds 32 columns a wave -- (row, query head) pairs that share a kv-head -- and takes the keys 64 at a time; all its
// waves multiply the same keys and values from LDS, the next 64 on their way through registers (which is where int8 becomes fp16, and
// where blocks that are not there become zeros: every block is read through a buffer descriptor of the rows that it has).
//   S^T = K Q^T     32x32x16, two tiles of 32 keys: lane (c = l & 31, h = l >> 5) holds keys 8 (i / 4) + 4 h + i % 4 of column c
//   O^T += V^T P^T  32x32x16: the lane's own 8 weights (keys 4 h .., 8 + 4 h .. of 16) are its operand; values by transposed LDS reads
// LDS rows are rotated by their number, 16 bytes at a time (keys) or 32 (values), so that neither read meets a bank twice as often as
// it must.  Scores, reference and sums as in paged_attn.hip.
//
// Heads of 256 dims: two waves have the same 32 columns, each the scores of half of a step's keys and the sums of half of the dimensions, so that both fit
// the registers of two waves a SIMD; they hand each other their weights through LDS, with a reference each (a whole number: moving to the larger is
// exact).  4000 rows of 16 heads on 8: 308 -> 220 us against one wave with all of it, one a SIMD.
//
// Bound: a wave's products and its softmax follow one another, and the other wave of its SIMD fills little of it: no unit is full.  4000 rows of 32 heads on
// 8 of 128: 148 - 153 us (860 - 890 TFLOP/s; 16000 rows 990, a library product 1218), matrix units busy 41 % of the cycles, vector instructions 48 %, LDS 37 %;
// with a cap 184 - 189 us, 31 % and 61 %; int8 164; heads of 256 186.  Waves of a SIMD a part of a step behind each other, by four steps in LDS and barriers
// at two places: 159 us for 159, 214 with a cap for 200; a barrier every second step 163, 201.  Not tried: the next step's scores among this one's softmax in
// the same wave, which needs both steps' scores in registers.
#include <math.h>

#include <atomic>

#include "paged_attn.hpp"

namespace ti {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x16 pmma32(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 pmma32(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

constexpr int kBlockKeys = 64;
constexpr float kPagedLeast = 0x1p-149f;
template <int D, int NW>   // NW: waves
struct BlockForm {
  static constexpr bool PAIR = D == 256;   // two waves a column: each half of a step's keys, and of the dimensions
  static constexpr int NT = 64 * NW, COLS = (PAIR ? 16 : 32) * NW;
  static constexpr int CH = D / 8, NP = kBlockKeys * CH / NT, RP = NT / CH;   // 16-byte chunks a row; a thread's chunks; rows of a pass
  static constexpr int kTile = kBlockKeys * D * 2, kLds = 4 * kTile + (PAIR ? NW * 2048 : 0);   // bytes: K and V, two steps; weights
};
// Chunk c of LDS row r.
template <int D>
__device__ __forceinline__ int key_at(int r, int c) { return r * (2 * D) + ((c ^ (D == 64 ? (r >> 1) & 7 : r & 15)) << 4); }
template <int D>
__device__ __forceinline__ int value_at(int r, int c) { return r * (2 * D) + ((((c >> 1) ^ (D == 64 ? (r >> 1) & 3 : r & 7)) << 5) | (c & 1) << 4); }

template <int D, int NW, class T, bool I8, int SHAPE>   // SHAPE: scores with 1: a near cap or slopes; 2: any other cap, slopes
__global__ __launch_bounds__(64 * NW, D == 64 && !I8 && SHAPE < 2 ? 3 : 2) void paged_block_kernel(const PagedAttn a, const XcdDeal deal) {
  typedef BlockForm<D, NW> F;
  typedef typename PagedMat<T, I8>::M M;
  typedef typename PagedMat<T, I8>::V8 V8;
  constexpr bool PAIR = F::PAIR, SHAPED = SHAPE > 0, FAR = SHAPE == 2;
  constexpr int NK = D / 16, NV = D / (PAIR ? 64 : 32), KT = PAIR ? 1 : 2, ES = I8 ? 1 : 2;   // this wave's: tiles of dimensions, of keys
  typedef std::conditional_t<I8, u32x2, u32x4> Raw;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ int odd, reach[4][NW];
  __shared__ float pair[2][PAIR ? 2 : 1][PAIR ? NW / 2 : 1][32];   // references, denominators of the halves
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 31, h = lane >> 5;
  const int half = PAIR ? wave / (NW / 2) : 0, group = PAIR ? wave % (NW / 2) : wave;
  const XcdWork work = xcd_work(deal, a.q, a.out);
  if (work.head < 0) return;
  const int kvh = work.head, split = work.j % a.splits;
  const long at_tile = (deal.n - 1 - work.j) / a.splits;   // (the last tiles, with the most keys, first)
  const PagedSeq s = paged_find(a.c, a.r, at_tile, [&](int start, int j) { return paged_tile0((long)start * a.G, j, F::COLS); });
  const int b = s.b;
  const long tile = at_tile - paged_tile0((long)s.row0 * a.G, b, F::COLS);
  if (tile < 0 || tile * F::COLS >= (long)s.n * a.G) return;
  const int ci = (int)tile * F::COLS + group * 32 + c, row = ci / a.G, head = kvh * a.G + (ci - row * a.G), m = s.row0 + row, p = s.pos0 + row;
  const bool live = row < s.n && p >= 0 && p < a.c.s.blocks * kPagedBlock;
  PagedSpan span = {1, 0};
  if (live) span = paged_span(a, s, m, p);
  const bool some = span.lo <= span.hi;
  int lo_any = some ? span.lo : INT32_MAX, hi_any = some ? span.hi : -1, lo_all = live ? span.lo : 0, hi_all = live ? span.hi : INT32_MAX;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    lo_any = min(lo_any, __shfl_xor(lo_any, o, 64));
    hi_any = max(hi_any, __shfl_xor(hi_any, o, 64));
    lo_all = max(lo_all, __shfl_xor(lo_all, o, 64));
    hi_all = min(hi_all, __shfl_xor(hi_all, o, 64));
  }
  lo_any = __builtin_amdgcn_readfirstlane(lo_any);
  hi_any = __builtin_amdgcn_readfirstlane(hi_any);
  lo_all = __builtin_amdgcn_readfirstlane(lo_all);
  hi_all = __builtin_amdgcn_readfirstlane(hi_all);
  if (lane == 0) {
    reach[0][wave] = lo_any;
    reach[1][wave] = hi_any;
    reach[2][wave] = lo_all;
    reach[3][wave] = hi_all;
  }
  if (threadIdx.x == 0) odd = 0;

  V8 qf[NK];
  float f = a.f, fx = fabsf(a.fx);
  {
    const T* qr = (const T*)a.q + (size_t)m * a.ldq + (size_t)head * D;
    u16x8 raw[NK];
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      raw[k] = (u16x8){};
      if (live) raw[k] = *(const u16x8*)(qr + 16 * k + 8 * h);
    }
    const uint16_t flip = f < 0.0f ? 0x8000 : 0;   // (a negative scale is the queries')
    f = fabsf(f);
    if constexpr (std::is_same_v<M, T>) {
#pragma unroll
      for (int k = 0; k < NK; ++k) qf[k] = __builtin_bit_cast(V8, raw[k] ^ flip);
    } else {   // bf16 as fp16 (paged_attn.hip)
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, raw[k][e] & 0x7f80u);
      top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
      const int ex = (int)(top >> 7) - 127;
      const bool scaled = top != 0 && top != 0x7f80u;
      const float up = scaled ? ldexpf(1.0f, -ex) : 1.0f;
      if (scaled) {
        f = ldexpf(f, ex);
        fx = ldexpf(fx, ex);
      }
#pragma unroll
      for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) qf[k][e] = (M)(__builtin_bit_cast(float, (uint32_t)(raw[k][e] ^ flip) << 16) * up);
    }
  }
  const float slope = SHAPED && a.slopes && live ? a.slopes[head] * kPagedLog2e : 0.0f;
  lds_sync();
  int wg_lo = INT32_MAX, wg_hi = -1, wg_lo_all = 0, wg_hi_all = INT32_MAX;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    wg_lo = min(wg_lo, reach[0][w]);
    wg_hi = max(wg_hi, reach[1][w]);
    wg_lo_all = max(wg_lo_all, reach[2][w]);
    wg_hi_all = min(wg_hi_all, reach[3][w]);
  }
  wg_lo = __builtin_amdgcn_readfirstlane(wg_lo);
  wg_hi = __builtin_amdgcn_readfirstlane(wg_hi);
  wg_lo_all = __builtin_amdgcn_readfirstlane(wg_lo_all);
  wg_hi_all = __builtin_amdgcn_readfirstlane(wg_hi_all);
  // this split's steps: an equal part of the tile's
  const int first_step = wg_hi < 0 ? 0 : wg_lo / kBlockKeys, n_steps = wg_hi < 0 ? 0 : wg_hi / kBlockKeys + 1 - first_step;
  const int each = (n_steps + a.splits - 1) / a.splits, s0 = first_step + split * each, s1 = min(s0 + each, first_step + n_steps);

  f32x16 o[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[v][i] = 0.0f;
  float mr = -INFINITY, lr = 0.0f;

  // 64 blocks' numbers (and int8 scales) at a time, a lane each: 16 steps; the next 64 are fetched with them
  int id = -1, id_next = -1;
  float ks = 1.0f, vs = 1.0f, ks_next = 1.0f, vs_next = 1.0f;
  auto fetch = [&](int step, int& to, float& k, float& v) {
    const int blk = step * 4 + lane;
    to = -1;
    if (step + (lane >> 2) < s1 && blk < a.c.s.blocks) to = paged_block(a.c.s, a.c.table[(size_t)b * a.c.table_ld + paged_column(a.c.s, blk)], kvh, blk);
    if constexpr (I8) {
      k = v = 1.0f;
      if (to >= 0) {
        k = a.c.ks[to];
        v = a.c.vs[to];
        v = v < kPagedTiny ? kPagedTiny : v;   // (a user's 0)
      }
    }
  };
  // when a step's successor goes to LDS: behind its keys' products, or (long softmaxes, which it would stand in front of) at its end
  constexpr bool late = D == 256 || SHAPED;
  Raw rk[F::NP], rv[F::NP];
  const int t_row = threadIdx.x / F::CH, t_ch = threadIdx.x % F::CH;
  // This thread's chunks of a step's keys and values.  (Blocks and sizes are the wave's, and said so: without, each load stands in a loop over the values
  // that its descriptor may have; 4000 rows 165 -> 157 us, capped 203 -> 196.)
  auto load = [&](int step) {
    const bool next = step - s0 >= 16 && ((step - s0) & 15) < 2;   // (two steps ahead: its numbers are the next ones still)
#pragma unroll
    for (int i = 0; i < F::NP; ++i) {
      const int blk = __builtin_amdgcn_readfirstlane((i * F::RP + t_row) >> 4), l = ((step - s0) & 15) * 4 + blk;
      const int ib_now = __builtin_amdgcn_readlane(id, l), ib_next = __builtin_amdgcn_readlane(id_next, l), ib = __builtin_amdgcn_readfirstlane(next ? ib_next : ib_now);
      const int have = __builtin_amdgcn_readfirstlane(ib < 0 ? 0 : max(0, min(16, s.len - 16 * (4 * step + blk))) * D * ES);
      const size_t off = (size_t)max(ib, 0) * (16 * D * ES);
      const int in = (((i * F::RP + t_row) & 15) * D + t_ch * 8) * ES;
      const auto krs = __builtin_amdgcn_make_buffer_rsrc((char*)a.c.k + off, 0, have, 0x00020000);
      const auto vrs = __builtin_amdgcn_make_buffer_rsrc((char*)a.c.v + off, 0, have, 0x00020000);
      if constexpr (I8) {
        rk[i] = __builtin_bit_cast(Raw, __builtin_amdgcn_raw_buffer_load_b64(krs, in, 0, 0));
        rv[i] = __builtin_bit_cast(Raw, __builtin_amdgcn_raw_buffer_load_b64(vrs, in, 0, 0));
      } else {
        rk[i] = __builtin_bit_cast(Raw, __builtin_amdgcn_raw_buffer_load_b128(krs, in, 0, 0));
        rv[i] = __builtin_bit_cast(Raw, __builtin_amdgcn_raw_buffer_load_b128(vrs, in, 0, 0));
      }
    }
  };
  auto wide = [](Raw x) {
    if constexpr (I8)
      return (u32x4){i8_of<false>(x[0]), i8_of<true>(x[0]), i8_of<false>(x[1]), i8_of<true>(x[1])};
    else
      return x;
  };
  auto part_seen = [&](int step) { return step * kBlockKeys < wg_lo_all || step * kBlockKeys + kBlockKeys - 1 > wg_hi_all; };
  auto store = [&](int step) {
    char* to = lds + ((step - s0) & 1) * 2 * F::kTile;
    if constexpr (!I8)
      if (part_seen(step)) {   // infinities and NaN that not every column sees (0 times them is NaN): 0 here, added at the end
        uint32_t bad = 0;
#pragma unroll
        for (int i = 0; i < F::NP; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            bad |= PagedOdd<M>::any(rv[i][j]);
            rv[i][j] = PagedOdd<M>::finite(rv[i][j]);
          }
        if (bad) odd = 1;
      }
#pragma unroll
    for (int i = 0; i < F::NP; ++i) {
      const int r = i * F::RP + t_row;
      *(u32x4*)(to + key_at<D>(r, t_ch)) = wide(rk[i]);
      *(u32x4*)(to + F::kTile + value_at<D>(r, t_ch)) = wide(rv[i]);
    }
  };
  if (s0 < s1) {
    fetch(s0, id, ks, vs);
    fetch(s0 + 16, id_next, ks_next, vs_next);
    load(s0);
    store(s0);
    load(s0 + 1);
  }
  for (int step = s0; step < s1; ++step) {
    if (step > s0 && ((step - s0) & 15) == 0) {
      id = id_next;
      ks = ks_next;
      vs = vs_next;
      fetch(step + 16, id_next, ks_next, vs_next);
    }
    lds_sync();   // this step's rows are there, and everyone has done with the other half
    const int key0 = step * kBlockKeys;
    const bool act = key0 <= hi_any && key0 + kBlockKeys - 1 >= lo_any;
    const char* st = lds + ((step - s0) & 1) * 2 * F::kTile;
    f32x16 sc[KT];
    if (act) {
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[t][i] = 0.0f;
#pragma unroll
      for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int t = 0; t < KT; ++t) sc[t] = pmma32(__builtin_bit_cast(V8, *(const u32x4*)(st + key_at<D>(32 * (t + half) + c, 2 * k + h))), qf[k], sc[t]);
      if constexpr (!PAIR) {   // four keys' fragments on their way in front of the products (one: 4000 capped rows 203 -> 197 us)
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
        for (int i = 0; i < NK * KT - 4; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x8, 4, 0);
      }
    }
    if (!late || !act) {
      store(step + 1);
      load(step + 2);
    }
    if (!act) {
      if constexpr (PAIR) lds_sync();
      continue;
    }
    int ids[2 * KT], no_block = 0;
    float fk[2 * KT], vl[2 * KT], vi[2 * KT];
    const int l0 = ((step - s0) & 15) * 4 + 2 * half, mine = key0 + 32 * half;   // this wave's first block and key
#pragma unroll
    for (int t = 0; t < 2 * KT; ++t) {
      ids[t] = __builtin_amdgcn_readlane(id, l0 + t);
      no_block |= ids[t];
      fk[t] = f;
      vl[t] = 0.0f;
      vi[t] = 1.0f;
      if constexpr (I8) {
        fk[t] *= __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ks), l0 + t));
        const float sv = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, vs), l0 + t));
        vl[t] = __builtin_amdgcn_logf(sv);
        vi[t] = __builtin_amdgcn_rcpf(sv) * kPagedUnit;
      }
    }
    const bool ragged = mine < lo_all || mine + 32 * KT - 1 > hi_all || no_block < 0;
    uint32_t see[KT];
#pragma unroll
    for (int t = 0; t < KT; ++t) see[t] = 0xffff;
    if (ragged) {
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        see[t] = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int j = mine + 32 * t + 8 * (i >> 2) + 4 * h + (i & 3);
          if (j >= span.lo && j <= span.hi && ids[2 * t + (i >> 3)] >= 0) see[t] |= 1u << i;
        }
      }
    }
    // exponents of 2: mul[block] s + add[block]
    float mul[2 * KT], add[2 * KT], mx = -INFINITY;
    if constexpr (FAR) {
      float fxk[2 * KT];
#pragma unroll
      for (int t = 0; t < 2 * KT; ++t) fxk[t] = I8 ? fx * __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ks), l0 + t)) : fx;
      paged_cap<8>(a.cap, sc, fk, fxk);
#pragma unroll
      for (int t = 0; t < 2 * KT; ++t) fk[t] = 1.0f;
    } else if (SHAPED && a.cap != 0.0f) {
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[t][i] = paged_capped(sc[t][i], fk[2 * t + (i >> 3)]);
#pragma unroll
      for (int t = 0; t < 2 * KT; ++t) fk[t] = a.cap;
    }
    if (SHAPED && a.slopes) {
      const float base = slope * (float)(mine + 4 * h - p);
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float more = fmaf(slope, (float)(32 * t + 8 * (i >> 2) + (i & 3)), base);
          if constexpr (I8) more += vl[2 * t + (i >> 3)];
          sc[t][i] = fmaf(sc[t][i], fk[2 * t + (i >> 3)], more);
        }
#pragma unroll
      for (int t = 0; t < 2 * KT; ++t) {
        mul[t] = 1.0f;
        add[t] = 0.0f;
      }
    } else {
#pragma unroll
      for (int t = 0; t < 2 * KT; ++t) {   // (what is masked stays -inf: a factor > 0, the least there is, which makes nothing of any score; none of a block that is not seen)
        const bool none = I8 && ragged && !(see[t >> 1] >> 8 * (t & 1) & 255);
        mul[t] = none ? 1.0f : fk[t] < kPagedLeast ? kPagedLeast : fk[t];
        add[t] = none ? 0.0f : vl[t];
      }
    }
    if (ragged) {
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (!(see[t] >> i & 1)) sc[t][i] = -INFINITY;
    }
#pragma unroll
    for (int t = 0; t < 2 * KT; ++t) {
      float x = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) x = fmaxf(x, sc[t >> 1][8 * (t & 1) + e]);
      mx = fmaxf(mx, I8 ? fmaf(x, mul[t], add[t]) : x);
    }
    mx = xor32_max(mx);
    if constexpr (!I8) mx *= mul[0];
    auto rescale = [&](float mn) {
      const float alpha = mn == mr ? 1.0f : __builtin_amdgcn_exp2f(mr - mn);
      mr = mn;
      lr *= alpha;
#pragma unroll
      for (int v = 0; v < NV; ++v) o[v] *= alpha;
    };
    // what this step's weights are relative to (PAIR: whole, the halves' weights move to a common one exactly)
    typedef PagedRef<M> Ref;
    float ref = mr, l_step = 0.0f;
    if constexpr (PAIR) {
      if (mx > mr + Ref::kUp) ref = floorf(mx) + Ref::kSet;
    } else {
      if (__builtin_amdgcn_ballot_w64(mx > mr + Ref::kUp) != 0) rescale(mx > mr + Ref::kUp ? mx + Ref::kSet : mr);
      ref = mr;
    }
    const float off = ref == -INFINITY ? 0.0f : ref;
    V8 pf[KT][2];   // weights of 16 keys each
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float l = 0.0f;
        const float m1 = mul[2 * t + u], a1 = add[2 * t + u] - off;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float w0 = __builtin_amdgcn_exp2f(fmaf(sc[t][8 * u + e], m1, a1)), w1 = __builtin_amdgcn_exp2f(fmaf(sc[t][8 * u + e + 1], m1, a1));
          l += w0 + w1;
          typedef M M2 __attribute__((ext_vector_type(2)));
          const M2 w = __builtin_convertvector((f32x2){w0, w1}, M2);
          pf[t][u][e] = w[0];
          pf[t][u][e + 1] = w[1];
        }
        const bool none = ragged && !(see[t] >> 8 * u & 255);   // (nothing of a block, whose scale may be NaN)
        float& sum = PAIR ? l_step : lr;
        sum = I8 ? fmaf(l, none ? 0.0f : vi[2 * t + u], sum) : sum + l;
      }
    // 8 keys of dims 32 v + c: keys 4 h .. and 8 + 4 h .. of the 16 that u says
    const int tr = ((lane & 15) >> 2) + 4 * h, tc = ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
    auto frag = [&](int u, int v) {
      u32x2 x[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = 16 * u + 8 * i + tr, byte = 64 * (v + half * NV) + tc;
        const char* src = st + F::kTile + value_at<D>(r, byte >> 4) + (byte & 15);
        x[i] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)src));
      }
      return (u32x4){x[0][0], x[0][1], x[1][0], x[1][1]};
    };
    if constexpr (PAIR) {
      // each half's weights and reference to the other
      u32x4* const mail = (u32x4*)(lds + 4 * F::kTile) + group * 4 * 64 + lane;
#pragma unroll
      for (int u = 0; u < 2; ++u) mail[(2 * half + u) * 64] = __builtin_bit_cast(u32x4, pf[0][u]);
      pair[0][half][group][c] = ref;
      lds_sync();
      V8 other[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) other[u] = __builtin_bit_cast(V8, mail[(2 - 2 * half + u) * 64]);
      const float ref_o = pair[0][1 - half][group][c], both = fmaxf(ref, ref_o);
      if (__builtin_amdgcn_ballot_w64(both != mr || ref != ref_o) != 0) {
        const float f0 = ref == both ? 1.0f : __builtin_amdgcn_exp2f(ref - both), f1 = ref_o == both ? 1.0f : __builtin_amdgcn_exp2f(ref_o - both);
        rescale(both);
        l_step *= f0;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            pf[0][u][e] = (M)((float)pf[0][u][e] * f0);
            other[u][e] = (M)((float)other[u][e] * f1);
          }
      }
      lr += l_step;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          o[v] = pmma32(__builtin_bit_cast(V8, frag(2 * half + u, v)), pf[0][u], o[v]);
          o[v] = pmma32(__builtin_bit_cast(V8, frag(2 - 2 * half + u, v)), other[u], o[v]);
        }
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int v = 0; v < NV; ++v) o[v] = pmma32(__builtin_bit_cast(V8, frag(u, v)), pf[(u >> 1) % KT][u & 1], o[v]);
    }
    if (late) {
      store(step + 1);
      load(step + 2);
    }
  }
  if constexpr (!I8) {
    lds_sync();
    if (odd) {
      for (int key = s0 * kBlockKeys; key < min(s1 * kBlockKeys, s.len); ++key) {
        if (!part_seen(key / kBlockKeys)) continue;
        const int blk = key / kPagedBlock, at = paged_block(a.c.s, a.c.table[(size_t)b * a.c.table_ld + paged_column(a.c.s, blk)], kvh, blk);
        if (at < 0 || key < span.lo || key > span.hi) continue;
        const M* x = (const M*)a.c.v + ((size_t)at * kPagedBlock + key % kPagedBlock) * D + 32 * NV * half + 4 * h;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float y = (float)x[32 * v + 8 * (i >> 2) + (i & 3)];
            if (!(fabsf(y) <= 3.4e38f)) o[v][i] += y;
          }
      }
    }
  }
  lr += lane_xor<32>(lr);
  if constexpr (PAIR) {
    pair[1][half][group][c] = lr;
    lds_sync();
    lr += pair[1][1 - half][group][c];
  }
  if (!live) return;
  const size_t rh = (size_t)m * a.heads + head;
  if (a.splits > 1) {
    const size_t at = rh * a.splits + split;
    if (h == 0 && half == 0) *(float2*)(a.part_ml + 2 * at) = make_float2(mr, lr);
    float* po = a.part_o + at * D + 32 * NV * half + 4 * h;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < 16; i += 4) *(f32x4*)(po + 32 * v + 2 * i) = (f32x4){o[v][i], o[v][i + 1], o[v][i + 2], o[v][i + 3]};
    return;
  }
  const float inv = a.unit / lr;
  T* out = (T*)a.out + (size_t)m * a.ldo + (size_t)head * D + 32 * NV * half + 4 * h;
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      typedef T Q4 __attribute__((ext_vector_type(4)));
      Q4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = (T)(lr == 0.0f ? 0.0f : o[v][i + e] * inv);
      *(Q4*)(out + 32 * v + 2 * i) = y;
    }
}

template <int D, int NW, class T>
static int launch_waves(const PagedAttn& a, long tiles, bool i8, hipStream_t s) {
  const int shape = a.far ? 2 : a.cap != 0.0f || a.slopes ? 1 : 0;
  static constexpr decltype(&paged_block_kernel<D, NW, T, true, 2>) kernels[2][3] = {
      {paged_block_kernel<D, NW, T, false, 0>, paged_block_kernel<D, NW, T, false, 1>, paged_block_kernel<D, NW, T, false, 2>},
      {paged_block_kernel<D, NW, T, true, 0>, paged_block_kernel<D, NW, T, true, 1>, paged_block_kernel<D, NW, T, true, 2>}};
  auto* fn = kernels[i8][shape];
  // (more than 64 KiB of LDS: said once per device)
  static std::atomic<uint64_t> said[6];
  const int which = 3 * i8 + shape;
  int dev = 0;
  TI_HIP_CHECK(hipGetDevice(&dev), "hipGetDevice");
  if (!(said[which].load(std::memory_order_relaxed) >> (dev & 63) & 1)) {
    TI_HIP_CHECK(hipFuncSetAttribute((const void*)fn, hipFuncAttributeMaxDynamicSharedMemorySize, BlockForm<D, NW>::kLds), "hipFuncSetAttribute");
    said[which].fetch_or(1ull << (dev & 63), std::memory_order_relaxed);
  }
  const XcdDeal deal = xcd_deal(a.c.s.kv_heads, (int)(tiles * a.splits));
  hipLaunchKernelGGL(fn, xcd_grid(deal), dim3(64 * NW), (BlockForm<D, NW>::kLds), s, a, deal);
  TI_LAUNCH_CHECK("paged_block_kernel");
  return TI_OK;
}
template <int D, class T>
static int launch(const PagedAttn& a, int waves, long tiles, bool i8, hipStream_t s) {
  if constexpr (D == 64) {
    return launch_waves<D, 4, T>(a, tiles, i8, s);
  } else {
    if constexpr (D == 128)
      if (waves == 4) return launch_waves<D, 4, T>(a, tiles, i8, s);
    return launch_waves<D, 8, T>(a, tiles, i8, s);
  }
}

int paged_block_run(const PagedAttn& a, const ti_paged_cache* c, int waves, long tiles, hipStream_t s) {
  return TI_PAGED_FORM(c, launch, a, waves, tiles, c->kv_type == TI_KV_I8, s);
}

}  // namespace ti
