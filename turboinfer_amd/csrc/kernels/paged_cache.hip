// paged_cache.hip -- writing rows into the paged key/value cache with the position rotation on the way, and reading them back
// (ti_paged_append, ti_paged_read).
//
// A thread holds 8 dimensions of a head.  Rotated pairs are inside them (TI_ROPE_PAIRS) or 8 dimensions half the rotated part
// away (TI_ROPE_HALVES), loaded again from the same cache lines, so that no thread needs another's values.  fp32 from the load to
// the one rounding.
//
// int8: one workgroup per (block of 16 tokens, kv-head, k or v) holds the whole block in registers, finds the largest new value,
// and writes new and moved old tokens once.
//
// Bound: of many rows HBM (16-bit caches, 8000 rows of 32 heads on 8 of 128: 43 us, 4.7 TB/s; read back 32000 tokens 43.6 us, 4.8 TB/s: a large copy's
// 4.9), int8 blocks by their chain of lookup, rows, maximum (52 us for the same rows, 3.5 TB/s; several heads a workgroup with the next one's rows
// ahead: 4 more); of a step its launch (32 streams 3.0 us).
#include <math.h>

#include "paged_device.hpp"

namespace ti {

struct AppendArgs {
  PagedCache c;
  PagedRows r;
  const void* x;
  void* q;
  const float* rope;
  int heads, ldx, ldq, rope_len, rot_dim, halves;
  int row_parts, chunks;   // workgroups of a row, 8-dimension chunks that it has (the other workgroups take int8 blocks, 2 a kv-head)
};

template <class X>
__device__ __forceinline__ void load8(const X* x, float* v) {
  if constexpr (sizeof(X) == 4) {
    const f32x4 a = *(const f32x4*)x, b = *(const f32x4*)(x + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = a[e];
      v[4 + e] = b[e];
    }
  } else {
    typedef X V __attribute__((ext_vector_type(8)));
    const V a = *(const V*)x;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)a[e];
  }
}

// Dimensions d .. d + 7 of a head at x and those that they are rotated with (rot_dim 0: not rotated), and their rotation by cs (this
// position's [rot_dim / 2] pairs).
struct Dims8 {
  float v[8], o[8];
};
template <class X>
__device__ __forceinline__ Dims8 dims8(const X* x, int d, int rot_dim, int halves) {
  Dims8 r;
  load8(x + d, r.v);
  if (halves && d < rot_dim) load8(x + (d < rot_dim >> 1 ? d + (rot_dim >> 1) : d - (rot_dim >> 1)), r.o);
  return r;
}
__device__ __forceinline__ void rotate8(Dims8& r, int d, const float* cs, int rot_dim, int halves) {
  if (d >= rot_dim) return;
  if (!halves) {
    float t[8];
    load8(cs + d, t);
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float a = r.v[e], b = r.v[e + 1];
      r.v[e] = a * t[e] - b * t[e + 1];
      r.v[e + 1] = a * t[e + 1] + b * t[e];
    }
    return;
  }
  const int half = rot_dim >> 1, i = d < half ? d : d - half;
  float t[16];
  load8(cs + 2 * i, t);
  load8(cs + 2 * i + 8, t + 8);
  const float sign = d < half ? -1.0f : 1.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) r.v[e] = r.v[e] * t[2 * e] + sign * (r.o[e] * t[2 * e + 1]);
}

// One int8 block of a kv-head: D * 2 threads, 8 dimensions of a token each.
template <int D, class X>
__device__ void append_block(const AppendArgs& a, int slot, int part, float* red) {
  constexpr int CH = D / 8;
  const int tid = threadIdx.x, kvh = part >> 1, is_v = part & 1;
  const PagedSeq s = paged_find(a.c, a.r, slot, [](int start, int j) { return paged_touch0(start, j); });
  const int b = s.b;
  const long at = a.r.start ? slot - paged_touch0(s.row0, b) : 0;
  const int pos_first = max(s.pos0, 0);
  const long blk = pos_first / kPagedBlock + at;
  if (s.n == 0 || at < 0 || blk * kPagedBlock >= (long)s.pos0 + s.n || blk >= a.c.s.blocks) return;
  if (a.rope && max(s.pos0, (int)blk * kPagedBlock) >= a.rope_len) return;   // (no fresh row: neither tokens nor scale change)
  const int id = paged_block(a.c.s, a.c.table[(size_t)b * a.c.table_ld + paged_column(a.c.s, (int)blk)], kvh, (int)blk);
  if (id < 0) return;
  const int tok = tid / CH, d = tid % CH * 8, pos = (int)blk * kPagedBlock + tok;
  const bool fresh = pos >= s.pos0 && pos < s.pos0 + s.n && (!a.rope || pos < a.rope_len), old = pos < s.pos0;
  // (a block with older tokens: its first token is one; a fresh row without a rotation leaves its place as it is)
  const bool has_old = (int)blk * kPagedBlock < s.pos0;
  float* scale = (is_v ? a.c.vs : a.c.ks) + id;
  int8_t* cell = (int8_t*)(is_v ? a.c.v : a.c.k) + (size_t)id * (kPagedBlock * D) + tok * D + d;
  const float s_old = has_old ? *scale : 0.0f;
  uint2 q = {0, 0};
  if (old) q = *(const uint2*)cell;
  Dims8 y = {};
  if (fresh) {
    const int rot = is_v ? 0 : a.rot_dim;
    y = dims8((const X*)a.x + (size_t)(s.row0 + (pos - s.pos0)) * a.ldx + (size_t)(a.heads + kvh + (is_v ? a.c.s.kv_heads : 0)) * D, d, rot, a.halves);
    rotate8(y, d, a.rope + (size_t)pos * a.rot_dim, rot, a.halves);
  }
  const float* v = y.v;
  // the largest magnitude by its bits: infinities and NaN are above every number
  uint32_t most = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) most = max(most, __builtin_bit_cast(uint32_t, v[e]) & 0x7fffffffu);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o, 64));
  if ((tid & 63) == 0) red[tid >> 6] = __builtin_bit_cast(float, most);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < D / 32; ++w) most = max(most, __builtin_bit_cast(uint32_t, red[w]));
  float sc = most >= 0x7f800000u ? __builtin_nanf("") : fmaxf(__builtin_bit_cast(float, most) / 127.0f, kPagedTiny);
  if (has_old && !(s_old <= sc)) sc = sc != sc ? sc : s_old;   // (NaN stays)
  if (tid == 0) *scale = sc;
  if (old) {
    if (!(s_old < sc)) return;
    const float f = s_old / sc;
    uint32_t w[2] = {q.x, q.y};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t n = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) n |= ((uint32_t)(int)rintf((float)(int8_t)(w[h] >> 8 * e) * f) & 255u) << 8 * e;
      w[h] = n;
    }
    *(uint2*)cell = make_uint2(w[0], w[1]);
  } else if (fresh) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t n = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) n |= ((uint32_t)(int)fminf(fmaxf(rintf(v[4 * h + e] / sc), -127.0f), 127.0f) & 255u) << 8 * e;
      w[h] = n;
    }
    *(uint2*)cell = make_uint2(w[0], w[1]);
  }
}

// Rows: q, and k and v of 16-bit caches.  D * 2 threads; a row's workgroups, then the int8 blocks'.
template <int D, class T, class X, bool I8>
__global__ __launch_bounds__(2 * D) void paged_append_kernel(const AppendArgs a) {
  constexpr int CH = D / 8;
  __shared__ float red[D / 32];
  const int row_groups = a.r.rows * a.row_parts;
  if (I8 && (int)blockIdx.x >= row_groups) {
    const int i = blockIdx.x - row_groups, n = 2 * a.c.s.kv_heads;
    append_block<D, X>(a, i / n, i % n, red);
    return;
  }
  const int m = blockIdx.x / a.row_parts, stride = a.row_parts * 2 * D;
  int at = (blockIdx.x - m * a.row_parts) * 2 * D + threadIdx.x;
  const X* x = (const X*)a.x + (size_t)m * a.ldx;
  // (the first values are asked for before it is known where they go)
  auto fetch = [&] { return dims8(x + at / CH * D, at % CH * 8, at / CH < a.heads + a.c.s.kv_heads ? a.rot_dim : 0, a.halves); };
  Dims8 y = {};
  if (at < a.chunks) y = fetch();
  const PagedSeq s = paged_find(a.c, a.r, m, [](int start, int) { return (long)start; });
  const int b = s.b;
  const int pos = s.pos0 + (m - s.row0);
  if (m < s.row0 || m >= s.row0 + s.n || pos < 0 || pos >= a.c.s.blocks * kPagedBlock || (a.rope && pos >= a.rope_len)) return;
  const int blk = pos / kPagedBlock, entry = I8 ? 0 : a.c.table[(size_t)b * a.c.table_ld + paged_column(a.c.s, blk)];
  for (; at < a.chunks; at += stride) {
    const int head = at / CH, d = at % CH * 8;
    const bool is_v = head >= a.heads + a.c.s.kv_heads;
    if (at >= stride) y = fetch();
    rotate8(y, d, a.rope + (size_t)pos * a.rot_dim, is_v ? 0 : a.rot_dim, a.halves);
    if (I8 || head < a.heads) {
      *(u16x8*)((T*)a.q + (size_t)m * a.ldq + head * D + d) = pack8<T>(y.v);
    } else {
      const int kvh = head - a.heads - (is_v ? a.c.s.kv_heads : 0), id = paged_block(a.c.s, entry, kvh, blk);
      if (id >= 0) *(u16x8*)((T*)(is_v ? a.c.v : a.c.k) + (size_t)id * (kPagedBlock * D) + (pos % kPagedBlock) * D + d) = pack8<T>(y.v);
    }
  }
}

struct ReadArgs {
  PagedCache c;
  PagedRows r;
  void* k;
  void* v;
  int ldk, ldv;
};

// Grid (rows, parts of [k | v] x kv-heads x D / 8); 256 threads.
template <int D, class T, bool I8>
__global__ __launch_bounds__(256) void paged_read_kernel(const ReadArgs a) {
  constexpr int CH = D / 8;
  const int m = blockIdx.x, at = blockIdx.y * 256 + threadIdx.x, d = at % CH * 8, hh = at / CH, is_v = hh >= a.c.s.kv_heads;
  const int kvh = hh - (is_v ? a.c.s.kv_heads : 0);
  const PagedSeq s = paged_find(a.c, a.r, m, [](int start, int) { return (long)start; });   // (all lanes)
  if (kvh >= a.c.s.kv_heads) return;
  const int b = s.b;
  const int pos = s.pos0 + (m - s.row0);
  if (m < s.row0 || m >= s.row0 + s.n || pos < 0 || pos >= a.c.s.blocks * kPagedBlock) return;
  const int blk = pos / kPagedBlock;
  const int id = paged_block(a.c.s, a.c.table[(size_t)b * a.c.table_ld + paged_column(a.c.s, blk)], kvh, blk);
  u16x8 o = {};
  if (id >= 0) {
    const size_t off = (size_t)id * (kPagedBlock * D) + (pos % kPagedBlock) * D + d;
    const void* cache = is_v ? a.c.v : a.c.k;
    if constexpr (I8) {
      const uint2 q = *(const uint2*)((const int8_t*)cache + off);
      const float sc = (is_v ? a.c.vs : a.c.ks)[id];
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (float)(int8_t)((e < 4 ? q.x : q.y) >> 8 * (e & 3)) * sc;
      o = pack8<T>(v);
    } else {
      o = *(const u16x8*)((const T*)cache + off);
    }
  }
  *(u16x8*)((T*)(is_v ? a.v : a.k) + (size_t)m * (is_v ? a.ldv : a.ldk) + kvh * D + d) = o;
}

template <int D, class T>
int append(AppendArgs a, const ti_paged_cache* c, int x_f32, hipStream_t s) {
  const bool i8 = c->kv_type == TI_KV_I8;
  a.chunks = (a.heads + (i8 ? 0 : 2 * c->kv_heads)) * (D / 8);
  // few rows: a chunk a thread; many: a row a workgroup, which looks its place up once.  us, 32 heads on 8 of 128: 32 rows 6.7 / 7.2, 512 6.4 /
  // 7.0, 2048 12.3 / 11.0, 8000 50.6 / 42.8 (4.7 TB/s, as a large copy)
  a.row_parts = (a.chunks + 2 * D - 1) / (2 * D);
  if (a.r.rows >= 1024 && a.row_parts > 1) a.row_parts = 1;
  const long slots = !i8 ? 0 : a.r.start ? paged_touches(a.r.rows, c->seqs) : a.r.rows;
  const long grid = (long)a.r.rows * a.row_parts + slots * 2 * c->kv_heads;
  if (grid > UINT32_MAX / (2 * D)) return ti_set_error(TI_ERR_ARG, "ti_paged_append: %d rows of %d heads in a call", a.r.rows, a.heads + 2 * c->kv_heads);
  auto* fn = i8 ? (x_f32 ? paged_append_kernel<D, T, float, true> : paged_append_kernel<D, T, T, true>)
                : (x_f32 ? paged_append_kernel<D, T, float, false> : paged_append_kernel<D, T, T, false>);
  hipLaunchKernelGGL(fn, dim3((unsigned)grid), dim3(2 * D), 0, s, a);
  TI_LAUNCH_CHECK("paged_append_kernel");
  return TI_OK;
}

template <int D, class T>
int read(const ReadArgs& a, const ti_paged_cache* c, hipStream_t s) {
  const dim3 grid(a.r.rows, (2 * c->kv_heads * (D / 8) + 255) / 256);
  if (c->kv_type == TI_KV_I8)
    hipLaunchKernelGGL((paged_read_kernel<D, T, true>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((paged_read_kernel<D, T, false>), grid, dim3(256), 0, s, a);
  TI_LAUNCH_CHECK("paged_read_kernel");
  return TI_OK;
}

static bool aligned(const void* p, int n) { return ((uintptr_t)p & (uintptr_t)(n - 1)) == 0; }

}  // namespace ti

int ti_paged_check(const ti_paged_cache* c, const char* who) {
  if (!c) return ti_set_error(TI_ERR_ARG, "%s: null cache", who);
  if (!c->k || !c->v || !c->table || !c->len) return ti_set_error(TI_ERR_ARG, "%s: null pointer in the cache", who);
  if (c->dtype != TI_PAGED_F16 && c->dtype != TI_PAGED_BF16) return ti_set_error(TI_ERR_ARG, "%s: dtype %d", who, c->dtype);
  if (c->kv_type != TI_KV_SAME && c->kv_type != TI_KV_I8) return ti_set_error(TI_ERR_ARG, "%s: kv_type %d", who, c->kv_type);
  if (c->kv_type == TI_KV_I8 && (!c->k_scale || !c->v_scale)) return ti_set_error(TI_ERR_ARG, "%s: int8 without scales", who);
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return ti_set_error(TI_ERR_UNSUPPORTED, "%s: head_dim %d not in {64, 128, 256}", who, c->head_dim);
  if (c->page < 16 || c->page > 256 || (c->page & (c->page - 1)))
    return ti_set_error(TI_ERR_UNSUPPORTED, "%s: pages of %d tokens, not 16, 32, 64, 128 or 256", who, c->page);
  if (c->seqs < 1 || c->seqs > (1 << 20) || c->kv_heads < 1 || c->kv_heads > 16384 || c->pages < 1 || c->table_ld < 1 ||
      (int64_t)c->pages * (c->page / 16) * c->kv_heads > INT32_MAX || (int64_t)c->table_ld * c->page > INT32_MAX)
    return ti_set_error(TI_ERR_ARG, "%s: bad sizes seqs=%d kv_heads=%d pages=%d page=%d table_ld=%d", who, c->seqs, c->kv_heads, c->pages,
                        c->page, c->table_ld);
  if (!ti::aligned(c->k, 16) || !ti::aligned(c->v, 16) || !ti::aligned(c->table, 4) || !ti::aligned(c->len, 4) || !ti::aligned(c->k_scale, 4) ||
      !ti::aligned(c->v_scale, 4))
    return ti_set_error(TI_ERR_ARG, "%s: pointers of the cache are not aligned", who);
  return TI_OK;
}

ti::PagedCache ti_paged_form(const ti_paged_cache* c) {
  const int lb = __builtin_ctz((unsigned)c->page) - 4;
  return {c->k, c->v, c->k_scale, c->v_scale, c->table, c->len, c->table_ld, c->seqs, {c->pages, c->kv_heads, lb, (int)((int64_t)c->table_ld << lb)}};
}

// Rows of a call: TI_OK, or the error set.
static int check_rows(const ti_paged_cache* c, const int32_t* start, int rows, const char* who) {
  if (rows < 0 || rows > ti::kPagedRows) return ti_set_error(TI_ERR_ARG, "%s: rows=%d", who, rows);
  if (!start && rows != c->seqs) return ti_set_error(TI_ERR_ARG, "%s: %d rows of %d sequences without row_start", who, rows, c->seqs);
  if (!ti::aligned(start, 4)) return ti_set_error(TI_ERR_ARG, "%s: row_start is not aligned", who);
  return TI_OK;
}

extern "C" int ti_paged_struct_bytes(int which) {
  return which == 0 ? (int)sizeof(ti_paged_cache) : which == 1 ? (int)sizeof(ti_paged_append_args) : which == 2 ? (int)sizeof(ti_paged_attn_args) : 0;
}

extern "C" int ti_paged_append(const ti_paged_cache* c, const ti_paged_append_args* p, ti_stream_t stream) {
  if (const int rc = ti_paged_check(c, "ti_paged_append")) return rc;
  if (!p || !p->x || (p->heads > 0 && !p->q)) return ti_set_error(TI_ERR_ARG, "ti_paged_append: null pointer");
  if (const int rc = check_rows(c, p->row_start, p->rows, "ti_paged_append")) return rc;
  const int D = c->head_dim;
  if (p->heads < 0 || p->heads > 16384 || p->ldx < (int64_t)(p->heads + 2 * c->kv_heads) * D || p->ldq < (int64_t)p->heads * D)
    return ti_set_error(TI_ERR_ARG, "ti_paged_append: bad sizes heads=%d ldx=%d ldq=%d", p->heads, p->ldx, p->ldq);
  if (!ti::aligned(p->x, 16) || !ti::aligned(p->q, 16) || p->ldx % (p->x_f32 ? 4 : 8) || (p->heads && p->ldq % 8) || !ti::aligned(p->rope_cs, 16))
    return ti_set_error(TI_ERR_ARG, "ti_paged_append: rows are not 16-byte aligned");
  if (p->rope_cs && (p->rot_dim < 16 || p->rot_dim > D || p->rot_dim % 16 || p->rope_len < 1 || (p->rope_kind != TI_ROPE_PAIRS && p->rope_kind != TI_ROPE_HALVES)))
    return ti_set_error(TI_ERR_ARG, "ti_paged_append: rotation of %d dimensions, %d positions, kind %d", p->rot_dim, p->rope_len, p->rope_kind);
  if (p->rows == 0) return TI_OK;
  const ti::AppendArgs a = {ti_paged_form(c), {p->row_start, p->rows}, p->x, p->q, p->rope_cs, p->heads, p->ldx, p->ldq, p->rope_len,
                            p->rope_cs ? p->rot_dim : 0, p->rope_kind == TI_ROPE_HALVES, 0, 0};
  using namespace ti;
  return TI_PAGED_FORM(c, ti::append, a, c, p->x_f32, (hipStream_t)stream);
}

extern "C" int ti_paged_read(const ti_paged_cache* c, const int32_t* row_start, int rows, void* k, int ldk, void* v, int ldv, ti_stream_t stream) {
  if (const int rc = ti_paged_check(c, "ti_paged_read")) return rc;
  if (!k || !v) return ti_set_error(TI_ERR_ARG, "ti_paged_read: null pointer");
  if (const int rc = check_rows(c, row_start, rows, "ti_paged_read")) return rc;
  const int64_t w = (int64_t)c->kv_heads * c->head_dim;
  if (ldk < w || ldv < w || ldk % 8 || ldv % 8 || !ti::aligned(k, 16) || !ti::aligned(v, 16))
    return ti_set_error(TI_ERR_ARG, "ti_paged_read: rows of pitch %d, %d for %ld values, or not 16-byte aligned", ldk, ldv, (long)w);
  if (rows == 0) return TI_OK;
  const ti::ReadArgs a = {ti_paged_form(c), {row_start, rows}, k, v, ldk, ldv};
  using namespace ti;
  return TI_PAGED_FORM(c, ti::read, a, c, (hipStream_t)stream);
}
