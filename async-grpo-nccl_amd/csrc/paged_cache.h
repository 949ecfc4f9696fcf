// A cache of keys and values in pages of `page` tokens, in bf16 or in e4m3 with one fp32 scale per (token, K/V head).
//   page p, place i of it, head h:  k + p k_st[0] + i k_st[1] + h k_st[2], D values one behind the other
// Sequence b's token j lies in page table[b][j / page], place j mod page.  The three calls that go by it (write, read, and the
// attention of paged_attn.h) share cu (the packed rows of each sequence), lens (its length, new tokens included) and table.
// What comes from device memory is held inside its arrays here: cu inside [0, T], lens inside [0, width * page], pages inside
// [0, num_pages).  Page sizes are powers of two of at least 16, so a place is a shift and a mask, and 16 tokens that start at a
// multiple of 16 lie in one page.
//
// Quantising: a = max over the finite |x| of the D values, s = max(a, 1e-30) / 448, code = e4m3(x * (448 / max(a, 1e-30))), rounded to
// nearest even.  A finite x becomes at most 448 (1 + 2^-23), which rounds to 448, so nothing overflows; the half step of e4m3 (3 bits
// behind the point) makes code * s off by at most 2^-4 |x| + 2^-10 s.  The floor keeps 448 / a finite for rows of zeros and
// of denormals.  Infinities and NaN become NaN, which the format has, and leave the rest of their row alone.
#pragma once
#include "attn_kernels.h"

namespace fgrpo {

constexpr float kFp8Max = 448.f, kFp8Floor = 1e-30f;

struct PagedView {
  char* k;
  char* v;
  float* k_scale;        // null: bf16
  float* v_scale;
  long long k_st[3], v_st[3], ks_st[3], vs_st[3];      // page, token, head; elements
  const int* table;      // [B][width], rows table_st apart (width >= 1: without a table, any readable address)
  const int* lens;       // [B]
  const int* cu;         // [B + 1]
  long long table_st;
  int B, T, width, reach, page_log2, num_pages, Hkv;      // reach: tokens that the table has blocks for
};

struct PagedSeq {
  int b, row0, rows, len;      // b < 0: the row belongs to no sequence
};
__device__ __forceinline__ int paged_len(const PagedView& c, int b) { return min(max(c.lens[b], 0), c.reach); }

// The sequence of packed row t (the same in all lanes): 64 ends at a time.  cu is taken to ascend; rows from cu[B] on belong to none.
__device__ __forceinline__ PagedSeq paged_find(const PagedView& c, int t, int lane) {
  int b = 0;
  for (int base = 0; base < c.B; base += 64) {
    const int i = base + lane;
    const bool past = i < c.B && c.cu[i + 1] <= t;
    const int n = __popcll(__ballot(past));
    b += n;
    if (n < 64) break;
  }
  b = __builtin_amdgcn_readfirstlane(b);
  if (b >= c.B) return PagedSeq{-1, 0, 0, 0};
  const int lo = min(max(c.cu[b], 0), c.T), hi = min(max(c.cu[b + 1], lo), c.T);
  if (t < lo) return PagedSeq{-1, 0, 0, 0};
  return PagedSeq{b, lo, hi - lo, paged_len(c, b)};
}
__device__ __forceinline__ int paged_page(const PagedView& c, int b, int j) {
  return min(max(c.table[(long long)b * c.table_st + (j >> c.page_log2)], 0), c.num_pages - 1);
}
__device__ __forceinline__ long long paged_offset(const long long (&st)[3], int page, int place, int head) {
  return (long long)page * st[0] + (long long)place * st[1] + (long long)head * st[2];
}

__device__ __forceinline__ float bf16_lo(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

// eight bf16 -> eight codes under the row's scale; LPR lanes hold a row
template <int LPR>
__device__ __forceinline__ uint2 paged_quantise(u32x4_t x, float& scale) {
  float f[8], a = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) f[2 * i] = bf16_lo(x[i]), f[2 * i + 1] = bf16_hi(x[i]);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float m = fabsf(f[i]);
    a = fmaxf(a, m < INFINITY ? m : 0.f);
  }
#pragma unroll
  for (int d = 1; d < LPR; d *= 2) a = fmaxf(a, __shfl_xor(a, d, 64));
  a = fmaxf(a, kFp8Floor);
  scale = a / kFp8Max;
  const float inv = kFp8Max / a;
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = fabsf(f[i]) < INFINITY ? f[i] * inv : NAN;
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[4], f[5], hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[6], f[7], hi, true);
  return make_uint2((uint32_t)lo, (uint32_t)hi);
}
// eight codes -> eight bf16 of code * scale
__device__ __forceinline__ u32x4_t paged_restore(uint2 x, float s) {
  u32x4_t r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int w = (int)(i ? x.y : x.x);
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    r[2 * i] = pack_bf16x2(a[0] * s, a[1] * s);
    r[2 * i + 1] = pack_bf16x2(b[0] * s, b[1] * s);
  }
  return r;
}

struct PagedWrite {
  PagedView c;
  const bf16_t* k;       // [T][Hkv][D] new rows
  const bf16_t* v;
  long long k_t, k_h, v_t, v_h;
};
struct PagedRead {
  PagedView c;
  bf16_t* k;             // [T][Hkv][D] contiguous
  bf16_t* v;
};

// Write and read: a wavefront takes one packed row (token), all its heads, 16 bytes of bf16 a lane; the rows of a K/V head are whole in a few lanes, so the maximum
// that e4m3 needs is a few lane moves.  Bound by memory, and for few tokens by the launch: 27000 tokens of 8 heads of 128 into e4m3 217 MB in 44 us (4.9 TB/s), 40
// sequences of e4m3 answers back into bf16 146 MB in 28 us (5.2 TB/s), 64 single tokens 5.5 us.
template <int HD, bool FP8>
static __global__ __launch_bounds__(256) void paged_write_kernel(PagedWrite p) {
  constexpr int LPR = HD / 8;
  const int lane = threadIdx.x & 63, t = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t >= p.c.T) return;
  const PagedSeq s = paged_find(p.c, t, lane);
  if (s.b < 0) return;
  const int j = s.len - s.rows + (t - s.row0);
  if (j < 0 || j >= s.len) return;
  const int page = paged_page(p.c, s.b, j), place = j & ((1 << p.c.page_log2) - 1);
  for (int i = lane; i < p.c.Hkv * LPR; i += 64) {
    const int h = i / LPR, d = i % LPR * 8;
    const u32x4_t xk = *(const u32x4_t*)(p.k + (long long)t * p.k_t + (long long)h * p.k_h + d);
    const u32x4_t xv = *(const u32x4_t*)(p.v + (long long)t * p.v_t + (long long)h * p.v_h + d);
    const long long ok = paged_offset(p.c.k_st, page, place, h) + d, ov = paged_offset(p.c.v_st, page, place, h) + d;
    if constexpr (FP8) {
      float sk, sv;
      *(uint2*)(p.c.k + ok) = paged_quantise<LPR>(xk, sk);
      *(uint2*)(p.c.v + ov) = paged_quantise<LPR>(xv, sv);
      if (d == 0) {
        p.c.k_scale[paged_offset(p.c.ks_st, page, place, h)] = sk;
        p.c.v_scale[paged_offset(p.c.vs_st, page, place, h)] = sv;
      }
    } else {
      *(u32x4_t*)(p.c.k + 2 * ok) = xk;
      *(u32x4_t*)(p.c.v + 2 * ov) = xv;
    }
  }
}

template <int HD, bool FP8>
static __global__ __launch_bounds__(256) void paged_read_kernel(PagedRead p) {
  constexpr int LPR = HD / 8;
  const int lane = threadIdx.x & 63, t = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t >= p.c.T) return;
  const PagedSeq s = paged_find(p.c, t, lane);
  if (s.b < 0) return;
  const int j = t - s.row0;
  if (j >= s.len) return;
  const int page = paged_page(p.c, s.b, j), place = j & ((1 << p.c.page_log2) - 1);
  for (int i = lane; i < p.c.Hkv * LPR; i += 64) {
    const int h = i / LPR, d = i % LPR * 8;
    const long long ok = paged_offset(p.c.k_st, page, place, h) + d, ov = paged_offset(p.c.v_st, page, place, h) + d;
    u32x4_t xk, xv;
    if constexpr (FP8) {
      xk = paged_restore(*(const uint2*)(p.c.k + ok), p.c.k_scale[paged_offset(p.c.ks_st, page, place, h)]);
      xv = paged_restore(*(const uint2*)(p.c.v + ov), p.c.v_scale[paged_offset(p.c.vs_st, page, place, h)]);
    } else {
      xk = *(const u32x4_t*)(p.c.k + 2 * ok);
      xv = *(const u32x4_t*)(p.c.v + 2 * ov);
    }
    const long long o = ((long long)t * p.c.Hkv + h) * HD + d;
    *(u32x4_t*)(p.k + o) = xk;
    *(u32x4_t*)(p.v + o) = xv;
  }
}

}  // namespace fgrpo
