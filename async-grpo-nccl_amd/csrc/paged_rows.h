// Attention over a paged cache for few rows a sequence (single tokens, drafts): all of its time is reading the cache, so the work is
// dealt out by what is read.  (What is computed: paged_attn.h.)
//
// A work-group is one wavefront.  It owns ROWS = 16 or 32 rows of a sequence and K/V head (G rows a token) and a stretch of the
// keys, which it walks in steps of KB = 32 or 64: a step's K and V travel global -> LDS directly, a step ahead.  No barriers.  The pages of a step are looked up by the scalar
// unit, a step ahead of their loads: 16 tokens that start at a multiple of 16 lie in one page, so each such group is one buffer descriptor, whose
// length ends with the stretch - rows behind it arrive as zeros, whatever lies there.
// Shares of the weights (paged_deal.h): what a wavefront begins or ends in the middle of leaves fp32 sums.
// One token each of 128 sequences of 128 .. 8192 keys, 28 / 4 heads of 128: 1.06 GB in 210 us (5.0 TB/s); of 48 of 1024 .. 32768, 64 / 8 heads, e4m3: 1.59 GB
// in 334 .. 354 us (4.5 .. 4.8 TB/s).  Two buffers and four wavefronts a CU: three and three take 206 and 339 us there, but 32.6 instead of 29.2 for 16
// sequences of 1000 .. 4000 in e4m3 and 29.7 instead of 25.3 for drafts at head dimension 64; four and two more still.  Short calls wait: 4 sequences of
// 128 .. 1024 keys take 11 us, of which two launches 8, the division 1.5, the first rows 2.
#pragma once
#include "paged_deal.h"

namespace fgrpo {

template <int RBY>
__device__ __forceinline__ int paged_swz(int row) {      // RBY: bytes of a row of the LDS tile; four rows of 64 bytes share the banks
  if constexpr (RBY == 64) return (row >> 2) & 3;
  else return attn_swz<RBY / 2>(row);
}
// LDS byte offsets of a lane's fragment reads (AttnLane, for rows of RBY bytes of either type)
template <int RBY>
struct PagedLane {
  uint32_t rowc[RBY / 32];
  uint32_t tr[RBY / 64][2];
};
template <int RBY>
__device__ __forceinline__ PagedLane<RBY> paged_lane(int lane, uint32_t lds0) {
  PagedLane<RBY> L;
  const int h = lane >> 5, g1 = (lane >> 4) & 1, j = lane & 15, r = lane & 31;
#pragma unroll
  for (int st = 0; st < RBY / 32; ++st) L.rowc[st] = lds0 + r * RBY + (((2 * st + h) ^ paged_swz<RBY>(r)) << 4);
#pragma unroll
  for (int nb = 0; nb < RBY / 64; ++nb)
#pragma unroll
    for (int rd = 0; rd < 2; ++rd) {
      const int row = 4 * h + (j >> 2) + 8 * rd, chunk = 4 * nb + 2 * g1 + ((j & 3) >> 1);
      L.tr[nb][rd] = lds0 + row * RBY + ((chunk ^ paged_swz<RBY>(row)) << 4) + 8 * (j & 1);
    }
  return L;
}

// Fragment reads of a 32-key block, in inline assembly (for an LDS access it sees, the compiler waits for every load that is on its way
// into LDS) that waits for them itself.
template <int OFF>
__device__ __forceinline__ void paged_read_rows(u32x4_t (&f)[8], const uint32_t (&a)[8]) {
  asm volatile("ds_read_b128 %0, %8 offset:%16\n\tds_read_b128 %1, %9 offset:%16\n\tds_read_b128 %2, %10 offset:%16\n\tds_read_b128 %3, %11 offset:%16\n\t"
               "ds_read_b128 %4, %12 offset:%16\n\tds_read_b128 %5, %13 offset:%16\n\tds_read_b128 %6, %14 offset:%16\n\tds_read_b128 %7, %15 offset:%16\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]), "=&v"(f[4]), "=&v"(f[5]), "=&v"(f[6]), "=&v"(f[7])
               : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7]), "i"(OFF) : "memory");
}
template <int OFF>
__device__ __forceinline__ void paged_read_rows(u32x4_t (&f)[4], const uint32_t (&a)[4]) {
  asm volatile("ds_read_b128 %0, %4 offset:%8\n\tds_read_b128 %1, %5 offset:%8\n\tds_read_b128 %2, %6 offset:%8\n\tds_read_b128 %3, %7 offset:%8\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]) : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "i"(OFF) : "memory");
}
template <int OFF>
__device__ __forceinline__ void paged_read_rows(u32x4_t (&f)[2], const uint32_t (&a)[2]) {
  asm volatile("ds_read_b128 %0, %2 offset:%4\n\tds_read_b128 %1, %3 offset:%4\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(f[0]), "=&v"(f[1]) : "v"(a[0]), "v"(a[1]), "i"(OFF) : "memory");
}
template <int OFF>
__device__ __forceinline__ void paged_read_scales(u32x4_t (&f)[4], uint32_t a) {      // keys 8 i + 4 h .. of the block
  asm volatile("ds_read_b128 %0, %4 offset:%5\n\tds_read_b128 %1, %4 offset:%6\n\tds_read_b128 %2, %4 offset:%7\n\tds_read_b128 %3, %4 offset:%8\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]) : "v"(a), "i"(OFF), "i"(OFF + 32), "i"(OFF + 64), "i"(OFF + 96) : "memory");
}
// the transposed fragments of 16 keys at OFF and of the next 16
template <int RBY, int OFF, int VB>
__device__ __forceinline__ void paged_read_columns(AttnTr (&f)[2][VB], const uint32_t (&a)[VB][2]) {
  static_assert(OFF + 16 * RBY < 65536, "DS offset field");
#pragma unroll
  for (int n = 0; n < VB; n += (VB == 1 ? 1 : 2)) {
    constexpr int NEXT = VB == 1 ? 0 : 1;
    if constexpr (VB == 1)
      asm volatile("ds_read_b64_tr_b16 %0, %4 offset:%6\n\tds_read_b64_tr_b16 %1, %5 offset:%6\n\t"
                   "ds_read_b64_tr_b16 %2, %4 offset:%7\n\tds_read_b64_tr_b16 %3, %5 offset:%7\n\ts_waitcnt lgkmcnt(0)"
                   : "=&v"(f[0][n].lo), "=&v"(f[0][n].hi), "=&v"(f[1][n].lo), "=&v"(f[1][n].hi)
                   : "v"(a[n][0]), "v"(a[n][1]), "i"(OFF), "i"(OFF + 16 * RBY) : "memory");
    else
      asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %9 offset:%12\n\t"
                   "ds_read_b64_tr_b16 %2, %10 offset:%12\n\tds_read_b64_tr_b16 %3, %11 offset:%12\n\t"
                   "ds_read_b64_tr_b16 %4, %8 offset:%13\n\tds_read_b64_tr_b16 %5, %9 offset:%13\n\t"
                   "ds_read_b64_tr_b16 %6, %10 offset:%13\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\ts_waitcnt lgkmcnt(0)"
                   : "=&v"(f[0][n].lo), "=&v"(f[0][n].hi), "=&v"(f[0][n + NEXT].lo), "=&v"(f[0][n + NEXT].hi),
                     "=&v"(f[1][n].lo), "=&v"(f[1][n].hi), "=&v"(f[1][n + NEXT].lo), "=&v"(f[1][n + NEXT].hi)
                   : "v"(a[n][0]), "v"(a[n][1]), "v"(a[n + NEXT][0]), "v"(a[n + NEXT][1]), "i"(OFF), "i"(OFF + 16 * RBY) : "memory");
  }
}

// ---- the same for blocks of 16 rows (16x16x32 instructions): lane l has row l % 16 of K or column l % 16 of the others, chunks 4 st + l / 16 and keys 4 (l / 16) .. + 3
// of 16.  Rows of 16 keys share 16 chunks of banks: conflict-free for 16 rows at one chunk and for 8 rows at two
template <int RBY>
__device__ __forceinline__ int paged_swz16(int row) {
  if constexpr (RBY == 256) return ((row & 7) << 1) | ((row >> 3) & 1);
  else if constexpr (RBY == 128) return (((row >> 1) & 3) << 1) | ((row >> 3) & 1);
  else return (((row >> 2) & 1) << 1) | ((row >> 3) & 1);
}
// N chunks of two rows OFF apart
template <int OFF>
__device__ __forceinline__ void paged_read_rows16(u32x4_t (&f)[2][4], const uint32_t (&a)[4]) {
  asm volatile("ds_read_b128 %0, %8\n\tds_read_b128 %1, %9\n\tds_read_b128 %2, %10\n\tds_read_b128 %3, %11\n\t"
               "ds_read_b128 %4, %8 offset:%12\n\tds_read_b128 %5, %9 offset:%12\n\tds_read_b128 %6, %10 offset:%12\n\tds_read_b128 %7, %11 offset:%12\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(f[0][0]), "=&v"(f[0][1]), "=&v"(f[0][2]), "=&v"(f[0][3]), "=&v"(f[1][0]), "=&v"(f[1][1]), "=&v"(f[1][2]), "=&v"(f[1][3])
               : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "i"(OFF) : "memory");
}
template <int OFF>
__device__ __forceinline__ void paged_read_rows16(u32x4_t (&f)[2][2], const uint32_t (&a)[2]) {
  asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\tds_read_b128 %2, %4 offset:%6\n\tds_read_b128 %3, %5 offset:%6\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(f[0][0]), "=&v"(f[0][1]), "=&v"(f[1][0]), "=&v"(f[1][1]) : "v"(a[0]), "v"(a[1]), "i"(OFF) : "memory");
}
template <int OFF>
__device__ __forceinline__ void paged_read_rows16(u32x4_t (&f)[2][1], const uint32_t (&a)[1]) {
  asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %2 offset:%3\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(f[0][0]), "=&v"(f[1][0]) : "v"(a[0]), "i"(OFF) : "memory");
}
// N blocks of 16 columns, four keys and the four OFF bytes behind
template <int OFF>
__device__ __forceinline__ void paged_read_columns16(AttnTr (&f)[8], const uint32_t (&a)[8]) {
#define TR16(n, k) "ds_read_b64_tr_b16 %" #n ", %" #k "\n\t"
#define TR16_OFF(n, k) "ds_read_b64_tr_b16 %" #n ", %" #k " offset:%24\n\t"
  asm volatile(TR16(0, 16) TR16(1, 17) TR16(2, 18) TR16(3, 19) TR16(4, 20) TR16(5, 21) TR16(6, 22) TR16(7, 23)
               TR16_OFF(8, 16) TR16_OFF(9, 17) TR16_OFF(10, 18) TR16_OFF(11, 19) TR16_OFF(12, 20) TR16_OFF(13, 21) TR16_OFF(14, 22) TR16_OFF(15, 23) "s_waitcnt lgkmcnt(0)"
               : "=&v"(f[0].lo), "=&v"(f[1].lo), "=&v"(f[2].lo), "=&v"(f[3].lo), "=&v"(f[4].lo), "=&v"(f[5].lo), "=&v"(f[6].lo), "=&v"(f[7].lo),
                 "=&v"(f[0].hi), "=&v"(f[1].hi), "=&v"(f[2].hi), "=&v"(f[3].hi), "=&v"(f[4].hi), "=&v"(f[5].hi), "=&v"(f[6].hi), "=&v"(f[7].hi)
               : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7]), "i"(OFF) : "memory");
#undef TR16
#undef TR16_OFF
}
template <int OFF>
__device__ __forceinline__ void paged_read_columns16(AttnTr (&f)[4], const uint32_t (&a)[4]) {
  asm volatile("ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %9\n\tds_read_b64_tr_b16 %2, %10\n\tds_read_b64_tr_b16 %3, %11\n\t"
               "ds_read_b64_tr_b16 %4, %8 offset:%12\n\tds_read_b64_tr_b16 %5, %9 offset:%12\n\tds_read_b64_tr_b16 %6, %10 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%12\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(f[0].lo), "=&v"(f[1].lo), "=&v"(f[2].lo), "=&v"(f[3].lo), "=&v"(f[0].hi), "=&v"(f[1].hi), "=&v"(f[2].hi), "=&v"(f[3].hi)
               : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "i"(OFF) : "memory");
}
template <int OFF>
__device__ __forceinline__ void paged_read_columns16(AttnTr (&f)[2], const uint32_t (&a)[2]) {
  asm volatile("ds_read_b64_tr_b16 %0, %4\n\tds_read_b64_tr_b16 %1, %5\n\tds_read_b64_tr_b16 %2, %4 offset:%6\n\tds_read_b64_tr_b16 %3, %5 offset:%6\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(f[0].lo), "=&v"(f[1].lo), "=&v"(f[0].hi), "=&v"(f[1].hi) : "v"(a[0]), "v"(a[1]), "i"(OFF) : "memory");
}
__device__ __forceinline__ void paged_read_scales16(u32x4_t (&f)[4], uint32_t k, uint32_t v) {      // keys 4 g .. and 16 + 4 g .., of K and of V
  asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:64\n\tds_read_b128 %2, %5\n\tds_read_b128 %3, %5 offset:64\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]) : "v"(k), "v"(v) : "memory");
}
__device__ __forceinline__ float paged_most_of_four(float x) {      // over the lanes l, l ^ 16, l ^ 32, l ^ 48
  float lo = x, hi = x;
  asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(lo), "+v"(hi));
  attn_halves(fmaxf(lo, hi), lo, hi);
  return fmaxf(lo, hi);
}
__device__ __forceinline__ float paged_sum_of_four(float x) {
  float lo = x, hi = x;
  asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(lo), "+v"(hi));
  attn_halves(lo + hi, lo, hi);
  return lo + hi;
}

// ---- the kernel ---------------------------------------------------------------------------------------------------------
template <int HD, bool FP8>
struct PagedRows {
  static constexpr int ES = FP8 ? 1 : 2, RBY = HD * ES, NB = RBY == 256 ? 1 : 2, KB = 32 * NB, NG = KB / 16;
  static constexpr int CPR = RBY / 16, RPI = 1024 / RBY, IPG = 16 / RPI;
  static constexpr int NBUF = 2, TILE = KB * RBY, BUF = 2 * TILE, SCALES = NBUF * BUF, LDS = NBUF * BUF + (FP8 ? NBUF * 2 * KB * 4 : 0);
  static constexpr int LOADS = 2 * NG * IPG + (FP8 ? 2 : 0);      // vector-memory instructions of a step
};

// eight codes of two registers of the transposing reads, one of two columns each -> bf16
__device__ __forceinline__ u32x4_t paged_codes_to_bf16(uint32_t a, uint32_t b) {      // codes 0 .. 3 and 4 .. 7
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  auto cvt = [](uint32_t x, auto hi) { return __builtin_bit_cast(uint32_t, (b2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, decltype(hi)::value)); };
  return u32x4_t{cvt(a, std::false_type{}), cvt(a, std::true_type{}), cvt(b, std::false_type{}), cvt(b, std::true_type{})};
}

// What the kernels share: a share of the weights, walked item by item, with `item()` for each stretch.
template <class C, int ROWS>
struct PagedWalk {
  const PagedAttn& p;
  const PagedSplit& sp;
  const int lane, w;
  uint32_t voff_k[C::IPG], voff_v[C::IPG];      // a lane's place in the rows of an instruction
  int first_pg[C::NBUF - 1][C::NG], pg[C::NG];      // as the table has them
  int head, b, q0, nq, len, rows, r0, k_end, all_see, k0, k1;      // the stretch at hand
  int first_tok, first_rem;      // row r0
  bool begins, ends;

  template <class Swz>
  __device__ __forceinline__ PagedWalk(const PagedAttn& p_, const PagedSplit& sp_, Swz swz)
      : p(p_), sp(sp_), lane(threadIdx.x), w((blockIdx.x & 7) * (sp_.W >> 3) + (blockIdx.x >> 3)) {      // neighbours in the order share an XCD's L2
#pragma unroll
    for (int i = 0; i < C::IPG; ++i) {
      const int row = i * C::RPI + lane / C::CPR, chunk = (lane % C::CPR) ^ swz(row);
      voff_k[i] = (uint32_t)(row * p.c.k_st[1] * C::ES) + chunk * 16;
      voff_v[i] = (uint32_t)(row * p.c.v_st[1] * C::ES) + chunk * 16;
    }
  }
  __device__ __forceinline__ void look_up(int (&to)[C::NG], int kb) const {
#pragma unroll
    for (int g = 0; g < C::NG; ++g) to[g] = paged_table_at(p.c, b, (kb + 16 * g) >> p.c.page_log2);
  }
  // the step at kb into buffer buf; behind the stretch: as many loads, of no rows
  __device__ __forceinline__ void fetch(char* smem, int buf, int kb, const int (&found)[C::NG]) {
    int pg[C::NG];
    char* t = smem + buf * C::BUF;
#pragma unroll
    for (int g = 0; g < C::NG; ++g) pg[g] = min(max(found[g], 0), p.c.num_pages - 1);      // here: in look_up it would wait for them
    if constexpr (C::ES == 1) {
      const int j = max(min(kb + (lane & (C::KB - 1)), k1 - 1), kb), g = (j - kb) >> 4, place = j & ((1 << p.c.page_log2) - 1);
      int page = pg[0];
#pragma unroll
      for (int i = 1; i < C::NG; ++i) page = g == i ? pg[i] : page;
      char* sc = smem + C::SCALES + buf * (2 * C::KB * 4);
      __builtin_amdgcn_global_load_lds(FGRPO_GLOBAL_PTR(p.c.k_scale + paged_offset(p.c.ks_st, page, place, head)), FGRPO_LDS_PTR(sc), 4, 0, 0);
      __builtin_amdgcn_global_load_lds(FGRPO_GLOBAL_PTR(p.c.v_scale + paged_offset(p.c.vs_st, page, place, head)), FGRPO_LDS_PTR(sc + C::KB * 4), 4, 0, 0);
    }
#pragma unroll
    for (int g = 0; g < C::NG; ++g) {
      const int j = kb + 16 * g, place = j & ((1 << p.c.page_log2) - 1), n = min(max(k1 - j, 0), 16);
      const __amdgpu_buffer_rsrc_t rk = make_rsrc(p.c.k + paged_offset(p.c.k_st, pg[g], place, head) * C::ES, n ? (uint32_t)((n - 1) * p.c.k_st[1] * C::ES) + C::RBY : 0);
      const __amdgpu_buffer_rsrc_t rv = make_rsrc(p.c.v + paged_offset(p.c.v_st, pg[g], place, head) * C::ES, n ? (uint32_t)((n - 1) * p.c.v_st[1] * C::ES) + C::RBY : 0);
#pragma unroll
      for (int i = 0; i < C::IPG; ++i) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, FGRPO_LDS_PTR(t + (g * C::IPG + i) * 1024), 16, (int)voff_k[i], 0, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, FGRPO_LDS_PTR(t + C::TILE + (g * C::IPG + i) * 1024), 16, (int)voff_v[i], 0, 0, 0);
      }
    }
  }
  // the pages of the first NBUF steps, asked for together
  __device__ __forceinline__ void look_ahead() {
#pragma unroll
    for (int i = 0; i < C::NBUF - 1; ++i) look_up(first_pg[i], k0 + i * C::KB);
    look_up(pg, k0 + (C::NBUF - 1) * C::KB);
  }
  __device__ __forceinline__ void prologue(char* smem) {
#pragma unroll
    for (int i = 0; i < C::NBUF - 1; ++i) fetch(smem, i, k0 + i * C::KB, first_pg[i]);
  }
  // the loads of the step NBUF - 1 ahead go out, and this one's have landed
  __device__ __forceinline__ void turn(char* smem, int next, int kb) {
    fetch(smem, next, kb + (C::NBUF - 1) * C::KB, pg);
    look_up(pg, kb + C::NBUF * C::KB);
    FGRPO_WAIT_VMCNT((C::NBUF - 1) * C::LOADS);
    __builtin_amdgcn_sched_barrier(0);
  }
  __device__ __forceinline__ void row(int i, int& tok, int& hq) const {      // of the tile: its token in the sequence, its query head
    const int n = first_rem + i < (1 << 20) ? small_div(first_rem + i, p.G) : (first_rem + i) / p.G;
    tok = first_tok + n, hq = head * p.G + first_rem + i - n * p.G;
  }
  __device__ __forceinline__ int slot() const { return 2 * w + (begins ? 1 : 0); }

  template <class Item>
  __device__ __forceinline__ void run(Item&& item) {
    PagedLanes<ROWS> lanes;
    const PagedTotal total = paged_total<ROWS>(p, lanes);
    const PagedShares sh = paged_shares(total, sp.W, sp.most_parts, (double)C::KB * p.G);
    const double hi = uniform(w < sh.used ? sh.bound(w + 1) : 0);
    double done = uniform(w < sh.used ? sh.bound(w) : 0);
    int4 rec = make_int4(0, 0, 0, 0);      // of the item that this wavefront begins and does not end
    int rec_head = 0;
    PagedItem s{0, 0, 0, 0, 0};
    if (done < hi) s = paged_item<ROWS, false>(p, lanes, done);
    while (done < hi) {
      const PagedWeight wt = lanes.of(p, s.b);
      const double weight = wt.of(s.t), x0 = done - s.at, x1 = fmin(hi - s.at, weight);
      b = s.b, head = s.head, q0 = wt.q0, nq = wt.nq, len = wt.len;
      rows = nq * p.G, r0 = s.t * ROWS;
      const PagedRowsAt at(r0, p.G);
      first_tok = at.tok, first_rem = at.rem;
      const PagedSight sight = paged_sight(p, wt, at, 0, ROWS, rows - r0);
      k_end = __builtin_amdgcn_readfirstlane(sight.most), all_see = __builtin_amdgcn_readfirstlane(sight.least);
      const PagedRange kr = paged_range<C::KB>(x0, x1, weight, k_end);
      k0 = kr.k0, k1 = kr.k1;
      begins = x0 <= 0, ends = x1 >= weight;
      if (begins && !ends) rec = make_int4(sh.holding(s.at + weight - 1) - w + 1, q0, r0, rows), rec_head = head;
      if (sp.items > 0 && begins && lane == 0) {
        const int i = min((int)s.index, sp.items - 1);
        sp.rec[2 * i] = ends ? make_int4(0, 0, 0, 0) : rec, sp.rec[2 * i + 1] = make_int4(head, 2 * w + 1, 0, 0);
      }
      look_ahead();
      item();
      s.at = done = uniform(s.at + weight);
      if (done >= hi) break;
      paged_next<ROWS>(p, lanes, s);
      if (s.b >= p.c.B) break;
    }
    if (sp.items > 0) {
      if (w == 0)
        for (int i = (int)total.items + lane; i < sp.items; i += 64) sp.rec[2 * i] = make_int4(0, 0, 0, 0);      // there are no more
    } else if (lane == 0) {
      sp.rec[2 * w] = rec, sp.rec[2 * w + 1] = make_int4(rec_head, 2 * w + 1, 0, 0);
    }
  }
};

// Blocks of 16 rows: a token of up to 16 query heads a K/V head.  Half the arithmetic of a block of 32, and half the registers (64 sequences of 1000 .. 4000
// keys, 12 / 2 heads, 38 us, in blocks of 32 42; e4m3 32.5 and 36).
template <int HD, bool FP8>
static __global__ __launch_bounds__(64) void paged_rows16_kernel(PagedAttn p, PagedSplit sp) {
  using C = PagedRows<HD, FP8>;
  constexpr int KS = HD / 32, DB = HD / 16, NK = C::RBY / 64, NV = C::RBY / 32;      // instructions of a score; blocks of columns; chunks and column blocks of a row as it lies
  __shared__ __attribute__((aligned(1024))) char smem[C::LDS];      // fragment addresses are formed by flipping bits below 1024
  const uint32_t lds0 = lds_addr(smem);
  PagedWalk<C, 16> W(p, sp, [](int row) { return paged_swz16<C::RBY>(row); });
  const int lane = W.lane, r16 = lane & 15, g = lane >> 4;
  const uint32_t row_at = lds0 + r16 * C::RBY + ((g ^ paged_swz16<C::RBY>(r16)) << 4);
  const int tr_row = 4 * g + (r16 >> 2);
  const uint32_t tr_at = lds0 + C::TILE + tr_row * C::RBY + ((((r16 & 3) >> 1) ^ paged_swz16<C::RBY>(tr_row)) << 4) + 8 * (r16 & 1);
  const float c = p.scale * kLog2e;
  W.run([&]() {
    int tok, hq;                 // lanes behind the last row repeat it
    W.row(min(r16, W.rows - W.r0 - 1), tok, hq);
    const int seen = p.causal ? min(max(W.len - W.nq + tok + 1, 0), W.len) : W.len;
    bf16x8_t qf[KS];             // chunks as the K fragments have theirs (e4m3: 16 bytes are two steps' worth)
    const bf16_t* src = p.q + (long long)(W.q0 + tok) * p.q_t + (long long)hq * p.q_h;
#pragma unroll
    for (int st = 0; st < KS; ++st) qf[st] = *(const bf16x8_t*)(src + (FP8 ? 8 * (st / 2) + 2 * g + st % 2 : 4 * st + g) * 8);
    __builtin_amdgcn_sched_barrier(0);
    W.prologue(smem);
#pragma unroll
    for (int st = 0; st < KS; ++st) {      // the rows have landed (they were asked for first); an empty statement makes the compiler wait for them here, not in the loop
      u32x4_t x = __builtin_bit_cast(u32x4_t, qf[st]);
      attn_settle(x);
      qf[st] = __builtin_bit_cast(bf16x8_t, x);
    }
    f32x4_t acc[DB];
    float m_run = -INFINITY, l_run = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    __builtin_amdgcn_sched_barrier(0);
    int buf = 0;
    for (int kb = W.k0; kb < W.k1; kb += C::KB, buf = (buf + 1) % C::NBUF) {
      W.turn(smem, (buf + C::NBUF - 1) % C::NBUF, kb);
      static_for<C::NB>([&](auto mbc) {
        constexpr int mb = decltype(mbc)::value;
        const uint32_t at = buf * C::BUF + mb * (32 * C::RBY);
        u32x4_t kf[2][NK], sk[4];
        uint32_t ka[NK], va[NV];
#pragma unroll
        for (int i = 0; i < NK; ++i) ka[i] = (row_at + at) ^ (i << 6);
#pragma unroll
        for (int i = 0; i < NV; ++i) va[i] = (tr_at + at) ^ (i << 5);
        paged_read_rows16<16 * C::RBY>(kf, ka);
        f32x4_t s[2] = {f32x4_t{0.f, 0.f, 0.f, 0.f}, f32x4_t{0.f, 0.f, 0.f, 0.f}};
        static_for<KS>([&](auto stc) {
          constexpr int st = decltype(stc)::value;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            u32x4_t a;
            if constexpr (FP8) a = paged_codes_to_bf16(kf[i][st / 2][2 * (st % 2)], kf[i][st / 2][2 * (st % 2) + 1]);
            else a = kf[i][st];
            s[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), qf[st], s[i], 0, 0, 0);
          }
        });
        AttnTr vf[NV];
        paged_read_columns16<16 * C::RBY>(vf, va);
        if constexpr (FP8) {
          const uint32_t sc = lds0 + C::SCALES + buf * (2 * C::KB * 4) + mb * 128 + 16 * g;
          paged_read_scales16(sk, sc, sc + C::KB * 4);
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[i][r] *= __uint_as_float(sk[i][r]);
        }
        const int k32 = kb + 32 * mb;
        if (k32 + 32 > W.all_see) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[i][r] = k32 + 16 * i + 4 * g + r < seen ? s[i][r] : -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[i][r]);
        const float m_new = fmaxf(m_run, paged_most_of_four(mx) * c), m_use = m_new == -INFINITY ? 0.f : m_new, alpha = fast_exp2(m_run - m_use);
        float sum = 0.f, e[8];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float x = fast_exp2(__builtin_fmaf(s[i][r], c, -m_use));
            sum += x;
            e[4 * i + r] = FP8 ? x * __uint_as_float(sk[2 + i][r]) : x;
          }
        l_run = l_run * alpha + sum;
        m_run = m_new;
        if (__any(alpha != 1.f)) {
#pragma unroll
          for (int db = 0; db < DB; ++db) acc[db] *= alpha;
        }
        const bf16x8_t pf = attn_pack8(e);
        static_for<NV>([&](auto nc) {
          constexpr int n = decltype(nc)::value;
          const u32x4_t v = {vf[n].lo.x, vf[n].lo.y, vf[n].hi.x, vf[n].hi.y};
          if constexpr (FP8) {
#pragma unroll
            for (int odd = 0; odd < 2; ++odd) {
              const uint32_t sel = odd ? 0x07050301u : 0x06040200u;
              const u32x4_t a = paged_codes_to_bf16(__builtin_amdgcn_perm(v[1], v[0], sel), __builtin_amdgcn_perm(v[3], v[2], sel));
              acc[2 * n + odd] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), pf, acc[2 * n + odd], 0, 0, 0);
            }
          } else {
            acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, v), pf, acc[n], 0, 0, 0);
          }
        });
        __builtin_amdgcn_sched_barrier(0);
      });
    }
    FGRPO_WAIT_VMCNT(0);         // the loads behind the stretch: the next one's go to the same buffers
    const float l = paged_sum_of_four(l_run);
    if (W.r0 + r16 >= W.rows) return;
    if (W.begins && W.ends) {
      const float mul = l > 0.f ? 1.f / l : 0.f;
      bf16_t* dst = p.out + ((long long)(W.q0 + tok) * p.Hq + hq) * HD;
      if constexpr (FP8) {
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          u32x4_t x;
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = pack_bf16x2(acc[2 * n][i] * mul, acc[2 * n + 1][i] * mul);
          *(u32x4_t*)(dst + paged_column<16, true>(2 * n, lane)) = x;
        }
      } else {
#pragma unroll
        for (int n = 0; n < DB; ++n) {
          uint2 x;
          x.x = pack_bf16x2(acc[n][0] * mul, acc[n][1] * mul), x.y = pack_bf16x2(acc[n][2] * mul, acc[n][3] * mul);
          *(uint2*)(dst + paged_column<16, false>(n, lane)) = x;
        }
      }
      if (p.lse && g == 0) p.lse[(long long)hq * p.c.T + W.q0 + tok] = paged_lse(m_run, l);
    } else {
      float* dst = sp.part + (long long)W.slot() * (16 * HD) + lane * 4;
#pragma unroll
      for (int n = 0; n < DB; ++n) *(f32x4_t*)(dst + 256 * n) = acc[n];
      if (g == 0) sp.ml[(long long)W.slot() * 16 + r16] = make_float2(m_run, l);
    }
  });
}

// Blocks of 32 rows: drafts.  Up to 64 rows a K/V head take two of them, which read the same keys out of one L2.  (64 rows a wavefront, K and V
// read once, need all registers of a SIMD and have their arithmetic in one wavefront: 1 to 8 drafts of 14 / 2 heads of 64 30 us
// against 25, of 40 / 8 heads of 128 54 against 52, in e4m3 63 against 43.)
template <int HD, bool FP8>
static __global__ __launch_bounds__(64) void paged_rows_kernel(PagedAttn p, PagedSplit sp) {
  using C = PagedRows<HD, FP8>;
  constexpr int KS = HD / 16, DB = HD / 32, VB = C::RBY / 64;
  __shared__ __attribute__((aligned(1024))) char smem[C::LDS];      // fragment addresses are formed by flipping bits below 1024
  const uint32_t lds0 = lds_addr(smem);
  PagedWalk<C, 32> W(p, sp, [](int row) { return paged_swz<C::RBY>(row); });
  const int lane = W.lane, h = lane >> 5;
  const PagedLane<C::RBY> L = paged_lane<C::RBY>(lane, lds0);
  const float c = p.scale * kLog2e;
  W.run([&]() {
    int tok, hq;                 // lanes behind the last row repeat it
    W.row(min(lane & 31, W.rows - W.r0 - 1), tok, hq);
    const int seen = p.causal ? min(max(W.len - W.nq + tok + 1, 0), W.len) : W.len;
    bf16x8_t qf[KS];             // chunks as the K fragments have theirs (e4m3: 16 bytes are two steps' worth)
    const bf16_t* src = p.q + (long long)(W.q0 + tok) * p.q_t + (long long)hq * p.q_h;
#pragma unroll
    for (int st = 0; st < KS; ++st) qf[st] = *(const bf16x8_t*)(src + (FP8 ? 4 * (st / 2) + 2 * h + st % 2 : 2 * st + h) * 8);
    __builtin_amdgcn_sched_barrier(0);
    W.prologue(smem);
#pragma unroll
    for (int st = 0; st < KS; ++st) {      // as in the kernel for 16
      u32x4_t x = __builtin_bit_cast(u32x4_t, qf[st]);
      attn_settle(x);
      qf[st] = __builtin_bit_cast(bf16x8_t, x);
    }
    f32x16_t acc[DB];
    float m_run = -INFINITY, l_run = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[db][r] = 0.f;
    __builtin_amdgcn_sched_barrier(0);
    auto step = [&](auto curc, int kb) {
      constexpr int cur = decltype(curc)::value, base = cur * C::BUF;
      W.turn(smem, (cur + C::NBUF - 1) % C::NBUF, kb);
      static_for<C::NB>([&](auto mbc) {
        constexpr int mb = decltype(mbc)::value;
        u32x4_t kf[C::RBY / 32], sk[4], sv[4];
        AttnTr vq[2][VB];
        paged_read_rows<base + mb * 32 * C::RBY>(kf, L.rowc);
        if constexpr (FP8) {
          paged_read_scales<cur * 2 * C::KB * 4 + mb * 128>(sk, lds0 + C::SCALES + 16 * h);
          paged_read_scales<cur * 2 * C::KB * 4 + C::KB * 4 + mb * 128>(sv, lds0 + C::SCALES + 16 * h);
        }
        f32x16_t s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
        static_for<KS>([&](auto stc) {
          constexpr int st = decltype(stc)::value;
          u32x4_t a;
          if constexpr (FP8) a = paged_codes_to_bf16(kf[st / 2][2 * (st % 2)], kf[st / 2][2 * (st % 2) + 1]);
          else a = kf[st];
          s = attn_mfma(a, __builtin_bit_cast(u32x4_t, qf[st]), s);
        });
        __builtin_amdgcn_sched_barrier(0);
        paged_read_columns<C::RBY, base + C::TILE + mb * 32 * C::RBY>(vq, L.tr);
        if constexpr (FP8) {
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] *= __uint_as_float(sk[r >> 2][r & 3]);
        }
        const int k32 = kb + 32 * mb;
        if (k32 + 32 > W.all_see) {
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = k32 + 4 * h + 8 * (r >> 2) + (r & 3) < seen ? s[r] : -INFINITY;
        }
        float mx = -INFINITY, mlo, mhi;
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[r]);
        attn_halves(mx, mlo, mhi);
        const float m_new = fmaxf(m_run, fmaxf(mlo, mhi) * c), m_use = m_new == -INFINITY ? 0.f : m_new, alpha = fast_exp2(m_run - m_use);
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float e = fast_exp2(__builtin_fmaf(s[r], c, -m_use));
          sum[r & 1] += e;
          s[r] = FP8 ? e * __uint_as_float(sv[r >> 2][r & 3]) : e;
        }
        l_run = l_run * alpha + (sum[0] + sum[1]);
        m_run = m_new;
        if (__any(alpha != 1.f)) {
#pragma unroll
          for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[db][r] *= alpha;
        }
        __builtin_amdgcn_sched_barrier(0);
        static_for<2>([&](auto qc) {
          constexpr int q = decltype(qc)::value;
          float tmp[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) tmp[j] = s[8 * q + j];
          const u32x4_t pf = __builtin_bit_cast(u32x4_t, attn_pack8(tmp));
          static_for<VB>([&](auto nc) {
            constexpr int n = decltype(nc)::value;
            const u32x4_t v = {vq[q][n].lo.x, vq[q][n].lo.y, vq[q][n].hi.x, vq[q][n].hi.y};
            if constexpr (FP8) {
#pragma unroll
              for (int odd = 0; odd < 2; ++odd) {
                const uint32_t sel = odd ? 0x07050301u : 0x06040200u;
                acc[2 * n + odd] = attn_mfma(paged_codes_to_bf16(__builtin_amdgcn_perm(v[1], v[0], sel), __builtin_amdgcn_perm(v[3], v[2], sel)), pf, acc[2 * n + odd]);
              }
            } else {
              acc[n] = attn_mfma(v, pf, acc[n]);
            }
          });
          __builtin_amdgcn_sched_barrier(0);
        });
      });
    };
    for (int kb = W.k0; kb < W.k1; kb += C::NBUF * C::KB)
      static_for<C::NBUF>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        if (kb + i * C::KB < W.k1) step(ic, kb + i * C::KB);
      });
    FGRPO_WAIT_VMCNT(0);         // the loads behind the stretch: the next one's go to the same buffers
    float l_lo, l_hi;
    attn_halves(l_run, l_lo, l_hi);
    const float l = l_lo + l_hi;
    if (W.r0 + (lane & 31) >= W.rows) return;
    if (W.begins && W.ends) {
      paged_store_row<HD, FP8>(acc, l > 0.f ? 1.f / l : 0.f, p.out + ((long long)(W.q0 + tok) * p.Hq + hq) * HD, h);
      if (p.lse && h == 0) p.lse[(long long)hq * p.c.T + W.q0 + tok] = paged_lse(m_run, l);
    } else {
      attn_store_partial(acc, sp.part + (long long)W.slot() * (32 * HD), lane);
      if (h == 0) sp.ml[(long long)W.slot() * 32 + lane] = make_float2(m_run, l);
    }
  });
}

}  // namespace fgrpo
