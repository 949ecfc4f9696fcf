// Attention over a paged cache for few rows a sequence (single tokens, drafts): all of its time is reading the cache, so the work is
// dealt out by what is read.  (What is computed: paged_attn.h.)
//
// A work-group is one wavefront.  It owns 32 RB rows of a sequence and K/V head (RB = 1 or 2; G rows a token) and a stretch of the
// keys, which it walks in steps of KB = 32 or 64: a step's K and V travel global -> LDS directly, a step ahead, 16 KiB in flight
// behind 16 KiB in use, four to five wavefronts a CU.  No barriers.  The pages of a step are looked up by the scalar unit, a step
// ahead of their loads: 16 tokens that start at a multiple of 16 lie in one page, so each such group is one buffer descriptor, whose
// length ends with the sequence - rows behind it arrive as zeros, whatever lies there.
// Shares of the weights (paged_deal.h): what a wavefront begins or ends in the middle of leaves fp32 sums.
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

// ---- the kernel ---------------------------------------------------------------------------------------------------------
template <int HD, bool FP8>
struct PagedRows {
  static constexpr int ES = FP8 ? 1 : 2, RBY = HD * ES, NB = RBY == 256 ? 1 : 2, KB = 32 * NB, NG = KB / 16;
  static constexpr int CPR = RBY / 16, RPI = 1024 / RBY, IPG = 16 / RPI;
  static constexpr int TILE = KB * RBY, BUF = 2 * TILE, SCALES = FP8 ? 4 * KB * 4 : 0, LDS = 2 * BUF + SCALES;
  static constexpr int LOADS = 2 * NG * IPG + (FP8 ? 2 : 0);      // vector-memory instructions of a step
};

// eight codes of two registers of the transposing reads, one of two columns each -> bf16
__device__ __forceinline__ u32x4_t paged_codes_to_bf16(uint32_t a, uint32_t b) {      // codes 0 .. 3 and 4 .. 7
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  auto cvt = [](uint32_t x, auto hi) { return __builtin_bit_cast(uint32_t, (b2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, decltype(hi)::value)); };
  return u32x4_t{cvt(a, std::false_type{}), cvt(a, std::true_type{}), cvt(b, std::false_type{}), cvt(b, std::true_type{})};
}

template <int HD, bool FP8, int RB>
static __global__ __launch_bounds__(64) void paged_rows_kernel(PagedAttn p, PagedSplit sp) {
  using C = PagedRows<HD, FP8>;
  constexpr int KS = HD / 16, DB = HD / 32, VB = C::RBY / 64, ROWS = 32 * RB;
  __shared__ __attribute__((aligned(16))) char smem[C::LDS];
  const uint32_t lds0 = lds_addr(smem);
  const int lane = threadIdx.x, h = lane >> 5;
  const int w = (blockIdx.x & 7) * (sp.W >> 3) + (blockIdx.x >> 3);      // neighbours in the order share an XCD's L2
  const PagedShares sh = paged_shares(paged_total<ROWS>(p), sp.W, 2.0 * C::KB * p.G);
  const double hi = uniform(w < sh.used ? sh.bound(w + 1) : 0);
  double done = uniform(w < sh.used ? sh.bound(w) : 0);
  int4 rec = make_int4(0, 0, 0, 0);      // of the item that this wavefront begins and does not end
  PagedItem s{0, 0, 0, 0, 0};
  if (done < hi) s = paged_item<ROWS, false>(p, done);
  const PagedLane<C::RBY> L = paged_lane<C::RBY>(lane, lds0);
  uint32_t voff_k[C::IPG], voff_v[C::IPG];
#pragma unroll
  for (int i = 0; i < C::IPG; ++i) {
    const int row = i * C::RPI + lane / C::CPR, chunk = (lane % C::CPR) ^ paged_swz<C::RBY>(row);
    voff_k[i] = (uint32_t)(row * p.c.k_st[1] * C::ES) + chunk * 16;
    voff_v[i] = (uint32_t)(row * p.c.v_st[1] * C::ES) + chunk * 16;
  }
  const float c = p.scale * kLog2e;
  while (done < hi) {
    const PagedWeight wt = paged_weight<ROWS>(p, s.b);
    const double weight = wt.of(s.t), x0 = done - s.at, x1 = fmin(hi - s.at, weight);
    const int q0 = __builtin_amdgcn_readfirstlane(wt.q0), nq = __builtin_amdgcn_readfirstlane(wt.nq), len = __builtin_amdgcn_readfirstlane(wt.len);
    const int rows = nq * p.G, r0 = s.t * ROWS;
    const PagedSight sight = paged_sight(p, wt, r0, ROWS);
    const int k_end = __builtin_amdgcn_readfirstlane(sight.most), all_see = __builtin_amdgcn_readfirstlane(sight.least);
    const PagedRange kr = paged_range<C::KB>(x0, x1, weight, k_end);
    const int k0 = kr.k0, k1 = kr.k1;
    const bool begins = x0 <= 0, ends = x1 >= weight;

    int pg[C::NG];
    auto look_up = [&](int kb) {
#pragma unroll
      for (int g = 0; g < C::NG; ++g) pg[g] = paged_table_at(p.c, s.b, (kb + 16 * g) >> p.c.page_log2);
    };
    auto fetch = [&](int buf, int kb) {
      char* t = smem + buf * C::BUF;
#pragma unroll
      for (int g = 0; g < C::NG; ++g) pg[g] = min(max(pg[g], 0), p.c.num_pages - 1);      // here: in look_up it would wait for them
      if constexpr (FP8) {
        const int j = min(kb + (lane & (C::KB - 1)), k_end - 1), g = (j - kb) >> 4, place = j & ((1 << p.c.page_log2) - 1);
        int page = pg[0];
#pragma unroll
        for (int i = 1; i < C::NG; ++i) page = g == i ? pg[i] : page;
        char* sc = smem + 2 * C::BUF + buf * (2 * C::KB * 4);
        __builtin_amdgcn_global_load_lds(FGRPO_GLOBAL_PTR(p.c.k_scale + paged_offset(p.c.ks_st, page, place, s.head)), FGRPO_LDS_PTR(sc), 4, 0, 0);
        __builtin_amdgcn_global_load_lds(FGRPO_GLOBAL_PTR(p.c.v_scale + paged_offset(p.c.vs_st, page, place, s.head)), FGRPO_LDS_PTR(sc + C::KB * 4), 4, 0, 0);
      }
#pragma unroll
      for (int g = 0; g < C::NG; ++g) {
        const int j = kb + 16 * g, place = j & ((1 << p.c.page_log2) - 1), n = min(max(k_end - j, 0), 16);
        const __amdgpu_buffer_rsrc_t rk = make_rsrc(p.c.k + paged_offset(p.c.k_st, pg[g], place, s.head) * C::ES, n ? (uint32_t)((n - 1) * p.c.k_st[1] * C::ES) + C::RBY : 0);
        const __amdgpu_buffer_rsrc_t rv = make_rsrc(p.c.v + paged_offset(p.c.v_st, pg[g], place, s.head) * C::ES, n ? (uint32_t)((n - 1) * p.c.v_st[1] * C::ES) + C::RBY : 0);
#pragma unroll
        for (int i = 0; i < C::IPG; ++i) {
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, FGRPO_LDS_PTR(t + (g * C::IPG + i) * 1024), 16, (int)voff_k[i], 0, 0, 0);
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, FGRPO_LDS_PTR(t + C::TILE + (g * C::IPG + i) * 1024), 16, (int)voff_v[i], 0, 0, 0);
        }
      }
    };
    if (k0 < k1) {
      look_up(k0);
      fetch(0, k0);
      look_up(k0 + C::KB);
    }
    // rows of this lane; the operand's chunks as the K fragments have theirs (e4m3: 16 bytes are two steps' worth)
    int seen[RB], least = all_see;
    bool valid[RB];
    bf16x8_t qf[RB][KS];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int row = r0 + 32 * rb + (lane & 31), tok = row / p.G;
      valid[rb] = row < rows;
      seen[rb] = !valid[rb] || !p.causal ? k_end : min(max(len - nq + tok + 1, 0), len);
      const bf16_t* src = p.q + (long long)(q0 + tok) * p.q_t + (long long)(s.head * p.G + row % p.G) * p.q_h;
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        const u32x4_t z = {0u, 0u, 0u, 0u};
        const int chunk = FP8 ? 4 * (st / 2) + 2 * h + st % 2 : 2 * st + h;
        const u32x4_t x = valid[rb] ? *(const u32x4_t*)(src + chunk * 8) : z;
        qf[rb][st] = __builtin_bit_cast(bf16x8_t, x);
      }
    }
    f32x16_t acc[RB][DB];
    float m_run[RB], l_run[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      m_run[rb] = -INFINITY, l_run[rb] = 0.f;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[rb][db][r] = 0.f;
    }
    FGRPO_WAIT_VMCNT(0);
    __builtin_amdgcn_sched_barrier(0);

    auto step = [&](auto curc, int kb) {
      constexpr int cur = decltype(curc)::value, base = cur * C::BUF;
      if (kb + C::KB < k1) {
        fetch(cur ^ 1, kb + C::KB);
        look_up(kb + 2 * C::KB);
        FGRPO_WAIT_VMCNT(C::LOADS);
      } else {
        FGRPO_WAIT_VMCNT(0);
      }
      __builtin_amdgcn_sched_barrier(0);
      static_for<C::NB>([&](auto mbc) {
        constexpr int mb = decltype(mbc)::value;
        u32x4_t kf[C::RBY / 32], sk[4], sv[4];
        AttnTr vq[2][VB];
        paged_read_rows<base + mb * 32 * C::RBY>(kf, L.rowc);
        if constexpr (FP8) {
          paged_read_scales<2 * C::BUF + cur * 2 * C::KB * 4 + mb * 128>(sk, lds0 + 16 * h);
          paged_read_scales<2 * C::BUF + cur * 2 * C::KB * 4 + C::KB * 4 + mb * 128>(sv, lds0 + 16 * h);
        }
        f32x16_t sc[RB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int r = 0; r < 16; ++r) sc[rb][r] = 0.f;
        static_for<KS>([&](auto sc_) {
          constexpr int st = decltype(sc_)::value;
          u32x4_t a;
          if constexpr (FP8) a = paged_codes_to_bf16(kf[st / 2][2 * (st % 2)], kf[st / 2][2 * (st % 2) + 1]);
          else a = kf[st];
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) sc[rb] = attn_mfma(a, __builtin_bit_cast(u32x4_t, qf[rb][st]), sc[rb]);
        });
        __builtin_amdgcn_sched_barrier(0);
        paged_read_columns<C::RBY, base + C::TILE + mb * 32 * C::RBY>(vq, L.tr);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          if constexpr (FP8) {
#pragma unroll
            for (int r = 0; r < 16; ++r) sc[rb][r] *= __uint_as_float(sk[r >> 2][r & 3]);
          }
          const int k32 = kb + 32 * mb;
          if (k32 + 32 > least) {
#pragma unroll
            for (int r = 0; r < 16; ++r) sc[rb][r] = k32 + 4 * h + 8 * (r >> 2) + (r & 3) < seen[rb] ? sc[rb][r] : -INFINITY;
          }
          float mx = -INFINITY;
#pragma unroll
          for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[rb][r]);
          float mlo, mhi;
          attn_halves(mx, mlo, mhi);
          const float m_new = fmaxf(m_run[rb], fmaxf(mlo, mhi) * c), m_use = m_new == -INFINITY ? 0.f : m_new, alpha = fast_exp2(m_run[rb] - m_use);
          float sum[2] = {0.f, 0.f};
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float e = fast_exp2(__builtin_fmaf(sc[rb][r], c, -m_use));
            sum[r & 1] += e;
            sc[rb][r] = FP8 ? e * __uint_as_float(sv[r >> 2][r & 3]) : e;
          }
          l_run[rb] = l_run[rb] * alpha + (sum[0] + sum[1]);
          m_run[rb] = m_new;
          if (__any(alpha != 1.f)) {
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
              for (int r = 0; r < 16; ++r) acc[rb][db][r] *= alpha;
          }
        }
        __builtin_amdgcn_sched_barrier(0);
        static_for<2>([&](auto qc) {
          constexpr int q = decltype(qc)::value;
          u32x4_t pf[RB];
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) {
            float tmp[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) tmp[j] = sc[rb][8 * q + j];
            pf[rb] = __builtin_bit_cast(u32x4_t, attn_pack8(tmp));
          }
          static_for<VB>([&](auto nc) {
            constexpr int n = decltype(nc)::value;
            const u32x4_t v = {vq[q][n].lo.x, vq[q][n].lo.y, vq[q][n].hi.x, vq[q][n].hi.y};
            if constexpr (FP8) {
#pragma unroll
              for (int odd = 0; odd < 2; ++odd) {
                const uint32_t sel = odd ? 0x07050301u : 0x06040200u;
                const u32x4_t a = paged_codes_to_bf16(__builtin_amdgcn_perm(v[1], v[0], sel), __builtin_amdgcn_perm(v[3], v[2], sel));
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) acc[rb][2 * n + odd] = attn_mfma(a, pf[rb], acc[rb][2 * n + odd]);
              }
            } else {
#pragma unroll
              for (int rb = 0; rb < RB; ++rb) acc[rb][n] = attn_mfma(v, pf[rb], acc[rb][n]);
            }
          });
          __builtin_amdgcn_sched_barrier(0);
        });
      });
    };
    for (int kb = k0; kb < k1; kb += 2 * C::KB) {
      step(std::integral_constant<int, 0>{}, kb);
      if (kb + C::KB < k1) step(std::integral_constant<int, 1>{}, kb + C::KB);
    }
    const int slot = 2 * w + (begins ? 1 : 0);
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      float l_lo, l_hi;
      attn_halves(l_run[rb], l_lo, l_hi);
      const float l = l_lo + l_hi;
      const int row = r0 + 32 * rb + (lane & 31), tok = q0 + row / p.G, hq = s.head * p.G + row % p.G;
      if (begins && ends) {
        if (valid[rb]) {
          paged_store_row<HD, FP8>(acc[rb], l > 0.f ? 1.f / l : 0.f, p.out + ((long long)tok * p.Hq + hq) * HD, h);
          if (p.lse && h == 0) p.lse[(long long)hq * p.c.T + tok] = paged_lse(m_run[rb], l);
        }
      } else if (valid[rb]) {
        attn_store_partial(acc[rb], sp.part + ((long long)slot * RB + rb) * (32 * HD), lane);
        if (h == 0) sp.ml[((long long)slot * RB + rb) * 32 + lane] = make_float2(m_run[rb], l);
      }
    }
    if (begins && !ends) rec = make_int4(s.b + 1, s.t, s.head, sh.holding(s.at + weight - 1) - w + 1);
    paged_next<ROWS>(p, s, paged_weight<ROWS>(p, s.b));
    done = s.at;
    if (s.b >= p.c.B) break;
  }
  if (lane == 0) sp.rec[2 * w] = make_int4(0, 0, 0, 0), sp.rec[2 * w + 1] = rec;
}

}  // namespace fgrpo
