// Attention over a paged cache for many rows a sequence (pieces of prompts, scored answers): bound by the matrix instructions and the
// vector arithmetic beside them.  (What is computed: paged_attn.h; how it is dealt out: paged_deal.h.)
//
// A work-group of four wavefronts has 128 rows of a sequence and K/V head, 32 a wavefront, and walks their keys 64 at a time through two
// LDS buffers, with one barrier a step and the fragment schedule of varlen_attn_fwd2_kernel (attn_kernels.h), two work-groups a CU.  Wavefront w fetches keys 16 w .. of
// a step, which lie in one page: one look-up by the scalar unit, a step ahead.
// bf16 travels global -> LDS directly.  e4m3 is converted once for the four wavefronts: codes wait in registers for a step (16 of them), and
// are written to LDS as bf16, which holds them exactly; the scales of a step's keys lie beside the tiles in LDS, a lane reads one of them, and the multiplications take
// them out of other lanes (each lane reading all of its own: 1 % more).
//
// Dealing out: a launch of W work-groups, all resident.  Where the heaviest item is more than two mean shares, or there are fewer items than
// work-groups, shares of the weights, cut inside items (a cut costs 64 KiB of sums written and read per part: 8 sequences of 682 tokens from the start 63 us in
// shares, 32 whole).  Else whole items, W / 8 a round for the W / 8 work-groups of an XCD, alternately from either end (under the causal mask weights
// ascend); what is left for the last round is cut into as many parts as make it shortest.  Work-groups me and me + W / 16 of an XCD share a CU: where there
// is one round, the heaviest items go beside the lightest (those 8 sequences 37 us without, 256 .. 1024 tokens over 2000 .. 3000 keys 110 and 105).
//
// What a step costs is its instructions: 1024 cycles of matrix instructions a wavefront (32 rows, 64 keys, head dimension 128) and about as many of vector ones, nearly one after the
// other though two wavefronts share a SIMD (bf16 2030 cycles a wavefront step, e4m3 2700; matrix pipes 0.5 busy).  The older of the two wins whatever both could issue,
// so both drift into the same phase; with the priority raised for the products, one's softmax runs beside the other's products (-4..-5 %), and
// sums that are rescaled only when the maximum has grown by 2^8 save the rest (-4..-8 %).  Memory is not what a step waits for: touching its
// lines two to four steps early costs 7..18 %.  40 / 8 heads, 4096 tokens over 32768 keys: bf16 2.36 ms (1.09 PFLOP/s), e4m3 2.80 ms (0.92); 8192 tokens
// from the start 0.67 ms; 14 / 2 heads of 64, 4096 over 32768, 0.57 ms.
#pragma once
#include "paged_rows.h"

namespace fgrpo {

constexpr int kPagedTileRB = kPagedRows / 32;

template <int HD, bool FP8>
struct PagedTiles {
  static constexpr int ES = FP8 ? 1 : 2, RBY = HD * ES;
  static constexpr int CPR = RBY / 16, RPI = 1024 / RBY, IPG = 16 / RPI;      // as the cache has its rows: 16-byte chunks, rows and instructions of 16 keys
  // Rows of the tiles in LDS.  What the direct loads write has no room between rows: chunks are swizzled (attn_swz).  What comes through registers has:
  // rows 16 bytes apart do not share banks where 16 of them are read at one chunk, rows 64 bytes apart where 4 are at 64 bytes, and every
  // fragment address is one register and a constant.
  static constexpr int KROW = HD * 2 + (FP8 ? 16 : 0), VROW = HD * 2 + (FP8 ? 64 : 0);
  static constexpr int KTILE = kAttnBK * KROW, BUF = KTILE + kAttnBK * VROW;
  static constexpr int T0 = FP8 ? 4 * kAttnBK * 4 : 0, LDS = T0 + 2 * BUF;      // the scales of both buffers lie in front (K, then V)
};

template <int OFF0, int OFF1>
__device__ __forceinline__ AttnTr paged_rd_tr(uint32_t a) {      // attn_rd_tr_asm from one address
  static_assert(OFF1 < 65536, "DS offset field");
  AttnTr f;
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(f.lo) : "v"(a), "i"(OFF0));
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(f.hi) : "v"(a), "i"(OFF1));
  return f;
}

template <int OFF>
__device__ __forceinline__ uint32_t paged_read_u32(uint32_t a) {
  uint32_t x;
  asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(x) : "v"(a), "i"(OFF));
  return x;
}
__device__ __forceinline__ void paged_settle_u32(uint32_t& x) { asm volatile("" : "+v"(x)); }

// Parts of the last, incomplete round of `left` items (fewer than n) on `n` work-groups: the shortest of rounds / parts, a cut taken for a 50th of an
// item (a 20th: the answers of the header 101.5 us, with it 100; 24 sequences of 200 .. 700 at head dimension 64 75.7 and 76.7).
__device__ __forceinline__ int paged_last_parts(int left, int n) {
  int best = 1;
  float cost = left > 0 ? 1.f : 0.f;
#pragma unroll
  for (int parts = 2; parts <= 8; ++parts) {
    const float c = (left * parts <= n ? 1.f : 2.f) * (1.f / parts) + 0.02f * parts;
    if (left * parts <= 2 * n && c < cost) cost = c, best = parts;
  }
  return best;
}

// Of items i0 .. i0 + count - 1 (at most 64, s the first of them), the one with `rank` heavier ones; its place among the weights is not found.  A lane weighs
// one; weights that differ by less than 2^-17 count as equal, and then the order decides.
template <int ROWS>
__device__ __forceinline__ PagedItem paged_ranked(const PagedAttn& p, PagedLanes<ROWS>& lanes, PagedItem s, int i0, int count, int rank) {
  const int lane = threadIdx.x & 63;
  int from = -1, b_l = 0, head_l = 0, t_l = 0;      // from: number of the sequence's first item
  uint32_t mine = 63 - lane;
  for (int b = s.b; b < p.c.B && from < i0 + count; ++b) {
    const PagedWeight w = lanes.of(p, b);
    if (from < 0) from = i0 - (s.head * w.tiles + s.t);
    const int at = i0 + lane - from;
    if (lane < count && at >= 0 && at < w.tiles * p.c.Hkv) b_l = b, head_l = at / w.tiles, t_l = at - head_l * w.tiles, mine = (__float_as_uint((float)w.of(t_l)) & ~63u) | (63 - lane);
    from += w.tiles * p.c.Hkv;
  }
  int heavier = 0;
#pragma unroll 16
  for (int j = 0; j < 64; ++j) heavier += (uint32_t)__builtin_amdgcn_readlane(mine, j) > mine;
  const int l = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(heavier == rank)) - 1);
  s.b = __builtin_amdgcn_readlane(b_l, l), s.head = __builtin_amdgcn_readlane(head_l, l), s.t = __builtin_amdgcn_readlane(t_l, l);
  return s;
}

template <int HD, bool FP8>
static __global__ __launch_bounds__(256, 2) void paged_tiles_kernel(PagedAttn p, PagedSplit sp) {
  using C = PagedTiles<HD, FP8>;
  constexpr int KS = HD / 16, DB = HD / 32, G4 = KS / 2, ROWS = kPagedRows;
  __shared__ __attribute__((aligned(1024))) char smem[C::LDS];      // fragment addresses are formed by flipping bits below 1024
  __shared__ double kept[6];
  const uint32_t lds0 = lds_addr(smem);
  const int lane = threadIdx.x & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int xcd = blockIdx.x & 7, n = sp.W >> 3, me = blockIdx.x >> 3, w = xcd * n + me;
  // fragment addresses.  bf16: of k step st the row's first with bits of its chunk flipped, of column block db likewise (AttnLane); e4m3: of buffer 0
  uint32_t row_at, tr_at[2];
  if constexpr (FP8) {
    row_at = lds0 + C::T0 + (lane & 31) * C::KROW + h * 16;
    tr_at[0] = lds0 + C::T0 + C::KTILE + (4 * h + ((lane & 15) >> 2)) * C::VROW + ((lane >> 4) & 1) * 32 + (lane & 3) * 8, tr_at[1] = 0;
  } else {
    const AttnLane<HD> L = attn_lane<HD>(lane);
    row_at = L.rowc[0] + lds0, tr_at[0] = L.tr[0][0] + lds0, tr_at[1] = L.tr[0][1] + lds0;
  }
  const uint32_t sc_at = lds0 + (8 * ((lane & 15) >> 2) + (lane & 3) + 4 * h) * 4;
  const float c = p.scale * kLog2e;
  // where this wavefront's lanes read: row lane / CPR of 16 and every RPI-th behind it, and of instruction i chunk `ch`, but for the bits of
  // the swizzle that i decides; and, codes, where they write
  const int row16 = lane / C::CPR, at16 = 16 * wave + row16, ch = FP8 ? lane % C::CPR : (lane % C::CPR) ^ attn_swz<HD>(at16);
  const uint32_t voff_k = (uint32_t)(row16 * p.c.k_st[1] * C::ES), voff_v = (uint32_t)(row16 * p.c.v_st[1] * C::ES);
  const uint32_t put_k = lds0 + C::T0 + at16 * C::KROW + ch * 32, put_v = lds0 + C::T0 + C::KTILE + at16 * C::VROW + ch * 32;
  auto flip = [](int i) { return attn_swz<HD>(i * C::RPI); };      // the swizzle of row16 + i RPI is that of row16 with these bits flipped: RPI is a power of two above row16

  // x0 .. x1 of an item's weight; whole: its output, else sums for `slot`
  auto walk = [&](const PagedItem& s, const PagedWeight& wt, double x0, double x1, int slot) {
    const double weight = wt.of(s.t);
    const bool whole = x0 <= 0 && x1 >= weight;
    const int q0 = wt.q0, nq = wt.nq, len = wt.len;
    const int rows = nq * p.G, r0 = s.t * ROWS, rw = r0 + 32 * wave;
    const int k_end = __builtin_amdgcn_readfirstlane(paged_sight(p, wt, PagedRowsAt(r0, p.G), 0, ROWS, rows - r0).most);
    const PagedRange kr = paged_range<kAttnBK>(x0, x1, weight, k_end);
    const int k0 = kr.k0, k1 = kr.k1;
    const bool wave_on = rw < rows;
    const PagedSight sight = paged_sight(p, wt, PagedRowsAt(r0, p.G), wave_on ? 32 * wave : 0, 32, rows - r0);
    const int w_most = wave_on ? __builtin_amdgcn_readfirstlane(sight.most) : 0, w_least = __builtin_amdgcn_readfirstlane(sight.least);

    int page = 0;
    auto look_up = [&](int kb) { page = paged_table_at(p.c, s.b, (kb + 16 * wave) >> p.c.page_log2); };
    u32x4_t raw[FP8 ? 2 * C::IPG : 1];
    uint32_t raw_scale[2] = {0u, 0u};
    // tile kb: into LDS (bf16), or into registers
    auto fetch = [&](int buf, int kb) {
      page = min(max(page, 0), p.c.num_pages - 1);
      const int j = kb + 16 * wave, place = j & ((1 << p.c.page_log2) - 1), m = min(max(k_end - j, 0), 16);
      const __amdgpu_buffer_rsrc_t rk = make_rsrc(p.c.k + paged_offset(p.c.k_st, page, place, s.head) * C::ES, m ? (uint32_t)((m - 1) * p.c.k_st[1] * C::ES) + C::RBY : 0);
      const __amdgpu_buffer_rsrc_t rv = make_rsrc(p.c.v + paged_offset(p.c.v_st, page, place, s.head) * C::ES, m ? (uint32_t)((m - 1) * p.c.v_st[1] * C::ES) + C::RBY : 0);
      if constexpr (FP8) {
        const __amdgpu_buffer_rsrc_t sk = make_rsrc(p.c.k_scale + paged_offset(p.c.ks_st, page, place, s.head), m ? (uint32_t)((m - 1) * p.c.ks_st[1] * 4) + 4 : 0);
        const __amdgpu_buffer_rsrc_t sv = make_rsrc(p.c.v_scale + paged_offset(p.c.vs_st, page, place, s.head), m ? (uint32_t)((m - 1) * p.c.vs_st[1] * 4) + 4 : 0);
        raw_scale[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_raw_buffer_load_b32(sk, (int)((lane & 15) * (uint32_t)p.c.ks_st[1] * 4), 0, 0));
        raw_scale[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_raw_buffer_load_b32(sv, (int)((lane & 15) * (uint32_t)p.c.vs_st[1] * 4), 0, 0));
#pragma unroll
        for (int i = 0; i < C::IPG; ++i) {
          raw[2 * i] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rk, (int)(voff_k + ch * 16), (int)(i * C::RPI * p.c.k_st[1]), 0));
          raw[2 * i + 1] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rv, (int)(voff_v + ch * 16), (int)(i * C::RPI * p.c.v_st[1]), 0));
        }
      } else {
        char* t = smem + buf * C::BUF + wave * (16 * C::RBY);
#pragma unroll
        for (int i = 0; i < C::IPG; ++i) {
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, FGRPO_LDS_PTR(t + i * 1024), 16, (int)(voff_k + (ch ^ flip(i)) * 16), (int)(i * C::RPI * p.c.k_st[1] * 2), 0, 0);
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, FGRPO_LDS_PTR(t + C::KTILE + i * 1024), 16, (int)(voff_v + (ch ^ flip(i)) * 16), (int)(i * C::RPI * p.c.v_st[1] * 2), 0, 0);
        }
      }
      look_up(kb + kAttnBK);
    };
    auto put_codes = [&](auto bufc) {      // registers -> LDS, as bf16
      constexpr int buf = decltype(bufc)::value;
      if constexpr (FP8) {
        static_for<C::IPG>([&](auto ic) {
          constexpr int i = decltype(ic)::value;
          static_for<2>([&](auto uc) {
            constexpr int u = decltype(uc)::value;
            lds_write_u128_asm<i * C::RPI * C::KROW + u * 16>(put_k + buf * C::BUF, paged_codes_to_bf16(raw[2 * i][2 * u], raw[2 * i][2 * u + 1]));
            lds_write_u128_asm<i * C::RPI * C::VROW + u * 16>(put_v + buf * C::BUF, paged_codes_to_bf16(raw[2 * i + 1][2 * u], raw[2 * i + 1][2 * u + 1]));
          });
        });
        if (lane < 16) {
          lds_write_u32_asm<buf * 2 * kAttnBK * 4>(lds0 + (16 * wave + lane) * 4, raw_scale[0]);
          lds_write_u32_asm<buf * 2 * kAttnBK * 4 + kAttnBK * 4>(lds0 + (16 * wave + lane) * 4, raw_scale[1]);
        }
      }
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I3 = std::integral_constant<int, 3>;

    const int row = rw + (lane & 31), tok = row / p.G, hq = s.head * p.G + row % p.G;
    const bool valid = row < rows;
    const int seen = !valid || !p.causal ? k_end : min(max(len - nq + tok + 1, 0), len);
    if (k0 < k1) {
      look_up(k0);
      fetch(0, k0);
    }
    bf16x8_t qf[KS];
    attn_row_operand(qf, p.q + (long long)(q0 + (valid ? tok : 0)) * p.q_t + (long long)hq * p.q_h, valid, h);
    f32x16_t acc[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[db][r] = 0.f;
    float m_run = -INFINITY, m_at = 0.f, l_run = 0.f;      // the maximum in powers of two, as the sums have it; the same, but 0 for none
    bool started = false;
    if constexpr (FP8) {
      if (k0 < k1) put_codes(I0{});
      if (k0 + kAttnBK < k1) fetch(0, k0 + kAttnBK);
      wait_lgkm<0>();
    } else {
      FGRPO_WAIT_VMCNT_LGKM0(0);
    }
    wg_barrier();
    auto step = [&](auto curc, int kb) {
      constexpr int cur = decltype(curc)::value, kt = cur * C::BUF, vt = kt + C::KTILE;
      if (kb + kAttnBK < k1) {
        if constexpr (FP8) {
          put_codes(std::integral_constant<int, cur ^ 1>{});
          if (kb + 2 * kAttnBK < k1) fetch(0, kb + 2 * kAttnBK);
        } else {
          fetch(cur ^ 1, kb + kAttnBK);
        }
      }
      if (kb < w_most) {
        u32x4_t kf[2][G4];
        AttnTr vq[2][DB];
        f32x16_t s2[2];
#pragma unroll
        for (int mb = 0; mb < 2; ++mb)
#pragma unroll
          for (int r = 0; r < 16; ++r) s2[mb][r] = 0.f;
        auto req_k = [&](auto gc) {
          constexpr int g = decltype(gc)::value;
          static_for<G4>([&](auto ic) {
            constexpr int i = decltype(ic)::value, st = G4 * (g % 2) + i;
            if constexpr (FP8) kf[g % 2][i] = lds_read_u128_asm<(g / 2) * 32 * C::KROW + st * 32>(row_at + kt);
            else kf[g % 2][i] = lds_read_u128_asm<kt + (g / 2) * 32 * C::KROW>(row_at ^ (st << 5));
          });
        };
        auto req_v = [&](auto qc) {
          constexpr int q = decltype(qc)::value;
          static_for<DB>([&](auto dc) {
            constexpr int db = decltype(dc)::value;
            if constexpr (FP8) vq[q % 2][db] = paged_rd_tr<16 * q * C::VROW + db * 64, 16 * q * C::VROW + db * 64 + 8 * C::VROW>(tr_at[0] + kt);
            else vq[q % 2][db] = attn_rd_tr_asm<vt + 16 * q * C::VROW>(tr_at[0] ^ (db << 6), tr_at[1] ^ (db << 6));
          });
        };
        auto mma_k = [&](auto gc) {
          constexpr int g = decltype(gc)::value;
#pragma unroll
          for (int i = 0; i < G4; ++i) {
            attn_settle(kf[g % 2][i]);
            s2[g / 2] = attn_mfma(kf[g % 2][i], __builtin_bit_cast(u32x4_t, qf[G4 * (g % 2) + i]), s2[g / 2]);
          }
        };
        // Scales of the 32 keys of a half, of K and of V: the lane has that of score lane % 16, and a row of 16 lanes hands them to each other as operands
        uint32_t sc[4];
        if constexpr (FP8)
          static_for<4>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            sc[i] = paged_read_u32<cur * 2 * kAttnBK * 4 + i * 128>(sc_at);
          });
        auto scale_half = [&](auto mbc, auto which) {
          constexpr int mb = decltype(mbc)::value, i = 2 * decltype(which)::value + mb;
          static_for<16>([&](auto rc) {
            constexpr int r = decltype(rc)::value;
            float x = s2[mb][r] * __uint_as_float(__builtin_amdgcn_mov_dpp(sc[i], 0x150 + r, 0xf, 0xf, true));      // row_newbcast
            asm volatile("" : "+v"(x));      // here, not in the blocks that use it: the broadcast is an operand only within one
            s2[mb][r] = x;
          });
        };
        __builtin_amdgcn_s_setprio(1);      // the other work-group's wavefront on this SIMD does its softmax beside the products
        req_k(I0{});
        req_k(I1{});
        wait_lgkm<G4>();
        __builtin_amdgcn_sched_barrier(0);
        mma_k(I0{});
        __builtin_amdgcn_sched_barrier(0);
        req_k(I2{});
        wait_lgkm<G4>();
        __builtin_amdgcn_sched_barrier(0);
        mma_k(I1{});
        __builtin_amdgcn_sched_barrier(0);
        req_k(I3{});
        req_v(I0{});
        wait_lgkm<G4 + 2 * DB>();
        __builtin_amdgcn_sched_barrier(0);
        mma_k(I2{});
        __builtin_amdgcn_sched_barrier(0);
        wait_lgkm<2 * DB>();
        __builtin_amdgcn_sched_barrier(0);
        mma_k(I3{});
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (FP8) {
#pragma unroll
          for (int i = 0; i < 4; ++i) paged_settle_u32(sc[i]);      // these landed first
          scale_half(I0{}, I0{});
          scale_half(I1{}, I0{});
        }
        __builtin_amdgcn_s_setprio(0);
        float mx = -INFINITY;
#pragma unroll
        for (int mb = 0; mb < 2; ++mb) {
          if (kb + 32 * mb + 32 > w_least) {
            const int at = kb + 32 * mb + 4 * h;
#pragma unroll
            for (int r = 0; r < 16; ++r) s2[mb][r] = at + 8 * (r >> 2) + (r & 3) < seen ? s2[mb][r] : -INFINITY;
          }
        }
#pragma unroll
        for (int mb = 0; mb < 2; ++mb)
#pragma unroll
          for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s2[mb][r]);
        {
          float mlo, mhi;
          attn_halves(mx, mlo, mhi);
          mx = fmaxf(mlo, mhi);
        }
        // The sums' power of two follows the maximum once it is 2^8 behind for some row: numerators stay below 2^8, and most steps have nothing to rescale
        const float m_new = fmaxf(m_run, mx * c);
        if (__any(m_new - m_run > 8.f)) {
          const float m_use = m_new == -INFINITY ? 0.f : m_new, alpha = fast_exp2(m_run - m_use);
          m_run = m_new, m_at = m_use, l_run *= alpha;
          if (started) {
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
              for (int r = 0; r < 16; ++r) acc[db][r] *= alpha;
          }
        }
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int mb = 0; mb < 2; ++mb)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float e = fast_exp2(__builtin_fmaf(s2[mb][r], c, -m_at));
            s2[mb][r] = e;
            sum[mb] += e;
          }
        l_run += sum[0] + sum[1];
        if constexpr (FP8) {
          scale_half(I0{}, I1{});
          scale_half(I1{}, I1{});
        }
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);
        static_for<4>([&](auto qc) {
          constexpr int q = decltype(qc)::value, mb = q / 2, half = q % 2;
          if constexpr (q < 3) req_v(std::integral_constant<int, q + 1>{});
          wait_lgkm<(q < 3 ? 2 * DB : 0)>();
          __builtin_amdgcn_sched_barrier(0);
          float tmp[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) tmp[j] = s2[mb][8 * half + j];
          const u32x4_t pf = __builtin_bit_cast(u32x4_t, attn_pack8(tmp));
#pragma unroll
          for (int db = 0; db < DB; ++db) acc[db] = attn_mfma(attn_settle_tr(vq[q % 2][db]), pf, acc[db]);
          __builtin_amdgcn_sched_barrier(0);
        });
        started = true;
      }
      if constexpr (!FP8) FGRPO_WAIT_VMCNT(0);
      wait_lgkm<0>();
      wg_barrier();
    };
    for (int kb = k0; kb < k1; kb += 2 * kAttnBK) {
      step(I0{}, kb);
      if (kb + kAttnBK < k1) step(I1{}, kb + kAttnBK);
    }
    float l_lo, l_hi;
    attn_halves(l_run, l_lo, l_hi);
    const float l = l_lo + l_hi;
    int lane_e = lane;
    asm volatile("" : "+v"(lane_e));      // the row's addresses formed anew: held across the loop, they would cost registers
    const int h_e = lane_e >> 5, row_e = rw + (lane_e & 31), tok_e = q0 + row_e / p.G, hq_e = s.head * p.G + row_e % p.G;
    if (row_e >= rows) return;
    if (whole) {
      attn_store_rowmajor(acc, l > 0.f ? 1.f / l : 0.f, p.out + ((long long)tok_e * p.Hq + hq_e) * HD, h_e);
      if (p.lse && h_e == 0) p.lse[(long long)hq_e * p.c.T + tok_e] = paged_lse(m_run, l);
    } else {
      attn_store_partial(acc, sp.part + ((long long)slot * kPagedTileRB + wave) * (32 * HD), lane_e);
      if (h_e == 0) sp.ml[((long long)slot * kPagedTileRB + wave) * 32 + lane_e] = make_float2(m_run, l);
    }
  };

  PagedLanes<ROWS> lanes;
  const PagedTotal total = paged_total<ROWS>(p, lanes);
  const int4 none = make_int4(0, 0, 0, 0);
  const bool shares = total.items < sp.W || total.most * sp.W > 2 * total.weight;
  PagedShares sh = paged_shares(total, sp.W, sp.most_parts, 2.0 * kAttnBK * p.G);
  double done = 0, hi = 0;                                    // shares: this one
  const int mine = me < n / 2 ? me : n + n / 2 - 1 - me;
  int first = 0, rounds = 0, left = 0, parts = 1, turn = 0;      // whole items: the XCD's first, rounds of n, those of the last round, their parts; this work-group's turn
  PagedItem s{0, 0, 0, 0, 0};
  if (shares) {
    if (threadIdx.x == 0) sp.rec[2 * w] = none;
    if (!(w < sh.used)) return;
    done = sh.bound(w), hi = sh.bound(w + 1);
    if (!(done < hi)) return;
    s = paged_item<ROWS, false>(p, lanes, done);
  } else {                       // those that begin in this XCD's eighth of the weights
    s = paged_item<ROWS, false>(p, lanes, floor(total.weight * xcd / 8));
    first = __builtin_amdgcn_readfirstlane((int)s.index);
    const int last = xcd == 7 ? (int)total.items : (int)paged_item<ROWS, false>(p, lanes, floor(total.weight * (xcd + 1) / 8)).index;
    const int items = __builtin_amdgcn_readfirstlane(last) - first;
    rounds = items / n, left = items - rounds * n, parts = __builtin_amdgcn_readfirstlane(paged_last_parts(left, n));
    if (threadIdx.x == 0 && (me >= left || parts == 1)) sp.rec[2 * w] = none;      // record `me` of the XCD is its item `me` of the last round's
  }
  if (threadIdx.x == 0) kept[0] = sh.total, kept[1] = sh.used, kept[2] = hi, kept[3] = sh.share;      // what the walks must not carry in registers
  __syncthreads();
  for (;;) {
    double x0 = 0, x1;
    int slot = 0, part = 0;
    if (!shares) {
      if (turn < rounds) {
        const int at = first + turn * n;
        s = rounds == 1 ? paged_ranked<ROWS>(p, lanes, s, at, n, mine) : paged_item<ROWS, true>(p, lanes, at + (turn & 1 ? n - 1 - me : me));
      } else {
        const int at = first + rounds * n, i = parts == 1 && rounds <= 1 ? rounds ? n - 1 - mine : mine : (turn - rounds) * n + me;
        if (i >= left * parts || turn - rounds > (parts > 1)) break;
        s = parts == 1 && rounds <= 1 ? paged_ranked<ROWS>(p, lanes, rounds ? paged_item<ROWS, true>(p, lanes, at) : s, at, left, i) : paged_item<ROWS, true>(p, lanes, at + i / parts);
        slot = 2 * n * xcd + i, part = i % parts;
      }
    }
    if (s.b >= p.c.B) break;
    const PagedWeight wt = lanes.of(p, s.b);
    const double weight = wt.of(s.t);
    int rec = 0;               // parts, where this is an item's first of several
    if (shares) {
      x0 = done - s.at, x1 = fmin(hi - s.at, weight);
      slot = 2 * w + (x0 <= 0);
      if (x0 <= 0 && x1 < weight) rec = sh.holding(s.at + weight - 1) - w + 1;
    } else if (turn >= rounds) {
      x0 = floor(weight * part / parts), x1 = floor(weight * (part + 1) / parts);
      if (parts > 1 && part == 0) rec = -parts;
    } else {
      x1 = weight;
    }
    if (rec != 0 && threadIdx.x == 0) {
      const int at = shares ? w : n * xcd + (slot - 2 * n * xcd) / parts;
      sp.rec[2 * at] = make_int4(rec, wt.q0, s.t * ROWS, wt.nq * p.G), sp.rec[2 * at + 1] = make_int4(s.head, slot, 0, 0);
    }
    ++turn;
    if (shares && threadIdx.x == 0) kept[4 + (turn & 1)] = s.at + weight;      // two places: a walk, with its barriers, lies between a write and the next to its place
    walk(s, wt, x0, x1, slot);
    lanes.b0 = -64;            // read again, as these are
    sh.total = uniform(kept[0]), sh.used = uniform(kept[1]), hi = uniform(kept[2]), sh.share = uniform(kept[3]);
    if (shares) {
      s.at = done = uniform(kept[4 + (turn & 1)]);
      if (!(done < hi)) break;
      paged_next<ROWS>(p, lanes, s);
    }
  }
}

}  // namespace fgrpo
