// Attention over a paged cache for few rows a sequence (single tokens, drafts): all of its time is reading the cache, so the work is
// dealt out by what is read.  (What is computed: paged_attn.h.)
//
// A work-group is one wavefront.  It owns 32 RB rows of a sequence and K/V head (RB = 1 or 2; G rows a token) and a stretch of the
// keys, which it walks in steps of KB = 32 or 64: a step's K and V travel global -> LDS directly, a step ahead, 16 KiB in flight
// behind 16 KiB in use, four to five wavefronts a CU.  No barriers.  The pages of a step are looked up by the scalar unit, a step
// ahead of their loads: 16 tokens that start at a multiple of 16 lie in one page, so each such group is one buffer descriptor, whose
// length ends with the sequence - rows behind it arrive as zeros, whatever lies there.
//
// Dealing out.  Every (sequence, head, tile of rows) has a weight, about its keys x G; W wavefronts take equal shares of the sum, one
// behind the other, cut inside items where need be.  All of it is computed by each wavefront from cu and lens (the lanes take a
// sequence each): nothing is known on the host but the shapes, nothing is waited for, and a captured call follows new lengths.
// An item that one wavefront walks whole is finished by it; parts of others leave fp32 sums, which paged_merge_kernel adds up
// in the order of the keys (no atomics: bit-reproducible).
#pragma once
#include "paged_attn.h"

namespace fgrpo {

constexpr int kPagedMaxParts = 128;      // of an item: what the merge reads one behind the other

struct PagedSplit {
  int W;                 // wavefronts of the launch, a multiple of 8
  float* part;           // [2 W][RB][32 x HD]
  float2* ml;            // [2 W][RB][32] maximum (in powers of two) and sum
  int4* rec;             // [2 W] {sequence + 1, tile, head, ends the item}; 0: none.  2 w: an item begun by an earlier wavefront, 2 w + 1: one begun here
};

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

// ---- dealing out ------------------------------------------------------------------------------------------------------
// Weight of tile t (ROWS rows) of a sequence: whole numbers in doubles, exact below 2^53.
struct PagedWeight {
  double base, slope;      // w_t = base + slope (t + 1)
  int tiles, len, nq;
  __device__ __forceinline__ double of(int t) const { return base + slope * (t + 1); }
  __device__ __forceinline__ double upto(int n) const { return base * n + slope * 0.5 * n * (n + 1.0); }      // tiles 0 .. n - 1
};
template <int ROWS>
__device__ __forceinline__ PagedWeight paged_weight(const PagedAttn& p, int b) {
  PagedWeight w;
  const int lo = min(max(p.c.cu[b], 0), p.c.T);
  w.nq = min(max(p.c.cu[b + 1], lo), p.c.T) - lo;
  w.len = paged_len(p.c, b);
  w.tiles = (int)(((long long)w.nq * p.G + ROWS - 1) / ROWS);
  w.base = (double)(p.causal ? max(w.len - w.nq, 0) : w.len) * p.G + ROWS;
  w.slope = p.causal ? ROWS : 0;
  return w;
}
struct PagedShare {
  double lo, hi;           // this wavefront's stretch of the weights; lo >= hi: none
  double at;               // where item (b, head, t) begins
  int b, head, t;
};
__device__ __forceinline__ double uniform(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)u), hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)(u >> 32));
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// The share of wavefront `at` of W.  steps_weight: weight of a step, min_steps: fewer are not worth a wavefront.
template <int ROWS>
__device__ __forceinline__ PagedShare paged_share(const PagedAttn& p, int at, int W, double step_weight) {
  const int lane = threadIdx.x & 63;
  double total = 0, most = 1;
  for (int b = lane; b < p.c.B; b += 64) {
    const PagedWeight w = paged_weight<ROWS>(p, b);
    if (w.tiles > 0) total += w.upto(w.tiles) * p.c.Hkv, most = fmax(most, w.of(w.tiles - 1));
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) total += __shfl_xor(total, d, 64), most = fmax(most, __shfl_xor(most, d, 64));
  total = uniform(total), most = uniform(most);
  const double used = fmax(fmin(fmin((double)W, ceil(total / step_weight)), floor(total * (kPagedMaxParts - 2) / most)), 1.0);
  PagedShare s{0, 0, 0, 0, 0, 0};
  if (at >= used) return s;
  s.lo = floor(total * at / used), s.hi = floor(total * (at + 1) / used);
  if (!(s.lo < s.hi)) return s;
  double before = 0;
  for (int b0 = 0; b0 < p.c.B; b0 += 64) {
    const int b = b0 + lane;
    double m = 0;
    if (b < p.c.B) {
      const PagedWeight w = paged_weight<ROWS>(p, b);
      m = w.upto(w.tiles) * p.c.Hkv;
    }
    double upto = m;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double y = __shfl_up(upto, d, 64);
      if (lane >= d) upto += y;
    }
    const unsigned long long past = __ballot(before + upto > s.lo);      // the first lane past it holds the sequence
    if (past) {
      const int l = __ffsll(past) - 1;
      s.b = b0 + l;
      s.at = uniform(before + __shfl(upto - m, l, 64));
      break;
    }
    before += __shfl(upto, 63, 64);
  }
  s.b = __builtin_amdgcn_readfirstlane(s.b);
  const PagedWeight w = paged_weight<ROWS>(p, s.b);
  const double one = w.upto(w.tiles);
  double r = s.lo - s.at;
  int head = (int)fmin(floor(r / one), p.c.Hkv - 1.0);
  if (head > 0 && one * head > r) --head;
  if (head + 1 < p.c.Hkv && one * (head + 1) <= r) ++head;
  r -= one * head;
  int t = 0;
  for (int n = w.tiles - 1, low = 0; low <= n;) {      // the last tile that begins at r or before
    const int mid = (low + n) / 2;
    if (w.upto(mid) <= r) t = mid, low = mid + 1;
    else n = mid - 1;
  }
  s.head = __builtin_amdgcn_readfirstlane(head), s.t = __builtin_amdgcn_readfirstlane(t);
  s.at = uniform(s.at + one * s.head + w.upto(s.t));
  return s;
}

// ---- the kernel ---------------------------------------------------------------------------------------------------------
template <int HD, bool FP8>
struct PagedRows {
  static constexpr int ES = FP8 ? 1 : 2, RBY = HD * ES, NB = RBY == 256 ? 1 : 2, KB = 32 * NB, NG = KB / 16;
  static constexpr int CPR = RBY / 16, RPI = 1024 / RBY, IPG = 16 / RPI;
  static constexpr int TILE = KB * RBY, BUF = 2 * TILE, SCALES = FP8 ? 4 * KB * 4 : 0, LDS = 2 * BUF + SCALES;
  static constexpr int LOADS = 2 * NG * IPG + (FP8 ? 2 : 0);      // vector-memory instructions of a step
};

__device__ __forceinline__ int paged_table_at(const PagedView& c, int b, int i) {      // by the scalar unit: b and i are the same in all lanes.  As it stands: not yet held inside the cache
  const auto* row = (const __attribute__((address_space(4))) int*)(c.table + (long long)b * c.table_st);
  return row[min(i, c.width - 1)];
}

// eight codes of two registers of the transposing reads, one of two columns each -> bf16
__device__ __forceinline__ u32x4_t paged_codes_to_bf16(uint32_t a, uint32_t b) {      // codes 0 .. 3 and 4 .. 7
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  auto cvt = [](uint32_t x, auto hi) { return __builtin_bit_cast(uint32_t, (b2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, decltype(hi)::value)); };
  return u32x4_t{cvt(a, std::false_type{}), cvt(a, std::true_type{}), cvt(b, std::false_type{}), cvt(b, std::true_type{})};
}

// Columns that a lane's accumulator values are.  bf16: block db, value r is column 32 db + 8 (r / 4) + 4 h + r % 4.  e4m3: the transposing
// reads move pairs of codes, so blocks 2 n and 2 n + 1 hold the even and the odd columns of 64: value r is column
// 64 n + 2 (8 (r / 4) + 4 h + r % 4) + (block % 2), and the values of both blocks with r / 4 = g are eight neighbours.
template <int HD, bool FP8>
__device__ __forceinline__ void paged_store_row(const f32x16_t (&acc)[HD / 32], float mul, bf16_t* row, int h) {
  if constexpr (!FP8) {
    attn_store_rowmajor(acc, mul, row, h);
  } else {
#pragma unroll
    for (int n = 0; n < HD / 64; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        u32x4_t x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = pack_bf16x2(acc[2 * n][4 * g + i] * mul, acc[2 * n + 1][4 * g + i] * mul);
        *(u32x4_t*)(row + 64 * n + 16 * g + 8 * h) = x;
      }
  }
}

template <int HD, bool FP8, int RB>
static __global__ __launch_bounds__(64) void paged_rows_kernel(PagedAttn p, PagedSplit sp) {
  using C = PagedRows<HD, FP8>;
  constexpr int KS = HD / 16, DB = HD / 32, VB = C::RBY / 64, ROWS = 32 * RB;
  __shared__ __attribute__((aligned(16))) char smem[C::LDS];
  const uint32_t lds0 = lds_addr(smem);
  const int lane = threadIdx.x, h = lane >> 5;
  const int w = (blockIdx.x & 7) * (sp.W >> 3) + (blockIdx.x >> 3);      // neighbours in the order share an XCD's L2
  PagedShare s = paged_share<ROWS>(p, w, sp.W, 2.0 * C::KB * p.G);
  int4 rec_in = make_int4(0, 0, 0, 0), rec_out = rec_in;
  const PagedLane<C::RBY> L = paged_lane<C::RBY>(lane, lds0);
  uint32_t voff_k[C::IPG], voff_v[C::IPG];
#pragma unroll
  for (int i = 0; i < C::IPG; ++i) {
    const int row = i * C::RPI + lane / C::CPR, chunk = (lane % C::CPR) ^ paged_swz<C::RBY>(row);
    voff_k[i] = (uint32_t)(row * p.c.k_st[1] * C::ES) + chunk * 16;
    voff_v[i] = (uint32_t)(row * p.c.v_st[1] * C::ES) + chunk * 16;
  }
  const float c = p.scale * kLog2e;
  double done = s.lo;
  while (done < s.hi) {
    const PagedWeight wt = paged_weight<ROWS>(p, s.b);
    const double weight = wt.of(s.t), x0 = done - s.at, x1 = fmin(s.hi - s.at, weight);
    const int q0 = __builtin_amdgcn_readfirstlane(min(max(p.c.cu[s.b], 0), p.c.T)), nq = __builtin_amdgcn_readfirstlane(wt.nq), len = __builtin_amdgcn_readfirstlane(wt.len);
    const int rows = nq * p.G, r0 = s.t * ROWS;
    const int first_tok = r0 / p.G, last_tok = (min(r0 + ROWS, rows) - 1) / p.G;
    const int k_end = p.causal ? min(max(len - nq + last_tok + 1, 0), len) : len;
    const int all_see = p.causal ? min(max(len - nq + first_tok + 1, 0), len) : len;      // keys that every row sees
    const int steps = (k_end + C::KB - 1) / C::KB;
    const int k0 = __builtin_amdgcn_readfirstlane((int)floor(x0 * steps / weight)) * C::KB;
    const int k1 = min(k_end, __builtin_amdgcn_readfirstlane((int)floor(x1 * steps / weight)) * C::KB);
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
          if (p.lse && h == 0) p.lse[(long long)hq * p.c.T + tok] = l > 0.f ? (m_run[rb] + __log2f(l)) * 0.6931471805599453f : -INFINITY;
        }
      } else if (valid[rb]) {
        attn_store_partial(acc[rb], sp.part + ((long long)slot * RB + rb) * (32 * HD), lane);
        if (h == 0) sp.ml[((long long)slot * RB + rb) * 32 + lane] = make_float2(m_run[rb], l);
      }
    }
    if (begins && !ends) rec_out = make_int4(s.b + 1, s.t, s.head, 0);
    else if (!begins) rec_in = make_int4(s.b + 1, s.t, s.head, ends);
    // the next item
    done = s.at = uniform(s.at + weight);
    if (done >= s.hi) break;
    if (++s.t >= wt.tiles) {
      s.t = 0;
      if (++s.head >= p.c.Hkv) {
        s.head = 0;
        do ++s.b; while (s.b < p.c.B && paged_weight<ROWS>(p, s.b).tiles == 0);
        s.b = __builtin_amdgcn_readfirstlane(s.b);
        if (s.b >= p.c.B) break;
      }
    }
  }
  if (lane == 0) sp.rec[2 * w] = rec_in, sp.rec[2 * w + 1] = rec_out;
}

// Adds up the parts of the item that wavefront blockIdx.x began and did not end, in the order of the keys: work-group y takes 32 rows and 32
// accumulator columns of them, a thread four columns of a row.
template <int HD, bool FP8, int RB>
static __global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttn p, PagedSplit sp) {
  constexpr int DB = HD / 32, ROWS = 32 * RB, WIDE = 4;
  const int w = blockIdx.x, lane = threadIdx.x & 63, h = lane >> 5;
  const int4 head = sp.rec[2 * w + 1];
  if (head.x == 0) return;
  int np = 1;              // parts: this one, and slots 2 (w + 1), 2 (w + 2) .. up to the one that ends the item
  for (int i0 = w + 1; i0 < sp.W && np < sp.W; i0 += 64) {
    const bool ends = i0 + lane < sp.W && sp.rec[2 * (i0 + lane)].w != 0;
    const unsigned long long m = __ballot(ends);
    np += m ? __ffsll(m) : min(64, sp.W - i0);
    if (m) break;
  }
  const int b = min(max(head.x - 1, 0), p.c.B - 1), rb = blockIdx.y / DB, db = blockIdx.y % DB, g = threadIdx.x >> 6;
  const int q0 = min(max(p.c.cu[b], 0), p.c.T), nq = min(max(p.c.cu[b + 1], q0), p.c.T) - q0;
  const int row = head.y * ROWS + 32 * rb + (lane & 31);
  if (row >= nq * p.G) return;
  const int tok = q0 + row / p.G, hq = head.z * p.G + row % p.G;
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  const float* part = sp.part + (long long)rb * (32 * HD) + (64 * (4 * db + g) + lane) * 4;
  const float2* ml = sp.ml + rb * 32 + (lane & 31);
  for (int i0 = 0; i0 < np; i0 += WIDE) {
    float2 x[WIDE];
    float4 y[WIDE];
#pragma unroll
    for (int i = 0; i < WIDE; ++i) {
      const int at = min(i0 + i, np - 1);
      const long long slot = (long long)RB * (at ? 2 * (w + at) : 2 * w + 1);
      x[i] = ml[slot * 32], y[i] = *(const float4*)(part + slot * (32 * HD));
    }
#pragma unroll
    for (int i = 0; i < WIDE; ++i) {
      if (i0 + i >= np) break;
      const float m_new = fmaxf(m, x[i].x), m_use = m_new == -INFINITY ? 0.f : m_new, a = fast_exp2(m - m_use), e = fast_exp2(x[i].x - m_use);
      l = l * a + x[i].y * e;
      o = make_float4(o.x * a + y[i].x * e, o.y * a + y[i].y * e, o.z * a + y[i].z * e, o.w * a + y[i].w * e);
      m = m_new;
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  bf16_t* dst = p.out + ((long long)tok * p.Hq + hq) * HD;
  if constexpr (FP8) {
    const int col = 64 * (db / 2) + 2 * (8 * g + 4 * h) + db % 2;
    dst[col] = f32_to_bf16_rn(o.x * inv), dst[col + 2] = f32_to_bf16_rn(o.y * inv), dst[col + 4] = f32_to_bf16_rn(o.z * inv), dst[col + 6] = f32_to_bf16_rn(o.w * inv);
  } else {
    uint2 x;
    x.x = pack_bf16x2(o.x * inv, o.y * inv), x.y = pack_bf16x2(o.z * inv, o.w * inv);
    *(uint2*)(dst + 32 * db + 8 * g + 4 * h) = x;
  }
  if (p.lse && db == 0 && g == 0 && h == 0) p.lse[(long long)hq * p.c.T + tok] = l > 0.f ? (m + __log2f(l)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace fgrpo
