// How the attention over a paged cache is dealt to work-groups (paged_rows.h, paged_tiles.h), computed by each of them from cu and lens,
// the lanes taking a sequence each: nothing is known on the host but the shapes, nothing is waited for, and a captured call follows new
// lengths.
//
// An item is a tile of ROWS rows of a sequence and K/V head with all its keys; items are in the order (sequence, head, tile).  Its weight
// is about its keys x G.  Shares: `used` work-groups take equal stretches of the sum of the weights, cut inside items where need be.
// Parts of an item leave fp32 sums in slots, which paged_merge_kernel adds up in the order of the keys (no atomics: bit-reproducible).
#pragma once
#include "paged_attn.h"

namespace fgrpo {

struct PagedSplit {
  int W;                 // work-groups of the launch, a multiple of 8
  int items;             // > 0: no more items than this, few enough for the merge to have work-groups for every unit of each: records go by item, not by work-group
  int most_parts;        // of an item
  float* part;           // [2 W][row blocks][units][64 lanes][4] sums of a part (paged_column)
  float2* ml;            // [2 W][rows] maximum (in powers of two) and sum
  int4* rec;             // [W][2] what the merge of an item needs, for each that a work-group begins and does not end: {parts (0: none; negative: their slots
                         // are neighbours), first packed row of the sequence, first row of the tile, rows of the sequence}, {head, slot of the first part}
};
// slot of part i of an item whose first is in `slot`.  Shares: work-group w has 2 w for an item that an earlier one began and 2 w + 1 for one
// that it begins and does not end.
__device__ __forceinline__ int paged_slot(int slot, int i, bool neighbours) { return neighbours ? slot + i : i ? slot - 1 + 2 * i : slot; }

// A sequence, and the weight of its tiles t (ROWS rows): whole numbers in doubles, exact below 2^53.
struct PagedWeight {
  int q0, nq, len;         // first packed row, rows, keys
  int tiles;
  double base, slope;      // w_t = base + slope (t + 1)
  __device__ __forceinline__ double of(int t) const { return base + slope * (t + 1); }
  __device__ __forceinline__ double upto(int n) const { return base * n + slope * 0.5 * n * (n + 1.0); }      // tiles 0 .. n - 1
};
// A parameter as if it were read here: what is made of it (its double, above all) is not carried in registers across the loops between its uses
__device__ __forceinline__ int at_hand(int x) {
  asm volatile("" : "+s"(x));
  return x;
}
template <int ROWS>
__device__ __forceinline__ PagedWeight paged_weight(const PagedAttn& p, int q0, int nq, int len) {
  PagedWeight w;
  w.q0 = q0, w.nq = nq, w.len = len;
  const int G = at_hand(p.G);
  w.tiles = (int)(((long long)nq * G + ROWS - 1) / ROWS);
  w.base = (double)(p.causal ? max(len - nq, 0) : len) * G + ROWS;
  w.slope = p.causal ? ROWS : 0;
  return w;
}
__device__ __forceinline__ double uniform(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)u), hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)(u >> 32));
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// inclusive sums and maxima over the lanes up to this one (values of at least 0), as wave_sum_upto moves them
template <int CTRL, int ROWS>
__device__ __forceinline__ double moved(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, false), hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <class F>
__device__ __forceinline__ double wave_upto(double x, F f) {
  x = f(x, moved<0x111, 0xf>(x)), x = f(x, moved<0x112, 0xf>(x)), x = f(x, moved<0x114, 0xf>(x)), x = f(x, moved<0x118, 0xf>(x));
  x = f(x, moved<0x142, 0xa>(x)), x = f(x, moved<0x143, 0xc>(x));
  return x;
}
__device__ __forceinline__ double wave_sums(double x) { return wave_upto(x, [](double a, double b) { return a + b; }); }
__device__ __forceinline__ double wave_most(double x) { return wave_upto(x, [](double a, double b) { return fmax(a, b); }); }
__device__ __forceinline__ double lane_of(double x, int l) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, l), hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), l);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// 64 sequences from b0 on, one a lane (behind the last: of no rows).  Read once; what a work-group needs of one of them comes out of the lane's registers.
template <int ROWS>
struct PagedLanes {
  int b0, q0, nq, len;
  __device__ __forceinline__ void load(const PagedAttn& p, int first) {
    b0 = first;
    const int b = first + (threadIdx.x & 63);
    q0 = nq = len = 0;
    if (b < p.c.B) {
      q0 = min(max(p.c.cu[b], 0), p.c.T);
      nq = min(max(p.c.cu[b + 1], q0), p.c.T) - q0;
      len = paged_len(p.c, b);
    }
  }
  __device__ __forceinline__ PagedWeight mine(const PagedAttn& p) const { return paged_weight<ROWS>(p, q0, nq, len); }
  __device__ __forceinline__ PagedWeight of(const PagedAttn& p, int b) {      // b, the same in all lanes, is below B
    if (b < b0 || b >= b0 + 64) load(p, b & ~63);
    const int l = b - b0;
    return paged_weight<ROWS>(p, __builtin_amdgcn_readlane(q0, l), __builtin_amdgcn_readlane(nq, l), __builtin_amdgcn_readlane(len, l));
  }
};
struct PagedTotal {
  double weight, most, items;      // of all items; the heaviest; how many
};
template <int ROWS>
__device__ __forceinline__ PagedTotal paged_total(const PagedAttn& p, PagedLanes<ROWS>& lanes) {      // leaves the first 64 sequences
  PagedTotal s{0, 1, 0};
  for (int b0 = (p.c.B - 1) & ~63; b0 >= 0; b0 -= 64) {
    lanes.load(p, b0);
    const PagedWeight w = lanes.mine(p);
    s.weight += lane_of(wave_sums(w.upto(w.tiles) * p.c.Hkv), 63);
    s.items += lane_of(wave_sums((double)w.tiles * p.c.Hkv), 63);
    s.most = fmax(s.most, lane_of(wave_most(w.tiles > 0 ? w.of(w.tiles - 1) : 0.0), 63));
  }
  return PagedTotal{uniform(s.weight), uniform(s.most), uniform(s.items)};
}

// No 64-bit divisions below: each is some thirty instructions in series before a work-group's first load.  Where a quotient decides on a border, all that
// matters is that everyone who asks gets the same, so an fp32 reciprocal serves; where it must be the floor, it is a guess that is put right.
__device__ __forceinline__ double about(double x, double y) { return x * (double)__builtin_amdgcn_rcpf((float)y); }

struct PagedItem {
  int b, head, t;          // b >= B: behind the last
  double at, index;        // weight and number of the items in front of it
};
// The item that holds place `x` of the weights, or of the numbers.
template <int ROWS, bool NUMBERS>
__device__ __forceinline__ PagedItem paged_item(const PagedAttn& p, PagedLanes<ROWS>& lanes, double x) {
  const int Hkv = at_hand(p.c.Hkv);
  PagedItem s{p.c.B, 0, 0, 0, 0};
  double weight = 0, number = 0;      // in front of the 64 at hand
  for (int b0 = 0; b0 < p.c.B; b0 += 64) {
    if (lanes.b0 != b0) lanes.load(p, b0);
    const PagedWeight w = lanes.mine(p);
    const double m = w.upto(w.tiles) * Hkv, n = (double)w.tiles * Hkv, upto_m = wave_sums(m), upto_n = wave_sums(n);
    const unsigned long long past = __ballot((NUMBERS ? number + upto_n : weight + upto_m) > x);      // the first lane past it holds the sequence
    if (past) {
      const int at = __ffsll(past) - 1;
      s.b = b0 + at;
      s.at = weight + lane_of(upto_m - m, at), s.index = number + lane_of(upto_n - n, at);
      break;
    }
    weight += lane_of(upto_m, 63), number += lane_of(upto_n, 63);
  }
  s.b = __builtin_amdgcn_readfirstlane(s.b);
  if (s.b >= p.c.B) return PagedItem{p.c.B, 0, 0, uniform(weight), uniform(number)};
  const PagedWeight w = lanes.of(p, s.b);
  const double one = NUMBERS ? (double)w.tiles : w.upto(w.tiles);      // of one head
  double r = x - (NUMBERS ? s.index : s.at);
  int head = (int)fmin(floor(about(r, one)), Hkv - 1.0), t = 0;
  while (head > 0 && one * head > r) --head;
  while (head + 1 < Hkv && one * (head + 1) <= r) ++head;
  r -= one * head;
  if (NUMBERS) {
    t = (int)fmin(r, w.tiles - 1.0);
  } else {
    // the last tile that begins at r or before: base n + slope n (n + 1) / 2 = r, solved in fp32 and put right
    const float m = (float)w.base + 0.5f * (float)w.slope, x = (float)r;
    t = (int)fminf(2.f * x * __builtin_amdgcn_rcpf(m + __builtin_amdgcn_sqrtf(m * m + 2.f * (float)w.slope * x)), (float)(w.tiles - 1));
    while (t > 0 && w.upto(t) > r) --t;
    while (t + 1 < w.tiles && w.upto(t + 1) <= r) ++t;
  }
  s.head = __builtin_amdgcn_readfirstlane(head), s.t = __builtin_amdgcn_readfirstlane(t);
  s.at = uniform(s.at + w.upto(w.tiles) * s.head + w.upto(s.t)), s.index = uniform(s.index + (double)w.tiles * s.head + s.t);
  return s;
}
// The next item; s.at already is where it begins.
template <int ROWS>
__device__ __forceinline__ void paged_next(const PagedAttn& p, PagedLanes<ROWS>& lanes, PagedItem& s) {
  s.index = uniform(s.index + 1);
  if (++s.t < lanes.of(p, s.b).tiles) return;
  s.t = 0;
  if (++s.head < p.c.Hkv) return;
  s.head = 0;
  do ++s.b; while (s.b < p.c.B && lanes.of(p, s.b).tiles == 0);
}

// Shares: work-group `at` of `used` has the weights [bound(at), bound(at + 1)).
struct PagedShares {
  double total, used, share;
  __device__ __forceinline__ double bound(int at) const { return uniform(at >= used ? total : floor(share * at)); }
  __device__ __forceinline__ int holding(double x) const {      // the share that holds place x
    int w = (int)fmin(floor(about(x, share)), used - 1);
    while (w > 0 && bound(w) > x) --w;
    while (w + 1 < used && bound(w + 1) <= x) ++w;
    return __builtin_amdgcn_readfirstlane(w);
  }
};
__device__ __forceinline__ PagedShares paged_shares(const PagedTotal& t, int W, int most_parts, double least) {      // least: weight that is worth a work-group
  const double some = fmin(fmin((double)W, ceil(about(t.weight, least))), floor(about(t.weight * (most_parts - 2), t.most))), used = uniform(fmax(some, 1.0));
  return PagedShares{t.weight, used, uniform(about(t.weight, used))};
}
// what a work-group walks of an item, in steps of KB keys: places x0 .. x1 of its weight
struct PagedRange {
  int k0, k1;
};
template <int KB>
__device__ __forceinline__ PagedRange paged_range(double x0, double x1, double weight, int k_end) {
  const int steps = (k_end + KB - 1) / KB;
  const double each = about((double)steps, weight);
  const int s0 = __builtin_amdgcn_readfirstlane(min((int)floor(x0 * each), steps)), s1 = x1 >= weight ? steps : __builtin_amdgcn_readfirstlane(min((int)floor(x1 * each), steps));
  return PagedRange{s0 * KB, min(k_end, s1 * KB)};
}
// Rows r0 .. of a sequence (r0 the same in all lanes): row r0 + i, i below 128, is token `token(i)`, head `head(i)` of the group.
struct PagedRowsAt {
  int tok, rem, G;
  __device__ __forceinline__ PagedRowsAt(int r0, int G_) : G(G_) { tok = __builtin_amdgcn_readfirstlane(r0 / G), rem = r0 - tok * G; }
  __device__ __forceinline__ void of(int i, int& token, int& head) const {
    const int n = rem + i < (1 << 20) ? small_div(rem + i, G) : (rem + i) / G;      // small_div reaches 2^21
    token = tok + n, head = rem + i - n * G;
  }
  __device__ __forceinline__ int token(int i) const {
    int t, h;
    of(i, t, h);
    return t;
  }
};
// the keys that rows i .. i + n - 1 behind `at` see at all, and those that all of them see; `rows` of the sequence's rows are behind `at`
struct PagedSight {
  int most, least;
};
__device__ __forceinline__ PagedSight paged_sight(const PagedAttn& p, const PagedWeight& w, const PagedRowsAt& at, int i, int n, int rows) {
  if (!p.causal) return PagedSight{w.len, w.len};
  const int first = at.token(i), last = at.token(max(min(i + n, rows) - 1, i));
  return PagedSight{min(max(w.len - w.nq + last + 1, 0), w.len), min(max(w.len - w.nq + first + 1, 0), w.len)};
}
__device__ __forceinline__ int paged_table_at(const PagedView& c, int b, int i) {      // by the scalar unit: b and i are the same in all lanes.  As it stands: not yet held inside the cache
  const auto* row = (const __attribute__((address_space(4))) int*)(c.table + (long long)b * c.table_st);
  return row[min(i, c.width - 1)];
}
__device__ __forceinline__ float paged_lse(float m, float l) { return l == 0.f ? -INFINITY : (m + __log2f(l)) * 0.6931471805599453f; }      // l NaN: so is this

// What a lane's accumulators hold.  SHAPE: rows of a block, 32 (v_mfma_f32_32x32x16_bf16) or 16 (16x16x32); the lane has row lane % SHAPE and, in unit u, four
// columns: in blocks of 32 columns value 4 g + i of block db is unit 4 db + g, in blocks of 16 value i of block u is unit u.  PAIRS (the transposing reads
// moved pairs of e4m3 codes): blocks 2 n and 2 n + 1 hold the even and the odd columns of a range.
template <int SHAPE, bool PAIRS>
__device__ __forceinline__ int paged_column(int u, int lane) {      // of the unit's first value; the others are 1 (PAIRS: 2) apart
  if constexpr (SHAPE == 32) {
    const int db = u / 4, g = u % 4, h = lane >> 5;
    return PAIRS ? 64 * (db / 2) + 16 * g + 8 * h + db % 2 : 8 * u + 4 * h;
  } else {
    return PAIRS ? 32 * (u / 2) + 8 * (lane >> 4) + u % 2 : 16 * u + 4 * (lane >> 4);
  }
}
template <int HD, bool PAIRS>
__device__ __forceinline__ void paged_store_row(const f32x16_t (&acc)[HD / 32], float mul, bf16_t* row, int h) {
  if constexpr (!PAIRS) {
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

struct PagedSum {
  float m, l;              // maximum (in powers of two) and sum
  float4 o;
};
__device__ __forceinline__ PagedSum paged_add(const PagedSum& a, const PagedSum& b) {
  const float m = fmaxf(a.m, b.m), m_use = m == -INFINITY ? 0.f : m, x = fast_exp2(a.m - m_use), y = fast_exp2(b.m - m_use);
  return PagedSum{m, a.l * x + b.l * y, make_float4(a.o.x * x + b.o.x * y, a.o.y * x + b.o.y * y, a.o.z * x + b.o.z * y, a.o.w * x + b.o.w * y)};
}
template <int SHAPE, bool PAIRS>
__device__ __forceinline__ void paged_store_unit(bf16_t* row, int unit, int lane, const float4& o, float inv) {
  bf16_t* dst = row + paged_column<SHAPE, PAIRS>(unit, lane);
  if constexpr (PAIRS) {
    dst[0] = f32_to_bf16_rn(o.x * inv), dst[2] = f32_to_bf16_rn(o.y * inv), dst[4] = f32_to_bf16_rn(o.z * inv), dst[6] = f32_to_bf16_rn(o.w * inv);
  } else {
    uint2 x;
    x.x = pack_bf16x2(o.x * inv, o.y * inv), x.y = pack_bf16x2(o.z * inv, o.w * inv);
    *(uint2*)dst = x;
  }
}

// The same for few items of perhaps many parts: work-group (item, unit of a block of rows), its wavefronts taking parts w, w + 4 ..
template <int HD, bool PAIRS, int SHAPE, int RB>
static __global__ __launch_bounds__(256) void paged_merge_items_kernel(PagedAttn p, PagedSplit sp) {
  constexpr int UNITS = HD / (SHAPE == 32 ? 8 : 16), WIDE = 8;
  __shared__ PagedSum sh[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rb = blockIdx.y / UNITS, unit = blockIdx.y % UNITS;
  const int4 rec = sp.rec[2 * blockIdx.x], place = sp.rec[2 * blockIdx.x + 1];
  if (rec.x == 0) return;
  const bool neighbours = rec.x < 0;
  const int np = neighbours ? -rec.x : rec.x, row = rec.z + SHAPE * rb + lane % SHAPE;
  const float* part = sp.part + (long long)rb * (SHAPE * HD) + (64 * unit + lane) * 4;
  const float2* ml = sp.ml + rb * SHAPE + lane % SHAPE;
  PagedSum sum{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
  if (row < rec.w)
    for (int i0 = wave; i0 < np; i0 += 4 * WIDE) {
      PagedSum x[WIDE];
#pragma unroll
      for (int i = 0; i < WIDE; ++i) {
        const long long slot = (long long)RB * min(paged_slot(place.y, min(i0 + 4 * i, np - 1), neighbours), 2 * sp.W - 1);
        const float2 y = ml[slot * SHAPE];
        x[i] = PagedSum{y.x, y.y, *(const float4*)(part + slot * (SHAPE * HD))};
      }
#pragma unroll
      for (int i = 0; i < WIDE; ++i)
        if (i0 + 4 * i < np) sum = paged_add(sum, x[i]);
    }
  sh[wave][lane] = sum;
  __syncthreads();
  if (wave != 0 || row >= rec.w) return;
  for (int i = 1; i < 4; ++i) sum = paged_add(sum, sh[i][lane]);
  const int tok = rec.y + row / p.G, hq = place.x * p.G + row % p.G;
  paged_store_unit<SHAPE, PAIRS>(p.out + ((long long)tok * p.Hq + hq) * HD, unit, lane, sum.o, sum.l > 0.f ? 1.f / sum.l : 0.f);
  if (p.lse && unit == 0 && lane < SHAPE) p.lse[(long long)hq * p.c.T + tok] = paged_lse(sum.m, sum.l);
}

// (Both are a launch of 3 to 5 us; 500 parts of 128 rows, 64 KiB each, take 9.)
// Adds up the parts of the item of record blockIdx.x in the order of the keys: work-group y takes block y of SHAPE rows, wavefront w the units w, w + 4 ..
// of their columns.  RB: blocks of a tile.
template <int HD, bool PAIRS, int SHAPE, int RB>
static __global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttn p, PagedSplit sp) {
  constexpr int NU = HD / (SHAPE == 32 ? 8 : 16) / 4, WIDE = 16 / NU < 8 ? 16 / NU : 8;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rb = blockIdx.y;
  const int4 rec = sp.rec[2 * blockIdx.x], place = sp.rec[2 * blockIdx.x + 1];
  if (rec.x == 0) return;
  const bool neighbours = rec.x < 0;
  const int np = neighbours ? -rec.x : rec.x, row = rec.z + SHAPE * rb + lane % SHAPE;
  if (row >= rec.w) return;
  const int tok = rec.y + row / p.G, hq = place.x * p.G + row % p.G;
  PagedSum sum[NU];
#pragma unroll
  for (int c = 0; c < NU; ++c) sum[c] = PagedSum{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
  const float* part = sp.part + (long long)rb * (SHAPE * HD) + (64 * wave + lane) * 4;
  const float2* ml = sp.ml + rb * SHAPE + lane % SHAPE;
  for (int i0 = 0; i0 < np; i0 += WIDE) {
    float2 x[WIDE];
    float4 y[WIDE][NU];
#pragma unroll
    for (int i = 0; i < WIDE; ++i) {
      const long long slot = (long long)RB * min(paged_slot(place.y, min(i0 + i, np - 1), neighbours), 2 * sp.W - 1);
      x[i] = ml[slot * SHAPE];
#pragma unroll
      for (int c = 0; c < NU; ++c) y[i][c] = *(const float4*)(part + slot * (SHAPE * HD) + 1024 * c);
    }
#pragma unroll
    for (int i = 0; i < WIDE; ++i)
      if (i0 + i < np)
#pragma unroll
        for (int c = 0; c < NU; ++c) sum[c] = paged_add(sum[c], PagedSum{x[i].x, x[i].y, y[i][c]});
  }
#pragma unroll
  for (int c = 0; c < NU; ++c)
    paged_store_unit<SHAPE, PAIRS>(p.out + ((long long)tok * p.Hq + hq) * HD, wave + 4 * c, lane, sum[c].o, sum[c].l > 0.f ? 1.f / sum[c].l : 0.f);
  if (p.lse && threadIdx.x < SHAPE) p.lse[(long long)hq * p.c.T + tok] = paged_lse(sum[0].m, sum[0].l);
}

}  // namespace fgrpo
