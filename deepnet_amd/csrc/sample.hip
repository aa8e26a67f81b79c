// Tokens drawn from columns of logits by given random numbers, with temperature, top-k, min-p and top-p (no counterpart in cudamat.cu; beside
// perturb_prob / choose_max, which draw from the whole distribution by a random number an entry).
#include "columns.h"
#include "tokens.h"
#include "wide_math.h"
#include <type_traits>

struct SampleArgs {
  const float *mat, *uniform, *temperature, *top_k, *top_p, *min_p;
  float *tokens, *logp;
  float all_temperature, all_top_k, all_top_p, all_min_p;
  int h, w;
  int shift;                       // weights are multiples of 2^-shift
};

// The weight e^((x - m) / T) of an entry, x <= m, as a whole multiple of 2^-shift: the same one wherever it is computed, and sums of
// them do not depend on their order, so a border between two sums is one border.  c = 256 log2(e) / T.  (x - m) c = n + f, n whole and |f| <= 1/2: 2^(n / 256) from
// a table of 256 steps (times 2^shift) and the whole part, 2^(f / 256) by its Taylor sum (remainder (ln 2 / 512)^5 / 5! < 4e-17).  Adding 2^52 leaves the rounded
// whole number in the low bits.  Entries that have none (too far from m) are not asked for.
// 2048 steps and one term less take as long, and 1.2 us more to fill the table.
#define SAMPLE_STEPS 256
__device__ __forceinline__ unsigned long long sample_weight(float x, float m, double c, const double* table) {
  const double d = (double)x - (double)m, b = fma(d, c, 6755399441055744.0), f = fma(d, c, 6755399441055744.0 - b);      // (3 * 2^51: the low bits are n)
  const int n = (int)__double_as_longlong(b);
  double p = 2.239395190875157e-12;            // (ln2 / 256)^4 / 4!
  p = fma(p, f, 3.308302680541371e-09);
  p = fma(p, f, 3.665565596910106e-06);
  p = fma(p, f, 0.0027076061740622863);
  const double step = table[n & (SAMPLE_STEPS - 1)], s = __hiloint2double(__double2hiint(step) + ((n >> 8) << 20), __double2loint(step));
  const double w = fma(s * f, p, s) + 4503599627370496.0;
  return (unsigned long long)__double_as_longlong(w) & 0xfffffffffffffull;
}
// 2^(n / 256), by its Taylor sum from the nearer end (remainder (ln 2 / 2)^13 / 13! < 2e-16)
__device__ __forceinline__ double sample_step(int n) {
  const double f = n <= 128 ? n / 256.0 : n / 256.0 - 1.0;
  double p = 2.5678435993488196e-11;    // ln2^12 / 12!
  p = fma(p, f, 4.44553827187081e-10);
  p = fma(p, f, 7.054911620801121e-09);
  p = fma(p, f, 1.0178086009239696e-07);
  p = fma(p, f, 1.3215486790144305e-06);
  p = fma(p, f, 1.5252733804059838e-05);
  p = fma(p, f, 0.00015403530393381606);
  p = fma(p, f, 0.0013333558146428441);
  p = fma(p, f, 0.009618129107628477);
  p = fma(p, f, 0.055504108664821576);
  p = fma(p, f, 0.2402265069591007);
  p = fma(p, f, 0.6931471805599453);
  p = fma(p, f, 1.0);
  return n <= 128 ? p : 2.0 * p;
}

// What a column is drawn with.
struct SampleRule {
  bool greedy;
  double c, top_p;                 // top_p: >= 1 for no limit
  int k;                           // h for no limit
  unsigned long long least;        // weight that min_p asks for
  float u;
};
__device__ __forceinline__ SampleRule sample_rule(const SampleArgs& a, int col) {
  SampleRule r;
  const float t = a.temperature ? a.temperature[col] : a.all_temperature, k = a.top_k ? a.top_k[col] : a.all_top_k;
  const float p = a.top_p ? a.top_p[col] : a.all_top_p, q = a.min_p ? a.min_p[col] : a.all_min_p;
  r.greedy = !(t > 0.f);
  r.c = 1.4426950408889634 / (double)t;
  r.k = k >= 1.f && k < (float)a.h ? (int)k : a.h;
  r.top_p = p < 1.f ? (double)p : 1.0;
  r.least = q > 0.f ? (unsigned long long)ceil(ldexp((double)fminf(q, 1.f), a.shift)) : 0;
  const float u = a.uniform[col];
  r.u = u > 0.f ? fminf(u, 1.f) : 0.f;
  return r;
}
// part * total as a whole number (total < 2^63)
__device__ __forceinline__ unsigned long long sample_part(double part, unsigned long long total) { return (unsigned long long)(part * (double)total); }
__device__ __forceinline__ unsigned long long sample_part_up(double part, unsigned long long total) { return (unsigned long long)ceil(part * (double)total); }

typedef unsigned long long u64;

// Sums of 64-bit numbers over the lanes before and including this one, by the cross-lane paths of the vector unit.
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 lane_add_u64(u64 v) {
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)(unsigned)v, CTRL, ROWS, 0xf, false), hi = __builtin_amdgcn_update_dpp(0, (int)(unsigned)(v >> 32), CTRL, ROWS, 0xf, false);
  return v + ((u64)hi << 32 | lo);
}
__device__ __forceinline__ u64 wave_scan_u64(u64 v) {
  v = lane_add_u64<0x111, 0xf>(v);           // rows of 16: one, two, four, eight lanes back
  v = lane_add_u64<0x112, 0xf>(v);
  v = lane_add_u64<0x114, 0xf>(v);
  v = lane_add_u64<0x118, 0xf>(v);
  v = lane_add_u64<0x142, 0xa>(v);           // the row before
  return lane_add_u64<0x143, 0xc>(v);        // the two rows before
}
__device__ __forceinline__ u64 lane_u64(u64 v, int lane) {
  return (u64)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)(v >> 32), lane) << 32 | (unsigned)__builtin_amdgcn_readlane((int)(unsigned)v, lane);
}

#define SAMPLE_SHORT 256           // candidates that are compared with each other
template <int LANES>
struct SampleShared {
  static constexpr int WAVES = LANES / 64, BINS = LANES, LIST = 4096;       // LIST: candidates
  double table[SAMPLE_STEPS];
  u64 few[2 * SAMPLE_SHORT];       // keys with their weights
  u64 list[LIST];                  // keys of candidates
  u64 masses[BINS];
  int counts[BINS];
  u64 wave_sum[WAVES];
  float wave_max[WAVES], wave_min[WAVES];
  int wave_bad[WAVES], listed, place, drawn;
  unsigned key_max, key_min;
  u64 border, base, before, total;
};

// Sums up to a lane (itself included) over a workgroup, and the sum of all.  Every lane calls it; what it uses is free again behind the next barrier.
template <int LANES>
__device__ __forceinline__ u64 sample_scan(u64 v, u64* wave_sum, u64* all) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  v = wave_scan_u64(v);
  __syncthreads();
  if (lane == 63) wave_sum[wv] = v;
  __syncthreads();
  u64 sum = 0;
#pragma unroll
  for (int k = 0; k < LANES / 64; ++k) { if (k == wv) v += sum; sum += wave_sum[k]; }
  *all = sum;
  return v;
}

// The entries of a column: a wavefront has a stretch of it, 256 rows a slab, four of them a lane; in registers (NV slabs) or, of columns that those do not hold
// (NV = 0), from memory, where eight slabs are on their way at once.  f(x, row, slab) for a lane's four, rows behind the column being -infinity.
template <int LANES, int NV>
struct SampleColumn {
  static constexpr int AHEAD = 8;
  const float* c;
  int h, from, slabs;              // behind the last row; the stretch's first row of this lane, slabs of a stretch
  float x[NV ? NV : 1][4];
  __device__ __forceinline__ void fetch(float (&v)[4], int row) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = -INFINITY;
    if (row + 4 <= h) col_load<false>(v, c + row);
    else {
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (row + e < h) v[e] = c[row + e];
    }
  }
  __device__ __forceinline__ void init(const float* column, int end, int first = 0) {
    c = column; h = end;
    slabs = (h - first + 4 * LANES - 1) / (4 * LANES);
    from = first + (int)(threadIdx.x >> 6) * slabs * 256 + 4 * (int)(threadIdx.x & 63);
    if (NV) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (k < slabs) fetch(x[k], from + 256 * k);
    }
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    if (NV) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (k < slabs) {
          float v[4];
          int row = from + 256 * k;
          // (what one pass makes of an entry or a row is not kept in registers for the next)
#pragma unroll
          for (int e = 0; e < 4; ++e) { v[e] = x[k][e]; asm volatile("" : "+v"(v[e])); }
          asm volatile("" : "+v"(row));
          f(v, row, k);
          __builtin_amdgcn_sched_barrier(0);
        }
    } else {
      for (int k = 0; k < slabs; k += AHEAD) {
        float v[AHEAD][4];
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) fetch(v[q], from + 256 * (k + q));
#pragma unroll
        for (int q = 0; q < AHEAD; ++q)
          if (k + q < slabs) { f(v[q], from + 256 * (k + q), k + q); __builtin_amdgcn_sched_barrier(0); }
      }
    }
  }
};

// Kept entries: those from the border on in the order of keys whose weight reaches `least`.
struct SampleKept {
  float m, far, x, above;          // the greatest entry; entries further from it than `far` have no weight; the last kept value (and the next greater),
  int row;                         // and of entries of that value the last kept row
  double c;                        // 256 log2(e) / temperature
  bool plain, bordered;            // plain: m - far is a number far enough from m
  u64 least;
  const double* table;
  __device__ __forceinline__ bool near(float v) const { return v > -INFINITY && m - v <= far; }
  __device__ __forceinline__ bool in(float v, int i) const { return near(v) && (v > x || (v == x && i <= row)); }
  __device__ __forceinline__ u64 weight(float v) const {
    const u64 w = sample_weight(v, m, c, table);
    return w >= least ? w : 0;
  }
  // of four rows; those of a wavefront without a kept entry are not computed
  __device__ __forceinline__ void weights(u64 (&w)[4], const float (&v)[4], int i) const {
    const float end = m - far;     // (entries from there on have no weight, nor has this)
    if (plain && !bordered && least == 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = sample_weight(fmaxf(v[e], end), m, c, table);
    } else if (plain) {
      // (rows up to the last kept one keep its value, those behind it the next greater)
      const float here = i <= row ? x : above;
      if (!__any(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) >= here || (i <= row && row < i + 3))) {
        w[0] = w[1] = w[2] = w[3] = 0;
        return;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = sample_weight(v[e] >= (e && i + e > row ? above : here) ? v[e] : end, m, c, table);
      if (least) {
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = w[e] >= least ? w[e] : 0;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = in(v[e], i + e) ? weight(v[e]) : 0;
    }
  }
  __device__ __forceinline__ void from(u64 border) {
    x = lp_key_value(border);
    row = lp_key_index(border);
    above = lp_key_value(((border >> 32) + 1) << 32);
    bordered = true;
  }
};
// What may be kept before any border is known.
__device__ __forceinline__ SampleKept sample_kept(const SampleArgs& a, const SampleRule& rule, float most, const double* table) {
  SampleKept kept;
  kept.m = most; kept.row = 0; kept.c = rule.c * 256.0; kept.least = rule.least; kept.table = table;
  kept.far = (float)((a.shift + 1.5) / rule.c);            // (2^-(shift + 1) is nothing; half an octave for the rounding of the distance)
  kept.plain = most - kept.far > -INFINITY && ((double)most - (double)(most - kept.far)) * rule.c >= a.shift + 1.0;
  kept.bordered = false;
  kept.x = kept.above = kept.plain ? most - kept.far : -INFINITY;
  return kept;
}
__device__ __forceinline__ void sample_out(const SampleArgs& a, int col, const SampleKept& kept, float v, int row, u64 total) {
  a.tokens[col] = (float)row;
  if (a.logp) a.logp[col] = (float)(((double)v - (double)kept.m) * (kept.c * (0.6931471805599453 / 256.0)) - dn_log_wide_pos(ldexp((double)total, -a.shift)));
}
__device__ __forceinline__ u64 sample_aim(const SampleRule& rule, u64 total) {
  const u64 at = sample_part((double)rule.u, total);
  return at < total ? at : total - 1;
}
// The weights that top_p asks for.
__device__ __forceinline__ u64 sample_ask(const SampleRule& rule, u64 total) {
  const u64 part = rule.top_p < 1.0 ? (rule.top_p > 0.0 ? sample_part_up(rule.top_p, total) : 0) : total;
  return part > 1 ? part : 1;
}

// The greatest border that leaves enough: bit by bit, a pass over the column each.  For more than LIST best ones, and for columns whose border lies among more than
// SAMPLE_SHORT entries that are alike or nearly so.  128003 x 64 by 6000 best 1390 us (by 4000 57), by top-p 0.9 of logits in steps of 1/64 2720 (54 of others): slower than
// elementary operations, and right.
template <int LANES, int NV, typename F>
__device__ __forceinline__ u64 sample_bisect(const SampleColumn<LANES, NV>& column, const SampleKept& kept, SampleShared<LANES>& sh, u64 enough, F value) {
  u64 border = 0;
  for (int bit = 63; bit >= 0; --bit) {
    const u64 trial = border | 1ull << bit;
    u64 sum = 0, all;
    column.each([&](const float (&v)[4], int row, int) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (kept.in(v[e], row + e) && lp_key(v[e], row + e) >= trial) sum += value(v[e]);
    });
    sample_scan<LANES>(sum, sh.wave_sum, &all);
    if (all >= enough) border = trial;
  }
  return border;
}

// Sums over the LANES / SAMPLE_SHORT lanes that have one of few entries together; every one of them gets it.
template <int TEAM>
__device__ __forceinline__ u64 team_sum_u64(u64 v) {
  static_assert(TEAM == 1 || TEAM == 4, "a lane or a quad");
  if (TEAM == 4) {
    auto move = [&](u64 x, auto step) __attribute__((always_inline)) {
      constexpr int CTRL = decltype(step)::value;
      const unsigned lo = __builtin_amdgcn_mov_dpp((int)(unsigned)x, CTRL, 0xf, 0xf, true), hi = __builtin_amdgcn_mov_dpp((int)(unsigned)(x >> 32), CTRL, 0xf, 0xf, true);
      return (u64)hi << 32 | lo;
    };
    v += move(v, std::integral_constant<int, 0xB1>());
    v += move(v, std::integral_constant<int, 0x4E>());
  }
  return v;
}
// Of the few (n2) entries in sh.few: how many are greater than that of this lane's team, and their weights.  (Lanes that have none are here too.)
template <int LANES>
__device__ __forceinline__ void sample_standing(int n2, SampleShared<LANES>& sh, u64 key, int* rank, u64* mass) {
  constexpr int TEAM = LANES / SAMPLE_SHORT;
  u64 r = 0, m = 0;
#pragma unroll 4
  for (int i = threadIdx.x % TEAM; i < n2; i += TEAM) {
    const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(sh.few + 2 * i);
    r += q.x > key ? 1 : 0;
    m += q.x > key ? q.y : 0;
  }
  *rank = (int)team_sum_u64<TEAM>(r);
  *mass = team_sum_u64<TEAM>(m);
}
// The weights of those of them that are kept and further up than a row.
template <int LANES>
__device__ __forceinline__ u64 sample_further_up(int n2, SampleShared<LANES>& sh, u64 border, int row) {
  constexpr int TEAM = LANES / SAMPLE_SHORT;
  u64 m = 0;
#pragma unroll 4
  for (int i = threadIdx.x % TEAM; i < n2; i += TEAM) {
    const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(sh.few + 2 * i);
    m += lp_key_index(q.x) < row && q.x >= border ? q.y : 0;
  }
  return team_sum_u64<TEAM>(m);
}

// From the n listed candidates: the border, of the first k (by_count: of those the first that have top_p of their weight) or where the weights, mass_before
// ahead of the list, reach `ask`.  `whole`: all that may be kept is in the list, which then draws.  More than a few are divided into bins of even width in the order
// of the keys, so that only the few of the bin that a border lies in are compared with each other.  Returns false where these are not few (many entries alike).
template <int LANES>
__device__ __forceinline__ bool sample_from_list(const SampleArgs& a, int col, int n, const SampleRule& rule, SampleKept& kept, SampleShared<LANES>& sh, bool by_count, bool whole,
                                                 u64 mass_before, u64 ask) {
  constexpr int BINS = SampleShared<LANES>::BINS;
  const int tid = threadIdx.x;
  constexpr int TEAM = LANES / SAMPLE_SHORT;
  const int who = tid / TEAM;      // (the entry that this lane has with its team)
  const bool leads = tid % TEAM == 0;
  if (n <= SAMPLE_SHORT) {
    u64 key = 0, w = 0, m;
    int rank;
    if (who < n) {
      key = sh.list[who];
      w = kept.weight(lp_key_value(key));
      if (leads) { sh.few[2 * who] = key; sh.few[2 * who + 1] = w; }
    }
    __syncthreads();
    sample_standing<LANES>(n, sh, key, &rank, &m);
    if (by_count) {
      if (leads && who < n && rank == (rule.k < n ? rule.k : n) - 1) { sh.border = key; sh.total = m + w; }
      __syncthreads();
      ask = sample_ask(rule, sh.total);
    }
    if (!by_count || rule.top_p < 1.0) {
      __syncthreads();
      if (leads && who < n && w && mass_before + m < ask && mass_before + m + w >= ask) { sh.border = key; sh.total = mass_before + m + w; }
    }
    __syncthreads();
    const u64 border = sh.border, total = sh.total;
    if (!whole) { kept.from(border); return true; }
    const u64 aim = sample_aim(rule, total);
    const int row = lp_key_index(key);
    const u64 sum = sample_further_up<LANES>(n, sh, border, row);
    if (leads && who < n && key >= border && w && sum <= aim && sum + w > aim) sample_out(a, col, kept, lp_key_value(key), row, total);
    sh.drawn = 1;
    return true;
  }
  if (tid == 0) { sh.key_max = 0; sh.key_min = ~0u; }
  sh.counts[tid] = 0;
  sh.masses[tid] = 0;
  __syncthreads();
  unsigned high = 0, low = ~0u;
  for (int i = tid; i < n; i += LANES) {
    const unsigned o = (unsigned)(sh.list[i] >> 32);
    high = o > high ? o : high;
    low = o < low ? o : low;
  }
  atomicMax(&sh.key_max, high);
  atomicMin(&sh.key_min, low);
  __syncthreads();
  const float most = lp_key_value((u64)sh.key_max << 32), scale = fminf((float)BINS / (most - lp_key_value((u64)sh.key_min << 32)), 3e38f);
  auto bin = [&](u64 key) __attribute__((always_inline)) { return (int)fminf((most - lp_key_value(key)) * scale, (float)(BINS - 1)); };
  u64 all_count, all_mass;
  for (int i = tid; i < n; i += LANES) {
    const u64 key = sh.list[i];
    const int b = bin(key);
    atomicAdd(&sh.counts[b], 1);
    const u64 w = kept.weight(lp_key_value(key));
    if (w) atomicAdd(&sh.masses[b], w);
  }
  __syncthreads();
  const u64 count = (u64)sh.counts[tid], mass = sh.masses[tid], up_count = sample_scan<LANES>(count, sh.wave_sum, &all_count), up_mass = sample_scan<LANES>(mass, sh.wave_sum, &all_mass);
  u64 border = 0, total = 0;
  // first the k-th, then the share of the weight
  for (int step = by_count ? 0 : 1; step < 2; ++step) {
    if (step == 1 && by_count) {
      if (rule.top_p >= 1.0) break;
      ask = sample_ask(rule, total);
    }
    const u64 want = step ? ask - mass_before : (u64)(rule.k < n ? rule.k : n);
    if (tid == 0) { sh.place = 0; sh.base = 0; sh.before = 0; sh.listed = 0; }
    __syncthreads();
    const u64 here = step ? mass : count, up = step ? up_mass : up_count;
    if (up >= want && up - here < want) { sh.place = tid; sh.base = up_mass - mass; sh.before = up_count - count; }      // (one lane)
    __syncthreads();
    const int place = sh.place;
    const u64 base = sh.base, before = sh.before;
    for (int i = tid; i < n; i += LANES) {
      const u64 key = sh.list[i];
      if (bin(key) == place) {
        const int at = atomicAdd(&sh.listed, 1);
        if (at < SAMPLE_SHORT) { sh.few[2 * at] = key; sh.few[2 * at + 1] = kept.weight(lp_key_value(key)); }
      }
    }
    __syncthreads();
    const int n2 = sh.listed;
    if (n2 > SAMPLE_SHORT) return false;
    {
      const u64 key = who < n2 ? sh.few[2 * who] : 0, w = who < n2 ? sh.few[2 * who + 1] : 0;
      int rank;
      u64 m;
      sample_standing<LANES>(n2, sh, key, &rank, &m);
      const bool it = step ? w && base + m < want && base + m + w >= want : before + (u64)rank == want - 1;
      if (it && leads && who < n2) { sh.border = key; sh.total = base + m + w + mass_before; }
    }
    __syncthreads();
    border = sh.border;
    total = sh.total;
  }
  if (!whole) { kept.from(border); return true; }
  // The row: the stretch of the column (one for every lane) in which the kept weights reach the aim, then those of its entries further up.
  const u64 aim = sample_aim(rule, total);
  const int stretch = (a.h + LANES - 1) / LANES;
  __syncthreads();
  if (tid == 0) sh.listed = 0;
  sh.masses[tid] = 0;
  __syncthreads();
  for (int i = tid; i < n; i += LANES) {
    const u64 key = sh.list[i], w = key >= border ? kept.weight(lp_key_value(key)) : 0;
    if (w) atomicAdd(&sh.masses[lp_key_index(key) / stretch], w);
  }
  __syncthreads();
  const u64 part = sh.masses[tid], up_part = sample_scan<LANES>(part, sh.wave_sum, &all_mass);
  if (part && up_part - part <= aim && up_part > aim) { sh.place = tid; sh.base = up_part - part; }      // (one lane)
  __syncthreads();
  const int place = sh.place;
  const u64 base = sh.base;
  for (int i = tid; i < n; i += LANES) {
    const u64 key = sh.list[i], w = key >= border && lp_key_index(key) / stretch == place ? kept.weight(lp_key_value(key)) : 0;
    if (w) {
      const int to = atomicAdd(&sh.listed, 1);
      if (to < SAMPLE_SHORT) { sh.few[2 * to] = key; sh.few[2 * to + 1] = w; }
    }
  }
  __syncthreads();
  const int n2 = sh.listed;
  if (n2 > SAMPLE_SHORT) { kept.from(border); sh.drawn = 0; return true; }      // (of tall columns: by a pass over the column)
  const u64 key = who < n2 ? sh.few[2 * who] : 0, w = who < n2 ? sh.few[2 * who + 1] : 0;
  const int row = lp_key_index(key);
  const u64 sum = base + sample_further_up<LANES>(n2, sh, border, row);
  if (leads && w && sum <= aim && sum + w > aim) sample_out(a, col, kept, lp_key_value(key), row, total);
  sh.drawn = 1;
  return true;
}

// Bins of even width by the distance to the greatest entry (one that overflows is in the last bin).
__device__ __forceinline__ float sample_scale(const SampleKept& kept, float least, int bins) {
  return fminf((float)bins / fminf(fminf(kept.far, kept.m - least), 3.402823466e38f), 3e38f);
}
__device__ __forceinline__ int sample_bin(const SampleKept& kept, float v, float scale, int bins) { return (int)fminf((kept.m - v) * scale, (float)(bins - 1)); }

// Lists the entries of the bins first to place, as long as there is room.  AHEAD: returns the weights of this lane's entries in the bins before them.
template <bool AHEAD, int LANES, int NV>
__device__ __forceinline__ u64 sample_list(const SampleColumn<LANES, NV>& column, const SampleKept& kept, float scale, int bins, int first, int place, int* listed, u64* list) {
  constexpr int LIST = SampleShared<LANES>::LIST;
  // (the values of these bins, with room for the roundings: two comparisons rule most entries out)
  const float slack = 1e-6f * fabsf(kept.m), end = place >= bins - 1 ? -INFINITY : kept.m - (float)(place + 1) / scale * 1.0001f - slack;
  const float start = !AHEAD && first > 0 ? kept.m - (float)first / scale * 0.9999f + slack : INFINITY;
  u64 sum = 0;
  column.each([&](const float (&v)[4], int row, int) __attribute__((always_inline)) {
    bool there[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) there[e] = v[e] >= end && v[e] <= start;
    if (!__any(there[0] || there[1] || there[2] || there[3]) || (!AHEAD && *(volatile int*)listed > LIST)) return;      // (too many already)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (AHEAD) there[e] = there[e] && kept.near(v[e]);
      int b = AHEAD ? sample_bin(kept, v[e], scale, bins) : 0;
      if (AHEAD) { const u64 w = kept.weight(there[e] ? v[e] : kept.m); sum += there[e] && b < first ? w : 0; }
      if (there[e] && (AHEAD || kept.near(v[e]))) {
        if (!AHEAD) b = sample_bin(kept, v[e], scale, bins);
        if (b >= first && b <= place) {
          const int at = atomicAdd(listed, 1);
          if (at < LIST) list[at] = lp_key(v[e], row + e);
        }
      }
    }
  });
  return sum;
}

// Finds what top-k and top-p keep: the border, for a pass over the column to draw by (true), or, where all that is kept has been listed and is little, draws.
// Candidates are chosen by the bin of their distance to the greatest entry.  At least k entries lie in the bins up to that of the k-th of 2 LANES maxima of
// parts of the column, and not many more.  Otherwise, and without a top-k, all entries are counted (weighed) bin by bin, and those of the bins up to
// the border's are listed, or where they are many those of its own.
template <int LANES, int NV>
__device__ __forceinline__ bool sample_border(const SampleArgs& a, int col, SampleColumn<LANES, NV>& column, const SampleRule& rule, SampleKept& kept, const float (&mine)[2],
                                              float least_x, SampleShared<LANES>& sh) {
  constexpr int BINS = SampleShared<LANES>::BINS, LIST = SampleShared<LANES>::LIST;
  const int tid = threadIdx.x;
  const bool by_count = rule.k < column.h;
  const float scale = sample_scale(kept, least_x, BINS);
  auto bin = [&](float v) __attribute__((always_inline)) { return sample_bin(kept, v, scale, BINS); };
  auto clear = [&](int place) __attribute__((always_inline)) {
    sh.counts[tid] = 0;
    sh.masses[tid] = 0;
    if (tid == 0) { sh.place = place; sh.listed = 0; }
    __syncthreads();
  };
  auto list_bins = [&](int first, int place) __attribute__((always_inline)) {
    sample_list<false>(column, kept, scale, BINS, first, place, &sh.listed, sh.list);
    __syncthreads();
    return sh.listed;
  };
  u64 ignored, mass_before = 0, ask = 0;
  int n = LIST + 1, place = BINS;
  bool whole = true;
  if (by_count && rule.k <= LANES) {
    clear(BINS - 1);
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (kept.near(mine[k])) atomicAdd(&sh.counts[bin(mine[k])], 1);
    __syncthreads();
    const u64 here = (u64)sh.counts[tid], up = sample_scan<LANES>(here, sh.wave_sum, &ignored);
    if (up >= (u64)rule.k && up - here < (u64)rule.k) sh.place = tid;
    __syncthreads();
    n = list_bins(0, sh.place);
    __syncthreads();
  }
  if (n > LIST) {
    clear(BINS);
    column.each([&](const float (&v)[4], int row, int) __attribute__((always_inline)) {
      if (by_count) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (kept.near(v[e])) atomicAdd(&sh.counts[bin(v[e])], 1);
      } else {
        u64 w[4];
        kept.weights(w, v, row);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (w[e]) atomicAdd(&sh.masses[bin(v[e])], w[e]);
      }
    });
    __syncthreads();
    const u64 here = by_count ? (u64)sh.counts[tid] : sh.masses[tid];
    u64 total;
    const u64 up = sample_scan<LANES>(here, sh.wave_sum, &total);
    ask = by_count ? 0 : sample_ask(rule, total);
    const u64 want = by_count ? (u64)rule.k : ask;
    if (up >= want && up - here < want) { sh.place = tid; sh.base = up - here; }      // (one lane at most)
    __syncthreads();
    place = sh.place;                                      // (BINS: fewer candidates than k)
    if (!by_count && column.slabs > 1) {                   // many, going by the first slab of every stretch: those of the border's bin alone
      float v[4];
      u64 some = 0;
      column.fetch(v, column.from);
#pragma unroll
      for (int e = 0; e < 4; ++e) some += kept.near(v[e]) && bin(v[e]) <= place ? 1 : 0;
      sample_scan<LANES>(some, sh.wave_sum, &some);
      whole = some * column.slabs <= LIST;
    }
    if (whole) n = list_bins(0, place);
    if (!by_count && (!whole || n > LIST)) {
      whole = false;
      mass_before = sh.base;
      __syncthreads();
      if (tid == 0) sh.listed = 0;
      __syncthreads();
      n = list_bins(place, place);
    }
  }
  if (n <= LIST && sample_from_list<LANES>(a, col, n, rule, kept, sh, by_count, whole, mass_before, ask)) return !whole || !sh.drawn;
  column.init(column.c, column.h);
  if (by_count) {
    const u64 border = sample_bisect(column, kept, sh, (u64)rule.k, [](float) { return (u64)1; });
    if (border) kept.from(border);                         // (none: fewer candidates than k)
  }
  if (rule.top_p < 1.0) {
    u64 sum = 0, total;
    column.each([&](const float (&v)[4], int row, int) __attribute__((always_inline)) {
      u64 w[4];
      kept.weights(w, v, row);
      sum += (w[0] + w[1]) + (w[2] + w[3]);
    });
    sample_scan<LANES>(sum, sh.wave_sum, &total);
    kept.from(sample_bisect(column, kept, sh, sample_ask(rule, total), [&](float v) __attribute__((always_inline)) { return kept.weight(v); }));
  }
  return true;
}

// The weights of a slab, `base` being those before it; draws if the aim is among them.
__device__ __forceinline__ u64 sample_slab(const SampleArgs& a, int col, const SampleKept& kept, const float (&v)[4], int row, u64 base, u64 aim, u64 total) {
  u64 w[4];
  kept.weights(w, v, row);
  const u64 own = (w[0] + w[1]) + (w[2] + w[3]), up = wave_scan_u64(own), all = lane_u64(up, 63);
  if (base + all > aim) {
    u64 up_to = base + up - own;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (w[e] && up_to <= aim && up_to + w[e] > aim) sample_out(a, col, kept, v[e], row + e, total);
      up_to += w[e];
    }
  }
  return all;
}

// Draws from one stretch of a column, whose first slab begins at `first` (of this lane) and which the aim is in; `base`: the weights before it.
// All wavefronts look for the part of the stretch (of one slab, or so many that there are at most as many parts as lanes), and one for the row in it.
template <int LANES, int NV>
__device__ __forceinline__ void sample_draw_stretch(const SampleArgs& a, int col, const SampleColumn<LANES, NV>& column, const SampleKept& kept, SampleShared<LANES>& sh, int first, u64 base,
                                                    u64 aim, u64 total) {
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, fold = (column.slabs + LANES - 1) / LANES;
  sh.masses[tid] = 0;
  __syncthreads();
  for (int part = wv; part * fold < column.slabs; part += LANES / 64) {
    u64 sum = 0;
    for (int k = part * fold; k < (part + 1) * fold && k < column.slabs; ++k) {
      float v[4];
      u64 w[4];
      column.fetch(v, first + 256 * k);
      kept.weights(w, v, first + 256 * k);
      sum += (w[0] + w[1]) + (w[2] + w[3]);
    }
    sum = lane_u64(wave_scan_u64(sum), 63);
    if (lane == 0) sh.masses[part] = sum;
  }
  __syncthreads();
  u64 all;
  const u64 here = sh.masses[tid], up = base + sample_scan<LANES>(here, sh.wave_sum, &all);
  if (here && up - here <= aim && up > aim) { sh.place = tid; sh.base = up - here; }      // (one lane)
  __syncthreads();
  if (wv) return;
  base = sh.base;
  for (int k = sh.place * fold; k < (sh.place + 1) * fold && k < column.slabs && base <= aim; ++k) {
    float v[4];
    column.fetch(v, first + 256 * k);
    base += sample_slab(a, col, kept, v, first + 256 * k, base, aim, total);
  }
}

// Draws from what is kept of a column.
template <int LANES, int NV>
__device__ __forceinline__ void sample_draw(const SampleArgs& a, int col, const SampleColumn<LANES, NV>& column, const SampleKept& kept, const SampleRule& rule, SampleShared<LANES>& sh) {
  constexpr int W = LANES / 64;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  // the weights of every wavefront's stretch, and the stretch that the aim is in
  u64 sum = 0;
  column.each([&](const float (&v)[4], int row, int) __attribute__((always_inline)) {
    u64 w[4];
    kept.weights(w, v, row);
    sum += (w[0] + w[1]) + (w[2] + w[3]);
  });
  sum = lane_u64(wave_scan_u64(sum), 63);
  __syncthreads();
  if (lane == 0) sh.wave_sum[wv] = sum;
  __syncthreads();
  u64 total = 0, base = 0;
  if (NV) {
#pragma unroll
    for (int k = 0; k < W; ++k) { if (k == wv) base = total; total += sh.wave_sum[k]; }
    const u64 aim = sample_aim(rule, total);
    if (aim < base || aim >= base + sum) return;
    // that wavefront looks for the slab, and the row in it
    column.each([&](const float (&v)[4], int row, int) __attribute__((always_inline)) {
      if (base > aim) return;
      base += sample_slab(a, col, kept, v, row, base, aim, total);
    });
    return;
  }
  int owner = 0;
#pragma unroll
  for (int k = 0; k < W; ++k) total += sh.wave_sum[k];
  const u64 aim = sample_aim(rule, total);
  u64 up_to = 0;
#pragma unroll
  for (int k = 0; k < W; ++k) {
    if (up_to <= aim) { owner = k; base = up_to; }
    up_to += sh.wave_sum[k];
  }
  sample_draw_stretch(a, col, column, kept, sh, owner * column.slabs * 256 + 4 * lane, base, aim, total);
}

// A workgroup a column, which it holds in registers, of up to 16384 rows, or reads again, from the caches (32768 x 512 takes as long either way).
// Weights are whole numbers (sample_weight), so every sum and with it every border is the same however it is added up.
// Bytes: 4 an entry.  32768 x 512 from the whole distribution 32 us (10 by the bytes): the first pass with the greatest entry takes as long as the greatest entries
// alone (19 with the search for them), the rest is the weights' arithmetic in 64 bits.  One column, 50000 x 1 with limits 15: its read by one CU and some
// twenty meetings of the workgroup.
template <int LANES, int NV, bool LIMITS>
__global__ void __launch_bounds__(LANES, LIMITS || LANES < 1024 || NV == 0 ? 1 : 8) k_sample_tokens(SampleArgs a) {
  constexpr int W = LANES / 64;
  __shared__ SampleShared<LANES> sh;
  const int col = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  SampleColumn<LANES, NV> column;
  column.init(a.mat + (size_t)col * a.h, a.h);
  const SampleRule rule = sample_rule(a, col);
  float mine[2] = {-INFINITY, -INFINITY}, least = INFINITY;
  bool bad = false;
  if (tid < SAMPLE_STEPS) sh.table[tid] = ldexp(sample_step(tid), a.shift);
  column.each([&](const float (&v)[4], int row, int slab) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      bad |= !(v[e] < INFINITY);
      mine[e & 1] = fmaxf(mine[e & 1], v[e]);
      least = fminf(least, v[e] > -INFINITY ? v[e] : INFINITY);
    }
  });
  float most = lanes_sum<64, true>(fmaxf(mine[0], mine[1]));
  least = -lanes_sum<64, true>(-least);
  bad = __any(bad);
  if (lane == 0) { sh.wave_max[wv] = most; sh.wave_min[wv] = least; sh.wave_bad[wv] = bad; }
  if (tid == 0) sh.place = a.h;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < W; ++k) { most = fmaxf(most, sh.wave_max[k]); least = fminf(least, sh.wave_min[k]); bad |= sh.wave_bad[k] != 0; }
  if (bad || !(most > -INFINITY)) {                        // (nothing to draw)
    if (tid == 0) { a.tokens[col] = -1.f; if (a.logp) a.logp[col] = bad ? NAN : 0.f; }
    return;
  }
  if (rule.greedy) {
    column.each([&](const float (&v)[4], int row, int) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 3; e >= 0; --e)
        if (v[e] == most) atomicMin(&sh.place, row + e);
    });
    __syncthreads();
    if (tid == 0) { a.tokens[col] = (float)sh.place; if (a.logp) a.logp[col] = 0.f; }
    return;
  }
  SampleKept kept = sample_kept(a, rule, most, sh.table);
  if constexpr (LIMITS) {
    if (rule.k < a.h || rule.top_p < 1.0) {
      __syncthreads();
      if (!sample_border<LANES, NV>(a, col, column, rule, kept, mine, least, sh)) return;
      column.init(column.c, a.h);                          // (the registers are the lists' meanwhile)
    }
  }
  sample_draw(a, col, column, kept, rule, sh);
}

// ------------------------------------------------------------------ few tall columns
// A column is divided into parts, a workgroup each, in four launches: the parts' greatest entries; their weights, bin by bin where top-p (or a large top-k)
// asks for a border; the candidates of the border's bins; and a workgroup a column that finds the border among those and draws, from the rows of
// one part.  The same sums of whole numbers, so the same tokens and bits as a workgroup a column gives.  What the lists do not hold
// (thousands of entries that are alike) that one does by itself.
// 128003 x 64, a rule of its own a column, 56 us (a workgroup a column 100): 6 to 10 for the greatest entries, 12 for the weights, 16 for the candidates, 19 for
// the borders; from the whole distribution 21 (37).
struct SamplePart { float most, least; int bad, first, listed; };      // first: row of the greatest entry (temperature 0)
struct SampleParts {
  int parts, rows;                 // of a column; of a part
  SamplePart* part;
  float* maxima;                   // one a lane, of every part
  u64 *bins, *lists, *sums;        // sums: of kept weights ahead of the list, 16 stretches a part
};
#define SAMPLE_PARTS 64            // of a column at most: a lane each where they meet
#define SAMPLE_BINS 2048           // two a lane: of 128003 logits a border's bin then has so few that they are compared with each other
typedef SampleShared<1024> SampleHere;
__device__ __forceinline__ SamplePart sample_meet(const SampleParts& s, int col) {
  const int lane = threadIdx.x & 63;
  const SamplePart* p = s.part + (size_t)col * s.parts + (lane < s.parts ? lane : 0);
  SamplePart o = {};
  const float most = p->most;
  o.most = lanes_sum<64, true>(most);
  o.least = -lanes_sum<64, true>(-p->least);
  o.bad = __any(p->bad);
  const unsigned long long who = __ballot(most == o.most);
  o.first = who ? __builtin_amdgcn_readlane(p->first, (int)__builtin_ctzll(who)) : 0;
  return o;
}
// Which of the ways a column goes: by a list of the first k, by bins of counts or weights, or only its weights' sum.
__device__ __forceinline__ bool sample_short(const SampleArgs& a, const SampleRule& rule) { return rule.k < a.h && rule.k <= 1024; }
__device__ __forceinline__ bool sample_whole(const SampleArgs& a, const SampleRule& rule) { return rule.k >= a.h && rule.top_p >= 1.0; }

// This lane's two bins of all parts.
__device__ __forceinline__ ulonglong2 sample_bins(const SampleParts& s, int col) {
  const ulonglong2* const bins = (const ulonglong2*)s.bins + (size_t)col * s.parts * (SAMPLE_BINS / 2) + threadIdx.x;
  ulonglong2 sum = {0, 0};
  for (int k = 0; k < s.parts; k += 4) {
    ulonglong2 x[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) x[q] = bins[SAMPLE_BINS / 2 * (k + q < s.parts ? k + q : k)];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (k + q < s.parts) { sum.x += x[q].x; sum.y += x[q].y; }
  }
  return sum;
}

template <bool LIMITS>
__global__ void __launch_bounds__(1024) k_sample_parts_most(SampleArgs a, SampleParts s) {
  __shared__ float wave_max[16], wave_min[16];
  __shared__ int wave_bad[16], place;
  const int col = blockIdx.x / s.parts, part = blockIdx.x - col * s.parts, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, first = part * s.rows;
  SampleColumn<1024, 0> column;
  column.init(a.mat + (size_t)col * a.h, first + s.rows < a.h ? first + s.rows : a.h, first);
  const SampleRule rule = sample_rule(a, col);
  float mine[2] = {-INFINITY, -INFINITY}, least = INFINITY;
  bool bad = false;
  column.each([&](const float (&v)[4], int row, int) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      bad |= !(v[e] < INFINITY);
      mine[e & 1] = fmaxf(mine[e & 1], v[e]);
      least = fminf(least, v[e] > -INFINITY ? v[e] : INFINITY);
    }
  });
  float most = fmaxf(mine[0], mine[1]);
  if (LIMITS && sample_short(a, rule)) s.maxima[(size_t)blockIdx.x * 1024 + tid] = most;
  most = lanes_sum<64, true>(most);
  least = -lanes_sum<64, true>(-least);
  bad = __any(bad);
  if (lane == 0) { wave_max[wv] = most; wave_min[wv] = least; wave_bad[wv] = bad; }
  if (tid == 0) place = a.h;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 16; ++k) { most = fmaxf(most, wave_max[k]); least = fminf(least, wave_min[k]); bad |= wave_bad[k] != 0; }
  if (rule.greedy) {
    column.each([&](const float (&v)[4], int row, int) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 3; e >= 0; --e)
        if (v[e] == most) atomicMin(&place, row + e);
    });
    __syncthreads();
  }
  if (tid == 0) s.part[blockIdx.x] = SamplePart{most, least, bad ? 1 : 0, place, 0};
}

template <bool LIMITS>
__global__ void __launch_bounds__(1024) k_sample_parts_weigh(SampleArgs a, SampleParts s) {
  __shared__ __align__(16) u64 bins[LIMITS ? SAMPLE_BINS : 2];
  __shared__ double table[SAMPLE_STEPS];
  const int col = blockIdx.x / s.parts, part = blockIdx.x - col * s.parts, tid = threadIdx.x, first = part * s.rows;
  const SampleRule rule = sample_rule(a, col);
  const SamplePart met = sample_meet(s, col);
  if (met.bad || !(met.most > -INFINITY) || rule.greedy || (LIMITS && sample_short(a, rule))) return;
  SampleColumn<1024, 0> column;
  column.init(a.mat + (size_t)col * a.h, first + s.rows < a.h ? first + s.rows : a.h, first);
  const SampleKept kept = sample_kept(a, rule, met.most, table);
  if (tid < SAMPLE_STEPS) table[tid] = ldexp(sample_step(tid), a.shift);
  if (LIMITS) reinterpret_cast<ulonglong2*>(bins)[tid] = ulonglong2{0, 0};
  __syncthreads();
  if (!LIMITS || sample_whole(a, rule)) {
    u64 sum = 0;
    column.each([&](const float (&v)[4], int row, int) __attribute__((always_inline)) {
      u64 w[4];
      kept.weights(w, v, row);
      sum += (w[0] + w[1]) + (w[2] + w[3]);
    });
    sum = lane_u64(wave_scan_u64(sum), 63);
    if ((tid & 63) == 0) s.sums[blockIdx.x * 16 + (tid >> 6)] = sum;
    return;
  }
  const bool by_count = rule.k < a.h;
  const float scale = sample_scale(kept, met.least, SAMPLE_BINS);
  column.each([&](const float (&v)[4], int row, int) __attribute__((always_inline)) {
    if (by_count) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (kept.near(v[e])) atomicAdd(&bins[sample_bin(kept, v[e], scale, SAMPLE_BINS)], 1ull);
    } else {
      u64 w[4];
      kept.weights(w, v, row);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (w[e]) atomicAdd(&bins[sample_bin(kept, v[e], scale, SAMPLE_BINS)], w[e]);
    }
  });
  __syncthreads();
  ((ulonglong2*)s.bins)[(size_t)blockIdx.x * 1024 + tid] = reinterpret_cast<ulonglong2*>(bins)[tid];
}

__global__ void __launch_bounds__(1024) k_sample_parts_list(SampleArgs a, SampleParts s) {
  __shared__ double table[SAMPLE_STEPS];
  __shared__ __align__(8) int counts[SAMPLE_BINS];
  __shared__ u64 wave_sum[16];
  __shared__ int found, listed;
  const int col = blockIdx.x / s.parts, part = blockIdx.x - col * s.parts, tid = threadIdx.x, first = part * s.rows;
  const SampleRule rule = sample_rule(a, col);
  const SamplePart met = sample_meet(s, col);
  if (met.bad || !(met.most > -INFINITY) || rule.greedy || sample_whole(a, rule)) return;
  SampleColumn<1024, 0> column;
  column.init(a.mat + (size_t)col * a.h, first + s.rows < a.h ? first + s.rows : a.h, first);
  const SampleKept kept = sample_kept(a, rule, met.most, table);
  const float scale = sample_scale(kept, met.least, SAMPLE_BINS);
  const bool by_count = rule.k < a.h, brief = sample_short(a, rule);
  if (!by_count && tid < SAMPLE_STEPS) table[tid] = ldexp(sample_step(tid), a.shift);
  reinterpret_cast<int2*>(counts)[tid] = int2{0, 0};
  if (tid == 0) { found = brief ? SAMPLE_BINS - 1 : SAMPLE_BINS; listed = 0; }
  __syncthreads();
  ulonglong2 here;
  if (brief) {
    const float* const maxima = s.maxima + (size_t)col * s.parts * 1024 + tid;
    for (int k = 0; k < s.parts; k += 8) {
      float x[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) x[q] = maxima[1024 * (k + q < s.parts ? k + q : k)];
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (k + q < s.parts && kept.near(x[q])) atomicAdd(&counts[sample_bin(kept, x[q], scale, SAMPLE_BINS)], 1);
    }
    __syncthreads();
    const int2 two = reinterpret_cast<const int2*>(counts)[tid];
    here = ulonglong2{(u64)two.x, (u64)two.y};
  } else here = sample_bins(s, col);
  u64 total;
  const u64 up = sample_scan<1024>(here.x + here.y, wave_sum, &total), want = by_count ? (u64)rule.k : sample_ask(rule, total), base = up - here.x - here.y;
  if (up >= want && base < want) found = 2 * tid + (base + here.x < want ? 1 : 0);      // (one lane at most)
  __syncthreads();
  const int place = found;
  u64* const list = s.lists + (size_t)blockIdx.x * SampleHere::LIST;
  if (by_count) sample_list<false>(column, kept, scale, SAMPLE_BINS, 0, place, &listed, list);
  else {
    const u64 sum = lane_u64(wave_scan_u64(sample_list<true>(column, kept, scale, SAMPLE_BINS, place, place, &listed, list)), 63);
    if ((tid & 63) == 0) s.sums[blockIdx.x * 16 + (tid >> 6)] = sum;
  }
  __syncthreads();
  if (tid == 0) s.part[blockIdx.x].listed = listed;
}

template <bool LIMITS>
__global__ void __launch_bounds__(1024) k_sample_parts_draw(SampleArgs a, SampleParts s) {
  __shared__ SampleHere sh;
  const int col = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), stretches = 16 * s.parts;
  const SampleRule rule = sample_rule(a, col);
  const SamplePart met = sample_meet(s, col);
  if (met.bad || !(met.most > -INFINITY)) {                // (nothing to draw)
    if (tid == 0) { a.tokens[col] = -1.f; if (a.logp) a.logp[col] = met.bad ? NAN : 0.f; }
    return;
  }
  if (rule.greedy) {
    if (tid == 0) { a.tokens[col] = (float)met.first; if (a.logp) a.logp[col] = 0.f; }
    return;
  }
  SampleKept kept = sample_kept(a, rule, met.most, sh.table);
  const bool by_count = rule.k < a.h, whole = !LIMITS || sample_whole(a, rule);
  u64 sum = !by_count && tid < stretches ? s.sums[(size_t)col * stretches + tid] : 0, before, total;
  if (tid < SAMPLE_STEPS) sh.table[tid] = ldexp(sample_step(tid), a.shift);
  SampleColumn<1024, 0> column;
  if constexpr (LIMITS) {
    if (!whole) {
      int up = lane < s.parts ? s.part[(size_t)col * s.parts + lane].listed : 0;      // (where a part's list ends)
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) { const int q = __shfl_up(up, o, WAVE); if (lane >= o) up += q; }
      const int n = __builtin_amdgcn_readlane(up, 63);
      bool found = false;
      if (n <= SampleHere::LIST) {
        for (int k = wv; k < s.parts; k += 16) {
          const int to = __builtin_amdgcn_readlane(up, k), from = k ? __builtin_amdgcn_readlane(up, k - 1) : 0;
          const u64* const list = s.lists + ((size_t)col * s.parts + k) * SampleHere::LIST;
          for (int i = from + lane; i < to; i += 64) sh.list[i] = list[i - from];
        }
        u64 ask = 0;
        before = 0;
        if (!by_count) {
          const ulonglong2 two = sample_bins(s, col);
          sample_scan<1024>(two.x + two.y, sh.wave_sum, &total);
          ask = sample_ask(rule, total);
          sample_scan<1024>(sum, sh.wave_sum, &before);
        }
        __syncthreads();
        found = sample_from_list<1024>(a, col, n, rule, kept, sh, by_count, by_count, before, ask);
        if (found && by_count && sh.drawn) return;
      }
      if (!found || by_count) {                            // by the whole column
        const float none[2] = {-INFINITY, -INFINITY};
        column.init(a.mat + (size_t)col * a.h, a.h);
        __syncthreads();
        if (found || sample_border<1024, 0>(a, col, column, rule, kept, none, met.least, sh)) sample_draw(a, col, column, kept, rule, sh);
        return;
      }
      // the listed ones that are kept, stretch by stretch
      const u64 border = sh.border;
      const int full = s.rows / 16, last = (a.h - (s.parts - 1) * s.rows + 4095) / 4096 * 256;
      __syncthreads();
      sh.masses[tid] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += 1024) {
        const u64 key = sh.list[i], w = key >= border ? kept.weight(lp_key_value(key)) : 0;
        const int row = lp_key_index(key), part = row / s.rows;
        if (w) atomicAdd(&sh.masses[16 * part + (row - part * s.rows) / (part == s.parts - 1 ? last : full)], w);
      }
      __syncthreads();
      sum += sh.masses[tid];
    }
  }
  // the stretch that the aim is in
  const u64 up = sample_scan<1024>(sum, sh.wave_sum, &total), aim = sample_aim(rule, total);
  if (sum && up - sum <= aim && up > aim) { sh.place = tid; sh.base = up - sum; }      // (one lane)
  __syncthreads();
  const int place = sh.place, first = (place >> 4) * s.rows;
  before = sh.base;
  column.init(a.mat + (size_t)col * a.h, first + s.rows < a.h ? first + s.rows : a.h, first);
  __syncthreads();
  sample_draw_stretch(a, col, column, kept, sh, first + (place & 15) * column.slabs * 256 + 4 * lane, before, aim, total);
}

extern "C" int sample_tokens(cudamat* mat, cudamat* uniform, cudamat* temperature, cudamat* top_k, cudamat* top_p, cudamat* min_p, cudamat* target,
                             cudamat* logp, float all_temperature, float all_top_k, float all_top_p, float all_min_p) {
  cudamat* const all[8] = {mat, uniform, temperature, top_k, top_p, min_p, target, logp};
  if (int e = tok_check_device(all)) return e;
  const int h = mat->size[0], w = mat->size[1];
  if (!uniform || !target) return ERROR_INCOMPATIBLE_DIMENSIONS;
  for (int i = 1; i < 8; ++i)
    if (!tok_shape(all[i], 1, w)) return ERROR_INCOMPATIBLE_DIMENSIONS;
  if (h > (1 << 24)) return ERROR_UNSUPPORTED;
  for (int i = 0; i < 6; ++i)
    if (!tok_apart(all[i], target) || !tok_apart(all[i], logp)) return ERROR_UNSUPPORTED;
  if (!tok_apart(target, logp)) return ERROR_UNSUPPORTED;
  if (w <= 0) return 0;
  int bits = 0;
  while ((1 << bits) < h) ++bits;
  // From the whole distribution, as the numbers say: without the lists two workgroups fit a CU.
  const bool limits = top_k || top_p || min_p || (all_top_k >= 1.f && all_top_k < (float)h) || all_top_p < 1.f || all_min_p > 0.f;
  const int slabs = (int)(((long long)h + 4095) / 4096);
  // Divided where that pays (us, a workgroup a column / divided: 65536 x 8 from the whole distribution 19.9 / 14.3, 32000 x 8 12.8 / 14.1; greatest entries 9.1 / 7.6,
  // 6.4 / 7.5; top-p 49.6 / 34.2, 30.7 / 29.9; in two parts, 65536 x 128, 20.8 / 19.5, 9.5 / 8.9, 51.5 / 50.9; 50 best, which take only one pass more,
  // 98304 x 8 17.3 / 20.7, 128003 x 64 22.2 / 21.4, 200000 x 8 27.3 / 21.3, x 128 39.0 / 45.6; 400 best 31.7 / 30.2, 37.6 / 33.0, 43.0 / 31.2, 50.1 / 56.7).
  const bool brief = !top_k && all_top_k >= 1.f && all_top_k < (float)h && all_top_k < 1025.f, greedy = !temperature && !(all_temperature > 0.f);
  int parts = dn_num_cus() / w;
  if (brief && !greedy ? slabs < 32 || parts < 4 : slabs <= 8) parts = 1;
  parts = parts < slabs ? parts : slabs;
  parts = parts < SAMPLE_PARTS ? parts : SAMPLE_PARTS;
  if (parts > 1) {
    SampleParts s;
    const int per = (slabs + parts - 1) / parts;
    s.rows = 4096 * per;
    s.parts = parts = (slabs + per - 1) / per;
    const size_t all_parts = (size_t)parts * w, each = sizeof(SamplePart) + 16 * sizeof(u64) + (limits ? 1024 * sizeof(float) + (SAMPLE_BINS + SampleHere::LIST) * sizeof(u64) : 0);
    if (char* scratch = (char*)dn_scratch(all_parts * each)) {
      s.sums = (u64*)scratch;
      s.lists = s.sums + 16 * all_parts;
      s.bins = s.lists + (limits ? all_parts * SampleHere::LIST : 0);
      s.maxima = (float*)(s.bins + (limits ? all_parts * SAMPLE_BINS : 0));
      s.part = (SamplePart*)(s.maxima + (limits ? all_parts * 1024 : 0));
      const SampleArgs a = {mat->data_device, tok_data(uniform), tok_data(temperature), tok_data(top_k), tok_data(top_p), tok_data(min_p), target->data_device, tok_data(logp),
                            all_temperature, all_top_k, all_top_p, all_min_p, h, w, 62 - bits < 45 ? 62 - bits : 45};
      const dim3 grid((unsigned)all_parts), block(1024);
      if (limits) hipLaunchKernelGGL(k_sample_parts_most<true>, grid, block, 0, dn_stream(), a, s);
      else hipLaunchKernelGGL(k_sample_parts_most<false>, grid, block, 0, dn_stream(), a, s);
      if (!greedy && !brief) {
        if (limits) hipLaunchKernelGGL(k_sample_parts_weigh<true>, grid, block, 0, dn_stream(), a, s);
        else hipLaunchKernelGGL(k_sample_parts_weigh<false>, grid, block, 0, dn_stream(), a, s);
      }
      if (!greedy && limits) hipLaunchKernelGGL(k_sample_parts_list, grid, block, 0, dn_stream(), a, s);
      if (limits) hipLaunchKernelGGL(k_sample_parts_draw<true>, dim3(w), block, 0, dn_stream(), a, s);
      else hipLaunchKernelGGL(k_sample_parts_draw<false>, dim3(w), block, 0, dn_stream(), a, s);
      return dn_launch_status();
    }
  }
  const long long most = h <= 4096 ? DN_MAX_GROUPS : DN_MAX_GROUPS / 4;            // columns of a launch
  for (long long c0 = 0; c0 < w; c0 += most) {
    const int n = (int)(w - c0 < most ? w - c0 : most);
    auto from = [c0](const cudamat* m) { return m ? m->data_device + c0 : nullptr; };
    const SampleArgs a = {mat->data_device + c0 * h, from(uniform), from(temperature), from(top_k), from(top_p), from(min_p), from(target), from(logp),
                          all_temperature, all_top_k, all_top_p, all_min_p, h, n, 62 - bits < 45 ? 62 - bits : 45};
#define SAMPLE_GO(LANES, NV) do { if (limits) hipLaunchKernelGGL((k_sample_tokens<LANES, NV, true>), dim3(n), dim3(LANES), 0, dn_stream(), a); \
                                  else hipLaunchKernelGGL((k_sample_tokens<LANES, NV, false>), dim3(n), dim3(LANES), 0, dn_stream(), a); } while (0)
    // (us, 256 / 1024 lanes: 2900 x 256 from the whole distribution 5.1 / 5.4, of 50 best 10.0 / 9.0, of 400 15.7 / 18.7; 4096 x 512 6.8 / 8.2, 11.1 / 16.6, 17.3 / 35.6.
    // Above 4096 rows, registers of 1024 lanes against memory and 256: 8192 x 128 6.5 / 7.8, 9.4 / 11.8, 19.5 / 21.3, but with limits in more columns than CUs
    // x 1000 34 / 24, 74 / 40, top-p 0.9 92 / 58; 16384 x 512 19.8 / 16.3, 42 / 31, 60 / 55; 32768 x 1000 54 / 52, 104 / 99, 135 / 147.)
    if (h <= 4096) SAMPLE_GO(256, 4);
    else if (h <= 16384 && limits && w > dn_num_cus()) hipLaunchKernelGGL((k_sample_tokens<256, 0, true>), dim3(n), dim3(256), 0, dn_stream(), a);
    else if (h <= 16384) SAMPLE_GO(1024, 4);
    else SAMPLE_GO(1024, 0);
#undef SAMPLE_GO
  }
  return dn_launch_status();
}
