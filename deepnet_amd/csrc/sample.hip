// Tokens drawn from columns of logits by given random numbers, with temperature, top-k, min-p and top-p (no counterpart in cudamat.cu; beside
// perturb_prob / choose_max, which draw from the whole distribution by a random number an entry).
#include "columns.h"
#include "tokens.h"
#include "wide_math.h"

struct SampleArgs {
  const float *mat, *uniform, *temperature, *top_k, *top_p, *min_p;
  float *tokens, *logp;
  float all_temperature, all_top_k, all_top_p, all_min_p;
  int h, w;
  int shift;                       // weights are multiples of 2^-shift
};

// The weight e^((x - m) / T) of an entry, x <= m, as a whole multiple of 2^-shift: the same one wherever it is computed, and sums of
// them do not depend on their order, so a border between two sums is one border.  c = log2(e) / T.  2^t with t = (n + f) / 256, n whole and |f| <= 1/2: 2^(n / 256) from
// a table of 256 steps and the whole part, 2^(f / 256) by its Taylor sum (remainder (ln 2 / 512)^5 / 5! < 4e-17).  Adding 2^52 leaves the rounded whole number in the low bits.
// Entries that have none (too far from m) are not asked for.
#define SAMPLE_STEPS 256
__device__ __forceinline__ unsigned long long sample_weight(float x, float m, double c, int shift, const double* table) {
  const double t = ((double)x - (double)m) * (c * 256.0), b = t + 6755399441055744.0, f = t - (b - 6755399441055744.0);      // (3 * 2^51: the low bits are n)
  const int n = (int)__double_as_longlong(b);
  double p = 2.239395190875157e-12;           // (ln2 / 256)^4 / 4!
  p = fma(p, f, 3.308302680541371e-09);
  p = fma(p, f, 3.665565596910106e-06);
  p = fma(p, f, 2.7076061740622863e-03);
  p = fma(p, f, 1.0) * table[n & 255];
  const double w = __hiloint2double(__double2hiint(p) + (((n >> 8) + shift) << 20), __double2loint(p)) + 4503599627370496.0;
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

#define SAMPLE_LIST 4096           // candidates that are sorted
#define SAMPLE_SHORT 256           // candidates whose places are counted instead, each by a lane
template <int LANES>
struct SampleShared {
  static constexpr int WAVES = LANES / 64, BINS = LANES;
  double table[SAMPLE_STEPS];
  u64 list[SAMPLE_LIST + 2];       // keys of candidates, or the weights of stretches of the column
  u64 masses[BINS];
  u64 sorted[SAMPLE_SHORT];
  int counts[BINS];
  u64 wave_sum[WAVES];
  float wave_max[WAVES], wave_min[WAVES];
  int wave_bad[WAVES], listed, place, cell;
  u64 border, base;
};

// Sums up to a lane (itself included) over a workgroup, and the sum of all.  Every lane calls it; what it uses is free again behind the next barrier.
template <int LANES>
__device__ __forceinline__ u64 sample_scan(u64 v, u64* wave_sum, u64* all) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) { const u64 q = __shfl_up(v, o, WAVE); if (lane >= o) v += q; }
  __syncthreads();
  if (lane == 63) wave_sum[wv] = v;
  __syncthreads();
  u64 sum = 0;
#pragma unroll
  for (int k = 0; k < LANES / 64; ++k) { if (k == wv) v += sum; sum += wave_sum[k]; }
  *all = sum;
  return v;
}

// The keys of a list, the greatest first: a bitonic sort of `size` (a power of two, at least the list's length) with zeros behind the list.
template <int LANES>
__device__ __forceinline__ void sample_sort(u64* list, int n, int size) {
  for (int i = n + threadIdx.x; i < size; i += LANES) list[i] = 0;
  __syncthreads();
  for (int run = 2; run <= size; run *= 2)
    for (int gap = run / 2; gap > 0; gap /= 2) {
      for (int i = threadIdx.x; i < size / 2; i += LANES) {
        const int x = 2 * i - (i & (gap - 1)), y = x + gap;
        const u64 p = list[x], q = list[y];
        if ((p < q) == ((x & run) == 0)) { list[x] = q; list[y] = p; }
      }
      __syncthreads();
    }
}

// The entries of a column, four rows a lane and slab: in registers (NV slabs) or, of columns that those do not hold (NV = 0), from memory, where
// eight slabs are on their way at once.  f(x, row) for a lane's four, rows behind the column being -infinity.
template <int LANES, int NV>
struct SampleColumn {
  const float* c;
  int h;
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
  __device__ __forceinline__ void init() {
    if (NV) {
#pragma unroll
      for (int k = 0; k < NV; ++k) fetch(x[k], 4 * (threadIdx.x + LANES * k));
    }
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    if (NV) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (4 * LANES * k < h) {
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) { v[e] = x[k][e]; asm volatile("" : "+v"(v[e])); }      // (what one pass makes of an entry is not kept for the next)
          int row = 4 * (int)(threadIdx.x + LANES * k);
          asm volatile("" : "+v"(row));
          f(v, row);
          __builtin_amdgcn_sched_barrier(0);
        }
    } else {
      for (int k = 0; 4 * LANES * k < h; k += 8) {
        float v[8][4];
#pragma unroll
        for (int q = 0; q < 8; ++q) fetch(v[q], 4 * (threadIdx.x + LANES * (k + q)));
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (4 * LANES * (k + q) < h) f(v[q], 4 * (int)(threadIdx.x + LANES * (k + q)));
      }
    }
  }
};

// Kept entries: those from `border` on in the order of keys whose weight reaches `least`.
struct SampleKept {
  float m, far, x;                 // the greatest entry; entries further from it than `far` have no weight; the last kept value,
  int row;                         // and of entries of that value the last kept row
  double c;
  int shift;
  u64 least;
  const double* table;
  __device__ __forceinline__ bool near(float v) const { return v > -INFINITY && m - v <= far; }
  __device__ __forceinline__ bool in(float v, int i) const { return near(v) && (v > x || (v == x && i <= row)); }
  __device__ __forceinline__ u64 weight(float v) const {
    const u64 w = sample_weight(v, m, c, shift, table);
    __builtin_amdgcn_sched_barrier(0);                     // (one at a time: registers)
    return w >= least ? w : 0;
  }
  __device__ __forceinline__ void from(u64 border) { x = lp_key_value(border); row = lp_key_index(border); }
};

__device__ __forceinline__ void sample_out(const SampleArgs& a, int col, const SampleKept& kept, float v, int row, u64 total) {
  a.tokens[col] = (float)row;
  if (a.logp) a.logp[col] = (float)(((double)v - (double)kept.m) * (kept.c * 0.6931471805599453) - dn_log_wide_pos(ldexp((double)total, -a.shift)));
}

// The greatest border that leaves enough: bit by bit, a pass over the column each.  For columns whose border lies among thousands of
// entries that are alike or nearly so.
template <int LANES, int NV, typename F>
__device__ __forceinline__ u64 sample_bisect(const SampleColumn<LANES, NV>& column, const SampleKept& kept, SampleShared<LANES>& sh, u64 enough, F value) {
  u64 border = 0;
  for (int bit = 63; bit >= 0; --bit) {
    const u64 trial = border | 1ull << bit;
    u64 sum = 0, all;
    column.each([&](const float (&v)[4], int row) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (kept.in(v[e], row + e) && lp_key(v[e], row + e) >= trial) sum += value(v[e]);
    });
    sample_scan<LANES>(sum, sh.wave_sum, &all);
    if (all >= enough) border = trial;
  }
  return border;
}

// From n listed candidates: the border, which the list contains, of the first k (by_count: of those the first that have top_p of their weight), or the one where
// the weights, mass_before ahead of the list, reach `ask`.  Returns 0 where they do not.  A lane has EACH neighbours of the sorted list.
template <int LANES, int EACH>
__device__ __forceinline__ u64 sample_cut(const u64* sorted, int n, const SampleRule& rule, const SampleKept& kept, SampleShared<LANES>& sh, bool by_count, u64 mass_before,
                                          u64 ask) {
  const int tid = threadIdx.x;
  u64 w[EACH], sum = 0, all;
#pragma unroll
  for (int k = 0; k < EACH; ++k) {
    const int i = EACH * tid + k;
    w[k] = i < n && (!by_count || i < rule.k) ? kept.weight(lp_key_value(sorted[i])) : 0;
    sum += w[k];
  }
  u64 up_to = sample_scan<LANES>(sum, sh.wave_sum, &all) - sum + mass_before;
  if (by_count) ask = rule.top_p < 1.0 ? (rule.top_p > 0.0 ? sample_part_up(rule.top_p, all) : 0) : all;
  if (ask < 1) ask = 1;
  if (tid == 0) sh.border = 0;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < EACH; ++k) {
    if (w[k] && up_to < ask && up_to + w[k] >= ask) { sh.border = sorted[EACH * tid + k]; sh.base = up_to + w[k]; }      // (one of them)
    up_to += w[k];
  }
  __syncthreads();
  return sh.border;
}

// The border that top-k and top-p set, for a pass over the column to draw by (true), or, where all that is kept has been listed and is little, the token
// itself.  Candidates are chosen by the bin of their distance to the greatest entry.
// At least k entries lie in the bins up to that of the k-th of the lanes' maxima, and not many more: these are listed.  Without a top-k 128 are, in the hope
// that they have enough of the weight.  Otherwise all entries are counted (without a top-k: weighed) bin by bin, and those of the bin of the
// border (with a top-k: of all up to it) are listed.
template <int LANES, int NV>
__device__ __forceinline__ bool sample_border(const SampleArgs& a, int col, const SampleColumn<LANES, NV>& column, const SampleRule& rule, SampleKept& kept, float mine, float least_x,
                                              SampleShared<LANES>& sh) {
  constexpr int BINS = SampleShared<LANES>::BINS;
  const int tid = threadIdx.x;
  const bool by_count = rule.k < column.h;
  const float scale = fminf((float)BINS / fminf(kept.far, kept.m - least_x), 3e38f);
  auto bin = [&](float v) __attribute__((always_inline)) { return (int)fminf((kept.m - v) * scale, (float)(BINS - 1)); };
  auto list_bins = [&](int first, int place) __attribute__((always_inline)) {
    if (tid == 0) sh.listed = 0;
    __syncthreads();
    column.each([&](const float (&v)[4], int row) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (kept.near(v[e])) {
          const int b = bin(v[e]);
          if (b >= first && b <= place) {
            const int at = atomicAdd(&sh.listed, 1);
            if (at < SAMPLE_LIST) sh.list[at] = lp_key(v[e], row + e);
          }
        }
    });
    __syncthreads();
    return sh.listed;
  };
  u64 total = 0, ask = 0;
  if (!by_count) {
    u64 sum = 0;
    column.each([&](const float (&v)[4], int row) __attribute__((always_inline)) {
      if (__any(kept.near(v[0]) || kept.near(v[1]) || kept.near(v[2]) || kept.near(v[3]))) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += kept.near(v[e]) ? kept.weight(v[e]) : 0;
      }
    });
    sample_scan<LANES>(sum, sh.wave_sum, &total);
    ask = rule.top_p > 0.0 ? sample_part_up(rule.top_p, total) : 1;
  }
  const int some = by_count ? rule.k : 128;
  if (some <= LANES / 2) {
    sh.counts[tid] = 0;
    if (tid == 0) sh.place = BINS - 1;
    __syncthreads();
    if (kept.near(mine)) atomicAdd(&sh.counts[bin(mine)], 1);
    __syncthreads();
    u64 all;
    const u64 here = (u64)sh.counts[tid], up = sample_scan<LANES>(here, sh.wave_sum, &all);
    if (up >= (u64)some && up - here < (u64)some) sh.place = tid;
    __syncthreads();
    const int n = list_bins(0, sh.place);
    if (n <= SAMPLE_SHORT) {
      // places by counting
      if (tid < 2) sh.list[n + tid] = 0;
      __syncthreads();
      if (tid < n) {
        const u64 key = sh.list[tid];
        int rank = 0;
#pragma unroll 4
        for (int i = 0; i < n; i += 2) {
          const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(sh.list + i);
          rank += (q.x > key ? 1 : 0) + (q.y > key ? 1 : 0);
        }
        sh.sorted[rank] = key;
      }
      __syncthreads();
      const u64 border = sample_cut<LANES, 1>(sh.sorted, n, rule, kept, sh, by_count, 0, ask);
      if (border) {
        // the kept ones draw: each adds the weights of those further up in the column
        const u64 key = tid < n ? sh.sorted[tid] : 0, kept_total = sh.base;
        const float v = lp_key_value(key);
        const int row = lp_key_index(key);
        const u64 w = key >= border ? kept.weight(v) : 0;
        if (tid < SAMPLE_SHORT) { sh.masses[tid] = w; sh.list[tid] = (u64)(unsigned)row; }
        __syncthreads();
        const u64 at = sample_part((double)rule.u, kept_total), aim = at < kept_total ? at : kept_total - 1;
        if (w) {
          u64 up_to = 0;
#pragma unroll 4
          for (int i = 0; i < n; ++i) up_to += (int)sh.list[i] < row ? sh.masses[i] : 0;
          if (up_to <= aim && up_to + w > aim) sample_out(a, col, kept, v, row, kept_total);
        }
        return false;
      }
    } else if (n <= SAMPLE_LIST) {
      int size = 512;
      while (size < n) size *= 2;
      sample_sort<LANES>(sh.list, n, size);
      const u64 border = sample_cut<LANES, SAMPLE_LIST / LANES>(sh.list, n, rule, kept, sh, by_count, 0, ask);
      if (border) { kept.from(border); return true; }
    }
    __syncthreads();
  }
  sh.counts[tid] = 0;
  sh.masses[tid] = 0;
  if (tid == 0) sh.place = BINS;
  __syncthreads();
  column.each([&](const float (&v)[4], int row) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (kept.near(v[e])) {
        const int b = bin(v[e]);
        atomicAdd(&sh.counts[b], 1);
        if (!by_count) atomicAdd(&sh.masses[b], kept.weight(v[e]));
      }
  });
  __syncthreads();
  u64 ignored;
  const u64 here = by_count ? (u64)sh.counts[tid] : sh.masses[tid], want = by_count ? (u64)rule.k : ask, up = sample_scan<LANES>(here, sh.wave_sum, &ignored);
  if (up >= want && up - here < want) { sh.place = tid; sh.base = up - here; }      // (one lane at most)
  __syncthreads();
  const int place = sh.place;                              // (BINS: fewer candidates than k)
  const u64 mass_before = by_count ? 0 : sh.base;
  const int n = list_bins(by_count ? 0 : place, place);
  if (n <= SAMPLE_LIST) {
    int size = 2;
    while (size < n) size *= 2;
    sample_sort<LANES>(sh.list, n, size);
    const u64 border = sample_cut<LANES, SAMPLE_LIST / LANES>(sh.list, n, rule, kept, sh, by_count, mass_before, ask);
    kept.from(border);
    return true;
  }
  if (by_count && place < BINS) kept.from(sample_bisect(column, kept, sh, (u64)rule.k, [](float) { return (u64)1; }));
  if (rule.top_p < 1.0) {
    u64 sum = 0;
    column.each([&](const float (&v)[4], int row) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (kept.in(v[e], row + e)) sum += kept.weight(v[e]);
    });
    sample_scan<LANES>(sum, sh.wave_sum, &total);
    const u64 p = rule.top_p > 0.0 ? sample_part_up(rule.top_p, total) : 0;
    kept.from(sample_bisect(column, kept, sh, p > 1 ? p : 1, [&](float v) __attribute__((always_inline)) { return kept.weight(v); }));
  }
  return true;
}

// A workgroup a column, which it holds in registers (of more than 65536 rows: reads again, from the caches).
// Weights are whole numbers (sample_weight), so every sum and with it every border is the same however it is added up.
template <int LANES, int NV>
__global__ void __launch_bounds__(LANES) k_sample_tokens(SampleArgs a) {
  constexpr int W = LANES / 64, CELLS = SAMPLE_LIST;
  __shared__ SampleShared<LANES> sh;
  const int col = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  SampleColumn<LANES, NV> column;
  column.c = a.mat + (size_t)col * a.h;
  column.h = a.h;
  column.init();
  const SampleRule rule = sample_rule(a, col);
  float most = -INFINITY, least = INFINITY;
  bool bad = false;
  column.each([&](const float (&v)[4], int row) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      bad |= !(v[e] < INFINITY);
      most = fmaxf(most, v[e]);
      least = fminf(least, v[e] > -INFINITY ? v[e] : INFINITY);
    }
  });
  const float mine = most;
  most = lanes_sum<64, true>(most);
  least = -lanes_sum<64, true>(-least);
  bad = __any(bad);
  if (lane == 0) { sh.wave_max[wv] = most; sh.wave_min[wv] = least; sh.wave_bad[wv] = bad; }
  if (tid == 0) sh.place = a.h;
  if (tid < SAMPLE_STEPS) sh.table[tid] = sample_step(tid);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < W; ++k) { most = fmaxf(most, sh.wave_max[k]); least = fminf(least, sh.wave_min[k]); bad |= sh.wave_bad[k] != 0; }
  if (bad || !(most > -INFINITY)) {                        // (nothing to draw)
    if (tid == 0) { a.tokens[col] = -1.f; if (a.logp) a.logp[col] = bad ? NAN : 0.f; }
    return;
  }
  if (rule.greedy) {
    column.each([&](const float (&v)[4], int row) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 3; e >= 0; --e)
        if (v[e] == most) atomicMin(&sh.place, row + e);
    });
    __syncthreads();
    if (tid == 0) { a.tokens[col] = (float)sh.place; if (a.logp) a.logp[col] = 0.f; }
    return;
  }
  SampleKept kept;
  kept.m = most; kept.x = -INFINITY; kept.row = 0; kept.c = rule.c; kept.shift = a.shift; kept.least = rule.least; kept.table = sh.table;
  kept.far = (float)((a.shift + 1.5) / rule.c);            // (2^-(shift + 1) is nothing; half an octave for the rounding of the distance)
  if ((rule.k < a.h || rule.top_p < 1.0) && !sample_border<LANES, NV>(a, col, column, rule, kept, mine, least, sh)) return;
  __syncthreads();
  // the kept weights of every wavefront's part of a slab (256 rows); of more slabs than there is room for, of several slabs
  const int slabs = (a.h + 4 * LANES - 1) / (4 * LANES), cells = slabs * W, fold = (cells + CELLS - 1) / CELLS;
  if (fold > 1)
    for (int k = tid; k < CELLS; k += LANES) sh.list[k] = 0;
  __syncthreads();
  column.each([&](const float (&v)[4], int row) __attribute__((always_inline)) {
    bool in[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) in[e] = kept.in(v[e], row + e);
    u64 sum = 0;
    if (__any(in[0] || in[1] || in[2] || in[3])) {
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += in[e] ? kept.weight(v[e]) : 0;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, WAVE);
    }
    if (lane == 0) {
      const int cell = row / 256;                          // (row: this wavefront's first one)
      if (fold == 1) sh.list[cell] = sum;
      else if (sum) atomicAdd(&sh.list[cell / fold], sum);
    }
  });
  __syncthreads();
  constexpr int EACH = CELLS / LANES;
  u64 w[EACH], sum = 0, total;
  const int used = (cells + fold - 1) / fold;
#pragma unroll
  for (int k = 0; k < EACH; ++k) {
    w[k] = EACH * tid + k < used ? sh.list[EACH * tid + k] : 0;
    sum += w[k];
  }
  u64 up_to = sample_scan<LANES>(sum, sh.wave_sum, &total) - sum;
  const u64 at = sample_part((double)rule.u, total), aim = at < total ? at : total - 1;
#pragma unroll
  for (int k = 0; k < EACH; ++k) {
    if (w[k] && up_to <= aim && up_to + w[k] > aim) { sh.cell = (EACH * tid + k) * fold; sh.base = up_to; }      // (one of them)
    up_to += w[k];
  }
  __syncthreads();
  if (wv > 0) return;
  // one wavefront: the entry among the 256 (or those of the folded slabs, 256 at a time)
  u64 base = sh.base;
  for (int cell = sh.cell; cell < sh.cell + fold; ++cell) {
    float v[4];
    const int row = 256 * cell + 4 * lane;
    column.fetch(v, row);
    u64 q[4], mine = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) { q[e] = kept.in(v[e], row + e) ? kept.weight(v[e]) : 0; mine += q[e]; }
    u64 up = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const u64 p = __shfl_up(up, o, WAVE); if (lane >= o) up += p; }
    u64 from = base + up - mine;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (q[e] && from <= aim && from + q[e] > aim) {
        sample_out(a, col, kept, v[e], row + e, total);
      }
      from += q[e];
    }
    base += __shfl(up, 63, WAVE);
  }
}

extern "C" int sample_tokens(cudamat* mat, cudamat* uniform, cudamat* temperature, cudamat* top_k, cudamat* top_p, cudamat* min_p, cudamat* target,
                             cudamat* logp, float all_temperature, float all_top_k, float all_top_p, float all_min_p) {
  cudamat* const all[8] = {mat, uniform, temperature, top_k, top_p, min_p, target, logp};
  if (int e = tok_check_device(all)) return e;
  const int h = mat->size[0], w = mat->size[1];
  for (int i = 1; i < 8; ++i)
    if (!tok_shape(all[i], 1, w)) return ERROR_INCOMPATIBLE_DIMENSIONS;
  if (h > (1 << 24)) return ERROR_UNSUPPORTED;
  for (int i = 0; i < 6; ++i)
    if (!tok_apart(all[i], target) || !tok_apart(all[i], logp)) return ERROR_UNSUPPORTED;
  if (!tok_apart(target, logp)) return ERROR_UNSUPPORTED;
  if (w <= 0) return 0;
  int bits = 0;
  while ((1 << bits) < h) ++bits;
  const SampleArgs a = {mat->data_device, uniform->data_device, tok_data(temperature), tok_data(top_k), tok_data(top_p), tok_data(min_p), target->data_device,
                        tok_data(logp), all_temperature, all_top_k, all_top_p, all_min_p, h, w, 62 - bits < 45 ? 62 - bits : 45};
#define SAMPLE_GO(LANES, NV) hipLaunchKernelGGL((k_sample_tokens<LANES, NV>), dim3(w), dim3(LANES), 0, dn_stream(), a)
  if (h <= 1024) SAMPLE_GO(256, 1);
  else if (h <= 4096) SAMPLE_GO(256, 4);
  else if (h <= 16384) SAMPLE_GO(1024, 4);
  else if (h <= 32768) SAMPLE_GO(1024, 8);
  else if (h <= 65536) SAMPLE_GO(1024, 16);
  else SAMPLE_GO(1024, 0);
#undef SAMPLE_GO
  return dn_launch_status();
}
