// A gated linear recurrence along the columns of sequences, and its gradients (no counterpart in cudamat.cu).  With the halves g, u of
// pre and a = sigmoid(g):  h_t = a_t h_{t-1} + (1 - a_t) u_t.
#include "columns.h"
#include "gated_act.h"
#include "scan_launch.h"
#include "tokens.h"

struct ScanArgs {
  const float *pre, *offsets, *state, *deriv, *out, *last_deriv;
  float *target, *last, *state_grad;
  int f, w, n, each;               // units, columns, sequences; columns of each where there are no offsets
};

// The first column of sequence q, q <= n; numbers that are out of place stay within the matrix.
__device__ __forceinline__ int scan_border(const ScanArgs& a, int q) {
  if (!a.offsets) return q * a.each;
  const float o = a.offsets[q];
  return o > 0.f ? (o < (float)a.w ? (int)o : a.w) : 0;
}

// sigmoid(g), and 1 - it, by e = 2^t with t = -|g| log2(e): the hardware's exp2 of the rounded product, times 1 + ln 2 of what the rounding (and that of the constant)
// left; 1 / (1 + e) by its estimate and a Newton step.  Each about 2 ulp; below the normal range (|g| > 87) 0.  Fewer instructions than
// gate_sigmoid: the recurrence is bound by them (1024 x 32768 114 us with that one).
__device__ __forceinline__ float scan_gate(float g, float* other) {
#pragma clang fp contract(off)      // (`low` is what the rounding of p left)
  const float L2E = 1.44269502162933349609375f, c = fminf(fabsf(g), 128.f), p = c * -L2E;
  const float low = __fmaf_rn(c, -1.925963033500011e-08f, __fmaf_rn(c, -L2E, -p));
  float e = __builtin_amdgcn_exp2f(fabsf(g) * -L2E);       // (of NaN NaN, of infinity 0)
  e = __fmaf_rn(e * low, 0.693147180559945309f, e);
  const float d = 1.f + e;
  float r = __builtin_amdgcn_rcpf(d);
  r = __fmaf_rn(r, __fmaf_rn(-d, r, 1.f), r);
  const float q = e * r;
  *other = g > 0.f ? q : r;
  return g > 0.f ? r : q;
}

// What a stretch of columns does to what comes into it: h -> p h + b, or b alone where a sequence begins in it, which the sign of p says.
struct ScanLink { float p, b; };
__device__ __forceinline__ bool scan_cuts(float p) { return (int)__float_as_uint(p) < 0; }
__device__ __forceinline__ ScanLink scan_join(ScanLink first, ScanLink then) {       // (a sign stays in a product with p >= 0)
  return scan_cuts(then.p) ? then : ScanLink{first.p * then.p, __fmaf_rn(then.p, first.b, then.b)};
}
__device__ __forceinline__ float scan_through(ScanLink l, float h) { return scan_cuts(l.p) ? l.b : __fmaf_rn(l.p, h, l.b); }

// How a call is cut.  A workgroup has 2^shift units (16, 32 or 64; its lanes with the same unit are `strands`) and strands * S columns, S of them
// a lane: a chunk, counted in the direction in which the recurrence runs.
struct ScanCut {
  int shift, strands, chunks, tiles, first_tile;
  unsigned long long* words;       // of more than one chunk: SCAN_WORDS for the launch, then 128 for every link
};
#define SCAN_GROUP 16
#define SCAN_TILES 1024            // of one launch
#define SCAN_WORDS (16 * SCAN_TILES)   // a counter a tile, each in a memory line of its own
#define SCAN_POLLS (1 << 20)       // (a wait lasts some microseconds; one that lasts this long, about a second, gives NaN)

// Which launch this is, and which of a tile's workgroups.  A tile's counter has the launches in its upper 36 bits; the last place taken moves it on,
// and those of tiles that this launch does not have, so that all of them always agree on the launch.
struct ScanPlace { unsigned long long launch; int chunk; };
__device__ __forceinline__ ScanPlace scan_take_place(unsigned long long* counters, int tile, int tiles, int chunks, ScanPlace* shared) {
  if (threadIdx.x == 0) {
    const unsigned long long t = __hip_atomic_fetch_add(counters + 16 * tile, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *shared = ScanPlace{t >> 28, (int)(t & 0xfffffff)};
  }
  __syncthreads();
  const ScanPlace o = *shared;
  if (o.chunk == chunks - 1)
    for (int k = tile + threadIdx.x * tiles; k < SCAN_TILES; k += blockDim.x * tiles)
      __hip_atomic_store(counters + 16 * k, scan_next(o.launch) << 28, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return o;
}
// A link as two words that each have the launch's number in their upper half: the words need no order between them, and nothing is cleared (what is
// there from before has another number, but where it has stayed unwritten for exactly as many launches as there are numbers, 2^32 - 1).
__device__ __forceinline__ void scan_put(unsigned long long* at, ScanLink l, unsigned tag) {
  __hip_atomic_store(at, (unsigned long long)tag << 32 | __float_as_uint(l.p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __hip_atomic_store(at + 64, (unsigned long long)tag << 32 | __float_as_uint(l.b), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// `count` links, `stride` words apart, joined.  Two are on their way at once, and again until they are there.
__device__ __forceinline__ ScanLink scan_get(const unsigned long long* at, size_t stride, int count, unsigned tag) {
  ScanLink l = {1.f, 0.f};
  for (int k = 0; k < count; k += 2) {
    unsigned long long w[4];
    bool there = false;
    for (int i = 0; i < SCAN_POLLS && !there; ++i) {
      if (i) __builtin_amdgcn_s_sleep(1);
#pragma unroll
      for (int q = 0; q < 4; ++q) w[q] = __hip_atomic_load(at + (k + (q >> 1) < count ? k + (q >> 1) : k) * stride + (q & 1) * 64, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      there = true;
#pragma unroll
      for (int q = 0; q < 4; ++q) there &= (unsigned)(w[q] >> 32) == tag;
    }
    if (!there) return ScanLink{NAN, NAN};
    l = scan_join(l, ScanLink{__uint_as_float((unsigned)w[0]), __uint_as_float((unsigned)w[1])});
    if (k + 1 < count) l = scan_join(l, ScanLink{__uint_as_float((unsigned)w[2]), __uint_as_float((unsigned)w[3])});
  }
  return l;
}

// One read of the inputs, one write of the results.  A lane holds S columns of its unit and reduces them to a link; the strands' links meet in
// LDS; the chunk's link is published for the workgroups of the chunks behind it; what comes into the chunk is joined, in the order of the chunks, from
// the links of its group (SCAN_GROUP chunks) and the state that the group before has left.  So results do not depend on which workgroup comes first.
// A workgroup takes its place among those of its units from a counter when it starts: all places before it have been taken by workgroups that run, and those
// publish their links before they wait for anything, so every wait ends.  A chunk that begins with a sequence waits for nothing.
// GRAD: columns run backwards, from the last of a sequence to its first.  With x_t, the derivative by h_t from outside, what goes on to
// column t - 1 is a_t (x_t + what comes from t + 1): the same recurrence.
// WIDE: 64 units, a strand is a wavefront and its columns' addresses are scalars.
// Bytes: 12 an entry, backward 24.  1024 x 32768 94 us (4.3 TB/s), of which waiting for links is 20 (71 without, wrong); backward 2048 x 8192 81 us
// (5.0 TB/s), 72 without the waits.  What was measured on the way, forward: one counter for all tiles 168 (80 ns a workgroup), blocks joined one after the other 168
// and 45 at 64 x 65536 (19 with links of blocks), gates of 2 ulp by the general routine 115.  Rows that do not start at a memory line
// are fetched half as often again, by XCDs that have neighbouring tiles: backward 515 x 10007 42 us (18.9 by the bytes; 38 without waits).  Every workgroup reads all
// offsets: 1024 x 32768 in 256 ragged sequences 83 us, in 16384 174, 64 x 1048576 in 262144 2100.
template <int S, bool WIDE, bool GRAD, bool STREAM>
__global__ void __launch_bounds__(1024) k_gated_scan(ScanArgs a, ScanCut cut) {
  __shared__ ScanLink links[1024];
  constexpr int MOST = (WIDE ? 16 : 64) * S;
  __shared__ int firsts[MOST], ends[MOST];      // of every column: 1 + the sequence that begins or ends with it
  __shared__ ScanPlace place;
  const int tid = threadIdx.x, lanes = blockDim.x, units = WIDE ? 64 : 1 << cut.shift, strand = WIDE ? __builtin_amdgcn_readfirstlane(tid >> 6) : tid >> cut.shift, strands = cut.strands, columns = strands * S;
  // Workgroups that follow each other are on different XCDs: neighbouring tiles, which have memory lines in common where rows do not start at one, are taken by
  // the same XCD, as far as the tiles can be dealt out evenly (2001 x 4099 41 -> 37 us, backward 2003 x 10007 156 -> 138, rows that do start there the same).
  const int deal = cut.tiles >> 3, tile = cut.tiles & 7 ? blockIdx.x % cut.tiles : (int)((blockIdx.x & 7) * deal + (blockIdx.x >> 3) % deal);
  const int unit_in = tid & (units - 1), unit = ((cut.first_tile + tile) << cut.shift) + unit_in;
  int chunk = 0;
  unsigned tag = 0;
  if (cut.chunks > 1) {
    const ScanPlace o = scan_take_place(cut.words, tile, cut.tiles, cut.chunks, &place);
    if (o.chunk >= cut.chunks) return;                     // (only where calls overlap, which they may not)
    chunk = __builtin_amdgcn_readfirstlane(o.chunk);
    tag = __builtin_amdgcn_readfirstlane(scan_tag(o.launch));
  }
  const bool live = unit < a.f;
  const size_t f = a.f, i = live ? unit : a.f - 1;
  // the chunk's first column, and this lane's among them
  const long long from = (long long)(GRAD ? cut.chunks - 1 - chunk : chunk) * columns;
  const int own = strand * S;
  auto column = [&](int j) __attribute__((always_inline)) { const long long c = from + own + j; return (size_t)(c < a.w ? c : a.w - 1); };
  auto ld = [](const float* p) __attribute__((always_inline)) { return STREAM ? __builtin_nontemporal_load(p) : *p; };
  auto st = [](float* p, float v) __attribute__((always_inline)) { if (STREAM) __builtin_nontemporal_store(v, p); else *p = v; };
  float g[S], u[S], x[GRAD ? S : 1], d[GRAD ? S : 1];
#pragma unroll
  for (int j = 0; j < S; ++j) {
    const size_t c = column(j);
    g[j] = ld(a.pre + 2 * f * c + i);
    u[j] = ld(a.pre + 2 * f * c + f + i);
    if (GRAD) {
      x[j] = ld(a.deriv + f * c + i);
      d[j] = a.out[f * (c > 0 ? c - 1 : 0) + i];           // (before the first column of a sequence: the state, below)
    }
  }
  const int first_col = scan_border(a, 0), end_col = scan_border(a, a.n);
  for (int k = tid; k < columns; k += lanes) {
    int first = 0, end = 0;
    if (!a.offsets && from + k < a.w) {
      const int c = (int)from + k, q = c / a.each, r = c - q * a.each;
      if (r == 0) first = q + 1;
      if (r == a.each - 1) end = q + 1;
    }
    firsts[k] = first;
    ends[k] = end;
  }
  __syncthreads();
  if (a.offsets) {
    for (int q = tid; q < a.n; q += lanes) {
      const int b = scan_border(a, q), e = scan_border(a, q + 1);
      if (b < e) {
        if (b >= from && b < from + columns) firsts[b - from] = q + 1;
        if (e > from && e <= from + columns) ends[e - 1 - from] = q + 1;
      }
    }
    __syncthreads();
  }
  // bits of the lane's columns: a sequence begins there, ends there, the column is in one
  unsigned begins = 0, finishes = 0, inside = 0;
#pragma unroll
  for (int j = 0; j < S; ++j) {
    const long long c = from + own + j;
    begins |= firsts[own + j] ? 1u << j : 0;
    finishes |= ends[own + j] ? 1u << j : 0;
    inside |= c >= first_col && c < end_col ? 1u << j : 0;
  }
  if (WIDE) { begins = __builtin_amdgcn_readfirstlane(begins); finishes = __builtin_amdgcn_readfirstlane(finishes); inside = __builtin_amdgcn_readfirstlane(inside); }
  // what the states give
  if (GRAD ? begins | finishes : 0) {
#pragma unroll
    for (int j = 0; j < S; ++j) {
      if (GRAD && (begins >> j & 1)) d[j] = a.state ? a.state[(firsts[own + j] - 1) * f + i] : 0.f;
      if (GRAD && (finishes >> j & 1) && a.last_deriv) x[j] += a.last_deriv[(ends[own + j] - 1) * f + i];
    }
  }
  // g becomes a column's factor, its sign set where it takes nothing from the column before it, u (x) what it adds; columns of no sequence hand on what comes
  float s[GRAD ? S : 1];
#pragma unroll
  for (int j = 0; j < S; ++j) {
    float other;
    g[j] = scan_gate(g[j], &other);
    if (GRAD) { s[j] = other; d[j] -= u[j]; }
    else u[j] *= other;
  }
  const unsigned cuts = GRAD ? finishes : begins, whole = (unsigned)((1ull << S) - 1);
  if (cuts || inside != whole) {
#pragma unroll
    for (int j = 0; j < S; ++j) {
      if (!GRAD && (begins >> j & 1) && a.state) u[j] = __fmaf_rn(g[j], a.state[(firsts[own + j] - 1) * f + i], u[j]);
      if (cuts >> j & 1) g[j] = -g[j];
      if (!(inside >> j & 1)) { g[j] = 1.f; if (GRAD) x[j] = 0.f; else u[j] = 0.f; }
    }
  }
  ScanLink own_link = {1.f, 0.f};
  auto step = [&](float h, int j, bool may_cut) __attribute__((always_inline)) {
    const bool cut_here = may_cut && scan_cuts(g[j]);
    if (GRAD) return fabsf(g[j]) * (cut_here ? x[j] : x[j] + h);
    return cut_here ? u[j] : __fmaf_rn(g[j], h, u[j]);
  };
  if (cuts) {
#pragma unroll
    for (int k = 0; k < S; ++k) {
      const int j = GRAD ? S - 1 - k : k;
      own_link = ScanLink{scan_cuts(g[j]) ? -1.f : own_link.p * g[j], step(own_link.b, j, true)};
    }
  } else {
#pragma unroll
    for (int k = 0; k < S; ++k) {
      const int j = GRAD ? S - 1 - k : k;
      own_link = ScanLink{own_link.p * g[j], step(own_link.b, j, false)};
    }
  }
  const int order = GRAD ? strands - 1 - strand : strand;
  links[order * units + unit_in] = own_link;
  __syncthreads();
  ScanLink before = {1.f, 0.f};
  for (int k = 0; k < order; ++k) before = scan_join(before, links[k * units + unit_in]);
  float in = 0.f;
  if (cut.chunks > 1) {
    const bool last_strand = order == strands - 1;
    ScanLink total = scan_join(before, own_link), past = {1.f, 0.f};      // of the chunk (in the last strand), and of what has been seen before it
    unsigned long long* words = cut.words + SCAN_WORDS;
    auto put = [&](int block) __attribute__((always_inline)) {
      unsigned long long* w = words + ((size_t)block * cut.tiles + tile) * 128 + unit_in;
      scan_put(w, total, tag);
    };
    if (last_strand) put(chunk);
    const int edge = GRAD ? columns - 1 : 0;
    const bool alone = from + edge < first_col || from + edge >= end_col || (GRAD ? ends[edge] : firsts[edge]);
    // Blocks of 16 chunks, of 16 blocks and so on have links too, which the workgroup of their last chunk publishes.
    int at_level = chunk;
    bool closes = true;
    for (int blocks = cut.chunks; blocks > 1; blocks = (blocks + SCAN_GROUP - 1) / SCAN_GROUP) {
      const int group = at_level / SCAN_GROUP, m = alone ? 0 : at_level - group * SCAN_GROUP;
      if (m > 0) {
        const int each = (m + strands - 1) / strands, used = (m + each - 1) / each;
        const int mine = m - strand * each, count = mine < 0 ? 0 : mine < each ? mine : each;
        ScanLink l = scan_get(words + ((size_t)(group * SCAN_GROUP + strand * each) * cut.tiles + tile) * 128 + unit_in, (size_t)cut.tiles * 128, count, tag);
        __syncthreads();                                   // (the links there have been read)
        links[strand * units + unit_in] = l;
        __syncthreads();
        l = ScanLink{1.f, 0.f};
        for (int k = 0; k < used; ++k) l = scan_join(l, links[k * units + unit_in]);
        past = scan_join(l, past);
        total = scan_join(l, total);
      }
      words += (size_t)blocks * cut.tiles * 128;
      closes = closes && at_level - group * SCAN_GROUP == SCAN_GROUP - 1;
      if (closes && last_strand && blocks > SCAN_GROUP) put(group);
      if (alone && !closes) break;
      at_level = group;
    }
    in = scan_through(past, 0.f);
  }
  float h = scan_through(before, in);
  auto write = [&](bool plain) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < S; ++k) {
      const int j = GRAD ? S - 1 - k : k;
      const size_t c = (size_t)(from + own + j);
      const bool there = plain || (live && (inside >> j & 1));
      if (GRAD) {
        const float all = !plain && scan_cuts(g[j]) ? x[j] : x[j] + h, du = s[j] * all;
        h = fabsf(g[j]) * all;
        if (there) {
          st(a.target + 2 * f * c + i, d[j] * (s[j] * h));
          st(a.target + 2 * f * c + f + i, du);
        }
        x[j] = h;
      } else {
        h = step(h, j, !plain);
        if (there) st(a.target + f * c + i, h);
        u[j] = h;
      }
    }
  };
  if (!cuts && inside == whole && live) write(true);
  else write(false);
  // last columns, derivatives of states; those of sequences without columns
  float* const states = GRAD ? a.state_grad : a.last;
  const float* const handed = GRAD ? a.last_deriv : a.state;
  if (states && live) {
    const unsigned done = GRAD ? begins : finishes;
    if (done) {
#pragma unroll
      for (int j = 0; j < S; ++j)
        if (done >> j & 1) states[((GRAD ? firsts : ends)[own + j] - 1) * f + i] = GRAD ? x[j] : u[j];
    }
  }
  if (states && a.offsets) {         // every wavefront of a tile looks through some of the sequences
    const int each = WIDE ? strands : strands << cut.shift >> 6, waves = cut.chunks * each;
    const int wave = chunk * each + (WIDE ? strand : __builtin_amdgcn_readfirstlane(strand << cut.shift >> 6));
    const int batch = (a.n + waves - 1) / waves < 64 ? (a.n + waves - 1) / waves : 64;
    for (long long q0 = (long long)batch * wave; q0 < a.n; q0 += (long long)batch * waves) {
      const int l = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0)), q = (int)q0 + l;
      unsigned long long none = __ballot(l < batch && q < a.n && scan_border(a, q < a.n ? q : a.n) >= scan_border(a, q < a.n ? q + 1 : a.n));
      while (none) {                 // two on their way at once (the first one again in the place of one that is not there)
        const size_t x = (size_t)(q0 + __builtin_ctzll(none)) * f + i;
        none &= none - 1;
        const size_t y = none ? (size_t)(q0 + __builtin_ctzll(none)) * f + i : x;
        none &= none - 1;            // (0 & -1: stays 0)
        const float v = handed ? handed[x] : 0.f, w = handed ? handed[y] : 0.f;
        if (live) { states[x] = v; states[y] = w; }
      }
    }
  }
}

// Sequences without any columns: states go through.
__global__ void __launch_bounds__(256) k_scan_states(const float* from, float* to, long long n) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i < n) to[i] = from ? from[i] : 0.f;
}

template <bool GRAD>
static int scan_launch(const ScanArgs& a) {
  if (a.w <= 0) {
    float* to = GRAD ? a.state_grad : a.last;
    const long long n = (long long)a.f * a.n;
    const float* from = GRAD ? a.last_deriv : a.state;
    const long long most = 256 * DN_MAX_GROUPS;
    for (long long i = 0; to && i < n; i += most)
      hipLaunchKernelGGL(k_scan_states, dim3((unsigned)(((n - i < most ? n - i : most) + 255) / 256)), dim3(256), 0, dn_stream(), from ? from + i : from, to + i, n - i);
    return dn_launch_status();
  }
  ScanCut cut;
  cut.shift = a.f <= 16 ? 4 : a.f <= 32 ? 5 : 6;
  const int tiles = (int)(((long long)a.f + (1 << cut.shift) - 1) >> cut.shift);
  // Strands are whole wavefronts, of at most 1024 lanes.
  const int least = 64 >> cut.shift;
  auto fit = [&](int s, int strands) {
    const long long want = (((long long)a.w + s - 1) / s + least - 1) / least * least;
    cut.strands = want < strands ? (int)want : strands;
    cut.chunks = (int)(((long long)a.w + (long long)cut.strands * s - 1) / ((long long)cut.strands * s));
    return s;
  };
  // Long chunks have fewer links to wait for, short ones give more workgroups, and the registers of S columns decide how many a CU has (us, S x strands, forward:
  // 1024 x 32768 16 x 16 103, 16 x 8 94, 8 x 8 123, 32 x 8 116; 2048 x 256 16 x 8 7.8, 8 x 8 6.6, 16 x 16 8.3; 512 x 2048 9.2, 8.9, 11.5.  Backward, whose
  // columns take twice the registers: 2048 x 8192 16 x 8 91, 8 x 8 85, 8 x 12 81, 8 x 16 89; 2048 x 256 8 x 8 7.5, 8 x 12 8.2).
  const bool wide = cut.shift == 6;
  int s;
  auto groups = [&] { return (long long)cut.chunks * tiles; };
  if (!wide) s = fit(4, 1024 >> cut.shift);
  else if (a.w <= 16) s = fit(1, 16);
  else if (a.w <= 64) s = fit(4, 16);
  else if (GRAD) { s = fit(8, 12); if (groups() < 2 * dn_num_cus()) s = fit(8, 8); }
  else { s = fit(16, 8); if (groups() < dn_num_cus()) s = fit(8, 8); }
  cut.words = nullptr;
  const int most_tiles = tiles < SCAN_TILES ? tiles : SCAN_TILES;
  if (cut.chunks > 1) {
    if (cut.chunks >= 1 << 28) return ERROR_UNSUPPORTED;
    size_t links = 0;
    for (size_t blocks = cut.chunks; blocks > 1; blocks = (blocks + SCAN_GROUP - 1) / SCAN_GROUP) links += blocks * most_tiles;
    cut.words = dn_tagged_words(SCAN_WORDS + links * 128);
    if (!cut.words) return CUDA_ERROR;
  }
  const bool stream = (long long)a.f * a.w >= DN_STREAM_MIN_ELEMS;
  for (cut.first_tile = 0; cut.first_tile < tiles; cut.first_tile += most_tiles) {
    cut.tiles = tiles - cut.first_tile < most_tiles ? tiles - cut.first_tile : most_tiles;
    const dim3 block((unsigned)(cut.strands << cut.shift));
    // (what one launch does not take goes on in the next: workgroups have the chunks in the order in which they start)
    const long long most = ((1ll << 32) - 1) / block.x / cut.tiles;
    for (long long c0 = 0; c0 < cut.chunks; c0 += most) {
      const dim3 grid((unsigned)((cut.chunks - c0 < most ? cut.chunks - c0 : most) * cut.tiles));
#define SCAN_GO(S, WIDE) do { if (stream) hipLaunchKernelGGL((k_gated_scan<S, WIDE, GRAD, true>), grid, block, 0, dn_stream(), a, cut); \
                              else hipLaunchKernelGGL((k_gated_scan<S, WIDE, GRAD, false>), grid, block, 0, dn_stream(), a, cut); } while (0)
      if (!wide) SCAN_GO(4, false);
      else if (s == 1) SCAN_GO(1, true);
      else if (s == 4) SCAN_GO(4, true);
      else if (s == 8) SCAN_GO(8, true);
      else if constexpr (!GRAD) SCAN_GO(16, true);
#undef SCAN_GO
    }
  }
  return dn_launch_status();
}

// Sequences: as many as are asked for, or (0) as the offsets or the states tell, or one.
static int scan_sequences(int asked, const cudamat* offsets, const cudamat* s0, const cudamat* s1, const cudamat* s2) {
  if (asked) return asked;
  if (offsets) return offsets->size[1] - 1;
  for (const cudamat* s : {s0, s1, s2})
    if (s) return s->size[1];
  return 1;
}

// Offsets are floats, and the kernel steps through the sequences by up to 2^22.
static bool scan_beyond(const cudamat* offsets, int w, int n) { return offsets && (w > (1 << 24) || (w > 0 && n > (1 << 30))); }

extern "C" {

int gated_scan(cudamat* pre, cudamat* offsets, cudamat* state, cudamat* target, cudamat* last, int sequences) {
  cudamat* const all[5] = {pre, offsets, state, target, last};
  if (int e = tok_check_device(all)) return e;
  const int f = target->size[0], w = target->size[1], n = scan_sequences(sequences, offsets, state, last, nullptr);
  if (pre->size[0] != 2 * (long long)f || pre->size[1] != w || n < 1 || !tok_shape(offsets, 1, n + 1) || (!offsets && w % n) ||
      !tok_shape(state, f, n) || !tok_shape(last, f, n))
    return ERROR_INCOMPATIBLE_DIMENSIONS;
  if (!tok_apart(pre, target) || !tok_apart(offsets, target) || !tok_apart(state, target) || !tok_apart(pre, last) || !tok_apart(offsets, last) ||
      !tok_apart(target, last) || (state && last && !tok_same_or_apart(state, last)) || scan_beyond(offsets, w, n))
    return ERROR_UNSUPPORTED;
  if (f <= 0 || (w <= 0 && !last)) return 0;
  const ScanArgs a = {pre->data_device, tok_data(offsets), tok_data(state), nullptr, nullptr, nullptr, target->data_device, tok_data(last), nullptr, f, w, n, w / n};
  return scan_launch<false>(a);
}

int gated_scan_grad(cudamat* deriv, cudamat* pre, cudamat* out, cudamat* offsets, cudamat* state, cudamat* last_deriv, cudamat* target,
                    cudamat* state_grad, int sequences) {
  cudamat* const all[8] = {deriv, pre, out, offsets, state, last_deriv, target, state_grad};
  if (int e = tok_check_device(all)) return e;
  const int f = deriv->size[0], w = deriv->size[1], n = scan_sequences(sequences, offsets, state, last_deriv, state_grad);
  if (pre->size[0] != 2 * (long long)f || pre->size[1] != w || !tok_shape(out, f, w) || target->size[0] != pre->size[0] || target->size[1] != w || n < 1 ||
      !tok_shape(offsets, 1, n + 1) || (!offsets && w % n) || !tok_shape(state, f, n) || !tok_shape(last_deriv, f, n) || !tok_shape(state_grad, f, n))
    return ERROR_INCOMPATIBLE_DIMENSIONS;
  if (!tok_same_or_apart(pre, target) || (last_deriv && state_grad && !tok_same_or_apart(last_deriv, state_grad)) || !tok_apart(pre, state_grad) ||
      !tok_apart(target, state_grad) || !tok_apart(last_deriv, target) || scan_beyond(offsets, w, n))
    return ERROR_UNSUPPORTED;
  for (const cudamat* m : {deriv, out, offsets, state})
    if (!tok_apart(m, target) || !tok_apart(m, state_grad)) return ERROR_UNSUPPORTED;
  if (f <= 0 || (w <= 0 && !state_grad)) return 0;
  const ScanArgs a = {pre->data_device, tok_data(offsets), tok_data(state), deriv->data_device, out->data_device, tok_data(last_deriv),
                      target->data_device, nullptr, tok_data(state_grad), f, w, n, w / n};
  return scan_launch<true>(a);
}

}  // extern "C"
