// Columns of a table by token, and the gradient of the table (no counterpart in cudamat.cu; selectRows has no scale and gives NaN for what is
// no token, accumulate_columns is for up to 512 columns).
#include "columns.h"
#include "tokens.h"

// ------------------------------------------------------------------ lookup
// target(:, c) = mult * mat(:, labels[c]), 0 where that is no token.  A lane has four groups of four rows (W = 1: rows) of the target on their way, at any 4-byte
// boundary; the last group of a column starts at h - 4, and rows that it has in common with the one before get the same value twice.
template <int W, bool STREAM>
__global__ void __launch_bounds__(256) k_embed(const float* mat, const float* labels, float* target, int h, int n, uint32_t groups, uint32_t total, FastDiv div, float mult) {
  const uint32_t first = blockIdx.x * 1024u + threadIdx.x;
  int t[4];
  uint32_t c[4], r[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t g = first + 256u * k < total ? first + 256u * k : total - 1;
    c[k] = fd_div(g, div);
    r[k] = (g - c[k] * groups) * W;
    if (W == 4 && r[k] + 4 > (uint32_t)h) r[k] = h - 4;
    t[k] = tok_label(labels[c[k]], n);
  }
  float v[4][4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float* p = mat + (size_t)(t[k] < 0 ? 0 : t[k]) * h + r[k];
    if (W == 4) col_load<false>(v[k], p);
    else v[k][0] = *p;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (first + 256u * k >= total) break;
    float* p = target + (size_t)c[k] * h + r[k];
#pragma unroll
    for (int e = 0; e < W; ++e) v[k][e] = t[k] < 0 ? 0.f : mult * v[k][e];
    if (W == 4) col_store<STREAM>(p, v[k]);
    else *p = v[k][0];
  }
}

// ------------------------------------------------------------------ gradient of the table
// Columns are first sorted by token (k_embed_sort), then every token's run of columns is added up (k_embed_sums), long runs in pieces whose
// sums k_embed_join adds: every order of addition follows from the labels alone.  Of a token with n > 16 columns a piece is up to sqrt(n / 2) of them, one
// after the other (n <= 2048: 16), and then up to sqrt(8 n) sums of pieces are added likewise, in 32 bits: at most 4608 roundings in a row for 2^21 columns.  In one launch
// (k_embed_few) these are n / 16 and 16, of up to 64 rows n / 64 and 64.
#define EMBED_RUN 16               // columns that one team adds for a token
#define EMBED_SLOT 8               // one slot for as many sorted columns: a run of more than EMBED_RUN has at least as many slots as pieces
#define EMBED_RANGE 512            // tokens of a workgroup that sorts
// The pieces of a long run: their length grows with the run, so that neither they nor their number get long (2048 columns: 128 pieces of 16, 2^21: 4096 of 512).
__device__ __forceinline__ int embed_piece(int count) {
  long long c = EMBED_RUN;
  while (8 * c * c < count) c *= 2;
  return (int)c;
}
__device__ __forceinline__ int embed_slot(int sorted) { return (int)(((unsigned)sorted + EMBED_SLOT - 1) / EMBED_SLOT); }

// Of the lanes in `all`, those with the same x (of `bits` bits): how many are before this one, and how many there are.  (The whole wavefront is here.)
__device__ __forceinline__ void embed_same(unsigned long long all, int x, int bits, int* rank, int* count) {
  unsigned lo = (unsigned)all, hi = (unsigned)(all >> 32);
  for (int b = 0; b < bits; ++b) {
    const int bit = (int)((unsigned)x << (31 - b)) >> 31;  // 0 or -1
    const unsigned long long set = __ballot(bit);
    lo &= ~((unsigned)set ^ bit);
    hi &= ~((unsigned)(set >> 32) ^ bit);
  }
  *rank = __builtin_amdgcn_mbcnt_hi(hi, __builtin_amdgcn_mbcnt_lo(lo, 0));
  *count = __popc(lo) + __popc(hi);
}

struct EmbedSlot { int from, count, token, pieces; };      // a piece of a long run; pieces: of its first one, how many there are (0 in the others)
struct EmbedSort {
  const float* labels;
  int w, n, range;                 // range: tokens of a workgroup
  int *starts, *sorted;            // of every token (and behind the last one) where its run begins; the columns in the order of their tokens
  EmbedSlot* slots;
};

// A workgroup sorts the columns of `range` tokens: it reads all labels, counts those below its range (where its columns begin) and, by
// wavefronts, each of which has a stretch of the columns, those of every token in it; then it goes through the labels again (up to 32768 stay in
// registers) and writes the columns down: by stretches, of 256 columns every fourth one first.  The labels come from the L2s; the workgroup of the most
// frequent tokens takes longest.  16384 columns of 32003 tokens 16 us, 32768 of 131072 28; with 4-byte loads 20 and 37, with a turn a token instead of its bits
// 40 and 171.  A call of 1024 x 16384 onto 32003 tokens 59 us: this, 38 for the sums (30 by the bytes) and 6 for the long runs.
__global__ void __launch_bounds__(1024) k_embed_sort(EmbedSort a) {
  __shared__ int counts[16][EMBED_RANGE], starts[EMBED_RANGE + 1], waves[2][16];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), lo = blockIdx.x * a.range;
  const int size = a.n - lo < a.range ? a.n - lo : a.range;
  const long long per = ((long long)a.w + 4095) / 4096 * 256, from = wv * per, to = from + per < a.w ? from + per : a.w;
  for (int k = tid; k < 16 * EMBED_RANGE; k += 1024) (&counts[0][0])[k] = 0;
  __syncthreads();
  float l[8][4];                     // labels of 2048 columns
  auto fetch = [&](long long c0) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const long long c = c0 + 256 * k + 4 * lane;
#pragma unroll
      for (int e = 0; e < 4; ++e) l[k][e] = -1.f;
      if (c0 + 256 * k >= to) continue;
      if (c + 4 <= to) col_load<false>(l[k], a.labels + c);
      else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
          if (c + e < to) l[k][e] = a.labels[c + e];
      }
    }
  };
  const float first = (float)lo, behind = (float)(lo + size);            // (whole numbers up to 2^24)
  int below = 0;                     // (of the wavefront)
  for (long long c0 = from; c0 < to; c0 += 2048) {
    fetch(c0);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (c0 + 256 * k >= to) break;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = l[k][e];
        if (x >= first && x < behind) atomicAdd(&counts[wv][(int)x - lo], 1);
        below += __popcll(__ballot(x >= 0.f && x < first));
      }
    }
  }
  if (lane == 0) waves[0][wv] = below;
  __syncthreads();
  int mine = 0, base = 0;
  if (tid < EMBED_RANGE)
    for (int k = 0; k < 16; ++k) mine += counts[k][tid];
  for (int k = 0; k < 16; ++k) base += waves[0][k];
  int up = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) { const int q = __shfl_up(up, o, WAVE); if (lane >= o) up += q; }
  if (lane == 63) waves[1][wv] = up;
  __syncthreads();
  int start = base + up - mine;
  for (int k = 0; k < wv; ++k) start += waves[1][k];
  if (tid < EMBED_RANGE) {
    starts[tid] = start;
    if (tid < size) a.starts[lo + tid] = start;
    if (tid == EMBED_RANGE - 1) starts[EMBED_RANGE] = start + mine;
    if (tid < size && lo + tid == a.n - 1) a.starts[a.n] = start + mine;
    for (int k = 0, at = start; k < 16; ++k) { const int q = counts[k][tid]; counts[k][tid] = at; at += q; }
  }
  __syncthreads();
  // the slots of these runs: the last token whose first slot is not behind it has it
  const int end = starts[EMBED_RANGE];
  for (int q = embed_slot(base) + tid; q < embed_slot(end); q += 1024) {
    int x = 0;
    for (int step = EMBED_RANGE / 2; step > 0; step /= 2)
      if (embed_slot(starts[x + step]) <= q) x += step;
    const int s = starts[x], count = starts[x + 1] - s, piece = embed_piece(count), k = q - embed_slot(s), pieces = (int)(((unsigned)count + piece - 1) / piece);
    EmbedSlot o = {0, 0, 0, 0};
    if (count > EMBED_RUN && k < pieces) o = EmbedSlot{s + k * piece, count - k * piece < piece ? count - k * piece : piece, lo + x, k ? 0 : pieces};
    a.slots[q] = o;
  }
  // lanes of the same token find each other by its bits
  volatile int* const next = counts[wv];
  const int bits = 32 - __builtin_clz(a.range);
  for (long long c0 = from; c0 < to; c0 += 2048) {
    if (per > 2048) fetch(c0);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (c0 + 256 * k >= to) break;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = l[k][e] >= first && l[k][e] < behind;
        const unsigned long long all = __ballot(in);
        if (all == 0) continue;
        const int x = in ? (int)l[k][e] - lo : 0;
        int rank, count;
        embed_same(all, x, bits, &rank, &count);
        if (in) {
          const int at = next[x];
          a.sorted[at + rank] = (int)(c0 + 256 * k + 4 * lane + e);
          if (rank == 0) next[x] = at + count;
        }
      }
    }
  }
}

struct EmbedSums {
  const float* deriv;
  float *target, *partials;        // partials: h a slot
  const int *starts, *sorted;
  const EmbedSlot* slots;
  int h, n, slot_count, tiles, rows;      // rows of a tile
  unsigned first;                  // item of a launch
  float beta, mult;
};
// A team (T lanes, NV groups of W rows each) and its rows of a column.
template <int T, int NV, int W, bool TAIL>
struct EmbedRows {
  ColGroups<NV, TAIL> at;
  __device__ __forceinline__ void init(int lane, int h) {
    if (W == 4) at.init(lane, T, h);
    else { at.row[0] = lane < h ? lane : h - 1; at.in[0] = lane < h; at.lap = 0; at.last = -1; }
  }
  template <bool STREAM>
  __device__ __forceinline__ void load(float (&v)[NV][4], const float* p) const {
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (W == 4) col_load<STREAM>(v[k], p + at.row[k]);
      else v[k][0] = p[at.row[k]];
  }
  template <bool STREAM>
  __device__ __forceinline__ void store(float* p, const float (&v)[NV][4]) const {
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (at.in[k]) {
        if (W == 4) col_store_group<STREAM, true>(at, k, p, v[k]);
        else p[at.row[k]] = v[k][0];
      }
  }
};
template <int NV, int W>
__device__ __forceinline__ void embed_add(float (&sum)[NV][4], const float (&v)[NV][4]) {
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < W; ++e) sum[k][e] += v[k][e];
}
// beta * old + mult * sum in the place of old (which is not read for beta = 0)
template <int T, int NV, int W, bool TAIL, bool STREAM>
__device__ __forceinline__ void embed_out(const EmbedRows<T, NV, W, TAIL>& rows, float* p, float (&sum)[NV][4], float beta, float mult) {
  float old[NV][4];
  if (beta != 0.f) rows.template load<STREAM>(old, p);
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < W; ++e) sum[k][e] = beta != 0.f ? __fmaf_rn(mult, sum[k][e], beta * old[k][e]) : mult * sum[k][e];
  rows.template store<STREAM>(p, sum);
}

// A team for every slot, then one for every token: the sum of a piece of a long run goes to the partial sums, that of a short run to the target,
// as does what a token without columns gets.  Four columns are on their way at once.  Bytes: the columns and, with beta = 0, the table.
template <int T, int NV, int W, bool TAIL, bool STREAM>
__global__ void __launch_bounds__(256) k_embed_sums(EmbedSums a) {
  const unsigned item = a.first + blockIdx.x * (256 / T) + (T == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / T) : threadIdx.x / T);
  const unsigned which = item / a.tiles, tile = item - which * a.tiles;
  if (which >= (unsigned)a.slot_count + a.n) return;
  const int row0 = tile * a.rows;
  EmbedRows<T, NV, W, TAIL> rows;
  rows.init(threadIdx.x % T, a.h - row0 < a.rows ? a.h - row0 : a.rows);
  int from, count;
  float* out;
  const bool piece = which < (unsigned)a.slot_count;
  if (piece) {
    if ((int)which >= embed_slot(a.starts[a.n])) return;   // (no columns that far)
    const EmbedSlot s = a.slots[which];
    from = s.from; count = s.count;
    if (count == 0) return;
    out = a.partials + (size_t)which * a.h + row0;
  } else {
    const int t = which - a.slot_count;
    from = a.starts[t];
    count = a.starts[t + 1] - from;
    if (count > EMBED_RUN || (count == 0 && a.beta == 1.f)) return;
    out = a.target + (size_t)t * a.h + row0;
  }
  float sum[NV][4];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[k][e] = 0.f;
  const float* const deriv = a.deriv + row0;
  int k = 0;
  for (; k + 4 <= count; k += 4) {
    float v[4][NV][4];
#pragma unroll
    for (int q = 0; q < 4; ++q) rows.template load<STREAM>(v[q], deriv + (size_t)a.sorted[from + k + q] * a.h);
#pragma unroll
    for (int q = 0; q < 4; ++q) embed_add<NV, W>(sum, v[q]);
  }
  if (k < count) {                                         // up to three more: the last one again in the place of those that are not there
    float v[3][NV][4];
#pragma unroll
    for (int q = 0; q < 3; ++q) rows.template load<STREAM>(v[q], deriv + (size_t)a.sorted[from + (k + q < count ? k + q : count - 1)] * a.h);
#pragma unroll
    for (int q = 0; q < 3; ++q)
      if (k + q < count) embed_add<NV, W>(sum, v[q]);
  }
  if (piece) rows.template store<false>(out, sum);
  else embed_out<T, NV, W, TAIL, STREAM>(rows, out, sum, a.beta, a.mult);
}

// The sums of the pieces of every long run, in their order, sixteen on their way at once.
template <int T, int W, bool TAIL>
__global__ void __launch_bounds__(256) k_embed_join(EmbedSums a) {
  const unsigned item = a.first + blockIdx.x * (256 / T) + (T == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / T) : threadIdx.x / T);
  const unsigned which = item / a.tiles, tile = item - which * a.tiles;
  if (which >= (unsigned)a.slot_count || (int)which >= embed_slot(a.starts[a.n])) return;
  const EmbedSlot s = a.slots[which];
  if (s.pieces == 0) return;
  const int row0 = tile * a.rows;
  EmbedRows<T, 1, W, TAIL> rows;
  rows.init(threadIdx.x % T, a.h - row0 < a.rows ? a.h - row0 : a.rows);
  float sum[1][4] = {{0.f, 0.f, 0.f, 0.f}};
  const float* p = a.partials + (size_t)which * a.h + row0;
  for (int k = 0; k < s.pieces; k += 16) {
    float v[16][1][4];
#pragma unroll
    for (int q = 0; q < 16; ++q) rows.template load<false>(v[q], p + (size_t)(k + q < s.pieces ? k + q : s.pieces - 1) * a.h);
#pragma unroll
    for (int q = 0; q < 16; ++q)
      if (k + q < s.pieces) embed_add<1, W>(sum, v[q]);
  }
  embed_out<T, 1, W, TAIL, false>(rows, a.target + (size_t)s.token * a.h + row0, sum, a.beta, a.mult);
}

// Few columns (at most EMBED_FEW): one launch.  A workgroup has a range of tokens and, of the table, 256 rows (T = 16: 64): it sorts its columns in LDS, its teams
// take the tokens of up to EMBED_RUN columns in turn, and all of them share those of more, whose parts meet in LDS in their order.
// 1001 x 4099 of 256 tokens 13 us (as three launches 18).
#define EMBED_FEW 8192
#define EMBED_FEW_RANGE 8
template <int T, int W, bool TAIL, bool STREAM>
__global__ void __launch_bounds__(1024) k_embed_few(EmbedSort a, EmbedSums b) {
  constexpr int WAVES = 16, TEAMS = 1024 / T, PER = EMBED_FEW / WAVES / 256;
  __shared__ int counts[WAVES][EMBED_FEW_RANGE], starts[EMBED_FEW_RANGE + 1], waves[WAVES], longs[EMBED_FEW_RANGE], long_count;
  __shared__ unsigned short list[EMBED_FEW];
  __shared__ float parts[TEAMS][T * 4];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int range = blockIdx.x / b.tiles, tile = blockIdx.x - range * b.tiles, lo = range * a.range, size = a.n - lo < a.range ? a.n - lo : a.range;
  const int per = (a.w + WAVES * 256 - 1) / (WAVES * 256) * 256, from = wv * per, to = from + per < a.w ? from + per : a.w;
  float l[PER][4];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int c = from + 256 * k + 4 * lane;
#pragma unroll
    for (int e = 0; e < 4; ++e) l[k][e] = -1.f;
    if (256 * k >= per) continue;
    if (c + 4 <= to) col_load<false>(l[k], a.labels + c);
    else {
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (c + e < to) l[k][e] = a.labels[c + e];
    }
  }
  for (int k = tid; k < WAVES * EMBED_FEW_RANGE; k += 1024) (&counts[0][0])[k] = 0;
  if (tid == 0) long_count = 0;
  __syncthreads();
  const float first = (float)lo, behind = (float)(lo + size);
#pragma unroll
  for (int k = 0; k < PER; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (l[k][e] >= first && l[k][e] < behind) atomicAdd(&counts[wv][(int)l[k][e] - lo], 1);
  __syncthreads();
  int mine = 0;
  if (tid < size)
    for (int k = 0; k < WAVES; ++k) mine += counts[k][tid];
  int up = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) { const int q = __shfl_up(up, o, WAVE); if (lane >= o) up += q; }
  if (lane == 63) waves[wv] = up;
  __syncthreads();
  int start = up - mine;
  for (int k = 0; k < wv; ++k) start += waves[k];
  if (tid < size) {
    starts[tid] = start;
    if (tid == size - 1) starts[size] = start + mine;
    if (mine > EMBED_RUN) longs[atomicAdd(&long_count, 1)] = tid;
    for (int k = 0, at = start; k < WAVES; ++k) { const int q = counts[k][tid]; counts[k][tid] = at; at += q; }
  }
  __syncthreads();
  volatile int* const next = counts[wv];
  const int bits = 32 - __builtin_clz(a.range);
#pragma unroll
  for (int k = 0; k < PER; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool in = l[k][e] >= first && l[k][e] < behind;
      const unsigned long long all = __ballot(in);
      if (all == 0) continue;
      const int x = in ? (int)l[k][e] - lo : 0;
      int rank, count;
      embed_same(all, x, bits, &rank, &count);
      if (in) {
        const int at = next[x];
        list[at + rank] = (unsigned short)(from + 256 * k + 4 * lane + e);
        if (rank == 0) next[x] = at + count;
      }
    }
  __syncthreads();
  const int row0 = tile * b.rows, team = T == 64 ? wv : tid / T;
  EmbedRows<T, 1, W, TAIL> rows;
  rows.init(tid % T, b.h - row0 < b.rows ? b.h - row0 : b.rows);
  const float* const deriv = b.deriv + row0;
  auto add = [&](float (&sum)[1][4], int at, int count) __attribute__((always_inline)) {
    for (int k = 0; k < count; k += 8) {                  // (the last one again in the place of those that are not there)
      float v[8][1][4];
#pragma unroll
      for (int q = 0; q < 8; ++q) rows.template load<STREAM>(v[q], deriv + (size_t)list[at + (k + q < count ? k + q : count - 1)] * b.h);
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (k + q < count) embed_add<1, W>(sum, v[q]);
    }
  };
  for (int t = team; t < size; t += TEAMS) {
    const int at = starts[t], count = starts[t + 1] - at;
    if (count > EMBED_RUN || (count == 0 && b.beta == 1.f)) continue;
    float sum[1][4] = {{0.f, 0.f, 0.f, 0.f}};
    add(sum, at, count);
    embed_out<T, 1, W, TAIL, STREAM>(rows, b.target + (size_t)(lo + t) * b.h + row0, sum, b.beta, b.mult);
  }
  const int many = long_count;
  for (int i = 0; i < many; ++i) {
    const int t = longs[i], at = starts[t], count = starts[t + 1] - at, each = (count + TEAMS - 1) / TEAMS, used = (count + each - 1) / each;
    float sum[1][4] = {{0.f, 0.f, 0.f, 0.f}};
    if (team < used) add(sum, at + team * each, count - team * each < each ? count - team * each : each);
#pragma unroll
    for (int e = 0; e < W; ++e) parts[team][tid % T * W + e] = sum[0][e];
    __syncthreads();
    if (team == i % TEAMS) {
      for (int k = 0; k < used; ++k)
#pragma unroll
        for (int e = 0; e < W; ++e) sum[0][e] = k ? sum[0][e] + parts[k][tid % T * W + e] : parts[0][tid % T * W + e];
      embed_out<T, 1, W, TAIL, false>(rows, b.target + (size_t)(lo + t) * b.h + row0, sum, b.beta, b.mult);
    }
    __syncthreads();
  }
}

// Tiles of at most `most` rows, a multiple of four; the last one has a group of four rows too.
static void embed_tiles(EmbedSums& s, int most) {
  const long long h = s.h;         // (h + most may pass 31 bits)
  long long tiles = (h + most - 1) / most, rows = tiles > 1 ? ((h + tiles - 1) / tiles + 3) / 4 * 4 : h;
  while (tiles > 1 && h % rows && h % rows < 4) rows -= 4;
  s.tiles = (int)((h + rows - 1) / rows);
  s.rows = (int)rows;
}

extern "C" {

int embed(cudamat* mat, cudamat* labels, cudamat* target, float mult) {
  cudamat* const all[3] = {mat, labels, target};
  if (int e = tok_check_device(all)) return e;
  const int h = mat->size[0], n = mat->size[1], w = target->size[1];
  if (target->size[0] != h || !tok_shape(labels, 1, w)) return ERROR_INCOMPATIBLE_DIMENSIONS;
  if (n > (1 << 24) || !tok_apart(mat, target) || !tok_apart(labels, target)) return ERROR_UNSUPPORTED;
  if (h <= 0 || w <= 0) return 0;
  const bool by4 = h >= 4, stream = (long long)h * w >= DN_STREAM_MIN_ELEMS;
  const uint32_t groups = by4 ? ((uint32_t)h + 3) / 4 : h;                              // (h + 3 may pass 31 bits)
  const FastDiv div = make_fastdiv(groups);
  const float* const from = n > 0 ? mat->data_device : target->data_device;            // (lanes without a token read its first entries)
  const long long most = (1ll << 31) / groups > 0 ? (1ll << 31) / groups : 1;           // columns of a launch
  for (long long c0 = 0; c0 < w; c0 += most) {
    const long long cols = w - c0 < most ? w - c0 : most, total = cols * groups;
    const dim3 grid((unsigned)((total + 1023) / 1024));
#define EMBED_GO(W, S) hipLaunchKernelGGL((k_embed<W, S>), grid, dim3(256), 0, dn_stream(), from, (const float*)labels->data_device + c0, \
                                          target->data_device + c0 * h, h, n, groups, (uint32_t)total, div, mult)
    if (!by4) EMBED_GO(1, false);
    else if (stream) EMBED_GO(4, true);
    else EMBED_GO(4, false);
#undef EMBED_GO
  }
  return dn_launch_status();
}

int embed_grad(cudamat* deriv, cudamat* labels, cudamat* target, float beta, float mult) {
  cudamat* const all[3] = {deriv, labels, target};
  if (int e = tok_check_device(all)) return e;
  const int h = deriv->size[0], n = target->size[1], w = deriv->size[1];
  if (target->size[0] != h || !tok_shape(labels, 1, w)) return ERROR_INCOMPATIBLE_DIMENSIONS;
  if (n > (1 << 24) || !tok_apart(deriv, target) || !tok_apart(labels, target)) return ERROR_UNSUPPORTED;
  if (h <= 0 || n <= 0) return 0;
  EmbedSums s;
  s.deriv = deriv->data_device; s.target = target->data_device; s.h = h; s.n = n; s.beta = beta; s.mult = mult;
  const bool stream = (long long)h * (w > n ? w : n) >= DN_STREAM_MIN_ELEMS;
  EmbedSort o;
  o.labels = labels->data_device; o.w = w; o.n = n;
  embed_tiles(s, h <= 64 ? 64 : 256);
  // One launch while the frequent tokens, which a workgroup has by itself, are not many columns (us, three launches / one: 1024 x 64 of 256 tokens 10.4 / 5.8, x 4000
  // 16.6 / 12.7, x 6000 21.6 / 21.5, x 8000 24.5 / 27.4; 64 x 8000 of 1000 18.4 / 11.2; 4096 x 1000 of 200 16.0 / 14.1, x 4000 30.3 / 38.7).  Fewer workgroups for few
  // columns (1024 x 64 in 1024 8.6, x 4000 in 512 15.4).
  if (w <= EMBED_FEW && (long long)h * w <= 1 << 22 && (long long)n * s.tiles <= 4096) {
    const int want = w <= 512 ? 512 : 1024;
    o.range = (int)(((long long)n * s.tiles + want - 1) / want);
    const long long groups = (long long)((n + o.range - 1) / o.range) * s.tiles;
#define FEW2(T, W, TAIL) do { if (stream) hipLaunchKernelGGL((k_embed_few<T, W, TAIL, true>), dim3((unsigned)groups), dim3(1024), 0, dn_stream(), o, s); \
                              else hipLaunchKernelGGL((k_embed_few<T, W, TAIL, false>), dim3((unsigned)groups), dim3(1024), 0, dn_stream(), o, s); } while (0)
#define FEW(T, W) do { if (h % 4 && W == 4) FEW2(T, W, true); else FEW2(T, W, false); } while (0)
    if (h < 4) FEW(16, 1);
    else if (h <= 64) FEW(16, 4);
    else FEW(64, 4);
#undef FEW
#undef FEW2
    return dn_launch_status();
  }
  s.slot_count = (int)(((long long)w + EMBED_SLOT - 1) / EMBED_SLOT);
  embed_tiles(s, 1024);
  const long long sums = ((long long)s.slot_count + n) * s.tiles;
  if (sums >= 1ll << 31) return ERROR_UNSUPPORTED;
  // starts, sorted columns, slots (16-byte ones), partial sums
  const size_t ints = ((size_t)n + 1 + w + 3) / 4 * 4, slots = (size_t)s.slot_count;
  char* scratch = (char*)dn_scratch(4 * ints + sizeof(EmbedSlot) * slots + 4 * (size_t)s.slot_count * h);
  if (!scratch) return CUDA_ERROR;
  o.starts = (int*)scratch; o.sorted = o.starts + n + 1; o.slots = (EmbedSlot*)(scratch + 4 * ints);
  s.starts = o.starts; s.sorted = o.sorted; s.slots = o.slots; s.partials = (float*)(o.slots + slots);
  // Few tokens a workgroup that sorts (its turns are as many as it has different tokens among 64 columns), unless the labels are so many that
  // reading them that often would take long.
  long long sorters = w > 0 ? (1ll << 25) / w : 512;
  sorters = sorters < 512 ? sorters : 512;
  const long long least = ((long long)n + EMBED_RANGE - 1) / EMBED_RANGE;
  sorters = sorters > least ? sorters : least;
  o.range = (int)((n + sorters - 1) / sorters);
  hipLaunchKernelGGL(k_embed_sort, dim3((unsigned)((n + o.range - 1) / o.range)), dim3(1024), 0, dn_stream(), o);
  // (items of one launch: teams of 16 or 64 lanes)
  auto launches = [&](long long items, int team, auto go) {
    const long long most = DN_MAX_GROUPS * (256 / team);
    for (long long i = 0; i < items; i += most) {
      s.first = (unsigned)i;
      go(dim3((unsigned)(((items - i < most ? items - i : most) + 256 / team - 1) / (256 / team))));
    }
  };
#define SUMS3(T, NV, W, TAIL, S) launches(sums, T, [&](dim3 grid) { hipLaunchKernelGGL((k_embed_sums<T, NV, W, TAIL, S>), grid, dim3(256), 0, dn_stream(), s); })
#define SUMS2(T, NV, W, TAIL) do { if (stream) SUMS3(T, NV, W, TAIL, true); else SUMS3(T, NV, W, TAIL, false); } while (0)
#define SUMS(T, NV, W) do { if (h % 4 && W == 4) SUMS2(T, NV, W, true); else SUMS2(T, NV, W, false); } while (0)
  if (h < 4) SUMS(16, 1, 1);
  else if (h <= 64) SUMS(16, 1, 4);
  else if (h <= 128) SUMS(16, 2, 4);
  else if (h <= 256) SUMS(64, 1, 4);
  else if (h <= 512) SUMS(64, 2, 4);
  else SUMS(64, 4, 4);
#undef SUMS
#undef SUMS2
#undef SUMS3
  {
    embed_tiles(s, 256);
    const long long joins = (long long)s.slot_count * s.tiles;
#define JOIN(T, W, TAIL) launches(joins, T, [&](dim3 grid) { hipLaunchKernelGGL((k_embed_join<T, W, TAIL>), grid, dim3(256), 0, dn_stream(), s); })
    if (h < 4) JOIN(16, 1, false);
    else if (h <= 64) { if (h % 4) JOIN(16, 4, true); else JOIN(16, 4, false); }
    else if (h % 4) JOIN(64, 4, true);
    else JOIN(64, 4, false);
#undef JOIN
  }
  return dn_launch_status();
}

}  // extern "C"
