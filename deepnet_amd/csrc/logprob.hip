// Log probabilities of given tokens, entropies and the best alternatives of columns of logits, and their gradient (no
// counterpart in cudamat.cu; softmax_ce_grad is the loss of a classifier, which stores its probabilities).
#include "columns.h"
#include "wide_math.h"
#include <float.h>

// e^t for t <= 0: t log2(e) in two terms, the hardware's exp2, a correction.  -inf gives 0, NaN stays NaN.
__device__ __forceinline__ float lp_exp(float t) {
  t = t < -128.f ? -128.f : t;      // (e^-128 is 0 in fp32; keeps -inf out of the correction)
  const float L2E = 1.44269502162933349609375f, L2E_LO = 1.925963033500011e-08f;
  const float p = t * L2E;
  const float lo = __fmaf_rn(t, L2E_LO, __fmaf_rn(t, L2E, -p));
  const float e = __builtin_amdgcn_exp2f(p);
  return __fmaf_rn(e, lo * 0.693147182464599609375f, e);
}

// Orders entries: the greater value first, of equal ones (0 and -0 are) the one further up; NaN ranks with -inf.
__device__ __forceinline__ unsigned long long lp_key(float x, int i) {
  x = x != x ? -INFINITY : x + 0.f;
  const unsigned u = __float_as_uint(x), v = u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
  return ((unsigned long long)v << 32) | (unsigned)~i;
}
__device__ __forceinline__ int lp_key_index(unsigned long long k) { return (int)~(unsigned)k; }

// log(1 + r), r >= 0 (NaN stays NaN); 1 + r itself would round a small r away.
__device__ __forceinline__ double lp_log1p(double u) {
  return u >= 1e-5 ? dn_log_wide_pos(1.0 + u) : u * fma(u, fma(u, 1.0 / 3.0, -0.5), 1.0);
}

struct LogProbArgs {
  const float *mat, *labels;
  float *logp, *entropy, *log_z, *top, *top_labels;
  int h, w, k;
  int segments, length;            // of a column: LogProbPart's and k keys of each in `parts` and `keys`
  float* parts;
  unsigned long long* keys;
  unsigned* arrived;
};

// What one pass over some entries keeps: their maximum m (at least the lowest finite number), how many are equal to it, and over the
// others r, the sum of e^(x - m), and t, that of (x - m) e^(x - m).  So log(sum of exponentials) = m + log(1 + (count - 1 + r)), to full
// precision however small r is beside the maximum's own 1, and entropy = log(1 + ..) - t / (1 + ..).  Entries of -inf count nothing: a
// column of nothing else has count 0.  NaN and +inf make r NaN.
struct LogProbPart { float m, count, r, t; };
__device__ __forceinline__ LogProbPart lp_none() { return LogProbPart{-FLT_MAX, 0.f, 0.f, 0.f}; }
// e^d, d <= 0: the hardware's exp2 of d log2(e) in two terms (d itself is off by half a step, that is what the result is off by).
__device__ __forceinline__ float lp_exp_fast(float d) { return __builtin_amdgcn_exp2f(__fmaf_rn(d, 1.925963033500011e-08f, d * 1.44269502162933349609375f)); }
// The part as seen from a maximum M >= m.
__device__ __forceinline__ void lp_raise(LogProbPart& p, float M) {
  if (M > p.m) {
    const float d = p.m - M, s = lp_exp_fast(d), all = p.r + p.count;
    p.t = s * __fmaf_rn(fmaxf(d, -200.f), all, p.t);
    p.r = s * all;
    p.count = 0.f;
    p.m = M;
  }
}
__device__ __forceinline__ void lp_take(LogProbPart& p, float x) {
  const float d = x - p.m, e = lp_exp_fast(d);
  p.count += d == 0.f ? 1.f : 0.f;
  p.r += d == 0.f ? 0.f : e;
  p.t = __fmaf_rn(fmaxf(d, -200.f), e, p.t);               // (-inf: e is 0; what is kept of d does not matter below -200)
}
// Over the 64 lanes of a wavefront; every lane gets it.
__device__ __forceinline__ LogProbPart lp_wave(LogProbPart p) {
  lp_raise(p, lanes_sum<64, true>(p.m));
  return LogProbPart{p.m, lanes_sum<64>(p.count), lanes_sum<64>(p.r), lanes_sum<64>(p.t)};
}

struct LogProbResult { float m, log_z; double lz; bool none; };
__device__ __forceinline__ LogProbResult lp_result(const LogProbPart& p) {
  LogProbResult o;
  o.m = p.m;
  o.none = p.count == 0.f && p.r == 0.f;
  o.lz = lp_log1p((double)(p.count - 1.f) + (double)p.r);
  o.log_z = o.none ? -INFINITY : p.r == p.r ? (float)((double)p.m + o.lz) : NAN;
  return o;
}
__device__ __forceinline__ float lp_of(const LogProbResult& o, float x) {
  return o.none ? -INFINITY : o.log_z != o.log_z ? NAN : (float)((double)x - (double)o.m - o.lz);
}
// The results of a column but for the top list, by one lane.
__device__ __forceinline__ void lp_finish(const LogProbArgs& a, int col, const LogProbPart& p, const LogProbResult& o) {
  if (a.log_z) a.log_z[col] = o.log_z;
  if (a.entropy) a.entropy[col] = o.none ? 0.f : o.log_z != o.log_z ? NAN : (float)(o.lz - (double)p.t / ((double)p.count + (double)p.r));
  if (a.logp) {
    const float l = a.labels[col];
    a.logp[col] = l >= 0.f && l < (float)a.h ? lp_of(o, a.mat[(size_t)col * a.h + (int)l]) : 0.f;
  }
}
__device__ __forceinline__ void lp_top_out(const LogProbArgs& a, int col, int rank, unsigned long long key, const LogProbResult& o) {
  const int i = lp_key_index(key);
  if (a.top) a.top[(size_t)col * a.k + rank] = lp_of(o, a.mat[(size_t)col * a.h + i]);
  if (a.top_labels) a.top_labels[(size_t)col * a.k + rank] = (float)i;
}
// How many of n keys in LDS (n even, 16-byte aligned) are greater.
__device__ __forceinline__ int lp_rank(unsigned long long key, const unsigned long long* keys, int n) {
  int r = 0;
#pragma unroll 4
  for (int i = 0; i < n; i += 2) {
    const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(keys + i);
    r += (q.x > key ? 1 : 0) + (q.y > key ? 1 : 0);
  }
  return r;
}

// The top list of a team.  The k greatest entries lie in the k lanes whose own greatest entries are the greatest: those lanes' entries
// from the k-th of these maxima on are the candidates (k and a few more, unless a few lanes have far more than their share), and a
// candidate's place is the number of greater ones.
#define LP_LIST 2048               // candidates that a workgroup holds

// ---- columns (or segments of them) by a workgroup of 256 lanes, four 16-byte groups a lane in flight
template <bool TOP>
__global__ void __launch_bounds__(256) k_log_probs(LogProbArgs a) {
  __shared__ LogProbPart parts[4];
  __shared__ __attribute__((aligned(16))) unsigned long long lane_keys[TOP ? 256 : 2], list[TOP ? LP_LIST + 2 : 2];
  __shared__ int winners[TOP ? 64 : 1], listed, last;
  __shared__ unsigned long long border;
  const int tid = threadIdx.x, col = blockIdx.x / a.segments, seg = blockIdx.x - col * a.segments;
  const int row0 = seg * a.length, n = a.h - row0 < a.length ? a.h - row0 : a.length, n4 = n >> 2, trips = (n4 + 1023) >> 10;
  const float* c = a.mat + (size_t)col * a.h + row0;
  LogProbPart p = lp_none();
  float best = -INFINITY;
  int best_at = 0;
  auto load = [&](float (&v)[4][4], int it) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = tid + 256 * u + 1024 * it;
      if (j < n4) col_load<false>(v[u], c + 4 * j);
      else v[u][0] = v[u][1] = v[u][2] = v[u][3] = -INFINITY;
    }
  };
  float v[4][4], next[4][4];
  load(v, 0);
  for (int it = 0; it < trips; ++it) {
    if (it + 1 < trips) load(next, it + 1);
    float m = v[0][0];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) m = fmaxf(m, v[u][e]);
    if (TOP && m > best) { best = m; best_at = it; }
    lp_raise(p, m);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) { lp_take(p, v[u][e]); v[u][e] = next[u][e]; }
  }
  const bool tail = tid < (n & 3);                         // the rows behind the last group: one a lane
  if (tail) {
    const float x = c[4 * n4 + tid];
    lp_raise(p, x);
    lp_take(p, x);
  }
  p = lp_wave(p);
  if (tid % 64 == 0) parts[tid >> 6] = p;
  if (TOP) {
    // this lane's greatest entry: the first of its trip's greatest, or its row of the tail
    unsigned long long key = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = tid + 256 * u + 1024 * best_at;
      if (j < n4) {
        col_load<false>(v[u], c + 4 * j);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned long long q = lp_key(v[u][e], row0 + 4 * j + e);
          key = q > key ? q : key;
        }
      }
    }
    if (tail) {
      const unsigned long long q = lp_key(c[4 * n4 + tid], row0 + 4 * n4 + tid);
      key = q > key ? q : key;
    }
    lane_keys[tid] = key;
    if (tid == 0) { listed = 0; border = 1; }
  }
  __syncthreads();
  auto all = [&]() __attribute__((always_inline)) {
    LogProbPart q = parts[tid & 3];
    float m = fmaxf(fmaxf(parts[0].m, parts[1].m), fmaxf(parts[2].m, parts[3].m));
    lp_raise(q, m);
    // (four neighbours have the four parts: sums over them)
    auto four = [](float x) __attribute__((always_inline)) { x += lane_move<0xB1>(x); return x + lane_move<0x4E>(x); };
    return LogProbPart{m, four(q.count), four(q.r), four(q.t)};
  };
  p = all();
  if (TOP) {
    const unsigned long long mine = lane_keys[tid];
    const int rank = lp_rank(mine, lane_keys, 256);
    if (mine && rank < a.k) {
      winners[rank] = tid;
      if (rank == a.k - 1) border = mine;
    }
    __syncthreads();
    const unsigned long long from = border;
    // (fewer lanes than k have entries only where there are fewer than 256 groups: then all of them take part)
    const int lanes = from > 1 ? a.k : 0;
    auto offer = [&](unsigned long long q) __attribute__((always_inline)) {
      if (q >= from) {
        const int at = atomicAdd(&listed, 1);
        if (at < LP_LIST) list[at] = q;
      }
    };
    if (lanes) {
      const int items = lanes * 4 * trips;
      for (int i = tid; i < items; i += 256) {
        const int q = i / (4 * trips), g = i - q * (4 * trips), j = winners[q] + 256 * (g & 3) + 1024 * (g >> 2);
        if (j < n4) {
          float x[4];
          col_load<false>(x, c + 4 * j);
#pragma unroll
          for (int e = 0; e < 4; ++e) offer(lp_key(x[e], row0 + 4 * j + e));
        }
      }
    } else {
      for (int j = tid; j < n4; j += 256) {
        float x[4];
        col_load<false>(x, c + 4 * j);
#pragma unroll
        for (int e = 0; e < 4; ++e) offer(lp_key(x[e], row0 + 4 * j + e));
      }
    }
    if (tail) offer(lp_key(c[4 * n4 + tid], row0 + 4 * n4 + tid));
    __syncthreads();
  }
  // one segment: the column's results; several: this one's part, and the last to arrive joins them
  LogProbResult o = lp_result(p);
  if (a.segments == 1 && tid == 0) lp_finish(a, col, p, o);
  unsigned long long* const keys = TOP ? a.keys + (size_t)blockIdx.x * a.k : nullptr;
  auto out = [&](int rank, unsigned long long key) __attribute__((always_inline)) {
    if (a.segments == 1) lp_top_out(a, col, rank, key, o);
    else __hip_atomic_store(keys + rank, key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  if (TOP) {
    const int count = listed;
    if (count <= LP_LIST) {
      if (tid < 2) list[count + tid] = 0;
      __syncthreads();
      for (int i = tid; i < count; i += 256) {
        const int rank = lp_rank(list[i], list, count + (count & 1));
        if (rank < a.k) out(rank, list[i]);
      }
      for (int i = count + tid; i < a.k; i += 256) out(i, 0);          // (a segment of fewer than k rows)
    } else {
      // more than fit: the greatest, the next one below it, and so on, a pass each
      unsigned long long above = ~0ull;
      for (int j = 0; j < a.k; ++j) {
        unsigned long long key = 0;
        for (int i = tid; i < n; i += 256) {
          const unsigned long long q = lp_key(c[i], row0 + i);
          key = q < above && q > key ? q : key;
        }
        __syncthreads();
        lane_keys[tid] = key;
        __syncthreads();
        if (lp_rank(key, lane_keys, 256) == 0 && key) { border = key; out(j, key); }
        __syncthreads();
        above = border;
      }
    }
  }
  if (a.segments == 1) return;
  if (tid < 4) {
    const float f[4] = {p.m, p.count, p.r, p.t};
    __hip_atomic_store(a.parts + 4 * (size_t)blockIdx.x + tid, f[tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __builtin_amdgcn_s_waitcnt(0);         // the stores of this wavefront have been acknowledged
  __syncthreads();
  if (tid == 0) {
    const unsigned old = __hip_atomic_fetch_add(a.arrived + col, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = old == (unsigned)a.segments - 1u;
    if (last) __hip_atomic_store(a.arrived + col, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last) return;
  // at most 64 segments: a lane each, in a fixed order whoever came last
  const float* f = a.parts + 4 * ((size_t)col * a.segments + (tid & 63));
  auto get = [&](int i) __attribute__((always_inline)) { return __hip_atomic_load(f + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
  p = lp_none();
  if ((tid & 63) < a.segments) p = LogProbPart{get(0), get(1), get(2), get(3)};
  p = lp_wave(p);
  o = lp_result(p);
  if (tid == 0) lp_finish(a, col, p, o);
  if (TOP) {
    const int count = a.segments * a.k;                    // (at most LP_LIST)
    const unsigned long long* from = a.keys + (size_t)col * count;
    for (int i = tid; i < count; i += 256) list[i] = __hip_atomic_load(from + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (tid < 2) list[count + tid] = 0;
    __syncthreads();
    for (int i = tid; i < count; i += 256) {
      const int rank = list[i] ? lp_rank(list[i], list, count + (count & 1)) : a.k;
      if (rank < a.k) lp_top_out(a, col, rank, list[i], o);
    }
  }
}

// ---- columns of 4 to 1024 rows by a wavefront, which holds them in registers
template <int NV, bool TAIL, bool TOP>
__global__ void __launch_bounds__(256) k_log_probs_wave(LogProbArgs a) {
  __shared__ __attribute__((aligned(16))) unsigned long long lane_keys[TOP ? 4 : 1][TOP ? 64 : 2], lists[TOP ? 4 : 1][TOP ? 256 * NV + 2 : 2];
  __shared__ int listed[4];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, col = blockIdx.x * 4 + wv;
  const bool live = col < a.w;
  const float* c = a.mat + (size_t)(live ? col : 0) * a.h;
  ColGroups<NV, TAIL> at;
  at.init(lane, 64, a.h);
  float v[NV][4], m = -FLT_MAX;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    if (at.row[k] >= 0) col_load<false>(v[k], c + at.row[k]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (at.row[k] < 0 || !at.own(k, e)) v[k][e] = -INFINITY;
      m = fmaxf(m, v[k][e]);
    }
  }
  LogProbPart p = lp_none();
  p.m = lanes_sum<64, true>(m);
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) lp_take(p, v[k][e]);
  p = LogProbPart{p.m, lanes_sum<64>(p.count), lanes_sum<64>(p.r), lanes_sum<64>(p.t)};
  const LogProbResult o = lp_result(p);
  if (live && lane == 0) lp_finish(a, col, p, o);
  if (!TOP) return;
  unsigned long long best = 0, border = 1;
  auto key_of = [&](int k, int e) __attribute__((always_inline)) { return at.row[k] >= 0 && at.own(k, e) ? lp_key(v[k][e], at.row[k] + e) : 0ull; };
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const unsigned long long q = key_of(k, e);
      best = q > best ? q : best;
    }
  // (a wavefront's own part of LDS, whose accesses are in order: the compiler has to keep them so)
  auto ordered = []() __attribute__((always_inline)) { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); __builtin_amdgcn_wave_barrier(); };
  unsigned long long *keys = lane_keys[wv], *list = lists[wv];
  keys[lane] = best;
  if (lane == 0) listed[wv] = 0;
  ordered();
  const int rank = lp_rank(best, keys, 64);
  const unsigned long long at_border = __ballot(best && rank == a.k - 1);
  if (at_border) border = keys[__builtin_ctzll(at_border)];
  ordered();
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const unsigned long long q = key_of(k, e);
      if (q >= border) list[atomicAdd(&listed[wv], 1)] = q;
    }
  ordered();
  const int count = listed[wv];
  if (lane < 2) list[count + lane] = 0;
  ordered();
  for (int i = lane; i < count; i += 64) {
    const int r = lp_rank(list[i], list, count + (count & 1));
    if (live && r < a.k) lp_top_out(a, col, r, list[i], o);
  }
}

// target = logp_weight (onehot(label) - p) - entropy_weight p (log p + entropy), log p = mat - log_z: one pass.
__global__ void __launch_bounds__(256)
k_log_probs_grad(const float* mat, const float* labels, const float* log_z, const float* logp_weight, const float* entropy,
                 const float* entropy_weight, float* target, int h) {
  const int col = blockIdx.x;
  const float z = log_z[col], l = labels ? labels[col] : -1.f;
  const bool token = l >= 0.f && l < (float)h;
  const int label = token ? (int)l : -1;
  const float lw = token ? (logp_weight ? logp_weight[col] : 1.f) : 0.f;
  const float ew = entropy_weight ? entropy_weight[col] : 0.f, ent = entropy ? entropy[col] : 0.f;
  const float* c = mat + (size_t)col * h;
  float* t = target + (size_t)col * h;
  for (int i = threadIdx.x; i < h; i += 256) {
    const float x = c[i], lp = x - z;
    const float p = x == -INFINITY ? 0.f : lp_exp(lp);
    const float q = p > 0.f || p != p ? p * (lp + ent) : 0.f;
    t[i] = lw * ((i == label ? 1.f : 0.f) - p) - ew * q;
  }
}

static inline long long end_of(const cudamat* a) { return dn_len(a); }
static inline bool apart(const cudamat* a, const cudamat* b) {
  return !a || !b || a->data_device + end_of(a) <= b->data_device || b->data_device + end_of(b) <= a->data_device;
}
// NULL, or rows x cols on the device
static int check_shape(const cudamat* m, int rows, int cols) {
  if (!m) return 0;
  if (!m->on_device) return ERROR_NOT_ON_DEVICE;
  if (m->is_trans) return ERROR_TRANSPOSED;
  return m->size[0] == rows && m->size[1] == cols ? 0 : ERROR_INCOMPATIBLE_DIMENSIONS;
}
#define LP_SEGMENT 4096           // rows of one trip of a workgroup
#define LP_JOIN 512               // keys that the last workgroup of a column ranks
#define DPTR(m) ((m) ? (m)->data_device : nullptr)

extern "C" {

int log_probs(cudamat* mat, cudamat* labels, cudamat* logp, cudamat* entropy, cudamat* log_z, cudamat* top, cudamat* top_labels) {
  const int h = mat->size[0], w = mat->size[1];
  if (!mat->on_device) return ERROR_NOT_ON_DEVICE;
  if (mat->is_trans) return ERROR_TRANSPOSED;
  cudamat* row[4] = {labels, logp, entropy, log_z};
  for (cudamat* m : row)
    if (int e = check_shape(m, 1, w)) return e;
  const int k = top ? top->size[0] : top_labels ? top_labels->size[0] : 0;
  if (int e = check_shape(top, k, w)) return e;
  if (int e = check_shape(top_labels, k, w)) return e;
  if (k > h || (logp && !labels)) return ERROR_INCOMPATIBLE_DIMENSIONS;
  if (k > LOG_PROBS_MAX_TOP || h > (1 << 24)) return ERROR_UNSUPPORTED;     // (whole numbers as floats)
  cudamat* out[5] = {logp, entropy, log_z, top, top_labels};
  for (int i = 0; i < 5; ++i) {
    if (!apart(out[i], mat) || !apart(out[i], labels)) return ERROR_UNSUPPORTED;
    for (int j = 0; j < i; ++j)
      if (!apart(out[i], out[j])) return ERROR_UNSUPPORTED;
  }
  if (h <= 0 || w <= 0) return 0;
  LogProbArgs a = {mat->data_device, DPTR(labels), DPTR(logp), DPTR(entropy), DPTR(log_z), DPTR(top), DPTR(top_labels), h, w, k, 1, h, nullptr, nullptr, nullptr};
  if (h >= 4 && h <= 1024) {
    const dim3 grid((unsigned)((w + 3) / 4));
#define LP_WAVE(NV, TAIL) do { if (k) hipLaunchKernelGGL((k_log_probs_wave<NV, TAIL, true>), grid, dim3(256), 0, dn_stream(), a); \
                               else hipLaunchKernelGGL((k_log_probs_wave<NV, TAIL, false>), grid, dim3(256), 0, dn_stream(), a); } while (0)
    if (h <= 256) { if (h % 4) LP_WAVE(1, true); else LP_WAVE(1, false); }
    else if (h <= 512) { if (h % 4) LP_WAVE(2, true); else LP_WAVE(2, false); }
    else if (h % 4) LP_WAVE(4, true);
    else LP_WAVE(4, false);
#undef LP_WAVE
    return dn_launch_status();
  }
  // few columns: segments of them, about two workgroups a CU, none shorter than LP_SEGMENT rows
  int segments = 2 * dn_num_cus() / (w < 2 * dn_num_cus() ? w : 2 * dn_num_cus());
  const int most[3] = {(h + LP_SEGMENT - 1) / LP_SEGMENT, 64, k ? LP_JOIN / k : 64};
  for (int m : most) segments = segments < m ? segments : m;
  if (segments > 1) {
    a.length = ((h + segments - 1) / segments + 3) / 4 * 4;
    a.segments = segments = (h + a.length - 1) / a.length;
    const size_t parts = (size_t)w * segments;
    a.keys = (unsigned long long*)dn_scratch(parts * (8 * k + 16));
    a.arrived = dn_zero_words(w);
    if (!a.keys || !a.arrived) return CUDA_ERROR;
    a.parts = (float*)(a.keys + parts * k);
  }
  const long long blocks = (long long)w * segments;
  if (blocks > 0x7fffffffll) return ERROR_UNSUPPORTED;
  if (k) hipLaunchKernelGGL(k_log_probs<true>, dim3((unsigned)blocks), dim3(256), 0, dn_stream(), a);
  else hipLaunchKernelGGL(k_log_probs<false>, dim3((unsigned)blocks), dim3(256), 0, dn_stream(), a);
  return dn_launch_status();
}

int log_probs_grad(cudamat* mat, cudamat* labels, cudamat* log_z, cudamat* logp_weight, cudamat* entropy, cudamat* entropy_weight,
                   cudamat* target) {
  const int h = mat->size[0], w = mat->size[1];
  if (!mat->on_device || !target->on_device || !log_z->on_device) return ERROR_NOT_ON_DEVICE;
  if (mat->is_trans || target->is_trans) return ERROR_TRANSPOSED;
  if (target->size[0] != h || target->size[1] != w) return ERROR_INCOMPATIBLE_DIMENSIONS;
  cudamat* row[5] = {labels, log_z, logp_weight, entropy, entropy_weight};
  for (cudamat* m : row)
    if (int e = check_shape(m, 1, w)) return e;
  if ((logp_weight && !labels) || (!entropy) != (!entropy_weight)) return ERROR_INCOMPATIBLE_DIMENSIONS;
  for (cudamat* m : row)
    if (!apart(m, target)) return ERROR_UNSUPPORTED;
  if ((!apart(mat, target) && mat->data_device != target->data_device) || h > (1 << 24)) return ERROR_UNSUPPORTED;
  if (h <= 0 || w <= 0) return 0;
  hipLaunchKernelGGL(k_log_probs_grad, dim3((unsigned)w), dim3(256), 0, dn_stream(), (const float*)mat->data_device, (const float*)DPTR(labels),
                     (const float*)log_z->data_device, (const float*)DPTR(logp_weight), (const float*)DPTR(entropy), (const float*)DPTR(entropy_weight),
                     target->data_device, h);
  return dn_launch_status();
}

}  // extern "C"
