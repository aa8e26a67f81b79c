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
// them do not depend on their order, so a border between two sums is one border.  c = log2(e) / T.  2^t = 2^n 2^f with |f| <= 1/2, the
// latter by its Taylor sum (remainder (ln 2 / 2)^12 / 12! < 7e-15); adding 2^52 leaves the rounded whole number in the low bits.
__device__ __forceinline__ unsigned long long sample_weight(float x, float m, double c, int shift) {
  const double t = fmax(((double)x - (double)m) * c, -80.0), n = rint(t), f = t - n;
  double p = 4.44553827187081e-10;    // ln2^11 / 11!
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
  const double w = ldexp(p, (int)n + shift) + 4503599627370496.0;
  return x > -INFINITY ? (unsigned long long)__double_as_longlong(w) & 0xfffffffffffffull : 0;
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

__device__ __forceinline__ unsigned long long wave_sum_u64(unsigned long long v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, WAVE);
  return v;
}
__device__ __forceinline__ unsigned long long wave_max_u64(unsigned long long v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { const unsigned long long q = __shfl_xor(v, o, WAVE); v = q > v ? q : v; }
  return v;
}
template <typename F>
__device__ __forceinline__ unsigned long long block_sum_u64(unsigned long long v, unsigned long long* red, F join) {
  v = join(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = (threadIdx.x & 63) < blockDim.x / 64 ? red[threadIdx.x & 63] : 0;
  return join(v);
}

// A workgroup of 1024 lanes a column.
__global__ void __launch_bounds__(1024) k_sample_tokens(SampleArgs a) {
  __shared__ unsigned long long red[16], lane_sums[16];
  __shared__ int drawn;
  const int col = blockIdx.x, tid = threadIdx.x, h = a.h;
  const float* c = a.mat + (size_t)col * h;
  const SampleRule r = sample_rule(a, col);
  auto sum = [&](unsigned long long v) __attribute__((always_inline)) { return block_sum_u64(v, red, wave_sum_u64); };
  unsigned long long best = 0, bad = 0;
  for (int i = tid; i < h; i += 1024) {
    const float x = c[i];
    const unsigned long long key = lp_key(x, i);
    best = key > best ? key : best;
    bad |= !(x < INFINITY) ? 1 : 0;
  }
  best = block_sum_u64(best, red, wave_max_u64);
  bad = sum(bad);
  const float m = lp_key_value(best);
  if (h == 0 || bad || !(m > -INFINITY)) {                // (nothing to draw)
    if (tid == 0) { a.tokens[col] = -1.f; if (a.logp) a.logp[col] = bad ? NAN : 0.f; }
    return;
  }
  if (r.greedy) {
    if (tid == 0) { a.tokens[col] = (float)lp_key_index(best); if (a.logp) a.logp[col] = 0.f; }
    return;
  }
  // Kept are the entries of keys from `border` on whose weight reaches `least`.
  auto weight = [&](int i) __attribute__((always_inline)) { const unsigned long long w = sample_weight(c[i], m, r.c, a.shift); return w >= r.least ? w : 0; };
  unsigned long long border = 0;
  auto greatest = [&](auto enough) __attribute__((always_inline)) {      // the greatest border that leaves enough
    unsigned long long b = 0;
    for (int bit = 63; bit >= 0; --bit)
      if (enough(b | 1ull << bit)) b |= 1ull << bit;
    return b;
  };
  if (r.k < h)
    border = greatest([&](unsigned long long b) {
      unsigned long long n = 0;
      for (int i = tid; i < h; i += 1024) n += lp_key(c[i], i) >= b ? 1 : 0;
      return sum(n) >= (unsigned long long)r.k;
    });
  auto mass = [&](unsigned long long b) __attribute__((always_inline)) {
    unsigned long long s = 0;
    for (int i = tid; i < h; i += 1024) s += lp_key(c[i], i) >= b ? weight(i) : 0;
    return sum(s);
  };
  unsigned long long total = mass(border);
  if (r.top_p < 1.0) {
    const unsigned long long part = r.top_p > 0.0 ? sample_part_up(r.top_p, total) : 0, ask = part > 1 ? part : 1;
    const unsigned long long b = greatest([&](unsigned long long b) { return mass(b) >= ask; });
    border = b > border ? b : border;
    total = mass(border);
  }
  const unsigned long long at = sample_part((double)r.u, total), aim = at < total ? at : total - 1;
  // the first entry behind whose weight the sums are over `aim`: 1024 entries a turn
  unsigned long long before = 0;
  for (int i0 = 0; i0 < h; i0 += 1024) {
    const int i = i0 + tid;
    const unsigned long long w = i < h && lp_key(c[i], i) >= border ? weight(i) : 0;
    unsigned long long up = w;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const unsigned long long q = __shfl_up(up, o, WAVE); if ((tid & 63) >= o) up += q; }
    __syncthreads();
    if ((tid & 63) == 63) lane_sums[tid >> 6] = up;
    __syncthreads();
    unsigned long long all = 0, base = before;
    for (int k = 0; k < 16; ++k) { if (k < tid >> 6) base += lane_sums[k]; all += lane_sums[k]; }
    if (w && base + up > aim && base + up - w <= aim) drawn = i;
    before += all;
    if (before > aim) break;
  }
  __syncthreads();
  if (tid == 0) {
    a.tokens[col] = (float)drawn;
    if (a.logp) a.logp[col] = (float)(((double)c[drawn] - (double)m) * (r.c * 0.6931471805599453) - dn_log_wide_pos(ldexp((double)total, -a.shift)));
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
  hipLaunchKernelGGL(k_sample_tokens, dim3(w), dim3(1024), 0, dn_stream(), a);
  return dn_launch_status();
}
