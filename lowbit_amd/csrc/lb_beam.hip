// Beam search's selection (lbd_beam_select): of every prompt's beams and their logits the W best
// continuations. No reference counterpart: the reference decodes greedily
// (src/lowbit/model.py:437-458).
//
// A beam of sum s and logits x offers s + x[v] - lse, lse = log sum exp x. Within a beam the order
// is that of x, so its W best are known without lse; they and lse meet in float64.
#include <math.h>

#include "lb_device.h"
#include "lb_internal.h"

namespace lbk {

// A row that offers tokens: its beam has not ended and there is one.
__device__ __forceinline__ bool beam_open(const BeamArgs &a, int row) {
  const float s = a.score[row];
  return !(a.done && a.done[row]) && s > -INFINITY;
}

// An offer's key: larger logit first, then the lower token; 0 for a logit of -inf, which is none.
__device__ __forceinline__ unsigned long long offer_key(float x, int v) { return x > -INFINITY ? argmax_key(x, v) : 0; }
__device__ __forceinline__ float offer_logit(unsigned long long key) {
  const uint32_t k = (uint32_t)(key >> 32);
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// float64 as an unsigned number of the same order (NaN does not occur).
__device__ __forceinline__ unsigned long long order_f64(double x) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(x + 0.0);  // -0 counts as 0
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

// ---- a row: its log-sum and its W best

__global__ __launch_bounds__(256) void beam_row_kernel(BeamArgs a, double *__restrict__ lse,
                                                       unsigned long long *__restrict__ best) {
  const int row = blockIdx.x, tid = threadIdx.x, wave = tid / kWave;
  if (!beam_open(a, row)) return;
  const float *x = a.logits + (size_t)row * a.ld;
  __shared__ float red[4];
  __shared__ unsigned long long top[4];
  float m = -INFINITY, bad = 0.0f, sum = 0.0f;
  for (int v = tid; v < a.V; v += 256) m = fmaxf(m, x[v]), bad += x[v] - x[v] == 0.0f || x[v] == -INFINITY ? 0.0f : 1.0f;
  m = wave_max(m);
  if (tid % kWave == 0) red[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  __syncthreads();
  for (int v = tid; v < a.V; v += 256) sum += expf(x[v] - m);
  sum = wave_sum(bad) > 0.0f ? NAN : wave_sum(sum);
  if (tid % kWave == 0) red[wave] = sum;
  __syncthreads();
  if (tid == 0) lse[row] = (double)m + log((double)(red[0] + red[1] + red[2] + red[3]));
  unsigned long long last = ~0ull;
  for (int w = 0; w < a.W; w++) {
    unsigned long long k = 0;
    for (int v = tid; v < a.V; v += 256) {
      const unsigned long long c = offer_key(x[v], v);
      k = c < last && c > k ? c : k;
    }
    k = wave_max_u64(k);
    if (tid % kWave == 0) top[wave] = k;
    __syncthreads();
    for (int i = 0; i < 4; i++) k = top[i] > k ? top[i] : k;
    __syncthreads();
    if (tid == 0) best[(size_t)row * a.W + w] = k;
    last = k ? k : 1;
  }
}

// ---- a prompt: the W best of its beams' offers

__global__ __launch_bounds__(64) void beam_merge_kernel(BeamArgs a, const double *__restrict__ lse,
                                                        const unsigned long long *__restrict__ best) {
  const int b = blockIdx.x, lane = threadIdx.x, W = a.W, base = b * W;
  __shared__ double sum[kMaxBeams * kMaxBeams];  // offer w W + n: beam w's n-th; -inf: none
  __shared__ int token[kMaxBeams * kMaxBeams];   // -1: the beam itself
  for (int i = lane; i < W * W; i += kWave) {
    const int row = base + i / W, n = i % W;
    double s = -INFINITY;
    int t = -1;
    if (beam_open(a, row)) {
      const unsigned long long k = best[(size_t)row * W + n];
      const double x = (double)a.score[row] + ((double)offer_logit(k) - lse[row]);
      t = argmax_key_index(k);
      if (k && x > -INFINITY) s = x;
    } else if (n == 0 && a.done && a.done[row] && a.score[row] > -INFINITY) {
      s = a.score[row];
    }
    sum[i] = s, token[i] = t;
  }
  __syncthreads();
  unsigned long long last = ~0ull;
  int last_i = -1;
  const int step = a.step ? a.step[b] : 0, none = a.eos >= 0 ? a.eos : 0;
  for (int w = 0; w < W; w++) {
    // the largest below the last one taken; of equals the lowest
    unsigned long long k = 0;
    int at = 0x7FFFFFFF;
    for (int i = lane; i < W * W; i += kWave) {
      if (!(sum[i] > -INFINITY)) continue;
      const unsigned long long c = order_f64(sum[i]);
      if (c > last || (c == last && i <= last_i)) continue;
      if (c > k || (c == k && i < at)) k = c, at = i;
    }
    const unsigned long long top = wave_max_u64(k);
    at = k == top && top ? at : 0x7FFFFFFF;
    for (int o = 1; o < kWave; o <<= 1) at = min(at, __shfl_xor(at, o));
    last = top, last_i = at;
    if (lane == 0) {
      const bool some = top != 0;
      const int t = some ? token[at] : -1, tok = t >= 0 ? t : none;
      const int parent = some ? base + at / W : -1;
      a.new_score[base + w] = some ? (float)sum[at] : -INFINITY;
      a.new_done[base + w] = some && (t < 0 || t == a.eos);
      a.tok[base + w] = tok;
      a.parent[base + w] = parent;
      if (a.step && step >= 0 && step < a.hist_len) {
        const size_t h = (size_t)step * a.B * W + base + w;
        a.hist_tok[h] = tok;
        a.hist_parent[h] = parent;
      }
    }
    if (!top) last = 0;
  }
  if (a.step && lane == 0) a.step[b] = step + 1;
}

size_t beam_select_work_bytes(int B, int W, int V) { return (size_t)B * W * (8 + 8 * W); }

hipError_t launch_beam_select(const BeamArgs &a, void *work, hipStream_t s) {
  const int rows = a.B * a.W;
  double *lse = static_cast<double *>(work);
  unsigned long long *best = reinterpret_cast<unsigned long long *>(lse + rows);
  hipLaunchKernelGGL(beam_row_kernel, dim3(rows), dim3(256), 0, s, a, lse, best);
  hipLaunchKernelGGL(beam_merge_kernel, dim3(a.B), dim3(kWave), 0, s, a, lse, best);
  return hipGetLastError();
}

}  // namespace lbk
