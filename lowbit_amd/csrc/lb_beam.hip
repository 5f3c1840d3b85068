// Beam search's selection (lbd_beam_select): of every prompt's beams and their logits the W best
// continuations. No reference counterpart: the reference decodes greedily
// (src/lowbit/model.py:437-458).
//
// A beam of sum s and logits x offers s + x[v] - lse, lse = log sum exp x. Within a beam the order
// is that of x, so a piece of a row gives its W largest logits and its part of the sum without
// knowing lse; a second launch, a workgroup a prompt, adds up lse and takes the W best offers in
// float64. An offer's key is the logit and the token in one number, so no two are equal and ties
// need no thought: a threshold key splits a row's offers exactly.
#include <math.h>

#include <algorithm>

#include "lb_device.h"
#include "lb_internal.h"

namespace lbk {

constexpr int kBeamWaves = 4;                            // of a workgroup
constexpr int kBeamLoads = 4;                            // 16-byte loads a lane has in flight
constexpr int kBeamChunk = 4 * kWave * kBeamLoads;       // logits a wave looks at a time
constexpr int kBeamStep = kBeamChunk * kBeamWaves;       // a workgroup
constexpr int kBeamRoom = 384;                           // keys that a wave has room for: 128, and 4 of every lane
constexpr int kBeamGridY = 1 << 15;                      // rows in the grid's second dimension
constexpr int kBeamHeads = 512;                          // pieces of a prompt's rows at most
constexpr float kBeamNone = -3.4028234663852886e38f;     // the maximum before any logit: finite

// What a workgroup leaves of its piece of a row: `best` keys, in descending order, 0 past the last.
struct BeamPiece {
  float max, sum;  // sum exp(x - max), NaN where the row offers nothing
};

__device__ __forceinline__ float offer_logit(unsigned long long key) {
  const uint32_t k = (uint32_t)(key >> 32);
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// float64 as an unsigned number of the same order, above 0 for all but NaN.
__device__ __forceinline__ unsigned long long order_f64(double x) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(x + 0.0);  // -0 counts as 0
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

// e^x by the hardware's 2^x: x log2 e rounded to float32, |x| 2^-24 of the result; where that is more
// than 2^-20 the term is below e^-16 of the sum's largest.
__device__ __forceinline__ float exp_below(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }

// A number that at least W of the lanes' reach and, if it can be, no more: found bit by bit from the top, as soon
// as exactly W reach it nothing larger is needed. 0 where fewer than W are above 0.
__device__ __forceinline__ uint32_t wave_reach(uint32_t k, int W) {
  uint32_t t = 0;
  for (int b = 31; b >= 0; b--) {
    const uint32_t c = t | 1u << b;
    const int n = __popcll((unsigned long long)__ballot(k >= c));
    if (n >= W) t = c;
    if (n == W) break;
  }
  return t;
}

// The same of n numbers in LDS, by the lanes' largest: W of them at least reach it, and few more.
__device__ __forceinline__ uint32_t beam_reach(const uint32_t *top, int n, int W) {
  uint32_t k = 0;
  for (int i = threadIdx.x & (kWave - 1); i < n; i += kWave) k = max(k, top[i]);
  return wave_reach(k, W);
}

// How many of n numbers (n a multiple of 4, all different but for zeros behind the last) are larger than one,
// by their high words `top`; where others have the same one, `before` compares what is left.
template <class F>
__device__ __forceinline__ int beam_place(const uint32_t *top, int n, uint32_t one, F before) {
  int place = 0, same = 0;
  for (int j = 0; j < n; j += 4) {
    const uint4 t = *reinterpret_cast<const uint4 *>(top + j);
    place += (t.x > one) + (t.y > one) + (t.z > one) + (t.w > one);
    same += (t.x == one) + (t.y == one) + (t.z == one) + (t.w == one);
  }
  if (same > 1)
    for (int j = 0; j < n; j++) place += top[j] == one && before(j);
  return place;
}

// ---------------------------------------------------------------- pieces of rows

// The W largest of n keys (n <= kBeamRoom, W <= n, all different), by one wave, to the front in descending
// order: a key's place is how many are larger. Returns the last of them. A function of its own, as a dozen places
// call it and hardly any call comes; by an LDS pointer, whose accesses happen in order.
typedef __attribute__((address_space(3))) unsigned long long LdsKey;
__device__ __attribute__((noinline)) unsigned long long beam_sort(LdsKey *keys, int n, int W) {
  constexpr int PER = kBeamRoom / kWave;
  const int lane = threadIdx.x & (kWave - 1);
  unsigned long long mine[PER];
  int place[PER];
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int at = lane + kWave * i;
    mine[i] = at < n ? keys[at] : 0;
    place[i] = 0;
  }
  for (int j = 0; j < n; j++) {
    const unsigned long long k = keys[j];
#pragma unroll
    for (int i = 0; i < PER; i++) place[i] += k > mine[i];
  }
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < PER; i++)
    if (mine[i] && place[i] < W) keys[place[i]] = mine[i];
  __builtin_amdgcn_wave_barrier();
  return keys[W - 1];
}

// The largest float that at least W of the lanes' values reach (all finite ones, where fewer are above -inf).
__device__ __forceinline__ float beam_threshold(float v, int W) {
  const uint32_t t = wave_reach((uint32_t)(argmax_key(v, 0) >> 32), W);  // (v is not NaN)
  return t < 0x00800000u ? kBeamNone : offer_logit((unsigned long long)t << 32);
}

// A workgroup a piece of `per` steps of a row. Every wave keeps the keys above its threshold in LDS: the first
// step's, for all waves, is the W-th largest of 64 lanes' maxima (W of them at least reach it, and few more),
// later ones come from a chunk of many larger logits, and from sorting the kept keys out where they run out of
// room. So most chunks end after a comparison of 16 logits' maximum. (128 rows of 151936: rising logits 26 us,
// 367 without a threshold for them; all equal ones, where keys differ by their tokens only, 81.)
//
// What bounds it: 128 rows of 151936 logits the instructions, 17 us = 4.3 TB/s (of a wave's 549 vector
// instructions 16 a chunk are exponentials and 48 their arguments and sum), and 2.85 steps a workgroup between its
// beginning and end; four such rows the launch and two loads one after the other, 4.8 us. The threshold of a
// wave's own first chunk kept four times as many keys (25.9 us), sixteen tests for room a chunk 20.8.
__global__ __launch_bounds__(kBeamWaves *kWave) void beam_piece_kernel(BeamArgs a, int per, int pieces,
                                                                       BeamPiece *__restrict__ piece,
                                                                       unsigned long long *__restrict__ best) {
  constexpr int N = 4 * kBeamLoads;  // logits of a lane and chunk
  const int row = (int)(blockIdx.y + blockIdx.z * kBeamGridY), at = blockIdx.x, lane = threadIdx.x & (kWave - 1), W = a.W;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  if (row >= a.B * W) return;
  const float score = a.score[row];
  const int over = a.done ? a.done[row] : 0;
  __shared__ unsigned long long keys[kBeamWaves][kBeamRoom], last[kBeamWaves * kBeamRoom];
  __shared__ __attribute__((aligned(16))) uint32_t high[kBeamWaves * kBeamRoom + 4];
  __shared__ float tops[kBeamWaves][kWave], smax[kBeamWaves], ssum[kBeamWaves], ssure[kBeamWaves];
  __shared__ int kept[kBeamWaves], count;
  const Rsrc x = make_rsrc(a.logits + (size_t)row * a.ld, 4u * (uint32_t)a.V);  // reads past the row give 0
  const int end = min(a.V, (at + 1) * per * kBeamStep);
  int v0 = at * per * kBeamStep + wave * kBeamChunk;
  unsigned long long *mine = keys[wave], low = 0;
  float m = kBeamNone, sum = 0.0f, least, sure;
  int n = 0;
  const auto load = [&](float *f, int v) {
#pragma unroll
    for (int i = 0; i < kBeamLoads; i++) {
      const float4 q = ld_f4(x, 4u * (uint32_t)(v + 4 * kWave * i + 4 * lane));
      f[4 * i] = q.x, f[4 * i + 1] = q.y, f[4 * i + 2] = q.z, f[4 * i + 3] = q.w;
    }
  };
  const auto token = [&](int i) { return v0 + 4 * kWave * (i >> 2) + 4 * lane + (i & 3); };
  // a chunk's part of the sum; the largest logit of each load in tops4, and of all
  const auto add = [&](float *f, float *tops4) {
    if (v0 + kBeamChunk > a.V) {
#pragma unroll
      for (int i = 0; i < N; i++) f[i] = token(i) < a.V ? f[i] : -INFINITY;
    }
    float top = -INFINITY;
#pragma unroll
    for (int g = 0; g < kBeamLoads; g++) {
      tops4[g] = fmaxf(fmaxf(f[4 * g], f[4 * g + 1]), fmaxf(f[4 * g + 2], f[4 * g + 3]));
      top = fmaxf(top, tops4[g]);
    }
    const float was = m;
    m = fmaxf(m, top);
    sum *= exp_below(was - m);
#pragma unroll
    for (int i = 0; i < N; i++) sum += exp_below(f[i] - m);
    return top;
  };
  // the chunk's keys that reach the threshold `least`; W of the workgroup's reach `sure`
  const auto keep = [&](const float *f, const float *tops4, float top) {
    // (a logit equal to the W-th best so far comes after it, by its token)
    if (low) least = fmaxf(least, offer_logit(((low >> 32) + 1) << 32));
    const int hits = __popcll((unsigned long long)__ballot(top >= least));
    if (!hits) return;
    if (hits > W + 8) {  // rising logits
      const float t = beam_threshold(top, W);
      least = fmaxf(least, t), sure = fmaxf(sure, t);
    }
#pragma unroll
    for (int g = 0; g < kBeamLoads; g++) {
      if (!__any(tops4[g] >= least)) continue;
      if (n > kBeamRoom - 4 * kWave) {
        __builtin_amdgcn_wave_barrier();
        low = beam_sort((LdsKey *)mine, n, W);
        n = W;
        least = fmaxf(least, offer_logit(low)), sure = fmaxf(sure, offer_logit(low));
      }
#pragma unroll
      for (int i = 4 * g; i < 4 * g + 4; i++) {
        if (!__any(f[i] >= least)) continue;
        const unsigned long long key = argmax_key(f[i], token(i)), push = __ballot(f[i] >= least && key > low);
        if (push >> lane & 1) mine[n + __popcll(push & ((1ull << lane) - 1))] = key;
        n += __popcll(push);
      }
    }
  };
  float f0[N], f1[N], t0[kBeamLoads], t1[kBeamLoads], top0 = -INFINITY;
  if (v0 < end) load(f0, v0);
  if (over || !(score > -INFINITY)) return;  // (known when the first logits are on their way)
  if (v0 < end) {
    if (v0 + kBeamStep < end) load(f1, v0 + kBeamStep);
    top0 = add(f0, t0);
  }
  // the first step's threshold: the W-th largest of 64 lanes' maxima over the waves
  tops[wave][lane] = fmaxf(top0, -INFINITY);
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  float first = tops[0][lane];
#pragma unroll
  for (int w = 1; w < kBeamWaves; w++) first = fmaxf(first, tops[w][lane]);
  least = sure = beam_threshold(first, W);
  if (v0 < end) keep(f0, t0, top0);
  for (v0 += kBeamStep; v0 < end; v0 += kBeamStep) {  // two chunks in turn, so that nothing is moved
    if (v0 + kBeamStep < end) load(f0, v0 + kBeamStep);
    const float top1 = add(f1, t1);
    keep(f1, t1, top1);
    v0 += kBeamStep;
    if (v0 >= end) break;
    if (v0 + kBeamStep < end) load(f1, v0 + kBeamStep);
    top0 = add(f0, t0);
    keep(f0, t0, top0);
  }
  // ---- the waves' sums and keys
  const float all = wave_max(m);
  const float part = wave_sum(sum * exp_below(m - all));
  if (lane == 0) smax[wave] = all, ssum[wave] = part, kept[wave] = n, ssure[wave] = sure;
  __syncthreads();
  const size_t to = (size_t)row * pieces + at;
  float top = smax[0], total = 0.0f, bar = ssure[0];
  int before[kBeamWaves + 1] = {0};
#pragma unroll
  for (int w = 0; w < kBeamWaves; w++) {
    top = fmaxf(top, smax[w]);
    bar = fmaxf(bar, ssure[w]);
    before[w + 1] = before[w] + kept[w];
  }
#pragma unroll
  for (int w = 0; w < kBeamWaves; w++) total += ssum[w] * exp_below(smax[w] - top);
  if (threadIdx.x == 0) piece[to] = {top, total};
  // W keys at least reach every wave's threshold; of those that reach the highest, a key's place is how many
  // are larger
  for (int i = threadIdx.x; i < before[kBeamWaves]; i += kBeamWaves * kWave) {
    int w = 0;
#pragma unroll
    for (int k = 1; k < kBeamWaves; k++) w += i >= before[k];
    const unsigned long long key = keys[w][i - before[w]];
    if (offer_logit(key) >= bar) {
      const int to = atomicAdd(&count, 1);
      last[to] = key, high[to] = (uint32_t)(key >> 32);
    }
  }
  __syncthreads();
  n = count;
  if (threadIdx.x < 4) high[n + threadIdx.x] = 0;
  __syncthreads();
  const uint32_t reach = n > kWave ? beam_reach(high, n, W) : 0;  // (many: only the best are put in order)
  for (int i = threadIdx.x; i < max(n, W); i += kBeamWaves * kWave) {
    if (i >= n) {
      best[to * W + i] = 0;
      continue;
    }
    const unsigned long long key = last[i];
    if ((uint32_t)(key >> 32) < reach) continue;
    const int place = beam_place(high, (n + 3) & ~3, (uint32_t)(key >> 32), [&](int j) { return j < n && last[j] > key; });
    if (place < W) best[to * W + place] = key;
  }
}

// ---------------------------------------------------------------- a prompt

// Offers in order: larger sums first (as order_f64's numbers, 0 for none), then the lower place, then the larger
// key; a key of ~0 is an ended beam itself. The W best lie in the W pieces whose first offers are the best: of
// those pieces the offers that reach the last of the W first ones are put in order by counting who comes before
// whom.
//
// What bounds it: three loads one after the other (sums and first offers, the chosen pieces' others, none of
// them near) and as many barriers, 4.6 us for 4 beams, 5.3 for 16 prompts' 8, 14 for 32. Counted among all 152
// first offers, not the few that reach the threshold, 6 us; all comparisons on 64-bit structures 20.
// (by_w and by_pieces: 2^16 / W and 2^20 / pieces and a bit more, for divisions of less than 1024 and 512.)
__global__ __launch_bounds__(kBeamHeads) void beam_merge_kernel(BeamArgs a, int pieces, uint32_t by_w, uint32_t by_pieces,
                                                                const BeamPiece *__restrict__ piece,
                                                                const unsigned long long *__restrict__ best) {
  constexpr int kOffers = kMaxBeams * (kMaxBeams + 1) / 2;
  const int b = blockIdx.x, tid = threadIdx.x, W = a.W, base = b * W;
  __shared__ double lse[kMaxBeams];
  __shared__ unsigned long long head_sum[kBeamHeads], head_key[kBeamHeads], sums[kOffers], keys[kOffers];
  __shared__ __attribute__((aligned(16))) uint32_t head_top[kBeamHeads], tops[kOffers + 4];
  __shared__ int beams[kOffers], chosen[kMaxBeams], count;
  __shared__ float scores[kMaxBeams];
  __shared__ int few[kBeamHeads], n_few;
  __shared__ __attribute__((aligned(16))) uint32_t few_top[kBeamHeads + 4];
  const int heads = W * pieces, beam = min((int)(tid * by_pieces >> 20), W - 1), row = base + beam;
  // (what closed rows' pieces hold is read and not used: nothing waits for another load here)
  const size_t list = ((size_t)base * pieces + min(tid, heads - 1)) * W;
  const unsigned long long key = best[list];
  const float score = a.score[row];
  const int over = a.done ? a.done[row] : 0;
  const bool alive = score > -INFINITY, here = tid < heads && alive && !over;
  const int step = a.step ? a.step[b] : 0, none = max(a.eos, 0);
  // lanes of a row: as many as there are, a power of two, at most a wave
  const int lane_bits = min(9 - (32 - __clz(W - 1)), 6), lanes = 1 << lane_bits, r = tid >> lane_bits;
  {
    float m = kBeamNone, s = 0.0f;
    if (r < W)
      for (int i = tid & (lanes - 1); i < pieces; i += lanes) {
        const BeamPiece p = piece[(size_t)(base + r) * pieces + i];
        const float top = fmaxf(m, p.max);
        s = s * exp_below(m - top) + p.sum * exp_below(p.max - top);
        m = top;
      }
    float all = m;
    if (lanes == kWave) {
      all = wave_max(m);
      s = wave_sum(s * exp_below(m - all));
    } else {
      for (int o = 1; o < lanes; o <<= 1) all = fmaxf(all, __shfl_xor(all, o));
      s *= exp_below(m - all);
      for (int o = 1; o < lanes; o <<= 1) s += __shfl_xor(s, o);
    }
    if (r < W && !(tid & (lanes - 1))) lse[r] = (double)all + log((double)s);
  }
  if (tid < W) chosen[tid] = -1;
  if (tid == 0) count = 0, n_few = 0;
  __syncthreads();
  const auto sum_of = [&](double lse_, float s, unsigned long long k) -> unsigned long long {
    const double x = (double)s + ((double)offer_logit(k) - lse_);
    return k && x > -INFINITY ? order_f64(x) : 0;
  };
  unsigned long long mine = here ? sum_of(lse[beam], score, key) : 0, own = key;
  if (tid < heads && alive && over && tid == beam * pieces) mine = order_f64(score), own = ~0ull;
  head_sum[tid] = mine, head_key[tid] = own, head_top[tid] = (uint32_t)(mine >> 32);
  if (tid < heads && tid == beam * pieces) scores[beam] = score;
  __syncthreads();
  // ---- the W best pieces: those that may be, then in order
  const uint32_t may = beam_reach(head_top, heads, W);
  if (mine && (uint32_t)(mine >> 32) >= may) {
    const int to = atomicAdd(&n_few, 1);
    few[to] = tid, few_top[to] = (uint32_t)(mine >> 32);
  }
  __syncthreads();
  const int some = n_few;
  if (tid < 4) few_top[some + tid] = 0;
  __syncthreads();
  if (tid < some) {
    const int h = few[tid], of = (int)(h * by_pieces >> 20);
    const unsigned long long sum = head_sum[h], k = head_key[h];
    const int place = beam_place(few_top, (some + 3) & ~3, (uint32_t)(sum >> 32), [&](int j) {
      if (j >= some) return false;
      const int g = few[j], other = (int)(g * by_pieces >> 20);
      if (head_sum[g] != sum) return head_sum[g] > sum;
      return other < of || (other == of && head_key[g] > k);
    });
    if (place < W) chosen[place] = h;
  }
  __syncthreads();
  // ---- their offers: the n-th of the q-th piece has at least q + n before it
  const int last = chosen[W - 1];
  const unsigned long long least = last >= 0 ? head_sum[last] : 1;
  constexpr int PER = kMaxBeams * kMaxBeams / kBeamHeads;
  unsigned long long next[PER];
#pragma unroll
  for (int p = 0; p < PER; p++) {  // all loads at once
    if (kBeamHeads * p >= W * W) break;
    const int i = tid + kBeamHeads * p, q = (int)(i * by_w >> 16), n = i - q * W, h = q + n < W ? chosen[q] : -1;
    next[p] = 0;
    if (h >= 0) next[p] = n ? best[((size_t)base * pieces + h) * W + n] : head_key[h];
  }
#pragma unroll
  for (int p = 0; p < PER; p++) {
    if (kBeamHeads * p >= W * W) break;
    const int i = tid + kBeamHeads * p, q = (int)(i * by_w >> 16), n = i - q * W, h = q + n < W ? chosen[q] : -1;
    if (h < 0 || (n && head_key[h] == ~0ull)) continue;
    const int from = (int)(h * by_pieces >> 20);
    const unsigned long long sum = n ? sum_of(lse[from], scores[from], next[p]) : head_sum[h];
    if (!sum || sum < least) continue;
    const int at = atomicAdd(&count, 1);
    sums[at] = sum, keys[at] = next[p], beams[at] = from, tops[at] = (uint32_t)(sum >> 32);
  }
  __syncthreads();
  const int n = count;
  if (tid < 4) tops[n + tid] = 0;
  __syncthreads();
  const auto put = [&](int w, float s, int end, int tok, int parent) {
    a.new_score[base + w] = s;
    a.new_done[base + w] = end;
    a.tok[base + w] = tok;
    a.parent[base + w] = parent;
    if (a.step && step >= 0 && step < a.hist_len) {
      const size_t h = (size_t)step * a.B * W + base + w;
      a.hist_tok[h] = tok;
      a.hist_parent[h] = parent;
    }
  };
  const uint32_t reach = n > kWave ? beam_reach(tops, n, W) : 0;
  for (int i = tid; i < n; i += kBeamHeads) {
    const unsigned long long u = sums[i], k = keys[i];
    if ((uint32_t)(u >> 32) < reach) continue;
    const int from = beams[i];
    const int place = beam_place(tops, (n + 3) & ~3, (uint32_t)(u >> 32), [&](int j) {
      if (j >= n || sums[j] != u) return j < n && sums[j] > u;
      return beams[j] < from || (beams[j] == from && keys[j] > k);
    });
    if (place >= W) continue;
    const double s = __longlong_as_double((long long)(u >> 63 ? u & 0x7FFFFFFFFFFFFFFFull : ~u));
    const int tok = k == ~0ull ? none : argmax_key_index(k);
    put(place, (float)s, k == ~0ull || tok == a.eos, tok, base + from);
  }
  if (tid >= n && tid < W) put(tid, -INFINITY, 0, none, -1);
  if (a.step && tid == 0) a.step[b] = step + 1;
}

// ---------------------------------------------------------------- launchers

// Pieces of a row and steps of each: at least a step a workgroup, eight workgroups a compute unit (128 rows of
// 151936: 22.1 us, four 24.2, two 29; 32 such beams of four prompts 44, 54, 64), and no more pieces of a prompt
// than its merge has threads.
static void beam_cut(int B, int W, int V, int &pieces, int &per) {
  const int steps = (V + kBeamStep - 1) / kBeamStep;
  const int most = std::min({steps, kBeamHeads / W, std::max(1, 2048 / (B * W))});
  per = (steps + most - 1) / most;
  pieces = (steps + per - 1) / per;
}

static size_t piece_bytes(int rows, int pieces) { return ((size_t)rows * pieces * sizeof(BeamPiece) + 15) & ~size_t(15); }

size_t beam_select_work_bytes(int B, int W, int V) {
  int pieces, per;
  beam_cut(B, W, V, pieces, per);
  return piece_bytes(B * W, pieces) + (size_t)B * W * pieces * W * 8;
}

hipError_t launch_beam_select(const BeamArgs &a, void *work, hipStream_t s) {
  int pieces, per;
  beam_cut(a.B, a.W, a.V, pieces, per);
  const int rows = a.B * a.W;
  BeamPiece *piece = static_cast<BeamPiece *>(work);
  auto *best = reinterpret_cast<unsigned long long *>(static_cast<char *>(work) + piece_bytes(rows, pieces));
  const dim3 grid(pieces, std::min(rows, kBeamGridY), (rows + kBeamGridY - 1) / kBeamGridY);
  hipLaunchKernelGGL(beam_piece_kernel, grid, dim3(kBeamWaves * kWave), 0, s, a, per, pieces, piece, best);
  hipLaunchKernelGGL(beam_merge_kernel, dim3(a.B), dim3(kBeamHeads), 0, s, a, pieces, 65536u / a.W + 1,
                     (1u << 20) / pieces + 1, piece, best);
  return hipGetLastError();
}

}  // namespace lbk
