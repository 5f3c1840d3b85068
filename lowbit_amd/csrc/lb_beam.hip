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
constexpr int kBeamRoom = 192;                           // keys that a wave keeps before it sorts them out
constexpr int kBeamGridY = 1 << 15;                      // rows in the grid's second dimension
constexpr int kBeamHeads = 256;                          // pieces of a prompt's rows at most
constexpr float kBeamNone = -3.4028234663852886e38f;     // the maximum before any logit: finite

// What a workgroup leaves of its piece of a row: `best` keys, in descending order, 0 past the last.
struct BeamPiece {
  float max, sum;  // sum exp(x - max), NaN where the row offers nothing
};

// A row that offers tokens: its beam has not ended and there is one.
__device__ __forceinline__ bool beam_open(const BeamArgs &a, int row) {
  const float s = a.score[row];
  return !(a.done && a.done[row]) && s > -INFINITY;
}

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

// ---------------------------------------------------------------- pieces of rows

// The W largest of n keys (n <= kBeamRoom, W <= n, all different), by one wave, to the front in descending
// order: a key's place is how many are larger. Returns the last of them.
__device__ __forceinline__ unsigned long long beam_sort(unsigned long long *keys, int n, int W) {
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

// The largest float that at least W of the lanes' values reach (-inf: fewer are above -inf), found bit by bit
// from the top on the values' ordered numbers; as soon as exactly W reach it nothing larger is needed.
__device__ __forceinline__ float beam_threshold(float v, int W) {
  const uint32_t k = (uint32_t)(argmax_key(v, 0) >> 32);  // (v is not NaN)
  uint32_t t = 0;
  for (int b = 31; b >= 0; b--) {
    const uint32_t c = t | 1u << b;
    const int n = __popcll((unsigned long long)__ballot(k >= c));
    if (n >= W) t = c;
    if (n == W) break;
  }
  return t < 0x00800000u ? kBeamNone : offer_logit((unsigned long long)t << 32);
}

// A workgroup a piece of `per` steps of a row. Every wave keeps the keys above its own threshold in LDS: the
// first chunk's comes from its lanes' maxima (the W-th largest of 64: W of them at least reach it, and few
// more), later ones from sorting the kept keys out, so that nearly all chunks of a row end after a comparison
// of 16 logits' maximum, and no wave waits for another before the end.
//
// What bounds it: see beam_merge_kernel.
__global__ __launch_bounds__(kBeamWaves *kWave) void beam_piece_kernel(BeamArgs a, int per, int pieces,
                                                                       BeamPiece *__restrict__ piece,
                                                                       unsigned long long *__restrict__ best) {
  const int row = (int)(blockIdx.y + blockIdx.z * kBeamGridY), at = blockIdx.x, lane = threadIdx.x & (kWave - 1), W = a.W;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  if (row >= a.B * W || !beam_open(a, row)) return;
  __shared__ unsigned long long keys[kBeamWaves][kBeamRoom];
  __shared__ unsigned long long floor_key[kBeamWaves];
  __shared__ float smax[kBeamWaves], ssum[kBeamWaves];
  __shared__ int kept[kBeamWaves];
  const Rsrc x = make_rsrc(a.logits + (size_t)row * a.ld, 4u * (uint32_t)a.V);  // reads past the row give 0
  const int end = min(a.V, (at + 1) * per * kBeamStep);
  int v0 = at * per * kBeamStep + wave * kBeamChunk;
  unsigned long long *mine = keys[wave], low = 0;
  float m = kBeamNone, sum = 0.0f, least = 0.0f;
  int n = 0;
  bool begun = false;
  float4 next[kBeamLoads];
  const auto load = [&](int v) {
#pragma unroll
    for (int i = 0; i < kBeamLoads; i++) next[i] = ld_f4(x, 4u * (uint32_t)(v + 4 * kWave * i + 4 * lane));
  };
  if (v0 < end) load(v0);
  for (; v0 < end; v0 += kBeamStep) {
    float f[4 * kBeamLoads];
#pragma unroll
    for (int i = 0; i < kBeamLoads; i++) f[4 * i] = next[i].x, f[4 * i + 1] = next[i].y, f[4 * i + 2] = next[i].z, f[4 * i + 3] = next[i].w;
    if (v0 + kBeamStep < end) load(v0 + kBeamStep);
    const auto token = [&](int i) { return v0 + 4 * kWave * (i >> 2) + 4 * lane + (i & 3); };
    if (v0 + kBeamChunk > a.V) {
#pragma unroll
      for (int i = 0; i < 4 * kBeamLoads; i++) f[i] = token(i) < a.V ? f[i] : -INFINITY;
    }
    float top = f[0];
#pragma unroll
    for (int i = 1; i < 4 * kBeamLoads; i++) top = fmaxf(top, f[i]);
    const float was = m;
    m = fmaxf(m, top);
    sum *= exp_below(was - m);
#pragma unroll
    for (int i = 0; i < 4 * kBeamLoads; i++) sum += exp_below(f[i] - m);
    if (!begun) least = beam_threshold(fmaxf(top, -INFINITY), W), begun = true;
    if (!__any(top >= least)) continue;
#pragma unroll
    for (int i = 0; i < 4 * kBeamLoads; i++) {
      if (!__any(f[i] >= least)) continue;
      const unsigned long long key = argmax_key(f[i], token(i)), push = __ballot(f[i] >= least && key > low);
      if (push >> lane & 1) mine[n + __popcll(push & ((1ull << lane) - 1))] = key;
      n += __popcll(push);
      if (n > kBeamRoom - kWave) {
        __builtin_amdgcn_wave_barrier();
        low = beam_sort(mine, n, W);
        n = W;
        least = offer_logit(low);
      }
    }
  }
  // ---- the waves' sums and keys
  const float all = wave_max(m);
  const float part = wave_sum(sum * exp_below(m - all));
  if (lane == 0) smax[wave] = all, ssum[wave] = part, kept[wave] = n, floor_key[wave] = low;
  __syncthreads();
  const size_t to = (size_t)row * pieces + at;
  float top = smax[0], total = 0.0f;
  int before[kBeamWaves + 1] = {0};
#pragma unroll
  for (int w = 0; w < kBeamWaves; w++) {
    top = fmaxf(top, smax[w]);
    low = floor_key[w] > low ? floor_key[w] : low;
    before[w + 1] = before[w] + kept[w];
  }
#pragma unroll
  for (int w = 0; w < kBeamWaves; w++) total += ssum[w] * exp_below(smax[w] - top);
  if (threadIdx.x == 0) piece[to] = {top, total};
  // a key's place is how many of the workgroup's are larger; a wave's W-th largest is no larger than theirs
  n = before[kBeamWaves];
  for (int i = threadIdx.x; i < max(n, W); i += kBeamWaves * kWave) {
    if (i >= n) {
      best[to * W + i] = 0;
      continue;
    }
    int w = 0;
#pragma unroll
    for (int k = 1; k < kBeamWaves; k++) w += i >= before[k];
    const unsigned long long key = keys[w][i - before[w]];
    if (key < low) continue;
    int place = 0;
#pragma unroll
    for (int k = 0; k < kBeamWaves; k++)
      for (int j = 0; j < kept[k]; j++) place += keys[k][j] > key;
    if (place < W) best[to * W + place] = key;
  }
}

// ---------------------------------------------------------------- a prompt

// An offer of the prompt's: larger sums first, then the lower place, then the larger key.
struct BeamOffer {
  unsigned long long sum, key;  // order_f64 of the sum (0: none); key of the logit, ~0: an ended beam itself
  int beam;
};
__device__ __forceinline__ bool beam_before(const BeamOffer &a, const BeamOffer &b) {
  return a.sum != b.sum ? a.sum > b.sum : a.beam != b.beam ? a.beam < b.beam : a.key > b.key;
}

// The W best offers lie in the W pieces whose first offers are the best: those and, of their further offers,
// the ones that reach the last of them are put in order by counting who comes before whom.
__global__ __launch_bounds__(kBeamHeads) void beam_merge_kernel(BeamArgs a, int pieces,
                                                                const BeamPiece *__restrict__ piece,
                                                                const unsigned long long *__restrict__ best) {
  constexpr int kOffers = kMaxBeams * (kMaxBeams + 1) / 2;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave, W = a.W, base = b * W;
  __shared__ double lse[kMaxBeams];
  __shared__ BeamOffer head[kBeamHeads], offer[kOffers];
  __shared__ int chosen[kMaxBeams], count;
  const int heads = W * pieces, beam = min(tid / pieces, W - 1), row = base + beam;
  const float score = a.score[row];
  const bool ended = a.done && a.done[row] && score > -INFINITY, open = beam_open(a, row);
  const bool here = tid < heads && open;
  const unsigned long long key = here ? best[((size_t)base * pieces + tid) * W] : 0;
  const int step = a.step ? a.step[b] : 0, none = max(a.eos, 0);
  for (int r = wave; r < W; r += kBeamHeads / kWave) {  // a wave a row
    float m = kBeamNone, s = 0.0f;
    if (beam_open(a, base + r))
      for (int i = lane; i < pieces; i += kWave) {
        const BeamPiece p = piece[(size_t)(base + r) * pieces + i];
        const float top = fmaxf(m, p.max);
        s = s * exp_below(m - top) + p.sum * exp_below(p.max - top);
        m = top;
      }
    const float all = wave_max(m);
    s = wave_sum(s * exp_below(m - all));
    if (lane == 0) lse[r] = (double)all + log((double)s);
  }
  if (tid < W) chosen[tid] = -1;
  if (tid == 0) count = 0;
  __syncthreads();
  const auto sum_of = [&](int w, float s, unsigned long long k) -> unsigned long long {
    const double x = (double)s + ((double)offer_logit(k) - lse[w]);
    return k && x > -INFINITY ? order_f64(x) : 0;
  };
  BeamOffer mine = {0, key, beam};
  if (here) mine.sum = sum_of(beam, score, key);
  if (tid < heads && ended && tid % pieces == 0) mine = {order_f64(score), ~0ull, beam};
  if (tid < heads) head[tid] = mine;
  __syncthreads();
  // ---- the W best pieces
  if (mine.sum) {
    int place = 0;
    for (int j = 0; j < heads; j++) place += beam_before(head[j], mine);
    if (place < W) chosen[place] = tid;
  }
  __syncthreads();
  // ---- their offers: the n-th of the q-th piece has q + n before it
  const int last = chosen[W - 1];
  const unsigned long long least = last >= 0 ? head[last].sum : 1;
  for (int i = tid; i < W * W; i += kBeamHeads) {
    const int q = i / W, n = i % W, h = chosen[q];
    if (h < 0 || q + n >= W) continue;
    BeamOffer o = head[h];
    if (n) {
      if (o.key == ~0ull) continue;
      o.key = best[((size_t)base * pieces + h) * W + n];
      o.sum = sum_of(o.beam, a.score[base + o.beam], o.key);
    }
    if (o.sum && o.sum >= least) offer[atomicAdd(&count, 1)] = o;
  }
  __syncthreads();
  const int n = count;
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
  for (int i = tid; i < n; i += kBeamHeads) {
    const BeamOffer o = offer[i];
    int place = 0;
    for (int j = 0; j < n; j++) place += beam_before(offer[j], o);
    if (place >= W) continue;
    const unsigned long long u = o.sum;
    const double s = __longlong_as_double((long long)(u >> 63 ? u & 0x7FFFFFFFFFFFFFFFull : ~u));
    const bool itself = o.key == ~0ull;
    const int tok = itself ? none : argmax_key_index(o.key);
    put(place, (float)s, itself || tok == a.eos, tok, base + o.beam);
  }
  if (tid >= n && tid < W) put(tid, -INFINITY, 0, none, -1);
  if (a.step && tid == 0) a.step[b] = step + 1;
}

// ---------------------------------------------------------------- launchers

// Pieces of a row and steps of each: at least a step a workgroup, four workgroups a compute unit, and no more
// pieces of a prompt than its merge has threads.
static void beam_cut(int B, int W, int V, int &pieces, int &per) {
  const int steps = (V + kBeamStep - 1) / kBeamStep;
  const int most = std::min({steps, kBeamHeads / W, std::max(1, 1024 / (B * W))});
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
  hipLaunchKernelGGL(beam_merge_kernel, dim3(a.B), dim3(kBeamHeads), 0, s, a, pieces, piece, best);
  return hipGetLastError();
}

}  // namespace lbk
