// The paged 8-bit key / value cache of several sequences: appending tokens to it
// (lbd_kv8_append) and attending over it (lbd_kv8_attention). No reference counterpart:
// its cache is one float32 array per sequence (src/lowbit/model.py:264-297).
//
// A block is the `page` tokens of one page and one KV head: E4M3 codes [page][D] and one
// E8M0 exponent e, value = code 2^(e - 127); e = 255 makes the block NaN. Relative rounding
// (2^-4 over 2^14 of range below the block's largest value) costs outlier channels nothing,
// and a power of two lets the exponent grow with later tokens of the block by a shift, which
// leaves normal codes as they are: what a block holds does not depend on how its tokens were
// cut into calls (but for codes among the subnormals, rounded once per growth).
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "lb_attn.h"
#include "lb_device.h"
#include "lb_internal.h"

namespace lbk {

// ---------------------------------------------------------------- the batch

// Inclusive sum over the lanes up to this one.
__device__ __forceinline__ int wave_scan(int v) {
  v += dpp_i<0x111>(v, 0);                   // row_shr:1
  v += dpp_i<0x112>(v, 0);                   // row_shr:2
  v += dpp_i<0x114>(v, 0);                   // row_shr:4
  v += dpp_i<0x118>(v, 0);                   // row_shr:8
  v += dpp_i<kDppRowBcast15, 0xA>(v, 0);
  v += dpp_i<kDppRowBcast31, 0xC>(v, 0);
  return v;
}

// One sequence's new tokens: rows row0 .. row0 + n - 1 at positions past ..
struct Kv8Seq {
  int b, row0, n, past;
};

// Sequence b of the batch (b < B) as this lane reads it, its rows kept inside [0, T) and its
// tokens to max_new; past < 0: no new tokens.
__device__ __forceinline__ Kv8Seq kv8_seq(const Kv8Args &a, int b) {
  Kv8Seq s = {b, 0, 0, 0};
  if (b < a.B) {
    const int r0 = a.q_start[b], r1 = a.q_start[b + 1], p = a.past[b];
    s.row0 = min(max(r0, 0), a.T);
    s.n = p < 0 ? 0 : min(max(min(r1, a.T) - s.row0, 0), a.max_new);
    s.past = min(max(p, 0), kKv8MaxPos);
  }
  return s;
}

__device__ __forceinline__ Kv8Seq kv8_lane(const Kv8Seq &s, int lane) {
  return {__builtin_amdgcn_readlane(s.b, lane), __builtin_amdgcn_readlane(s.row0, lane),
          __builtin_amdgcn_readlane(s.n, lane), __builtin_amdgcn_readlane(s.past, lane)};
}

// Unit u of the batch's units (sequence b has units(its Kv8Seq) of them, in order): its
// sequence in s, its index there in `at` and, where asked, the sum of weight(..) over the
// sequences before it. False past the last. By the whole wave, 64 sequences a step, the first
// of them in `first` already.
struct Kv8None {
  __device__ int operator()(const Kv8Seq &) const { return 0; }
};
template <class F, class W = Kv8None>
__device__ __forceinline__ bool kv8_locate(const Kv8Args &a, const Kv8Seq &first, int u, F units, Kv8Seq &s, int &at,
                                           W weight = W(), int *before = nullptr) {
  const int lane = threadIdx.x & (kWave - 1);
  int base = 0, sum = 0;
  for (int b0 = 0; b0 < a.B; b0 += kWave) {
    const Kv8Seq q = b0 ? kv8_seq(a, b0 + lane) : first;
    const int c = units(q), inc = wave_scan(c), all = __builtin_amdgcn_readlane(inc, 63);
    const int wt = before ? weight(q) : 0, winc = before ? wave_scan(wt) : 0;
    if (u < base + all) {
      const int l = __ffsll((unsigned long long)__ballot(u - base < inc)) - 1;
      s = kv8_lane(q, l);
      at = u - base - __builtin_amdgcn_readlane(inc - c, l);
      if (before) *before = sum + __builtin_amdgcn_readlane(winc - wt, l);
      return true;
    }
    base += all;
    if (before) sum += __builtin_amdgcn_readlane(winc, 63);
  }
  return false;
}

// The sequence that row belongs to; false for a row of none.
__device__ __forceinline__ bool kv8_find_row(const Kv8Args &a, int row, Kv8Seq &s) {
  const int lane = threadIdx.x & (kWave - 1);
  for (int b0 = 0; b0 < a.B; b0 += kWave) {
    const Kv8Seq q = kv8_seq(a, b0 + lane);
    const unsigned long long in = __ballot(row >= q.row0 && row - q.row0 < q.n);
    if (in) {
      s = kv8_lane(q, __ffsll(in) - 1);
      return true;
    }
  }
  return false;
}

// ---------------------------------------------------------------- append

// Smallest e with |x| <= 448 2^(e - 127) for the float32 bits of |x| (448 = 1.75 2^8);
// 255 where x is not finite.
__device__ __forceinline__ int kv8_exponent(int bits) {
  if (bits >= 0x7F800000) return 255;
  return max((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000), 0);
}

__device__ __forceinline__ uint32_t e4m3x4(float4 v, float s) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(v.x * s, v.y * s, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(v.z * s, v.w * s, w, true);
  return (uint32_t)w;
}

__device__ __forceinline__ float4 e4m3x4_f32(uint32_t w) {
  const v2f a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return make_float4(a.x, a.y, b.x, b.y);
}

__device__ __forceinline__ int abs_bits(float x) { return __float_as_int(x) & 0x7FFFFFFF; }
__device__ __forceinline__ int abs_bits(float4 v) {
  return max(max(abs_bits(v.x), abs_bits(v.y)), max(abs_bits(v.z), abs_bits(v.w)));
}

__device__ __forceinline__ float4 add4(float4 a, float4 b) {
  return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}

__device__ __forceinline__ void rope4_pair(float4 &a, float4 &b, float4 c, float4 s) {
  rope_pair(a.x, b.x, c.x, s.x, a.x, b.x);
  rope_pair(a.y, b.y, c.y, s.y, a.y, b.y);
  rope_pair(a.z, b.z, c.z, s.z, a.z, b.z);
  rope_pair(a.w, b.w, c.w, s.w, a.w, b.w);
}

// One launch, two kinds of workgroups (NT threads):
//   the first nkv 2 KV: block (page, KV head) of K or V that new tokens fall into, the whole
//     block's tokens of this call at once, so that its exponent is settled by one reduction
//     and nobody else writes it. A thread takes IT items of 8 elements: 4 of each half of a
//     token's head row, a rotation's partners (page D / 8 items at most).
//   the others: 8 NT elements of a row's query heads, rotated into q_out.
//
// What bounds it: a step, the launch and three loads one after the other (the batch, the page, the
// block's exponent): one token of 14 heads on 2 2.6 us, 64 sequences of 32 heads on 8 3.2 us.
// Prompts, the bytes: 4 sequences of up to 1000 tokens, 32 heads on 8, 45.8 MB in 10.6 us = 4.3
// TB/s (a large copy reaches 5.2). A block is one workgroup's so that its largest element costs no
// second pass over the rows and no atomic, and codes leave as whole words.
//
// Rounding: rotation as lbd_qkv_rope's, every product and sum to float32; a code to the nearest
// E4M3, ties to even, once, and once more for each later growth of its block's exponent.
template <int D, int NT, int IT>
__global__ __launch_bounds__(NT) void kv8_append_kernel(Kv8Args a, const float *qkv, int stride,
                                                        const float *__restrict__ bias, int H,
                                                        const float *__restrict__ cosT,
                                                        const float *__restrict__ sinT, int max_pos, float *q_out,
                                                        int q_stride, int nkv) {
  constexpr int half = D / 2, PER = D / 8;  // items of a head row
  const int tid = threadIdx.x;
  const int page = 1 << a.page_shift, cap = a.max_pages << a.page_shift;
  const int id = (int)blockIdx.x, per_page = 2 * a.KV;
  const auto angle = [&](int p) { return (size_t)min(p, max_pos - 1) * half; };  // past the tables: the last angle
  if (id >= nkv * per_page) {
    const int chunks = (H * PER + NT - 1) / NT, at = id - nkv * per_page;
    const int row = at / chunks, item = at % chunks * NT + tid;
    const int h = item / PER, e = 4 * (item % PER);
    const bool in = h < H;
    const float *x = qkv + (size_t)row * stride + (in ? h * D + e : 0);
    float4 x1 = *reinterpret_cast<const float4 *>(x), x2 = *reinterpret_cast<const float4 *>(x + half);
    Kv8Seq s;
    if (!kv8_find_row(a, row, s) || !in) return;
    if (bias) {
      x1 = add4(x1, *reinterpret_cast<const float4 *>(bias + h * D + e));
      x2 = add4(x2, *reinterpret_cast<const float4 *>(bias + h * D + half + e));
    }
    const size_t an = angle(s.past + row - s.row0) + e;
    rope4_pair(x1, x2, *reinterpret_cast<const float4 *>(cosT + an), *reinterpret_cast<const float4 *>(sinT + an));
    float *y = q_out + (size_t)row * q_stride + h * D + e;
    *reinterpret_cast<float4 *>(y) = x1;
    *reinterpret_cast<float4 *>(y + half) = x2;
    return;
  }
  const int unit = id / per_page, kv = (id % per_page) >> 1;
  const bool isv = id & 1;
  Kv8Seq s;
  int at;
  const auto pages_of = [&](const Kv8Seq &q) {
    const int end = min(q.past + q.n, cap);
    return end > q.past ? ((end - 1) >> a.page_shift) - (q.past >> a.page_shift) + 1 : 0;
  };
  if (!kv8_locate(a, kv8_seq(a, tid & (kWave - 1)), unit, pages_of, s, at)) return;
  const int pi = (s.past >> a.page_shift) + at;
  const int t0 = max(s.past, pi << a.page_shift), t1 = min(min(s.past + s.n, cap), (pi + 1) << a.page_shift);
  const int lo = t0 & (page - 1), items = (t1 - t0) * PER;
  const int pg = a.table[(size_t)s.b * a.max_pages + pi];
  if ((unsigned)pg >= (unsigned)a.pages) return;  // no such page: its tokens are dropped
  uint8_t *ep = (isv ? a.ve : a.ke) + (size_t)pg * a.KV + kv;
  uint8_t *codes = (isv ? a.v : a.k) + (((size_t)pg * a.KV + kv) << a.page_shift) * D;
  // a page begun in this call holds nothing yet; read (and waited for) before any thread writes it
  const int e_old = lo ? __builtin_amdgcn_readfirstlane((int)*ep) : 0;
  const int col = (H + (isv ? a.KV : 0) + kv) * D;
  float4 x1[IT], x2[IT];
  int big = 0;
#pragma unroll
  for (int i = 0; i < IT; i++) {
    const int it = tid + NT * i, tok = it / PER, e = 4 * (it % PER);
    if (it >= items) break;
    const int p = t0 + tok;
    const float *x = qkv + (size_t)(s.row0 + p - s.past) * stride + col + e;
    x1[i] = *reinterpret_cast<const float4 *>(x);
    x2[i] = *reinterpret_cast<const float4 *>(x + half);
    if (bias) {
      x1[i] = add4(x1[i], *reinterpret_cast<const float4 *>(bias + col + e));
      x2[i] = add4(x2[i], *reinterpret_cast<const float4 *>(bias + col + half + e));
    }
    if (!isv) {
      const size_t an = angle(p) + e;
      rope4_pair(x1[i], x2[i], *reinterpret_cast<const float4 *>(cosT + an),
                 *reinterpret_cast<const float4 *>(sinT + an));
    }
    big = max(big, max(abs_bits(x1[i]), abs_bits(x2[i])));
  }
  big = wave_max_i32(big);
  if constexpr (NT > kWave) {
    __shared__ int red[NT / kWave];
    if ((tid & (kWave - 1)) == 0) red[tid / kWave] = big;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / kWave; w++) big = max(big, red[w]);
  }
  const int e = max(e_old, kv8_exponent(big));
  const bool bad = e == 255;
  if (!bad && e != e_old && lo) {  // the earlier tokens' codes in the new unit
    const int f = 127 + e_old - e;
    const float shift = __int_as_float(f > 0 ? f << 23 : 0);  // below 2^-126 of E4M3 values: zeros
    for (int i = 16 * tid; i < lo * D; i += 16 * NT) {
      uint4 w = *reinterpret_cast<const uint4 *>(codes + i);
      w.x = e4m3x4(e4m3x4_f32(w.x), shift);
      w.y = e4m3x4(e4m3x4_f32(w.y), shift);
      w.z = e4m3x4(e4m3x4_f32(w.z), shift);
      w.w = e4m3x4(e4m3x4_f32(w.w), shift);
      *reinterpret_cast<uint4 *>(codes + i) = w;
    }
  }
  // codes y 2^(127 - e), exact but for the rounding to E4M3; zeros in a NaN block
  const float inv = __int_as_float(e < 254 ? (254 - e) << 23 : 0x00400000);  // 2^-127 is a subnormal
#pragma unroll
  for (int i = 0; i < IT; i++) {
    const int it = tid + NT * i, tok = it / PER, el = 4 * (it % PER);
    if (it >= items) break;
    uint8_t *c = codes + (lo + tok) * D + el;
    *reinterpret_cast<uint32_t *>(c) = bad ? 0u : e4m3x4(x1[i], inv);
    *reinterpret_cast<uint32_t *>(c + half) = bad ? 0u : e4m3x4(x2[i], inv);
  }
  if (tid == 0 && (e != e_old || !lo)) *ep = (uint8_t)e;
}

// ---------------------------------------------------------------- attention
//
// A sequence's query rows of one KV head are its new tokens' G = H / KV heads, row
// r = token G + head, cut into row blocks of R; a row block's keys are cut into slices, each
// one workgroup's. Slices that share a row block leave partial sums that a second launch adds.
//
// Scores are kept in base 2: x = q k log2(e) / sqrt(D). A block's V exponent ev joins the
// exponential: a row's reference m is a whole number (so rescaling by 2^(m - m') is exact) at most
// kKv8Head below the largest x + ev so far, and its weights w = 2^(x + ev - m) multiply V's codes
// as they are, so that what a row sees of V decides its precision, however far apart the blocks'
// exponents are. The denominator is sum w 2^(mid - ev), in the unit 2^(m - mid), with
// mid 50 below the slice's largest ev: every factor stays within 2^+-50. Blocks of V more than
// 2^100 below the largest count as zeros.
//
// An E4M3 code is exact in float16 and in bf16, so the matrix products take codes as they are and
// q and w in terms whose sum they are. q, two float16 terms: 22 bits of an element, and 2^-38 of its
// row's largest where that is more (the matrix cores take float16's subnormals as they are). w, three
// bf16 terms: all 24 bits however far it lies below the largest, as the keys that it outweighs may
// hold the larger values (two float16 terms lost weights e^-17 below the row's largest, and those
// e^-30 below it altogether; three bf16 terms made 2048 tokens of 32 heads 9 % slower. Two of them,
// rounded: 1 % faster, but errors of 2e-6 to 7e-6 in place of 4e-7 to 1.2e-6).

constexpr int kKv8GridY = 1 << 15;  // units of a call in the grid's second dimension
constexpr float kKv8Head = 8.0f;  // x + ev may lie this far above the reference: few new ones are needed
constexpr int kKv8Waves = 4;       // of an attention workgroup
// Floats before a class's sums: 256 bytes, as sums 16 bytes off the cache lines cost 61 steps 0.8 of 59 us.
constexpr int kKv8CutHead = 64;
constexpr int kKv8Spread = 100;    // exponents of V below the largest that still count
// The reference before any key: finite, so that masked scores of -inf weigh exp2(-inf) = 0 under it.
constexpr float kKv8None = -3.4028234663852886e38f;
constexpr float kKv8Log2e = 1.4426950408889634f;

// How a launch cuts its rows and keys: the sequences of rows_min .. rows_max rows a KV head, in
// row blocks of R = 1 << r_shift rows, their keys in slices of at least min_keys; see
// kv8_slice_keys for the rest.
struct Kv8Cut {
  int G, R, r_shift, rows_min, rows_max, min_keys;
  unsigned g_inv;  // ceil(2^32 / G)
  int few_blocks, slots_few, slots;  // slices a KV head: with at most few_blocks row blocks, and with more
  float units, fits;  // many rows: compute units a KV head, and workgroups that they hold; else 0
  int span;           // keys that a row block reads at most
};

// One class of a call's sequences, by their rows, and where its slices' sums lie in the workspace:
// `sums` floats of them from `at` on, their scalars behind, and kKv8CutHead floats before them the
// keys of a slice, which the first launch decides and the merge reads: the merge finds the sums
// where they were written, whatever the compiler makes of the decision's float arithmetic.
// Of a KV head at most `blocks` row blocks and `units` slices. merge: workgroups a row block of the
// second launch, 0: one a row.
struct Kv8Part {
  Kv8Cut cut;
  int blocks, units, merge;
  size_t at, sums;
};

__device__ __forceinline__ void kv8_put_cut(float *work, const Kv8Part &pt, int slice_keys) {
  *reinterpret_cast<int *>(work + pt.at - kKv8CutHead) = slice_keys;
}
__device__ __forceinline__ int kv8_cut_of(const float *work, const Kv8Part &pt) {
  // (whatever it holds, a number that kv8_slices takes)
  return max(*reinterpret_cast<const int *>(work + pt.at - kKv8CutHead) & ~127, 128);
}

// r / G for 0 <= r < 2^32 / 2: the product is at most one too large.
__device__ __forceinline__ int kv8_token(const Kv8Cut &c, int r) {
  if (c.G == 1) return r;
  const int t = (int)__umulhi((unsigned)r, c.g_inv);
  return t * c.G > r ? t - 1 : t;
}

__device__ __forceinline__ int kv8_row_blocks(const Kv8Cut &c, const Kv8Seq &s) {
  const int rows = s.n * c.G;  // T H <= 2^30
  return rows >= c.rows_min && rows <= c.rows_max ? (rows + (1 << c.r_shift) - 1) >> c.r_shift : 0;
}
// The most keys that a row block of the sequence reads.
template <bool WIN>
__device__ __forceinline__ int kv8_keys(const Kv8Args &a, const Kv8Cut &c, const Kv8Seq &s) {
  const int all = min(s.past + s.n, a.max_pages << a.page_shift);
  return WIN ? min(all, c.span) : all;
}

// Rows of a row block, by the column blocks of 16 a wave takes (0: 8 rows, both terms in one).
__host__ __device__ constexpr int kv8_rows(int nc) { return nc ? 16 * nc : 8; }

// How many keys a slice has, in steps of 128 (a chunk of each wave). `first`: sequences 0 .. 63 by lane.
//
// Few rows (the cache's bytes bound them): the batch's row blocks times keys over the slots, so
// that however the lengths differ the slices are alike. Few row blocks (alike, mostly) get 512
// slices in all, two a compute unit: 60000 keys of 8 KV heads 28.6 us, with 1024 32.5 (more sums to
// merge); many get 2048: 61 sequences of 50 to 4096 keys 59.0 us, with 1024 60.1, with 512 61.9.
//
// Many rows (the instructions bound them): the mean row block's keys in ns slices, lane ns - 1
// weighing what they cost, in keys. For one sequence, whose slices are alike: a slice's keys and
// 512 for a workgroup's beginning and end, times 0.72 k + 0.25 with k workgroups on the fullest
// compute unit (measured 1, 1.5, 2.4), and the sums' way to the merge. (200 tokens behind 8000, 25
// row blocks of 8 KV heads: five slices 74.9 us, four 87.4, three 82.1; 64 behind 8000, 8 row
// blocks: four 33.0 us, six 36.6, three 39.1; 300 behind 2000 on 2 KV heads: three even slices 20.5
// us, 1024 + 1024 + 252 keys 25.0; 1000 tokens, 219 row blocks of 2: one 17.1 us, two 22.3.) For
// several, whose slices fill the units as they come: the rounds that the device takes, the last two
// thirds where it fills half of it (3 of up to 100 tokens behind 6000, 32 heads on 8: 41.6 us, by
// the other rule 45.2; 16 of up to 40 behind 3000: 38.6 and 44.3).
//
// Slices are never more than slots and row blocks together: the few's sum in float 1 % up, the
// many's product 2 %.
template <bool WIN>
__device__ __forceinline__ int kv8_slice_keys(const Kv8Args &a, const Kv8Cut &c, const Kv8Seq &first) {
  if (WIN && c.span <= c.min_keys) return c.min_keys;
  const int lane = threadIdx.x & (kWave - 1);
  float blocks = (float)kv8_row_blocks(c, first), sum = blocks * (float)kv8_keys<WIN>(a, c, first);
  for (int b0 = kWave; b0 < a.B; b0 += kWave) {
    const Kv8Seq s = kv8_seq(a, b0 + lane);
    const float n = (float)kv8_row_blocks(c, s);
    blocks += n;
    sum += n * (float)kv8_keys<WIN>(a, c, s);
  }
  blocks = fmaxf(wave_sum(blocks), 1.0f), sum = wave_sum(sum);
  if (c.units > 0.0f) {
    const bool one = a.B == 1;
    const float mean = (one ? 1.0f : 1.01f) * sum / blocks;
    const auto keys_of = [&](float ns) {  // (for one, an exact multiple stays)
      const float x = one ? 128.0f * ceilf(mean / ns * 0x1p-7f - 0x1p-11f) : 256.0f * ceilf(mean / ns * 0x1p-8f);
      return fmaxf(x, (float)c.min_keys);
    };
    const float ns = (float)(lane + 1), load = blocks * ns / c.units, full = blocks * ns / c.fits;
    const float k = load <= 4.0f ? ceilf(load) : load + 0.5f, whole = floorf(full), rest = full - whole;
    const float rounds = full < 3.0f ? whole + (rest == 0.0f ? 0.0f : rest <= 0.5f ? 0.67f : 1.0f) : full + 0.5f;
    float cost = one ? (0.72f * k + 0.25f) * (keys_of(ns) + 512.0f) : rounds * (mean / ns + 512.0f);
    if (lane) cost += 256.0f + (one ? 180.0f * load : 16.0f * ns);
    if (lane && (mean < ns * (float)c.min_keys || 1.02f * blocks * ns > (float)c.slots)) cost = INFINITY;
    const int best = __ffsll((unsigned long long)__ballot(cost == -wave_max(-cost)));
    // one: only sequences well longer than the mean are cut, the fewer the more row blocks there are
    // (and no more than there are slots for)
    const float per = best > 1 ? keys_of((float)best)
                               : fmaxf(keys_of(blocks > 1.5f * c.fits ? 0.5f : 0.8f), keys_of((float)c.slots / blocks));
    return (int)fminf(per, (float)kKv8MaxPos);
  }
  const float per = 1.01f * sum / (float)(blocks <= (float)c.few_blocks ? c.slots_few : c.slots);
  return max(c.min_keys, ((int)fminf(per, (float)kKv8MaxPos) | 255) + 1);
}

// ceil(keys / SL) for SL a multiple of 128 and keys <= 2^30, by way of float: both counts of
// 128 keys are exact there, the quotient is at most one off.
__device__ __forceinline__ int kv8_slices(int keys, int slice_keys) {
  const int s = slice_keys >> 7, n = ((keys + 127) >> 7) + s - 1;
  int d = (int)((float)n * __builtin_amdgcn_rcpf((float)s));
  const int rest = n - d * s;
  d += rest < 0 ? -1 : rest >= s ? 1 : 0;
  return d;
}

// Row block and slice of unit u; or, u a row block, that row block and the units before its
// sequence's. By slices of w.slice_keys keys.
struct Kv8Unit {
  Kv8Seq s;
  int rb, slice, slices, slice_keys, before, at;
};
template <bool BLOCK, bool WIN>
__device__ __forceinline__ bool kv8_unit(const Kv8Args &a, const Kv8Cut &c, const Kv8Seq &first, int u, Kv8Unit &w) {
  const auto blocks = [&](const Kv8Seq &s) { return kv8_row_blocks(c, s); };
  const auto slices = [&](const Kv8Seq &s) { return kv8_slices(kv8_keys<WIN>(a, c, s), w.slice_keys); };
  const auto units = [&](const Kv8Seq &s) { return blocks(s) * slices(s); };
  if constexpr (BLOCK) {
    if (!kv8_locate(a, first, u, blocks, w.s, w.at, units, &w.before)) return false;
    w.slices = slices(w.s);
    w.rb = w.at;
  } else {  // the last row blocks, which see the most keys, first
    if (!kv8_locate(a, first, u, units, w.s, w.at)) return false;
    w.slices = slices(w.s);
    const int back = w.slices == 1 ? w.at : w.at / w.slices;
    w.rb = blocks(w.s) - 1 - back;
    w.slice = w.at - back * w.slices;
  }
  return true;
}

__device__ __forceinline__ v8h e4m3x8_h(uint32_t lo, uint32_t hi) {
  const h2v a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
  const h2v b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
  const h2v c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
  const h2v d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
  return v8h{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

__device__ __forceinline__ h2v pk_half(float a, float b) {  // toward zero: lo keeps what is left
  return __builtin_bit_cast(h2v, __builtin_amdgcn_cvt_pkrtz(a, b));
}
// The other term: x - hi (exact), rounded, in one instruction (v_fma_mixlo_f16); minus1 is -1
// in a register that the compiler cannot see through, or it makes a conversion and two more.
__device__ __forceinline__ _Float16 half_rest(float x, _Float16 hi, float minus1) {
  return (_Float16)__builtin_fmaf((float)hi, minus1, x);
}
__device__ __forceinline__ float minus_one() { return __uint_as_float(opaque(0xBF800000u)); }

// max(a, |x|, |y|), in one instruction (NaN never wins).
__device__ __forceinline__ float max3_abs(float a, float x, float y) {
  float r;
  asm("v_max3_f32 %0, %1, |%2|, |%3|" : "=v"(r) : "v"(a), "v"(x), "v"(y));
  return r;
}

// 2^(13 - exponent of a row's largest |q|), which brings it into [2^13, 2^14), and the inverse.
// (An element that is not finite has a lo term of NaN, so its row's scores are NaN.)
__device__ __forceinline__ void kv8_q_scale(int big, float &up, float &down) {
  const int e = min(267 - (big >> 23), 253);
  up = __int_as_float(e << 23);
  down = __int_as_float((254 - e) << 23);
}

// Two weights in three bf16 terms each, 8 significant bits a term and all 24 together (the first of
// a pair in the low half).
struct Kv8Terms {
  uint32_t hi, mid, lo;
};
__device__ __forceinline__ Kv8Terms kv8_terms(float a, float b) {
  const auto top = [](float x) { return __uint_as_float(__float_as_uint(x) & 0xFFFF0000u); };
  const auto pack = [](float x, float y) { return pack_bf16(__float_as_uint(x), __float_as_uint(y)); };
  const float ra = a - top(a), rb = b - top(b);
  return {pack(a, b), pack(ra, rb), pack(ra - top(ra), rb - top(rb))};
}

// Sum (or larger) of a value over the four lanes c, c + 16, c + 32, c + 48.
__device__ __forceinline__ float quarters_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}
__device__ __forceinline__ float quarters_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}

// The unit 2^(m - mid) of a denominator. m may be too large for m - mid to keep mid, so units
// are compared by it but differences are taken of m and mid apart.
struct Kv8Unit2 {
  float m, mid;
};
__device__ __forceinline__ Kv8Unit2 kv8_larger(Kv8Unit2 a, Kv8Unit2 b) { return b.m - b.mid > a.m - a.mid ? b : a; }

// Waits for every load of the wave. After loads on a path that is seldom taken: without it the
// compiler waits for all loads wherever the paths have joined, the common one included.
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0F70); }  // vmcnt(0)

// A tile of 16 keys as a wave holds it.
struct Kv8Tile {
  bool held;     // there is such a page
  bool unused;   // its V codes are not to be used
  bool nan;      // K's or V's block is NaN
  float kscale;  // 2^ke of K
  float ev;      // V's exponent
  float unit;    // 2^(mid - ev), what a weight counts in the denominator
};

// A row block's slice of keys. Four waves share it in chunks of 32 keys, two 16-key tiles, each
// wave with its own running reference and sums, merged in LDS. Everything is transposed,
// scores^T = K Q^T and out^T = V^T W^T, so a lane keeps one query row (lane % 16) of each column
// block and what it gets from the first product (keys 4 (lane / 16) + r of either tile) is the
// operand of the second as it is.
//   NC 0: 8 rows; columns 8 .. 15 hold the second terms of the rows in 0 .. 7, one matrix
//     instruction for both, and a row rotation by 8 adds them.
//   NC 1: 16 rows, a matrix instruction a term.
//   NC 2: 32 rows, two column blocks of 16, for which K and V are made float16 once. Their two
//     terms are made once too, a part by each wave, and read from LDS in every chunk: the 64
//     registers of a wave's own copy at D = 128 would leave room for two waves a SIMD, not three
//     (24 sequences of prompts and steps, 14 heads on 2 of 64, took 19 % longer with them).
// K is read 16 bytes a lane (8 at D = 32), V D / 16 bytes a lane of eight keys: a lane's bytes
// of two keys are interleaved by v_perm on their way to float16, which is all the transposing
// that V needs, and its output elements come out contiguous. The next chunk's K is requested
// once the scores are made, its V once the outputs are: loads are always in flight, and no
// LDS lies between them and the matrix cores.
//
// What bounds it. Few rows, the cache's bytes: 61 sequences of 50 to 4096 keys, 32 heads on 8 of
// 128, 254 MB in 54 us and 5 for the merge, 4.7 TB/s; one of 60000 keys 25 us and 5. (Three waves a
// SIMD at D = 128: with registers for four the loop spills, 22 % slower.) Short ones, the launch and
// four loads one after the other (batch, page, exponents beside codes): 700 keys 7.8 us.
// Many rows, the instructions: 2048 tokens of 32 heads on 8 of 128 91 us, 376 TFLOP/s of the
// formula, 2.5 times that in products of terms (a large float16 product reaches 1180). The matrix
// cores are busy for 38 % of the time; a wave issues 2300 vector instructions, 370 of them matrix
// ones, more than a third of the others in its beginning and end; the two kinds hardly overlap.
// Tried and slower or alike: products of 32 x 32 x 16 (0 to 6 %), the next chunk's scores
// beside this one's weights (0 to 40 %, it spills), matrix and vector instructions alternated by
// scheduling barriers, both column blocks' weights in one stretch (3 %), two waves a workgroup (1
// to 15 %), the place of a workgroup found by one of its waves (1 %).
template <int D, int NC, int NW>
struct Kv8Lds {
  union {
    float sh[NC < 2 ? NW : NW == 4 ? 2 : 1][kv8_rows(NC)][D + 4];
    uint4 q[NC == 2 ? D / 8 : 1][kWave];  // NC 2: the query rows' operands, [column block][product][term]
    v4f ex[NC == 2 && NW == 2 ? 2 : 1][D / 16][kWave];  // what the waves hand to each other
  };
  float cx[2][16];
  float sm[NW][kv8_rows(NC)], sl[NW][kv8_rows(NC)], smid[NW];
};

//
// WIN: a window. A row block's keys are those that a row of it may see, counted without the gap
// behind the sinks (positions come back in load_tiles and in the mask), and everything else is as
// it is for a short sequence. What bounds it: 61 steps in windows of 4096 behind up to 30000, 32 heads on
// 8 of 128, the bytes, 498 MB in 98 us and 5 for the merge (whole caches masked: 200 us); 2048 tokens in
// 512 the instructions, 55 us: 18 chunks a row block, and a third of them in the waves' beginnings and
// ends (whole caches masked: 104). Tried for those: one wave a workgroup (15 to 20 % faster at windows of
// 128 and 2000 row blocks, as much slower at 1024), eight (8 to 15 % faster at D = 64 and up to 256 row
// blocks, 20 to 80 % slower else), and output stored straight from the matrix layout, 16 of a line's 128
// bytes at a time (10 to 20 % slower).
template <int D, int NC, bool WIN, int NW>
__device__ __forceinline__ void kv8_attend(const Kv8Args &a, const Kv8Part &pt, int kv, int unit,
                                           const float *__restrict__ q, int q_stride, float *__restrict__ out,
                                           int out_stride, float *__restrict__ work, Kv8Lds<D, NC, NW> &lds) {
  constexpr bool SEP = NC > 0;
  constexpr int NB = SEP ? NC : 1, R = kv8_rows(NC), KS = D / 32, CK = 32;
  constexpr int KB = D >= 64 ? 16 : 8, KL = D / (4 * KB);  // bytes of a K load, loads per lane and tile
  constexpr int VB = D / 16;                               // bytes of a V load (a key's)
  const Kv8Cut &cut = pt.cut;
  float *part = work + pt.at;
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int c = lane & 15, g = lane >> 4;
  const Kv8Seq first = kv8_seq(a, lane);
  Kv8Unit w;
  w.slice_keys = kv8_slice_keys<WIN>(a, cut, first);
  if (!kv8_unit<false, WIN>(a, cut, first, unit, w)) return;
  const int place = unit - w.at + w.rb * w.slices + w.slice;  // in the workspace
  if (place >= pt.units) return;  // (rows of several sequences at once, which is not allowed)
  const int G = cut.G, rows = w.s.n * G, cap = a.max_pages << a.page_shift, page = 1 << a.page_shift;
  // this lane's query rows, the keys they see (a window: from low on), and those that the block's
  // last row sees
  int lim[NB], low[NB];
  const float *qr[NB];
#pragma unroll
  for (int y = 0; y < NB; y++) {
    const int r = w.rb * R + (SEP ? 16 * y + c : c & 7), rc = min(r, rows - 1), tok = kv8_token(cut, rc);
    lim[y] = r < rows ? min(w.s.past + tok + 1, cap) : 0;
    if constexpr (WIN) low[y] = w.s.past + tok + 1 - a.window;
    qr[y] = q + (size_t)(w.s.row0 + tok) * q_stride + (kv * G + rc - tok * G) * D;
  }
  const int tok_last = kv8_token(cut, min(w.rb * R + R, rows) - 1), tok_first = kv8_token(cut, w.rb * R);
  // A window: keys are counted without the `gap` positions between the tiles of the sinks, `sinks` of
  // them, and the tile that the first row's window begins in.
  const int sinks = WIN ? (a.sinks + 15) & ~15 : 0;
  const int gap = WIN ? max((min(max(w.s.past + tok_first + 1 - a.window, 0), cap) & ~15) - sinks, 0) : 0;
  const int k_begin = w.slice * w.slice_keys;
  const int k_end = min(min(w.s.past + tok_last + 1, cap) - gap, k_begin + w.slice_keys);
  const int k_full = min(w.s.past + tok_first + 1, cap) - gap;  // keys below: every row sees them
  // (a window: those below the sinks and from k_low on; positions from the sinks to `begin` no row sees)
  const int begin = WIN ? w.s.past + tok_first + 1 - a.window : 0;
  const int k_low = WIN && w.s.past + tok_last + 1 - a.window > a.sinks ? w.s.past + tok_last + 1 - a.window - gap : 0;
  const int chunks = max(0, (k_end - k_begin - CK * wave + CK * NW - 1) / (CK * NW));
  const int32_t *table = a.table + (size_t)w.s.b * a.max_pages;

  // ---- tiles of the wave's next 32 chunks, one a lane (t_ve -1: no such page), with what a chunk
  // needs of them made here, so that it only reads lanes (in the chunk's scalar code: 4 to 7 % slower)
  int t_ke = 0, t_ve = 0;
  size_t t_at = 0;  // the tile's first code row, in bytes
  float t_kscale = 0.f, t_ev = 0.f, t_unit = 0.f;
  uint64_t t_held = 0, t_unused = 0, t_nan = 0;  // a bit a tile
  const auto tile_key = [&](int i) { return k_begin + CK * (wave + NW * (i >> 1)) + 16 * (i & 1); };
  const auto load_tiles = [&](int i0) {
    int key = tile_key(i0 + lane);
    const bool mine = key < k_end;
    if constexpr (WIN) key += key < sinks ? 0 : gap;
    const int pg = mine ? table[key >> a.page_shift] : -1;
    const bool in = (unsigned)pg < (unsigned)a.pages;
    const size_t block = (size_t)(in ? pg : 0) * a.KV + kv;
    t_at = ((block << a.page_shift) + (key & (page - 1))) * D;
    t_ke = a.ke[block];
    t_ve = a.ve[block];
    t_ve = in ? t_ve : -1;
  };
  constexpr bool BIG = NC == 2;  // the query rows laid out by the waves together, in LDS
  constexpr int QB = BIG ? 1 : NB;
  v8h qh[QB][KS], ql[QB][SEP ? KS : 1];
  float4 qf[QB][KS][2];
  if constexpr (BIG) qr[0] = wave & 1 ? qr[1] : qr[0];
#pragma unroll
  for (int y = 0; y < QB; y++)
#pragma unroll
    for (int s = 0; s < KS; s++) {
      const int d = D == 32 ? 8 * g : 64 * (s >> 1) + 16 * g + 8 * (s & 1);
      qf[y][s][0] = *reinterpret_cast<const float4 *>(qr[y] + d);
      qf[y][s][1] = *reinterpret_cast<const float4 *>(qr[y] + d + 4);
    }
  load_tiles(0);

  // ---- codes of a chunk's two tiles (no page: page 0's, not used)
  uint4 kf[2][KL];
  uint2 vf[2][4];
  size_t at[2];  // of the tiles requested last
  const auto locate = [&](int i) {
#pragma unroll
    for (int x = 0; x < 2; x++) {
      const int o = (i + x) & (kWave - 1);
      at[x] = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)t_at, o) |
              (size_t)(uint32_t)__builtin_amdgcn_readlane((int)(t_at >> 32), o) << 32;
    }
  };
  const auto load_k = [&]() {
#pragma unroll
    for (int x = 0; x < 2; x++) {
      const uint8_t *p = a.k + at[x] + c * D + KB * g;
      if constexpr (D == 32) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        kf[x][0] = make_uint4(v.x, v.y, 0, 0);
      } else {
#pragma unroll
        for (int l = 0; l < KL; l++) kf[x][l] = *reinterpret_cast<const uint4 *>(p + 64 * l);
      }
    }
  };
  const auto load_v = [&]() {
#pragma unroll
    for (int x = 0; x < 2; x++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const uint8_t *p = a.v + at[x] + (4 * g + e) * D + VB * c;
        if constexpr (VB == 8) vf[x][e] = *reinterpret_cast<const uint2 *>(p);
        if constexpr (VB == 4) vf[x][e].x = *reinterpret_cast<const uint32_t *>(p);
        if constexpr (VB == 2) vf[x][e].x = *reinterpret_cast<const uint16_t *>(p);
      }
  };
  if (chunks) {
    locate(0);
    load_k();
    load_v();
  }

  // ---- the wave's largest V exponent
  int biggest = wave_max_i32(t_ve == 255 ? -1 : t_ve);
  if (2 * chunks > kWave) {
    for (int i = kWave; i < 2 * chunks; i += kWave) {
      load_tiles(i);
      biggest = max(biggest, wave_max_i32(t_ve == 255 ? -1 : t_ve));
    }
    load_tiles(0);
    wait_loads();
  }
  const int least = max(biggest - kKv8Spread, 0);  // E8M0 exponents of V below count as zeros
  const int imid = max(biggest, 0) - kKv8Spread / 2;
  const float mid = (float)(imid - 127);
  const auto weigh_tiles = [&]() {
    const int ve = max(t_ve, least);
    t_held = __ballot(t_ve >= 0);
    t_nan = __ballot(t_ke == 255 || t_ve == 255);
    t_unused = __ballot(t_ve < least);
    t_kscale = e8m0_to_f32((uint32_t)t_ke);
    t_ev = t_ve == 255 ? __builtin_nanf("") : (float)(ve - 127);
    t_unit = t_ve == 255 ? __builtin_nanf("") : __int_as_float((127 + imid - ve) << 23);
  };
  weigh_tiles();

  // ---- the query rows in two terms
  const float minus1 = minus_one();
  float cx[NB];
#pragma unroll
  for (int y = 0; y < QB; y++) {
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int e = 0; e < 2; e++) top = max3_abs(max3_abs(top, qf[y][s][e].x, qf[y][s][e].y), qf[y][s][e].z, qf[y][s][e].w);
    int big = __float_as_int(top);
    big = max(big, __shfl_xor(big, 16));
    big = max(big, __shfl_xor(big, 32));
    float up, down;
    kv8_q_scale(big, up, down);
    cx[y] = down * (kKv8Log2e / sqrtf((float)D));
#pragma unroll
    for (int s = 0; s < KS; s++) {
      if (BIG && s * NW / 2 / KS != wave / 2) continue;  // another wave's
      const float4 a0 = qf[y][s][0], a1 = qf[y][s][1];
      const float x[8] = {a0.x * up, a0.y * up, a0.z * up, a0.w * up, a1.x * up, a1.y * up, a1.z * up, a1.w * up};
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const h2v hi = pk_half(x[e], x[e + 1]);
        const h2v lo = {half_rest(x[e], hi.x, minus1), half_rest(x[e + 1], hi.y, minus1)};
        if constexpr (SEP) {
          qh[y][s][e] = hi.x, qh[y][s][e + 1] = hi.y;
          ql[y][s][e] = lo.x, ql[y][s][e + 1] = lo.y;
        } else {
          const h2v two =
              __builtin_bit_cast(h2v, c < 8 ? __builtin_bit_cast(uint32_t, hi) : __builtin_bit_cast(uint32_t, lo));
          qh[y][s][e] = two.x, qh[y][s][e + 1] = two.y;
        }
      }
      if constexpr (BIG) {
        lds.q[((wave & 1) * KS + s) * 2][lane] = __builtin_bit_cast(uint4, qh[0][s]);
        lds.q[((wave & 1) * KS + s) * 2 + 1][lane] = __builtin_bit_cast(uint4, ql[0][s]);
      }
    }
  }
  if constexpr (BIG) {
    if (g == 0 && wave < 2) lds.cx[wave][c] = cx[0];
    __syncthreads();
    cx[0] = lds.cx[0][c], cx[NB - 1] = lds.cx[1][c];
  }

  float m[NB], l[NB];
  v4f acc[NB][VB];
#pragma unroll
  for (int y = 0; y < NB; y++) {
    m[y] = kKv8None, l[y] = 0.0f;
#pragma unroll
    for (int j = 0; j < VB; j++) acc[y][j] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  bool huge = false;  // |m| with few bits left for fractions: x has to be rounded as it was for m
  const auto q_at = [&](int y, int k, int term) {
    if constexpr (BIG)
      return __builtin_bit_cast(v8h, lds.q[(y * KS + k) * 2 + term][lane]);
    else
      return term ? ql[y][SEP ? k : 0] : qh[y][k];
  };
  const auto chunk = [&](int i, auto more) {
    const int key0 = tile_key(2 * i);
    Kv8Tile now[2];
#pragma unroll
    for (int x = 0; x < 2; x++) {
      const int o = (2 * i + x) & (kWave - 1);
      const auto of = [&](float v) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), o)); };
      now[x].held = t_held >> o & 1;
      now[x].unused = t_unused >> o & 1;
      now[x].nan = t_nan >> o & 1;
      now[x].kscale = of(t_kscale);
      now[x].ev = of(t_ev);
      now[x].unit = of(t_unit);
    }
    // ---- scores of 32 keys
    v4f s[NB][2];
#pragma unroll
    for (int y = 0; y < NB; y++)
#pragma unroll
      for (int x = 0; x < 2; x++) s[y][x] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < KS; k++) {
      v8h kk[2];
#pragma unroll
      for (int x = 0; x < 2; x++) {
        const uint4 kw = kf[x][k >> 1];
        kk[x] = k & 1 ? e4m3x8_h(kw.z, kw.w) : e4m3x8_h(kw.x, kw.y);
      }
#pragma unroll
      for (int x = 0; x < 2; x++)
#pragma unroll
        for (int y = 0; y < NB; y++) s[y][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk[x], q_at(y, k, 0), s[y][x], 0, 0, 0);
      if constexpr (SEP) {
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
          for (int y = 0; y < NB; y++)
            s[y][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk[x], q_at(y, k, 1), s[y][x], 0, 0, 0);
      }
    }
    if constexpr (more) {
      if (((2 * i + 2) & (kWave - 1)) == 0) {
        load_tiles(2 * i + 2);
        wait_loads();
        weigh_tiles();
      }
      locate(2 * i + 2);
      load_k();
    }
    if constexpr (!SEP) {
#pragma unroll
      for (int x = 0; x < 2; x++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[0][x][e] += dpp_f<0x128>(s[0][x][e], 0.0f);  // row_ror:8
    }
    // ---- what some row does not see: scores -inf, and V's codes, which may be anything, 0
    bool edge = key0 + CK > k_full || now[0].unused || now[1].unused;
    if constexpr (WIN) edge = edge || (key0 < k_low && key0 + CK > a.sinks);
    bool careful = false;  // a score of -inf may meet a factor of NaN or 0
    if (edge) {
      bool zero = false;
#pragma unroll
      for (int y = 0; y < NB; y++) zero = zero || cx[y] * fminf(now[0].kscale, now[1].kscale) == 0.0f;
      careful = careful || now[0].nan || now[1].nan || __any(zero);
#pragma unroll
      for (int x = 0; x < 2; x++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int key = key0 + 16 * x + 4 * g + e;
#pragma unroll
          for (int y = 0; y < NB; y++) {
            if constexpr (WIN) {
              const int at = key + (key0 + 16 * x < sinks ? 0 : gap);
              // (bit by bit: && and || become branches, two an element)
              const bool seen = (at < lim[y]) & ((at >= low[y]) | (at < a.sinks)) & now[x].held;
              s[y][x][e] = seen ? s[y][x][e] : -INFINITY;
            } else {
              s[y][x][e] = key < lim[y] && now[x].held ? s[y][x][e] : -INFINITY;
            }
          }
          bool none = key >= k_end || now[x].unused;
          if constexpr (WIN) {
            const int at = key + (key0 + 16 * x < sinks ? 0 : gap);
            none = none | ((at < begin) & (at >= a.sinks));
          }
          if (none) vf[x][e] = make_uint2(0, 0);
        }
    }
    constexpr int NT = SEP ? 3 : 2;  // matrix instructions for a weight's terms
    v4u pw[NT][NB];
#pragma unroll
    for (int y = 0; y < NB; y++) {
      // ---- the running reference
      const float c0 = cx[y] * now[0].kscale, c1 = cx[y] * now[1].kscale;
      const v4f s0 = s[y][0], s1 = s[y][1];
      const float t0 = fmaxf(fmaxf(s0[0], s0[1]), fmaxf(s0[2], s0[3]));
      const float t1 = fmaxf(fmaxf(s1[0], s1[1]), fmaxf(s1[2], s1[3]));
      const float top = fmaxf(__builtin_fmaf(t0, c0, now[0].ev), __builtin_fmaf(t1, c1, now[1].ev));
      if (__any(top > m[y] + kKv8Head)) {
        const float mnew = fmaxf(m[y], ceilf(quarters_max(top)));
        const float alpha = __builtin_amdgcn_exp2f(m[y] - mnew);
        m[y] = mnew;
        huge = huge || __any(fabsf(mnew) > 0x1p22f && mnew != kKv8None);
        l[y] *= alpha;
#pragma unroll
        for (int j = 0; j < VB; j++)
#pragma unroll
          for (int e = 0; e < 4; e++) acc[y][j][e] *= alpha;
      }
      // ---- weights, their sum, and their terms
      const auto weights = [&](auto slow) {
#pragma unroll
        for (int x = 0; x < 2; x++) {
          const float cc = x ? c1 : c0, off = now[x].ev - m[y];
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            p[e] = __builtin_fmaf(s[y][x][e], cc, off);
            if constexpr (slow) {
              if (huge) p[e] = __builtin_fmaf(s[y][x][e], cc, now[x].ev) - m[y];
              p[e] = __builtin_amdgcn_exp2f(p[e]);
              // a block whose exponent is NaN counts where it is seen
              const bool seen = s[y][x][e] != -INFINITY;
              p[e] = seen ? p[e] : 0.0f;
              l[y] = __builtin_fmaf(p[e], seen ? now[x].unit : 0.0f, l[y]);
            } else {
              p[e] = __builtin_amdgcn_exp2f(p[e]);
              l[y] = __builtin_fmaf(p[e], now[x].unit, l[y]);
            }
          }
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const Kv8Terms t = kv8_terms(p[e], p[e + 1]);
            if constexpr (SEP) {
              pw[0][y][2 * x + e / 2] = t.hi, pw[1][y][2 * x + e / 2] = t.mid, pw[NT - 1][y][2 * x + e / 2] = t.lo;
            } else {
              pw[0][y][2 * x + e / 2] = c < 8 ? t.hi : t.mid;
              pw[1][y][2 * x + e / 2] = c < 8 ? t.lo : 0u;
            }
          }
        }
      };
      if (careful || huge)
        weights(std::true_type());
      else
        weights(std::false_type());
    }
    // ---- out^T += V^T W^T, two output tiles (bytes 2 b, 2 b + 1 of a V load) at a time
#pragma unroll
    for (int b = 0; b < VB / 2; b++) {
      uint32_t z[2][2];  // [tile][key pair]: both bytes of keys 0, 1 and 2, 3
#pragma unroll
      for (int x = 0; x < 2; x++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const uint32_t u0 = b < 2 ? vf[x][2 * e].x : vf[x][2 * e].y;
          const uint32_t u1 = b < 2 ? vf[x][2 * e + 1].x : vf[x][2 * e + 1].y;
          z[x][e] = __builtin_amdgcn_perm(u1, u0, b & 1 ? 0x07030602u : 0x05010400u);
        }
#pragma unroll
      for (int y = 0; y < 2; y++) {
        const auto two = [&](uint32_t v) {
          return y ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, 1.0f, true)
                   : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, 1.0f, false);
        };
        const v2bf e0 = two(z[0][0]), e1 = two(z[0][1]), e2 = two(z[1][0]), e3 = two(z[1][1]);
        const v8bf vv = {e0.x, e0.y, e1.x, e1.y, e2.x, e2.y, e3.x, e3.y};
        const int o = 2 * b + y;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int n = 0; n < NB; n++)
            acc[n][o] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vv, __builtin_bit_cast(v8bf, pw[t][n]), acc[n][o], 0, 0, 0);
      }
    }
    if constexpr (more) load_v();
  };
  // the last chunk apart, so that every wait in the loop counts the same loads behind it
  for (int i = 0; i + 1 < chunks; i++) chunk(i, std::true_type());
  if (chunks) chunk(chunks - 1, std::false_type());

  // ---- the waves' sums, merged; element 4 VB g + VB e + j of row c is acc[.][j][e]
  const auto put = [&](int at) {
#pragma unroll
    for (int y = 0; y < NB; y++)
#pragma unroll
      for (int e = 0; e < 4; e++)
#pragma unroll
        for (int j = 0; j < VB; j++) lds.sh[at][16 * y + c][4 * VB * g + VB * e + j] = acc[y][j][e];
  };
#pragma unroll
  for (int y = 0; y < NB; y++) {
    l[y] = quarters_sum(l[y]);
    if constexpr (!SEP) {
#pragma unroll
      for (int j = 0; j < VB; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) acc[y][j][e] += dpp_f<0x128>(acc[y][j][e], 0.0f);
    }
    if (SEP || c < 8) {
      if constexpr (!BIG) put(wave);
      if (g == 0) {
        lds.sm[wave][16 * y + c] = m[y];
        lds.sl[wave][16 * y + c] = l[y];
      }
    }
  }
  if (lane == 0) lds.smid[wave] = mid;
  if (unit == 0 && kv == 0 && threadIdx.x == 0) kv8_put_cut(work, pt, w.slice_keys);
  __syncthreads();
  const size_t pu = (size_t)place * a.KV + kv;
  float *po = part + pu * R * D;
  // a thread a row: the waves' factors, and the sums' common unit
  for (int rr = threadIdx.x; rr < R; rr += NW * kWave) {
    float M = lds.sm[0][rr], den = 0.0f, f[NW];
    Kv8Unit2 u = {M, lds.smid[0]};
#pragma unroll
    for (int x = 1; x < NW; x++) {
      M = fmaxf(M, lds.sm[x][rr]);
      u = kv8_larger(u, {lds.sm[x][rr], lds.smid[x]});
    }
#pragma unroll
    for (int x = 0; x < NW; x++) {
      f[x] = __builtin_amdgcn_exp2f(lds.sm[x][rr] - M);  // 0 for a wave without keys
      den = __builtin_fmaf(lds.sl[x][rr], __builtin_amdgcn_exp2f((lds.sm[x][rr] - u.m) - (lds.smid[x] - u.mid)), den);
    }
    if (w.slices > 1) {
      reinterpret_cast<float4 *>(part + pt.sums)[pu * R + rr] = make_float4(M, u.m, u.mid, den);
    } else {
      const float inv = den == 0.0f ? 0.0f : 1.0f / den;
#pragma unroll
      for (int x = 0; x < NW; x++) f[x] *= inv;
    }
#pragma unroll
    for (int x = 0; x < NW; x++) lds.sm[x][rr] = f[x];
    lds.sl[0][rr] = (M - u.m) + u.mid;
  }
  __syncthreads();
  if constexpr (BIG && NW == 2) {
    // each wave adds up one column block's rows; in LDS a row's elements lie side by side
#pragma unroll
    for (int y = 0; y < NB; y++) {
      const float f = lds.sm[wave][16 * y + c];
#pragma unroll
      for (int j = 0; j < VB; j++) acc[y][j] *= f;
    }
#pragma unroll
    for (int j = 0; j < VB; j++) lds.ex[wave][j][lane] = wave ? acc[0][j] : acc[1][j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < VB; j++) acc[0][j] = (wave ? acc[1][j] : acc[0][j]) + lds.ex[1 - wave][j][lane];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 4; e++) {
      float *row = &lds.sh[0][16 * wave + c][4 * VB * g + VB * e];
      if constexpr (VB >= 4) {
#pragma unroll
        for (int j = 0; j < VB; j += 4)
          *reinterpret_cast<float4 *>(row + j) =
              make_float4(acc[0][j][e], acc[0][j + 1][e], acc[0][j + 2][e], acc[0][j + 3][e]);
      } else {
        *reinterpret_cast<float2 *>(row) = make_float2(acc[0][0][e], acc[0][1][e]);
      }
    }
    __syncthreads();
  } else if constexpr (BIG) {
    float fy[NB];
#pragma unroll
    for (int y = 0; y < NB; y++) fy[y] = lds.sm[wave][16 * y + c];
#pragma unroll
    for (int y = 0; y < NB; y++)
#pragma unroll
      for (int j = 0; j < VB; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) acc[y][j][e] *= fy[y];
    // half of the waves to the other half, twice (half the LDS of all at once, which three workgroups share)
#pragma unroll
    for (int half = NW / 2; half; half /= 2) {
      if (wave >= half && wave < 2 * half) put(wave - half);
      __syncthreads();
      if (wave < half) {
#pragma unroll
        for (int y = 0; y < NB; y++)
#pragma unroll
          for (int e = 0; e < 4; e++)
#pragma unroll
            for (int j = 0; j < VB; j++) acc[y][j][e] += lds.sh[wave][16 * y + c][4 * VB * g + VB * e + j];
      }
      __syncthreads();
    }
    if (wave == 0) put(0);
    __syncthreads();
  }
  for (int i = threadIdx.x; i < R * D / 4; i += NW * kWave) {
    const int rr = i / (D / 4), d = 4 * (i % (D / 4)), ro = w.rb * R + rr;
    if (ro >= rows) break;
    float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
    if constexpr (BIG) num = *reinterpret_cast<const float4 *>(&lds.sh[0][rr][d]);
#pragma unroll
    for (int x = 0; x < (BIG ? 0 : NW); x++) {
      const float f = lds.sm[x][rr];
      const float4 v = *reinterpret_cast<const float4 *>(&lds.sh[x][rr][d]);
      num.x = __builtin_fmaf(v.x, f, num.x);
      num.y = __builtin_fmaf(v.y, f, num.y);
      num.z = __builtin_fmaf(v.z, f, num.z);
      num.w = __builtin_fmaf(v.w, f, num.w);
    }
    if (w.slices > 1) {
      *reinterpret_cast<float4 *>(po + rr * D + d) = num;
    } else {
      const int e = (int)lds.sl[0][rr], t = kv8_token(cut, ro);
      *reinterpret_cast<float4 *>(out + (size_t)(w.s.row0 + t) * out_stride + (kv * G + ro - t * G) * D + d) =
          make_float4(ldexpf(num.x, e), ldexpf(num.y, e), ldexpf(num.z, e), ldexpf(num.w, e));
    }
  }
}

// One class of sequences, or (MIXED) two in one launch, of many rows (NC = 2) and then of few
// (NC = 1), so that the cache streaming of the ones runs beside the matrix products of the others
// (24 sequences of prompts and steps, 14 heads on 2: 36.6 us; two launches and two merges one after
// the other took 27 % longer, 8 of up to 1100, 32 heads on 8, 25 %, and few rows first 29 %).
template <int D, int NC, bool MIXED, bool WIN, int NW>
__global__ __launch_bounds__(NW *kWave, D == 128 ? 3 : 4) void kv8_attend_kernel(
    Kv8Args a, Kv8Part p0, Kv8Part p1, const float *__restrict__ q, int q_stride, float *__restrict__ out,
    int out_stride, float *__restrict__ work) {
  union Lds {
    Kv8Lds<D, NC, NW> one;
    Kv8Lds<D, 1, NW> few;
  };
  __shared__ Lds lds;
  const int kv = blockIdx.x;
  const int unit = (int)(blockIdx.y + blockIdx.z * kKv8GridY);
  if constexpr (MIXED) {
    if (unit >= p0.units) {
      kv8_attend<D, 1, WIN, NW>(a, p1, kv, unit - p0.units, q, q_stride, out, out_stride, work, lds.few);
      return;
    }
  }
  kv8_attend<D, NC, WIN, NW>(a, p0, kv, unit, q, q_stride, out, out_stride, work, lds.one);
}

// Partial sums of a row block's slices -> out, two ways: few rows of many slices, many rows of few.
//
// Few rows: a workgroup a row. Lane s of every wave holds slice s's scalars (m, the denominator's
// unit and it), and the D-element sums, 256 / D slices to a wave load, go round the four waves,
// eight loads requested before the scalars are waited for (64 slices of 8 KV heads' rows: 4.7 us; a
// wave a row took 3.5 times as long).
template <int D, bool WIN>
__device__ __forceinline__ void kv8_merge_long(const Kv8Args &a, const Kv8Part &pt, int block,
                                               const float *__restrict__ work, float4 (*sh)[D / 4],
                                               float *__restrict__ out, int out_stride) {
  constexpr int W = 4, LPR = D / 4, SP = kWave / LPR, U = 8;
  const Kv8Cut &cut = pt.cut;
  const int lane = threadIdx.x & (kWave - 1), e4 = lane % LPR;
  const int wr = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int rr = block % cut.R, idx = block / cut.R, kv = idx % a.KV;
  Kv8Unit w;
  w.slice_keys = kv8_cut_of(work, pt);
  if (!kv8_unit<true, WIN>(a, cut, kv8_seq(a, lane), idx / a.KV, w)) return;
  const int ns = w.slices, ro = w.rb * cut.R + rr;
  if (ns < 2 || ro >= w.s.n * cut.G || w.before + (w.rb + 1ll) * ns > pt.units) return;
  const size_t pu = (size_t)(w.before + w.rb * ns) * a.KV + kv, step = (size_t)a.KV * cut.R;
  const float4 *sc = reinterpret_cast<const float4 *>(work + pt.at + pt.sums) + pu * cut.R + rr;
  const float4 *v = reinterpret_cast<const float4 *>(work + pt.at) + (pu * cut.R + rr) * LPR + e4;
  const float4 none = make_float4(kKv8None, kKv8None, 0.f, 0.f);
  float4 x[U];
  const auto load = [&](int i0) {  // this wave's next slices, past the last the last again
#pragma unroll
    for (int i = 0; i < U; i++) x[i] = v[(size_t)min(i0 + SP * W * i + lane / LPR, ns - 1) * step * LPR];
  };
  float M = kKv8None;
  Kv8Unit2 u = {kKv8None, 0.0f};
  float4 my = none;  // (conditional loads, not a choice between addresses)
  if (lane < ns) my = sc[(size_t)lane * step];
  load(SP * wr);
  const float4 head = my;
  for (int s0 = 0; s0 < ns; s0 += kWave) {
    if (s0) {
      my = none;
      if (s0 + lane < ns) my = sc[(size_t)(s0 + lane) * step];
    }
    M = fmaxf(M, my.x);
    u = kv8_larger(u, {my.y, my.z});
  }
  M = wave_max(M);
  const float at = u.m - u.mid;
  const int best = __ffsll((unsigned long long)__ballot(at == wave_max(at))) - 1;
  u.m = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(u.m), best));
  u.mid = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(u.mid), best));
  float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
  float den = 0.0f;
  my = head;
  for (int s0 = 0; s0 < ns; s0 += kWave) {  // 64 slices' scalars in the lanes
    if (s0) {
      my = none;
      if (s0 + lane < ns) my = sc[(size_t)(s0 + lane) * step];
    }
    const float f = __builtin_amdgcn_exp2f(my.x - M);  // 0 for a slice without keys, and past the last
    den = __builtin_fmaf(my.w, __builtin_amdgcn_exp2f((my.y - u.m) - (my.z - u.mid)), den);
    const int n = min(ns - s0, kWave);
    for (int i0 = SP * wr; i0 < n; i0 += SP * W * U) {
      if (s0 || i0 > SP * wr) load(s0 + i0);
#pragma unroll
      for (int i = 0; i < U; i++) {
        const int k = i0 + SP * W * i + lane / LPR;
        const float fk = __shfl(f, k & (kWave - 1));
        if (k < n) {
          num.x = __builtin_fmaf(x[i].x, fk, num.x);
          num.y = __builtin_fmaf(x[i].y, fk, num.y);
          num.z = __builtin_fmaf(x[i].z, fk, num.z);
          num.w = __builtin_fmaf(x[i].w, fk, num.w);
        }
      }
    }
  }
  den = wave_sum(den);
#pragma unroll
  for (int o = LPR; o < kWave; o <<= 1) {
    num.x += __shfl_xor(num.x, o);
    num.y += __shfl_xor(num.y, o);
    num.z += __shfl_xor(num.z, o);
    num.w += __shfl_xor(num.w, o);
  }
  if (lane < LPR) sh[wr][lane] = num;
  __syncthreads();
  if (wr) return;
  num = sh[0][e4];
#pragma unroll
  for (int k = 1; k < W; k++) num = add4(num, sh[k][e4]);
  if (lane >= LPR) return;
  const float f = den == 0.0f ? 0.0f : 1.0f / den;
  const int e = (int)((M - u.m) + u.mid), t = kv8_token(cut, ro);
  *reinterpret_cast<float4 *>(out + (size_t)(w.s.row0 + t) * out_stride + (kv * cut.G + ro - t * cut.G) * D + 4 * e4) =
      make_float4(ldexpf(num.x * f, e), ldexpf(num.y * f, e), ldexpf(num.z * f, e), ldexpf(num.w * f, e));
}

// Many rows: D / 4 lanes a row, 1024 / D rows a workgroup at a time, `groups` workgroups a row
// block. Eight slices at a time, all of their loads in flight together and nothing exchanged
// between lanes (200 rows of 8200 keys in five slices, 32 heads: 7.4 us; a wave a row took twice as
// long).
template <int D>
__device__ __forceinline__ void kv8_merge_row(const Kv8Args &a, const Kv8Part &pt, const Kv8Unit &w, int kv, int rr,
                                              const float *__restrict__ work, float *__restrict__ out,
                                              int out_stride) {
  const Kv8Cut &cut = pt.cut;
  constexpr int LPR = D / 4, U = 8;
  const int e4 = threadIdx.x % LPR, ns = w.slices, ro = w.rb * cut.R + rr;
  const size_t pu = (size_t)(w.before + w.rb * ns) * a.KV + kv, step = (size_t)a.KV * cut.R;
  const float4 *sc = reinterpret_cast<const float4 *>(work + pt.at + pt.sums) + pu * cut.R + rr;
  const float4 *v = reinterpret_cast<const float4 *>(work + pt.at) + (pu * cut.R + rr) * LPR + e4;
  float M = kKv8None, den = 0.0f;
  Kv8Unit2 u = {kKv8None, 0.0f};
  float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < ns; s0 += U) {
    float4 my[U], x[U];
#pragma unroll
    for (int i = 0; i < U; i++) {
      my[i] = make_float4(kKv8None, kKv8None, 0.f, 0.f);
      x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (s0 + i < ns) {
        my[i] = sc[(size_t)(s0 + i) * step];
        x[i] = v[(size_t)(s0 + i) * step * LPR];
      }
    }
    float Mn = M;
    Kv8Unit2 un = u;
#pragma unroll
    for (int i = 0; i < U; i++) {
      Mn = fmaxf(Mn, my[i].x);
      un = kv8_larger(un, {my[i].y, my[i].z});
    }
    const float fm = __builtin_amdgcn_exp2f(M - Mn), fd = __builtin_amdgcn_exp2f((u.m - un.m) - (u.mid - un.mid));
    num = make_float4(num.x * fm, num.y * fm, num.z * fm, num.w * fm);
    den *= fd;
#pragma unroll
    for (int i = 0; i < U; i++) {
      const float f = __builtin_amdgcn_exp2f(my[i].x - Mn);  // 0 for a slice without keys, and past the last
      num.x = __builtin_fmaf(x[i].x, f, num.x);
      num.y = __builtin_fmaf(x[i].y, f, num.y);
      num.z = __builtin_fmaf(x[i].z, f, num.z);
      num.w = __builtin_fmaf(x[i].w, f, num.w);
      den = __builtin_fmaf(my[i].w, __builtin_amdgcn_exp2f((my[i].y - un.m) - (my[i].z - un.mid)), den);
    }
    M = Mn, u = un;
  }
  const float f = den == 0.0f ? 0.0f : 1.0f / den;
  const int e = (int)((M - u.m) + u.mid), t = kv8_token(cut, ro);
  *reinterpret_cast<float4 *>(out + (size_t)(w.s.row0 + t) * out_stride + (kv * cut.G + ro - t * cut.G) * D + 4 * e4) =
      make_float4(ldexpf(num.x * f, e), ldexpf(num.y * f, e), ldexpf(num.z * f, e), ldexpf(num.w * f, e));
}

template <int D, bool WIN>
__device__ __forceinline__ void kv8_merge(const Kv8Args &a, const Kv8Part &pt, int block,
                                          const float *__restrict__ work, float4 (*sh)[D / 4],
                                          float *__restrict__ out, int out_stride) {
  constexpr int ROWS = 1024 / D;
  if (!pt.merge) {
    kv8_merge_long<D, WIN>(a, pt, block, work, sh, out, out_stride);
    return;
  }
  const int idx = block / pt.merge, kv = idx % a.KV;
  Kv8Unit w;
  w.slice_keys = kv8_cut_of(work, pt);
  if (!kv8_unit<true, WIN>(a, pt.cut, kv8_seq(a, threadIdx.x & (kWave - 1)), idx / a.KV, w) || w.slices < 2) return;
  if (w.before + (w.rb + 1ll) * w.slices > pt.units) return;
  const int rows = min(pt.cut.R, w.s.n * pt.cut.G - w.rb * pt.cut.R);
  for (int rr = block % pt.merge * ROWS + threadIdx.x / (D / 4); rr < rows; rr += pt.merge * ROWS)
    kv8_merge_row<D>(a, pt, w, kv, rr, work, out, out_stride);
}

template <int D, bool MIXED, bool WIN>
__global__ __launch_bounds__(256) void kv8_merge_kernel(Kv8Args a, Kv8Part p0, Kv8Part p1, int blocks0,
                                                        const float *__restrict__ work, float *__restrict__ out,
                                                        int out_stride) {
  __shared__ float4 sh[4][D / 4];
  const int block = blockIdx.x;
  if constexpr (MIXED) {
    if (block >= blocks0) {
      kv8_merge<D, WIN>(a, p1, block - blocks0, work, sh, out, out_stride);
      return;
    }
  }
  kv8_merge<D, WIN>(a, p0, block, work, sh, out, out_stride);
}

// ---------------------------------------------------------------- launchers

hipError_t launch_kv8_append(const Kv8Args &a, int D, const float *qkv, int stride, const float *bias, int H,
                             const float *cosT, const float *sinT, int max_pos, float *q_out, int q_stride,
                             hipStream_t s) {
  const int page = 1 << a.page_shift;
  // pages that n tokens of a sequence can touch: at most (n + 2 page - 2) / page, and n
  const long long nkv = std::min<long long>(a.T, (long long)a.T / page + 2LL * a.B);
  const auto go = [&](auto kern, int nt) {
    const long long chunks = ((long long)H * (D / 8) + nt - 1) / nt;
    const long long grid = nkv * 2 * a.KV + chunks * a.T;
    if (grid > 0xFFFFFFFFll / nt) return hipErrorInvalidValue;  // threads of a launch are counted in 32 bits
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(nt), 0, s, a, qkv, stride, bias, H, cosT, sinT, max_pos, q_out,
                       q_stride, (int)nkv);
    return hipGetLastError();
  };
  const auto pick = [&](auto d) {
    constexpr int DD = decltype(d)::value;
    const int most = std::min(page, a.max_new) * (DD / 8);  // items of a block
    if (most <= kWave) return go(kv8_append_kernel<DD, 64, 1>, 64);
    if (most <= 256) return go(kv8_append_kernel<DD, 256, 1>, 256);
    if (most <= 512) return go(kv8_append_kernel<DD, 256, 2>, 256);
    if constexpr (DD >= 64)
      if (most <= 1024) return go(kv8_append_kernel<DD, 256, 4>, 256);
    if constexpr (DD >= 128) return go(kv8_append_kernel<DD, 256, 8>, 256);
    return hipErrorInvalidValue;
  };
  if (D == 32) return pick(std::integral_constant<int, 32>());
  if (D == 64) return pick(std::integral_constant<int, 64>());
  if (D == 128) return pick(std::integral_constant<int, 128>());
  return hipErrorInvalidValue;
}

// ---- how a call's attention is cut

// Sequences of more rows a KV head than this take row blocks of 32.
constexpr int kKv8FewRows = 16;
constexpr int kKv8Whole = 2304;  // a window of at most so many keys may be taken whole by its row blocks

struct Kv8Plan {
  Kv8Part p[2];  // the call's classes: with both, many rows first
  int parts, nc;  // nc: column blocks of the first one's kernel
  size_t floats;         // of the workspace
};

// false: the grid would not hold it.
static bool kv8_plan(const Kv8Args &a, int D, int H, Kv8Plan &plan) {
  const int G = H / a.KV, cap = a.max_pages << a.page_shift;
  const long long most = (long long)a.max_new * G;
  const unsigned g_inv = (unsigned)(((1ull << 32) + G - 1) / G);  // (G = 1: not used)
  const auto each = [&](int groups) { return std::max(1, groups / a.KV); };
  const bool many = most > kKv8FewRows;
  plan = {};
  const auto add = [&](int nc, int rows_min, int rows_max) {
    Kv8Part &p = plan.p[plan.parts];
    const int R = kv8_rows(nc);
    // a window: the sinks' tiles, the first row's window from its tile on, and the block's further tokens
    const long long seen = ((a.sinks + 15) & ~15) + 15ll + a.window + (R - 2 + G) / G;
    const int span = a.window ? (int)std::min<long long>(cap, seen) : cap;
    long long blocks;
    if (nc < 2) {
      blocks = std::min(a.B, a.T);  // a row block each
      // A window's few keys may be taken whole: no slots for slices, no second launch. One step of 32 heads
      // on 8 of 128 in a window of 512: 10.6 -> 9.3 us, of 1000: 10.6, whole 11.0; 16 and 64 of them of 1500:
      // 16.2 -> 14.8 and 35.6 -> 29.6.
      const bool whole = a.window && (span <= 768 || (span <= 1664 && blocks * a.KV >= 128));
      p.cut = {G, R, nc + 3, rows_min, rows_max, whole ? kKv8Whole : !a.window && cap <= 1024 ? 1024 : 256, g_inv,
               each(256), each(512), whole ? 0 : each(many ? 512 : 2048), 0.0f, 0.0f, span};
    } else {
      blocks = std::min((long long)a.T * G / R + a.B, (long long)a.T * ((G + R - 1) / R));
      const int fits = 256 * (D == 128 ? 3 : 4);  // workgroups that the device holds
      // A window of few keys, or row blocks enough for half of the compute units: taken whole, so that
      // nobody decides on slices and no second launch looks for them (2048 tokens, 32 heads on 8 of 128,
      // windows of 512 and 1024: 64.3 -> 57.9 us and 85.5 -> 78.7; 200 tokens of them in 1024, 208 row blocks,
      // 26.1 -> 22.1, 80 tokens, 88 row blocks: 19.4, whole 21.6; 40 tokens in 600, 48 row blocks, 18.6 -> 15.6).
      const bool whole = a.window && (span <= 768 || (span <= kKv8Whole && blocks * a.KV >= 128));
      p.cut = {G, R, nc + 3, rows_min, rows_max, whole ? kKv8Whole : 256, g_inv, 0, 0, whole ? 0 : each(2 * fits),
               256.0f / (float)a.KV, (float)fits / (float)a.KV, span};
    }
    const long long units = blocks + p.cut.slots, rows = blocks * a.KV * R;
    if (blocks * a.KV >= 1 << 23) return false;  // threads of a launch are counted in 32 bits
    p.blocks = (int)blocks;
    p.units = (int)units;
    // Few rows (of many slices): a workgroup a row (but 16 sequences of up to 2000
    // keys and 4 tokens, 32 heads on 8, 2048 rows: 16.0 us, a workgroup a row 20.6). Many: 1024 / D rows at
    // a time, and where there are workgroups enough a whole row block one after the other, as each
    // finds its place anew (1000 tokens, 32 heads on 8: 37.6 us, with four a row block 40.2).
    p.merge = rows <= 512 ? 0 : blocks * a.KV >= 256 ? 1 : std::max(1, R * D / 1024);
    p.at = plan.floats + kKv8CutHead;
    const size_t slots = p.cut.min_keys == kKv8Whole ? 0 : units;  // one slice each: no sums to hand on
    p.sums = slots * a.KV * R * D;
    plan.floats = p.at + p.sums + slots * a.KV * R * 4;
    plan.parts++;
    return true;
  };
  plan.nc = many ? 2 : most > 8 ? 1 : 0;
  // a batch of one sequence is taken whole by the kernel that its largest size calls for
  if (!many) return add(plan.nc, 1, kKv8FewRows);
  return add(2, a.B > 1 ? kKv8FewRows + 1 : 1, 0x7FFFFFFF) && (a.B == 1 || add(1, 1, kKv8FewRows));
}

size_t kv8_attention_work_bytes(const Kv8Args &a, int D, int H) {
  Kv8Plan p;
  return kv8_plan(a, D, H, p) ? p.floats * sizeof(float) : 0;
}

template <int D, bool WIN>
static hipError_t kv8_attention(const Kv8Args &a, const float *q, int q_stride, int H, float *out, int out_stride,
                                float *work, hipStream_t s) {
  Kv8Plan plan;
  if (!kv8_plan(a, D, H, plan)) return hipErrorInvalidValue;
  const Kv8Part &p0 = plan.p[0], &p1 = plan.p[1];
  const int units = p0.units + p1.units;
  const dim3 grid(a.KV, std::min(units, kKv8GridY), (units + kKv8GridY - 1) / kKv8GridY);
  const auto go = [&](auto kern, int waves) {
    hipLaunchKernelGGL(kern, grid, dim3(waves * kWave), 0, s, a, p0, p1, q, q_stride, out, out_stride, work);
  };
  constexpr int W4 = kKv8Waves;
  if (plan.nc == 0) go(kv8_attend_kernel<D, 0, false, WIN, W4>, W4);
  if (plan.nc == 1) go(kv8_attend_kernel<D, 1, false, WIN, W4>, W4);
  if (plan.nc == 2) {
    const bool one = plan.parts == 1;
    // Two waves a workgroup, each with more chunks between its beginning and end, where a window is short or
    // row blocks are many (2048 tokens, 32 heads on 8 of 128, a window of 256: 47.3 -> 43.1 us, 8192 tokens of
    // 512: 226.9 -> 203.3; of 2048 tokens and 14 heads on 2 of 64, 898 row blocks, 256: 17.0 -> 16.1, 512:
    // 20.1, two waves 21.5; 658 row blocks, 256: 15.0, two waves 15.5).
    const long long groups = (long long)p0.blocks * a.KV;
    const bool two = WIN && p0.cut.min_keys == kKv8Whole && groups >= 768 && (p0.cut.span <= 384 || (one && groups >= 3000));
    if constexpr (WIN) {
      if (two) one ? go(kv8_attend_kernel<D, 2, false, WIN, 2>, 2) : go(kv8_attend_kernel<D, 2, true, WIN, 2>, 2);
    }
    if (!two) one ? go(kv8_attend_kernel<D, 2, false, WIN, W4>, W4) : go(kv8_attend_kernel<D, 2, true, WIN, W4>, W4);
  }
  const hipError_t e = hipGetLastError();
  const bool cut = p0.cut.span > p0.cut.min_keys || (plan.parts == 2 && p1.cut.span > p1.cut.min_keys);
  if (e != hipSuccess || !cut) return e;
  const auto groups = [&](const Kv8Part &p) { return p.blocks * a.KV * (p.merge ? p.merge : p.cut.R); };
  const auto merge = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3(groups(p0) + groups(p1)), dim3(256), 0, s, a, p0, p1, groups(p0), work, out,
                       out_stride);
  };
  plan.parts == 1 ? merge(kv8_merge_kernel<D, false, WIN>) : merge(kv8_merge_kernel<D, true, WIN>);
  return hipGetLastError();
}

hipError_t launch_kv8_attention(const Kv8Args &a, int D, const float *q, int q_stride, int H, float *out,
                                int out_stride, void *work, hipStream_t s) {
  float *w = static_cast<float *>(work);
  const auto go = [&](auto d) {
    constexpr int DD = decltype(d)::value;
    return a.window ? kv8_attention<DD, true>(a, q, q_stride, H, out, out_stride, w, s)
                    : kv8_attention<DD, false>(a, q, q_stride, H, out, out_stride, w, s);
  };
  if (D == 32) return go(std::integral_constant<int, 32>());
  if (D == 64) return go(std::integral_constant<int, 64>());
  if (D == 128) return go(std::integral_constant<int, 128>());
  return hipErrorInvalidValue;
}

}  // namespace lbk
