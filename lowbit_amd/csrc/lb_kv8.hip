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

__device__ __forceinline__ int wave_max_i32(int v) {
  v = max(v, dpp_i<kDppQuad1032>(v, v));
  v = max(v, dpp_i<kDppQuad2301>(v, v));
  v = max(v, dpp_i<kDppRowHalfMirror>(v, v));
  v = max(v, dpp_i<kDppRowMirror>(v, v));
  v = max(v, dpp_i<kDppRowBcast15, 0xA>(v, v));
  v = max(v, dpp_i<kDppRowBcast31, 0xC>(v, v));
  return __builtin_amdgcn_readlane(v, 63);
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
// sequence in s and its index there in `at`. False past the last. By the whole wave: 64
// sequences a step, one round trip of loads each.
template <class F>
__device__ __forceinline__ bool kv8_locate(const Kv8Args &a, int u, F units, Kv8Seq &s, int &at) {
  const int lane = threadIdx.x & (kWave - 1);
  int base = 0;
  for (int b0 = 0; b0 < a.B; b0 += kWave) {
    const Kv8Seq q = kv8_seq(a, b0 + lane);
    const int c = units(q), inc = wave_scan(c), all = __builtin_amdgcn_readlane(inc, 63);
    if (u < base + all) {
      const int l = __ffsll((unsigned long long)__ballot(u - base < inc)) - 1;
      s = kv8_lane(q, l);
      at = u - base - __builtin_amdgcn_readlane(inc - c, l);
      return true;
    }
    base += all;
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
  if (!kv8_locate(a, unit, pages_of, s, at)) return;
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
  const float inv = __int_as_float((254 - min(e, 253)) << 23);
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

// One wave a row and head: a key per lane and round, the round's weights in LDS, then the
// lanes own output elements.
template <int D>
__global__ __launch_bounds__(kWave) void kv8_attend_kernel(Kv8Args a, const float *__restrict__ q, int q_stride,
                                                           int H, float *__restrict__ out, int out_stride) {
  constexpr int DPL = (D + kWave - 1) / kWave;
  __shared__ float qs[D], ps[kWave];
  __shared__ size_t rows[kWave];
  const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, kv = h / (H / a.KV);
  Kv8Seq s;
  if (!kv8_find_row(a, row, s)) return;
  const int cap = a.max_pages << a.page_shift, page = 1 << a.page_shift;
  const int S = min(s.past + row - s.row0 + 1, cap);
  for (int e = lane; e < D; e += kWave) qs[e] = q[(size_t)row * q_stride + h * D + e];
  __syncthreads();
  float m = -INFINITY, l = 0.0f, acc[DPL];
#pragma unroll
  for (int j = 0; j < DPL; j++) acc[j] = 0.0f;
  for (int k0 = 0; k0 < S; k0 += kWave) {
    const int key = k0 + lane;
    const int pg = key < S ? a.table[(size_t)s.b * a.max_pages + (key >> a.page_shift)] : -1;
    const bool in = (unsigned)pg < (unsigned)a.pages;
    const size_t block = (size_t)(in ? pg : 0) * a.KV + kv, at = (block << a.page_shift) + (key & (page - 1));
    float sc = -INFINITY, vs = 0.0f;
    if (in) {
      float d = 0.0f;
      for (int e = 0; e < D; e += 4) {
        const float4 k4 = e4m3x4_f32(*reinterpret_cast<const uint32_t *>(a.k + at * D + e));
        d = __builtin_fmaf(qs[e], k4.x, d);
        d = __builtin_fmaf(qs[e + 1], k4.y, d);
        d = __builtin_fmaf(qs[e + 2], k4.z, d);
        d = __builtin_fmaf(qs[e + 3], k4.w, d);
      }
      sc = d * e8m0_to_f32(a.ke[block]) / sqrtf((float)D);
      vs = e8m0_to_f32(a.ve[block]);
    }
    const float mnew = fmaxf(m, wave_max(sc)), ref = mnew == -INFINITY ? 0.0f : mnew;
    const float alpha = expf(m - ref), p = in ? expf(sc - ref) : 0.0f;
    m = mnew;
    l = __builtin_fmaf(l, alpha, wave_sum(p));
    __syncthreads();
    ps[lane] = in ? p * vs : 0.0f;
    rows[lane] = in ? at : ~(size_t)0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < DPL; j++) acc[j] *= alpha;
    for (int i = 0; i < kWave; i++) {
      if (rows[i] == ~(size_t)0) continue;
#pragma unroll
      for (int j = 0; j < DPL; j++) {
        const int e = lane + kWave * j;
        if (e < D)
          acc[j] = __builtin_fmaf(ps[i], __builtin_amdgcn_cvt_f32_fp8((int)a.v[rows[i] * D + e], 0), acc[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < DPL; j++) {
    const int e = lane + kWave * j;
    if (e < D) out[(size_t)row * out_stride + h * D + e] = l == 0.0f ? 0.0f : acc[j] / l;
  }
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
    if (grid > 0x7FFFFFFF) return hipErrorInvalidValue;
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

hipError_t launch_kv8_attention(const Kv8Args &a, int D, const float *q, int q_stride, int H, float *out,
                                int out_stride, void *work, hipStream_t s) {
  const auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3(a.T, H), dim3(kWave), 0, s, a, q, q_stride, H, out, out_stride);
    return hipGetLastError();
  };
  if (D == 32) return go(kv8_attend_kernel<32>);
  if (D == 64) return go(kv8_attend_kernel<64>);
  if (D == 128) return go(kv8_attend_kernel<128>);
  return hipErrorInvalidValue;
}

size_t kv8_attention_work_bytes(const Kv8Args &a, int D, int H) { return 0; }

}  // namespace lbk
