// Pages of the paged 8-bit cache moved about: copies within every layer's pool
// (lbd_kv8_copy_pages), and the sequences of a beam search put in their new order
// (lbd_kv8_reorder). No reference counterpart: its cache is one float32 array per sequence
// (src/lowbit/model.py:264-297).
#include <algorithm>

#include "lb_device.h"
#include "lb_internal.h"

namespace lbk {

constexpr int kCopyBytes = 1 << 14;  // of a page's K or V codes that a workgroup copies at a time
constexpr long long kCopyGroups = 1ll << 32;  // workgroups of a call and 64 layers: pages of 1 KB and more that
                                              // fill the card, at most 2^24 of them, take fewer

// ---------------------------------------------------------------- copies of pages

// A workgroup a part of one page's K or V in one layer. What bounds it: the bytes; 250 pages of 128 KB in 16
// layers, 524 MB read and written, 100 us = 5.2 TB/s, what a large copy reaches; 3 pages of 4 KB in 24 layers
// the launch, 2.8 us.
__global__ __launch_bounds__(256) void kv8_copy_kernel(Kv8Layers l, const int32_t *__restrict__ src,
                                                       const int32_t *__restrict__ dst, int parts) {
  const Kv8Codes c = l.of[blockIdx.y];
  const int pair = (int)blockIdx.x / (2 * parts), rest = (int)blockIdx.x % (2 * parts);
  const bool isv = rest >= parts;
  const int part = isv ? rest - parts : rest, from = src[pair], to = dst[pair];
  if ((unsigned)from >= (unsigned)l.pages || (unsigned)to >= (unsigned)l.pages || from == to) return;
  const size_t bytes = (size_t)l.KV << (l.page_shift + l.d_shift);
  uint8_t *codes = isv ? c.v : c.k, *exps = isv ? c.ve : c.ke;
  const size_t end = min(bytes, ((size_t)part + 1) * kCopyBytes);
  for (size_t i = (size_t)part * kCopyBytes + 16 * threadIdx.x; i < end; i += 16 * 256)
    *reinterpret_cast<uint4 *>(codes + to * bytes + i) = *reinterpret_cast<const uint4 *>(codes + from * bytes + i);
  if (part == 0)
    for (int i = threadIdx.x; i < l.KV; i += 256) exps[(size_t)to * l.KV + i] = exps[(size_t)from * l.KV + i];
}

// ---------------------------------------------------------------- beams in their new order

// The places of a prompt, one a lane: what each continues (parent -1: no sequence) and the tokens that it holds;
// the index of the page that is being written, its tokens (0: it is begun next) and the parent's page there, which
// the first of a parent's children keeps.
struct Kv8Family {
  int parent, length, tail, used, was;
  bool first;
};

__device__ __forceinline__ Kv8Family kv8_family(const Kv8Order &o, int page_shift, int base) {
  const int lane = threadIdx.x & (kWave - 1), cap = o.max_pages << page_shift;
  Kv8Family f = {-1, 0, 0, 0, -1, false};
  if (lane < o.W) {
    const int p = o.parent[base + lane];
    if (p >= base && p < base + o.W && !(o.done && o.done[base + lane])) {
      const int past = o.past[p];
      if (past >= 0) f.parent = p, f.length = (int)min((long long)past + o.add, (long long)kKv8MaxPos);
    }
  }
  f.tail = min(f.length, cap) >> page_shift, f.used = f.length < cap ? f.length & ((1 << page_shift) - 1) : 0;
  f.first = f.parent >= 0 && f.used;
  if (f.first) f.was = o.table[(size_t)f.parent * o.max_pages + f.tail];
  const unsigned long long writes = __ballot(f.first);
  for (int k = 0; k < o.W; k++) {
    const int theirs = __builtin_amdgcn_readlane(f.parent, k);
    if ((writes >> k & 1) && k < lane && theirs == f.parent) f.first = false;
  }
  return f;
}

// The page that place base + me, whose sequence holds none at index j, gets there, by the whole wave: its own
// where no sequence of the prompt holds one, else of own's pages that none holds, in order, the next one. (There
// are W of them, and a place holds one or gets one, so they suffice whatever the sequences' lengths.)
__device__ __forceinline__ int kv8_page_at(const Kv8Order &o, const Kv8Family &f, int pages, int base, int me, int j) {
  const int lane = threadIdx.x & (kWave - 1);
  const bool holds = f.parent >= 0 && (f.tail > j || (f.tail == j && f.first));
  const int spare = lane < o.W ? o.own[(size_t)(base + lane) * o.max_pages + j] : -1;
  const unsigned long long held = __ballot(holds);
  if (!held) return __builtin_amdgcn_readlane(spare, me);
  int page = f.was;
  if (holds && f.tail > j) page = o.table[(size_t)f.parent * o.max_pages + j];
  bool free = (unsigned)spare < (unsigned)pages;
  for (int k = 0; k < o.W; k++) {
    const int kept = __builtin_amdgcn_readlane(page, k);
    if ((held >> k & 1) && kept == spare) free = false;
  }
  unsigned long long left = __ballot(free);
  for (unsigned long long before = __ballot(f.parent >= 0 && !holds && lane < me); before; before &= before - 1)
    left &= left - 1;
  return left ? __builtin_amdgcn_readlane(spare, __ffsll(left) - 1) : -1;
}

// What becomes of one place, the same in every lane of a wave.
struct Kv8Move {
  int parent, length, tail, used;  // as above
  int from, page;                  // the page in writing: the parent's and the place's (the parent's own: no copy)
};

// The move of place base + me, by the whole wave.
__device__ __forceinline__ Kv8Move kv8_move(const Kv8Order &o, const Kv8Family &f, int pages, int base, int me) {
  const auto mine = [&](int v) { return __builtin_amdgcn_readlane(v, me); };
  Kv8Move m = {mine(f.parent), mine(f.length), mine(f.tail), mine(f.used), mine(f.was), mine(f.was)};
  if (m.parent >= 0 && m.used && !mine(f.first)) m.page = kv8_page_at(o, f, pages, base, me, m.tail);
  return m;
}

// A workgroup takes one place's part of K or V in every `step`-th layer, so that it finds the place's move once
// (four loads one after the other) for several copies. What bounds it: a few places those loads and the launch
// (4 beams in 24 layers of 14 heads on 2 of 64 4.4 us); many the bytes: 8 prompts' 5 beams in 32 layers of 8 heads
// of 128, 50 MB read and written, 13.2 us = 3.8 TB/s.
__global__ __launch_bounds__(256) void kv8_reorder_kernel(Kv8Layers l, Kv8Order o, int copies, int parts, int step) {
  const int tid = threadIdx.x, id = (int)blockIdx.x;
  if (id >= copies) {  // a place's row of the table
    if (blockIdx.y) return;
    const int place = id - copies, base = place / o.W * o.W;
    const Kv8Family f = kv8_family(o, l.page_shift, base);
    const Kv8Move m = kv8_move(o, f, l.pages, base, place - base);
    const size_t row = (size_t)place * o.max_pages;
    // up to here other sequences of the prompt, longer ones, hold pages
    const int last = m.parent >= 0 ? wave_max_i32(f.parent < 0 ? -1 : f.first ? f.tail : f.tail - 1) : -1;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave), next = m.used ? m.tail + 1 : m.tail;
    for (int j = next + wave; j <= last; j += 256 / kWave) {
      const int p = kv8_page_at(o, f, l.pages, base, place - base, j);
      if (tid % kWave == 0) o.new_table[row + j] = p;
    }
    for (int j = tid; j < o.max_pages; j += 256) {
      if (j >= next && j <= last) continue;
      int p = -1;
      if (m.parent >= 0) {
        p = j < m.tail ? o.table[(size_t)m.parent * o.max_pages + j] : o.own[row + j];
        if (j == m.tail && m.used) p = m.page;
      }
      o.new_table[row + j] = p;
    }
    if (tid == 0) o.new_past[place] = m.parent >= 0 ? m.length : -1;
    return;
  }
  const int place = id / (2 * parts), rest = id % (2 * parts);
  const bool isv = rest >= parts;
  const int part = isv ? rest - parts : rest;
  const int base = place / o.W * o.W;
  const Kv8Move m = kv8_move(o, kv8_family(o, l.page_shift, base), l.pages, base, place - base);
  if (m.parent < 0 || !m.used || m.page == m.from) return;
  if ((unsigned)m.page >= (unsigned)l.pages || (unsigned)m.from >= (unsigned)l.pages) return;
  const size_t bytes = (size_t)l.KV << (l.page_shift + l.d_shift);
  constexpr int N = kCopyBytes / (16 * 256);
  bool mine[N];  // of the part's slots those that hold tokens
  size_t at[N];
#pragma unroll
  for (int k = 0; k < N; k++) {
    at[k] = (size_t)part * kCopyBytes + 16 * (tid + 256 * k);
    mine[k] = at[k] < bytes && ((int)(at[k] >> l.d_shift) & ((1 << l.page_shift) - 1)) < m.used;
  }
  for (int y = blockIdx.y; y < l.n; y += step) {
    const Kv8Codes c = l.of[y];
    uint8_t *codes = isv ? c.v : c.k, *exps = isv ? c.ve : c.ke;
    v4u w[N];  // (an array of the struct uint4 ends up in LDS)
#pragma unroll
    for (int k = 0; k < N; k++) w[k] = *reinterpret_cast<const v4u *>(codes + m.from * bytes + (mine[k] ? at[k] : 0));
#pragma unroll
    for (int k = 0; k < N; k++)
      if (mine[k]) *reinterpret_cast<v4u *>(codes + m.page * bytes + at[k]) = w[k];
    if (part == 0)
      for (int i = tid; i < l.KV; i += 256) exps[(size_t)m.page * l.KV + i] = exps[(size_t)m.from * l.KV + i];
  }
}

// ---------------------------------------------------------------- launchers

static int copy_parts(const Kv8Layers &l) {
  const long long bytes = (long long)l.KV << (l.page_shift + l.d_shift);
  return (int)((bytes + kCopyBytes - 1) / kCopyBytes);
}

// Threads of a launch are counted in 32 bits.
static bool fits(long long blocks, int layers) { return blocks * layers <= 0xFFFFFFFFll / 256; }

hipError_t launch_kv8_copy_pages(const Kv8Layers &l, const int32_t *src, const int32_t *dst, int n, hipStream_t s) {
  const int parts = copy_parts(l);
  if (2ll * n * parts * l.n > kCopyGroups) return hipErrorInvalidValue;
  const int most = (int)(0xFFFFFFFFll / 256 / l.n / (2 * parts));  // pairs of a launch
  for (int at = 0; at < n; at += most) {
    const int pairs = std::min(n - at, most);
    hipLaunchKernelGGL(kv8_copy_kernel, dim3(2 * pairs * parts, l.n), dim3(256), 0, s, l, src + at, dst + at, parts);
  }
  return hipGetLastError();
}

hipError_t launch_kv8_reorder(const Kv8Layers &l, const Kv8Order &o, bool write, hipStream_t s) {
  const int parts = copy_parts(l);
  const long long places = (long long)o.B * o.W, copies = 2 * places * parts, grid = copies + (write ? places : 0);
  // Workgroups in all, so that a place's move is found for several layers where there are many: ten a compute unit.
  // us a call at 1600, 2560, 3200 and 4096 of them (rows of workgroups), heads of 128, a page's K codes of
  //   64 KB: 40 places in 32 layers 15.0 (5), 14.5 (8), 14.0 (10), 14.1 (13), and 38.7 with one row; 16 places 8.4
  //          (13), 8.5 (20), 8.7 (25), 9.9 (32); 130 places 59.4 (2), 54.5 (3), 51.7 (4), 51.6 (4)
  //   128 KB: 40 places in 32 layers 45.0 (3), 40.8 (4), 40.5 (5), 38.7 (7); 128 places 135 (1), 103 (2), 103 (2), 103 (2)
  //   16 KB: 128 places in 28 layers 15.5 (7), 14.5 (10), 16.1 (13), 16.5 (16)
  // Of 4 KB, whose parts leave lanes idle: 128 places in 24 layers 10.6 with 1024 in all, 11.2 with 2560; 32 places 6.2, 6.3.
  const long long want = ((long long)l.KV << (l.page_shift + l.d_shift)) < kCopyBytes ? 1024 : 2560;
  const int rows = (int)std::min<long long>(l.n, std::max<long long>(1, (want + copies - 1) / copies));
  if (!fits(grid, rows)) return hipErrorInvalidValue;
  hipLaunchKernelGGL(kv8_reorder_kernel, dim3((unsigned)grid, rows), dim3(256), 0, s, l, o, (int)copies, parts, rows);
  return hipGetLastError();
}

}  // namespace lbk
