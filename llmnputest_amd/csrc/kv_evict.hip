// Caches cut down to the positions that were given the most attention and the newest ones. No reference
// counterpart (its cache never shrinks).
//
// Per (sequence, kv head) with n = lens[b] > budget positions: of the first n - recent those budget - recent
// of the greatest weights (ties to the lowest position), then the `recent` last, in the order of their
// positions. With n <= budget all are kept. First which ones, by a radix selection of the weights' keys, then
// the rows. Up to 16384 positions the selection is one workgroup's for a (sequence, kv head), the keys in
// registers (8 sequences of 5000 / 16384: 13.2 / 19.7 us, by parts 21.7 / 22.6 and two launches more). Beyond,
// that is bound by its own instructions on a quarter of the chip (8 sequences of 32771: 33.7 us of 25.6), so
// parts of 4096 share it: histograms of the keys' upper 11 bits; where the wanted number is reached, and the
// keys of that bin, among which the last part to arrive looks for the rest; then the positions, in order.
//
// Rows move towards the front. Into other memory they move all at once. In place, row i comes from a
// position >= i, so a workgroup that takes rows in order, a block at a time, only overwrites rows that it
// has read: a block's sources lie at or behind the block's own first row, and every later block's behind it.
// K and V have a workgroup each, a chain of blocks: for one sequence of 8 kv heads, 4096 of 16384 rows of 64,
// turned, 28.5 us (into other memory 5.0), for 8 of 32771 66.5 (33.4).
//
// With a RoPE table K is turned to its new place: a key that was rotated by position o and now stands at i
// is rotated back by o - i places, in fp32, rounded once.

#include <math.h>

#include "common.h"

namespace q4nx {

struct EvictArgs {
  const uint16_t* k;
  const uint16_t* v;
  const float* weights;
  const int32_t* lens;
  const float* tab;        // [max_pos][2][D/2], or nullptr: keys move as they are
  uint16_t* k_out;
  uint16_t* v_out;
  float* weights_out;
  int32_t* lens_out;
  int32_t* kept;           // [batch][hkv][budget]
  int32_t* n_old;          // [batch * hkv]: lengths, for the later launches
  unsigned* counters;      // the next five: selection by parts, index bk * parts + part
  uint16_t* hist;          // [..][kPickBins]
  uint32_t* cand;          // [..][kPickPart]: keys in the bin where the wanted number is reached
  int32_t* part_info;      // [..][4]: keys above the bin, keys in it; then its first place, equal keys before it
  uint32_t* cut;           // [batch * hkv][2]: the last wanted key, and how many of its like
  int64_t b_stride, h_stride, w_b_stride, w_h_stride;
  int64_t ob_stride, oh_stride, ow_b_stride, ow_h_stride;
  int batch, hkv, max_len, budget, recent, room;
  int parts;               // of 4096 positions
  int blocks;              // workgroups for a (sequence, kv head)'s rows of K, and of V
};

// Greater weights have greater keys; a NaN's is the greatest; -0 and 0 are one value.
__device__ __forceinline__ uint32_t weight_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  const uint32_t key = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
  return (u & 0x7fffffffu) > 0x7f800000u ? 0xffffffffu : key;
}
__device__ __forceinline__ float weight_at(const float* w, int p) {   // p below 2^24: a base and 32 bits
  return *(const float*)((const char*)w + (uint32_t)p * 4u);
}

constexpr int kPickThreads = 1024;
constexpr int kPickWaves = kPickThreads / 64;
constexpr int kPickBins = 2048;    // 11 bits a pass: 32 bits in three
constexpr int kPickFew = 4 * kPickThreads, kPickHeld = 16 * kPickThreads;   // positions held in 4, in 16 registers
constexpr int kPickCopies = 4;     // of the histogram, by lane: weights crowd in few bins

// Sum over the lanes up to and with this one.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);   // row_shr:1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);   // row_bcast:31 into rows 2 and 3
  return v;
}

// The waves take equal shares of the positions in a row, at most KPT * 64 each. HELD: that is all of them,
// and their keys stay in registers; otherwise each pass reads the weights again, KPT * 1024 at a time.
// put(i, p): kept position i is p.
template <int KPT, bool HELD, typename Put>
__device__ __forceinline__ void evict_pick(const EvictArgs& a, int bk, int n, Put put) {
  __shared__ __attribute__((aligned(16))) int s_hist[kPickBins * kPickCopies];
  __shared__ int s_sum[kPickWaves], s_gt[kPickWaves], s_eq[kPickWaves];
  __shared__ uint32_t s_key;
  __shared__ int s_left;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int b = bk / a.hkv, h = bk - b * a.hkv;
  if (n <= a.budget) {
    for (int i = tid; i < a.budget; i += kPickThreads) put(i, i < n ? i : -1);
    return;
  }
  const int old = n - a.recent, want = a.budget - a.recent;   // want < old
  for (int i = tid; i < a.recent; i += kPickThreads) put(want + i, old + i);
  if (want == 0) return;
  const float* w = a.weights + (size_t)b * a.w_b_stride + (size_t)h * a.w_h_stride;

  uint32_t key[KPT];
  const int share = HELD ? (old + kPickThreads - 1) / kPickThreads * 64 : KPT * 64;   // a wave's
  const int first = wave * share;
  auto load = [&](int p0) {   // key 0 (below that of every weight) past the end
    float x[KPT];
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
      x[i] = 64 * i < share ? weight_at(w, min(p0 + 64 * i + lane, old - 1)) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < KPT; ++i) key[i] = 64 * i < share && p0 + 64 * i + lane < old ? weight_key(x[i]) : 0u;
  };
  auto each = [&](auto f) {
    if constexpr (HELD) {
      f();
    } else {
      for (int p0 = 0; p0 < old; p0 += KPT * kPickThreads) {
        load(p0 + first);
        f();
      }
    }
  };
  if constexpr (HELD) load(first);

  // ---- the key of the want-th greatest, 11, 11 and 10 bits at a time; `left`: how many of the keys that
  // share the bits found so far are wanted
  uint32_t found = 0;
  int left = want;
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t mask = pass < 2 ? 2047u : 1023u;
    const uint32_t known = pass == 0 ? 0u : pass == 1 ? ~0u << 21 : ~0u << 10;
    for (int i = tid; i < kPickBins * kPickCopies; i += kPickThreads) s_hist[i] = 0;
    __syncthreads();
    each([&] {
#pragma unroll
      for (int i = 0; i < KPT; ++i)
        if (64 * i < share && (key[i] & known) == found)   // (no weight's key is in key 0's bin)
          atomicAdd(&s_hist[((key[i] >> shift) & mask) * kPickCopies + lane % kPickCopies], 1);
    });
    __syncthreads();
    // the bin where the sum from the greatest on reaches `left`: two bins a thread, the greatest first
    const int hi = kPickBins - 1 - 2 * tid;
    const int4 h0 = *(const int4*)(s_hist + 4 * hi), h1 = *(const int4*)(s_hist + 4 * hi - 4);
    const int c0 = h0.x + h0.y + h0.z + h0.w, c1 = h1.x + h1.y + h1.z + h1.w;
    const int upto = wave_scan(c0 + c1);
    if (lane == 63) s_sum[wave] = upto;
    __syncthreads();
    int before = 0;
#pragma unroll
    for (int i = 0; i < kPickWaves; ++i) before += i < wave ? s_sum[i] : 0;
    const int from = before + upto - c0 - c1;   // keys above this thread's bins
    if (from < left && left <= from + c0 + c1) {
      const bool one = left <= from + c0;
      s_key = found | (uint32_t)(one ? hi : hi - 1) << shift;
      s_left = left - (one ? from : from + c0);
    }
    __syncthreads();
    found = s_key;
    left = s_left;
  }

  // ---- positions in order: the waves count theirs, then write them
  int done = 0, ties = 0;   // written, and equal keys seen, before the block of positions at hand
  const uint64_t below = (1ull << lane) - 1;
  for (int p0 = 0; p0 < old; p0 += kPickWaves * share) {
    if constexpr (!HELD) load(p0 + first);
    int gt = 0, eq = 0;
#pragma unroll
    for (int i = 0; i < KPT; ++i)
      if (64 * i < share) {
        gt += __popcll(__ballot(key[i] > found));
        eq += __popcll(__ballot(key[i] == found));
      }
    __syncthreads();
    if (lane == 0) {
      s_gt[wave] = gt;
      s_eq[wave] = eq;
    }
    __syncthreads();
    int at = done, seen = ties;
#pragma unroll
    for (int i = 0; i < kPickWaves; ++i) {
      const int g = s_gt[i], e = s_eq[i], t = min(e, max(left - ties, 0));
      done += g + t;
      ties += e;
      if (i < wave) {
        at = done;
        seen = ties;
      }
    }
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
      if (64 * i >= share) break;
      const uint64_t same = __ballot(key[i] == found);
      const bool take = key[i] > found || (key[i] == found && seen + __popcll(same & below) < left);
      const uint64_t who = __ballot(take);
      if (take) put(at + __popcll(who & below), p0 + first + 64 * i + lane);
      at += __popcll(who);
      seen += __popcll(same);
    }
  }
}

template <int KPT, bool HELD>
__global__ __launch_bounds__(kPickThreads) void evict_pick_kernel(EvictArgs a) {
  const int bk = blockIdx.x;
  const int n = min(max(a.lens[bk / a.hkv], 0), a.max_len);
  if (threadIdx.x == 0) a.n_old[bk] = n;
  int32_t* const kept = a.kept + (size_t)bk * a.budget;
  evict_pick<KPT, HELD>(a, bk, n, [&](int i, int p) { kept[i] = p; });
}

// ---- by parts of 4096 positions, 256 threads each: a wave holds 1024 of them in a row
constexpr int kPickPart = 4096;
constexpr int kPartThreads = 256;
constexpr int kPartKeys = kPickPart / kPartThreads;

struct PartJob {
  int bk, part, n, old, want, p0;   // p0: the wave's first position
  const float* w;
};
__device__ __forceinline__ PartJob part_job(const EvictArgs& a) {
  PartJob j;
  j.bk = blockIdx.x / a.parts;
  j.part = blockIdx.x % a.parts;
  const int b = j.bk / a.hkv, h = j.bk - b * a.hkv;
  j.n = min(max(a.lens[b], 0), a.max_len);
  j.old = j.n - a.recent;
  j.want = a.budget - a.recent;
  j.p0 = j.part * kPickPart + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 64 * kPartKeys;
  j.w = a.weights + (size_t)b * a.w_b_stride + (size_t)h * a.w_h_stride;
  return j;
}
// Whether there is a choice to make, and this part has some of it.
__device__ __forceinline__ bool part_chooses(const EvictArgs& a, const PartJob& j) {
  return j.n > a.budget && j.want > 0 && j.part * kPickPart < j.old;
}
__device__ __forceinline__ void part_keys(const PartJob& j, int lane, uint32_t (&key)[kPartKeys]) {
  float x[kPartKeys];
#pragma unroll
  for (int i = 0; i < kPartKeys; ++i) x[i] = weight_at(j.w, min(j.p0 + 64 * i + lane, j.old - 1));
#pragma unroll
  for (int i = 0; i < kPartKeys; ++i) key[i] = j.p0 + 64 * i + lane < j.old ? weight_key(x[i]) : 0u;
}

__global__ __launch_bounds__(kPartThreads) void evict_hist_kernel(EvictArgs a) {
  __shared__ __attribute__((aligned(16))) int s_hist[kPickBins];
  const int tid = threadIdx.x, lane = tid & 63;
  const PartJob j = part_job(a);
  if (j.part == 0 && tid == 0) a.n_old[j.bk] = j.n;
  if (!part_chooses(a, j)) return;
  uint32_t key[kPartKeys];
  part_keys(j, lane, key);
  for (int i = tid; i < kPickBins; i += kPartThreads) s_hist[i] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPartKeys; ++i)
    if (key[i] != 0) atomicAdd(&s_hist[key[i] >> 21], 1);
  __syncthreads();
  uint32_t* const to = (uint32_t*)(a.hist + (size_t)blockIdx.x * kPickBins);
  for (int i = tid; i < kPickBins / 2; i += kPartThreads)
    to[i] = (uint32_t)s_hist[2 * i] | (uint32_t)s_hist[2 * i + 1] << 16;
}

// With eight bins' counts a thread (c[0] the lowest bin's; thread t has bins 8 (255 - t) ..): the bin where the
// sum from the greatest on reaches `left`, and what is left of it there.
__device__ __forceinline__ void find_bin(const int (&c)[8], int left, int* s_sum, int* s_found) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int total = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) total += c[i];
  const int upto = wave_scan(total);
  if (lane == 63) s_sum[wave] = upto;
  __syncthreads();
  int from = upto - total;
#pragma unroll
  for (int i = 0; i < kPartThreads / 64; ++i) from += i < wave ? s_sum[i] : 0;
#pragma unroll
  for (int i = 7; i >= 0; --i) {
    if (from < left && left <= from + c[i]) {
      s_found[0] = 8 * (kPartThreads - 1 - tid) + i;
      s_found[1] = left - from;
    }
    from += c[i];
  }
  __syncthreads();
}

constexpr int kHeldKeys = 4096;
__global__ __launch_bounds__(kPartThreads) void evict_cut_kernel(EvictArgs a) {
  __shared__ __attribute__((aligned(16))) int s_hist[kPickBins];
  __shared__ int s_sum[kPartThreads / 64], s_found[2], s_gt, s_eq, s_last, s_end[kPartThreads];
  __shared__ int s_above[kPartThreads], s_same[kPartThreads];   // the first parts' (the others' go through memory)
  __shared__ uint32_t s_held[kHeldKeys];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const PartJob j = part_job(a);
  if (!part_chooses(a, j)) return;
  const int parts = (j.old + kPickPart - 1) / kPickPart;   // that take part
  const size_t row0 = (size_t)j.bk * a.parts;
  uint32_t key[kPartKeys];
  part_keys(j, lane, key);
  if (tid == 0) s_gt = s_eq = 0;
  int c[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 4
  for (int p = 0; p < parts; ++p) {
    const uint4 h = *(const uint4*)(a.hist + (row0 + p) * kPickBins + 8 * (kPartThreads - 1 - tid));
    const uint32_t x[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[2 * i] += (int)(x[i] & 0xffffu);
      c[2 * i + 1] += (int)(x[i] >> 16);
    }
  }
  find_bin(c, j.want, s_sum, s_found);
  const uint32_t bin = (uint32_t)s_found[0];
  int left = s_found[1];
  // thread p: part p's keys in the bin, on its way beside the arrivals
  const int many = tid < parts ? a.hist[(row0 + tid) * kPickBins + bin] : 0;

  // ---- this part's keys above the bin, and those in it (in any order), for whoever arrives last
  uint32_t* const mine = a.cand + (row0 + j.part) * kPickPart;
  int gt = 0;
#pragma unroll
  for (int i = 0; i < kPartKeys; ++i) {
    gt += __popcll(__ballot(key[i] >> 21 > bin));
    const bool in = key[i] != 0 && key[i] >> 21 == bin;
    const uint64_t who = __ballot(in);
    if (who == 0) continue;
    int at = 0;
    if (lane == 0) at = atomicAdd(&s_eq, __popcll(who));
    at = __builtin_amdgcn_readfirstlane(at);
    if (in)
      __hip_atomic_store(mine + at + __popcll(who & ((1ull << lane) - 1)), key[i], __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_SYSTEM);
  }
  if (lane == 0) atomicAdd(&s_gt, gt);
  __syncthreads();
  int32_t* const info = a.part_info + row0 * 4;
  if (tid == 0) {
    __hip_atomic_store(info + 4 * j.part, s_gt, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    __hip_atomic_store(info + 4 * j.part + 1, s_eq, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
  }
  wait_vm();
  __syncthreads();
  if (tid == 0) s_last = ticket(a.counters + j.bk, parts) ? 1 : 0;
  __syncthreads();
  if (!s_last) return;

  // ---- the last: the wanted key's lower 21 bits, from the keys of the bin. They are few unless weights are
  // much alike: then they are held in LDS, where they are looked at three times (131072 positions of one
  // sequence: 30 to 25 us)
  uint32_t found = bin << 21;
  const uint32_t* const all = a.cand + row0 * kPickPart;
  auto load = [&](const uint32_t* p) {
    return __hip_atomic_load(const_cast<uint32_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
  };
  auto load_i = [&](const int32_t* p) {
    return __hip_atomic_load(const_cast<int32_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
  };
  // where part p's keys end
  const int above_bin = tid < parts ? load_i(info + 4 * tid) : 0;
  int upto = wave_scan(many);
  if (lane == 63) s_sum[wave] = upto;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPartThreads / 64; ++i) upto += i < wave ? s_sum[i] : 0;
  s_end[tid] = upto;
  __syncthreads();
  const bool held = parts <= kPartThreads && s_end[kPartThreads - 1] <= kHeldKeys;
  if (held) {
    for (int p = wave; p < parts; p += kPartThreads / 64) {
      const int end = s_end[p], begin = p > 0 ? s_end[p - 1] : 0;
      for (int i = begin + lane; i < end; i += 64) s_held[i] = load(all + (size_t)p * kPickPart + (i - begin));
    }
    __syncthreads();
  }
  // f(key) of part p's keys, by a wave
  auto keys_of = [&](int p, auto f) {
    if (held) {
      const int end = s_end[p], begin = p > 0 ? s_end[p - 1] : 0;
      for (int i = begin + lane; i < end; i += 64) f(s_held[i]);
    } else {
      const int m = load_i(info + 4 * p + 1);
#pragma unroll 4
      for (int i = lane; i < m; i += 64) f(load(all + (size_t)p * kPickPart + i));
    }
  };
  for (int pass = 0; pass < 2; ++pass) {
    const int shift = pass == 0 ? 10 : 0;
    const uint32_t mask = pass == 0 ? 2047u : 1023u, known = pass == 0 ? ~0u << 21 : ~0u << 10;
    for (int i = tid; i < kPickBins; i += kPartThreads) s_hist[i] = 0;
    __syncthreads();
    for (int p = wave; p < parts; p += kPartThreads / 64)
      keys_of(p, [&](uint32_t k) {
        if ((k & known) == found) atomicAdd(&s_hist[k >> shift & mask], 1);
      });
    __syncthreads();
    int d[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] = s_hist[8 * (kPartThreads - 1 - tid) + i];
    find_bin(d, left, s_sum, s_found);
    found |= (uint32_t)s_found[0] << shift;
    left = s_found[1];
    __syncthreads();
  }
  // ---- how many each part writes, and from where on: its first place, and the equal keys before it
  for (int p = wave; p < parts; p += kPartThreads / 64) {
    int above = 0, same = 0;
    keys_of(p, [&](uint32_t k) {
      above += k > found;
      same += k == found;
    });
    above = wave_scan(above);
    same = wave_scan(same);
    if (lane == 63) {
      (p < kPartThreads ? s_above[p] : info[4 * p + 2]) = above;
      (p < kPartThreads ? s_same[p] : info[4 * p + 3]) = same;
    }
  }
  wait_vm();
  __syncthreads();
  int at = 0, ties = 0;   // before the parts at hand
  for (int p0 = 0; p0 < parts; p0 += kPartThreads) {
    const int p = p0 + tid;
    int g = 0, e = 0;
    if (p < parts) {
      g = p0 == 0 ? above_bin + s_above[p] : load_i(info + 4 * p) + info[4 * p + 2];
      e = p0 == 0 ? s_same[p] : info[4 * p + 3];
    }
    int eq_upto = wave_scan(e);
    if (lane == 63) s_sum[wave] = eq_upto;
    __syncthreads();
    int eq_all = 0;
#pragma unroll
    for (int i = 0; i < kPartThreads / 64; ++i) {
      eq_upto += i < wave ? s_sum[i] : 0;
      eq_all += s_sum[i];
    }
    __syncthreads();
    const int before = ties + eq_upto - e;
    const int n = g + min(e, max(left - before, 0));
    int n_upto = wave_scan(n);
    if (lane == 63) s_sum[wave] = n_upto;
    __syncthreads();
    int n_all = 0;
#pragma unroll
    for (int i = 0; i < kPartThreads / 64; ++i) {
      n_upto += i < wave ? s_sum[i] : 0;
      n_all += s_sum[i];
    }
    __syncthreads();
    if (p < parts) {
      info[4 * p + 2] = at + n_upto - n;
      info[4 * p + 3] = before;
    }
    at += n_all;
    ties += eq_all;
  }
  if (tid == 0) {
    a.cut[2 * j.bk] = found;
    a.cut[2 * j.bk + 1] = (uint32_t)left;
  }
}

__global__ __launch_bounds__(kPartThreads) void evict_list_kernel(EvictArgs a) {
  __shared__ int s_gt[kPartThreads / 64], s_eq[kPartThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const PartJob j = part_job(a);
  int32_t* const kept = a.kept + (size_t)j.bk * a.budget;
  const int stride = a.parts * kPartThreads;
  if (j.n <= a.budget) {
    for (int i = j.part * kPartThreads + tid; i < a.budget; i += stride) kept[i] = i < j.n ? i : -1;
    return;
  }
  for (int i = j.part * kPartThreads + tid; i < a.recent; i += stride) kept[j.want + i] = j.old + i;
  if (!part_chooses(a, j)) return;
  const uint32_t found = a.cut[2 * j.bk];
  const int left = (int)a.cut[2 * j.bk + 1];
  const int32_t* const info = a.part_info + ((size_t)j.bk * a.parts + j.part) * 4;
  int at = info[2], ties = info[3];
  uint32_t key[kPartKeys];
  part_keys(j, lane, key);
  int gt = 0, eq = 0;
#pragma unroll
  for (int i = 0; i < kPartKeys; ++i) {
    gt += __popcll(__ballot(key[i] > found));
    eq += __popcll(__ballot(key[i] == found));
  }
  if (lane == 0) {
    s_gt[wave] = gt;
    s_eq[wave] = eq;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPartThreads / 64; ++i)
    if (i < wave) {
      at += s_gt[i] + min(s_eq[i], max(left - ties, 0));
      ties += s_eq[i];
    }
  const uint64_t below = (1ull << lane) - 1;
#pragma unroll
  for (int i = 0; i < kPartKeys; ++i) {
    const uint64_t same = __ballot(key[i] == found);
    const bool take = key[i] > found || (key[i] == found && ties + __popcll(same & below) < left);
    const uint64_t who = __ballot(take);
    if (take) kept[at + __popcll(who & below)] = j.p0 + 64 * i + lane;
    at += __popcll(who);
    ties += __popcll(same);
  }
}

// A row's K or V in 16-byte pieces. K in pairs: piece c of the first half of the channels and of the second.
__device__ __forceinline__ void turn_back(uint4& a, uint4& z, const float* cs, int half, int c) {
  uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {z.x, z.y, z.z, z.w};
  float co[8], si[8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    *(float4*)(co + 4 * i) = *(const float4*)(cs + 8 * c + 4 * i);
    *(float4*)(si + 4 * i) = *(const float4*)(cs + half + 8 * c + 4 * i);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a0 = bf16lo(x[i]), a1 = bf16hi(x[i]), z0 = bf16lo(y[i]), z1 = bf16hi(y[i]);
    x[i] = pack_bf16x2(fmaf(a0, co[2 * i], z0 * si[2 * i]), fmaf(a1, co[2 * i + 1], z1 * si[2 * i + 1]));
    y[i] = pack_bf16x2(fmaf(z0, co[2 * i], -(a0 * si[2 * i])), fmaf(z1, co[2 * i + 1], -(a1 * si[2 * i + 1])));
  }
  a = make_uint4(x[0], x[1], x[2], x[3]);
  z = make_uint4(y[0], y[1], y[2], y[3]);
}

constexpr int kMoveThreads = 512;

// The rows of K (`which` 0) or V (1) and with V's the weights, TH / (D / 16) of them a step, two 16-byte pieces
// a thread; workgroup `block` of `blocks`, in place one for all. n: the old length.
template <int D, bool IN_PLACE, int TH>
__device__ __forceinline__ void evict_move(const EvictArgs& a, int bk, int n, int which, int block, int blocks,
                                           const int32_t* kept) {
  constexpr int L = D / 16, STEP = TH / L;   // threads of a row, rows of a step
  const int tid = threadIdx.x, c = tid % L, sub = tid / L;
  const int b = bk / a.hkv, h = bk - b * a.hkv;
  const int m = min(n, a.budget);
  if (IN_PLACE && n <= a.budget) return;
  const uint16_t* from = (which ? a.v : a.k) + (size_t)b * a.b_stride + (size_t)h * a.h_stride;
  uint16_t* to = (which ? a.v_out : a.k_out) + (size_t)b * a.ob_stride + (size_t)h * a.oh_stride;
  const float* w = a.weights + (size_t)b * a.w_b_stride + (size_t)h * a.w_h_stride;
  float* w_to = a.weights_out + (size_t)b * a.ow_b_stride + (size_t)h * a.ow_h_stride;
  const bool turn = which == 0 && a.tab != nullptr;
  // K's second piece is half a row on (its partner of a rotation), V's the next sixteen bytes
  const int e0 = which ? 16 * c : 8 * c, e1 = which ? 16 * c + 8 : D / 2 + 8 * c;

  struct Row {
    int src;
    uint4 x[2];
    float w;
  };
  auto load = [&](int i0, Row& r) {
    const int i = i0 + sub;
    r.src = i < m ? kept[i] : -1;
    if (r.src >= 0) {
      r.x[0] = *(const uint4*)(from + (size_t)r.src * D + e0);
      r.x[1] = *(const uint4*)(from + (size_t)r.src * D + e1);
      if (which && c == 0) r.w = w[r.src];
    }
  };
  auto store = [&](int i0, Row& r) {
    const int i = i0 + sub;
    if (r.src < 0) return;
    if (turn && r.src != i) turn_back(r.x[0], r.x[1], a.tab + (size_t)(r.src - i) * D, D / 2, c);
    *(uint4*)(to + (size_t)i * D + e0) = r.x[0];
    *(uint4*)(to + (size_t)i * D + e1) = r.x[1];
    if (which && c == 0) w_to[i] = r.w;
  };
  Row r;
  if constexpr (!IN_PLACE) {
    for (int i0 = block * STEP; i0 < m; i0 += blocks * STEP) {
      load(i0, r);
      store(i0, r);
    }
    if (which)
      for (int i = m + block * TH + tid; i < a.room; i += blocks * TH) w_to[i] = 0.f;
  } else {
    // the next step's rows are read before this step's are written
    Row next;
    load(0, r);
    for (int i0 = 0; i0 < m; i0 += STEP) {
      next.src = -1;
      if (i0 + STEP < m) load(i0 + STEP, next);
      wait_vm();          // this step's rows (with those read ahead) are there for every thread before any is written
      __syncthreads();
      store(i0, r);
      r = next;
    }
    if (which) {
      wait_vm();
      __syncthreads();
      for (int i = m + tid; i < n; i += TH) w_to[i] = 0.f;
    }
  }
}

template <int D, bool IN_PLACE>
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictArgs a) {
  // K first, which takes longer with a table; with 8 blocks or more an XCD has the same blocks of every (sequence,
  // kv head), and so about the same rows of the table (8 sequences, 4096 rows: 33 to 31 us)
  const int per = gridDim.x / 2;
  const int which = (int)blockIdx.x < per ? 0 : 1;
  const int blk = blockIdx.x - which * per;
  const int bk = blk / a.blocks, block = blk % a.blocks;
  const int n = a.n_old[bk];
  if (which == 1 && block == 0 && bk % a.hkv == 0 && threadIdx.x == 0) a.lens_out[bk / a.hkv] = min(n, a.budget);
  evict_move<D, IN_PLACE, kMoveThreads>(a, bk, n, which, block, a.blocks, a.kept + (size_t)bk * a.budget);
}

// Short caches cut down to few rows: a workgroup picks its (sequence, kv head)'s and moves them. The lengths
// stay as they are until the last workgroup of a sequence has read its own.
constexpr int kWholeRows = 1024;
template <int D, bool IN_PLACE, int KPT>
__global__ __launch_bounds__(kPickThreads) void evict_whole_kernel(EvictArgs a) {
  __shared__ int32_t s_kept[kWholeRows];
  const int bk = blockIdx.x, b = bk / a.hkv;
  const int n = min(max(a.lens[b], 0), a.max_len);
  int32_t* const kept = a.kept + (size_t)bk * a.budget;
  evict_pick<KPT, true>(a, bk, n, [&](int i, int p) {
    kept[i] = p;
    if (i < kWholeRows) s_kept[i] = p;
  });
  __syncthreads();
  if (threadIdx.x == 0 && ticket(a.counters + b, a.hkv)) a.lens_out[b] = min(n, a.budget);
  evict_move<D, IN_PLACE, kPickThreads>(a, bk, n, 0, 0, 1, s_kept);
  evict_move<D, IN_PLACE, kPickThreads>(a, bk, n, 1, 0, 1, s_kept);
}

template <int D, bool IN_PLACE>
static void whole_launch(const EvictArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.batch * a.hkv)), threads(kPickThreads);
  if (a.max_len <= kPickFew) hipLaunchKernelGGL((evict_whole_kernel<D, IN_PLACE, 4>), grid, threads, 0, s, a);
  else hipLaunchKernelGGL((evict_whole_kernel<D, IN_PLACE, 16>), grid, threads, 0, s, a);
}

static bool evict_shape_ok(int batch, int hkv, int d, int max_len, int budget, int recent) {
  return batch >= 1 && hkv >= 1 && (long long)batch * hkv <= (1 << 24) && (d == 64 || d == 128) && max_len >= 1 &&
         max_len < (1 << 24) && budget >= 1 && recent >= 0 && recent <= budget;
}

// Parts of a (sequence, kv head)'s selection; 0: one workgroup's, with few positions and where there are more
// (sequence, kv head)s than counters.
static int evict_parts(size_t bh, int max_len) {
  return max_len <= kPickHeld || bh > Q4NX_WS_COUNTER_BYTES / 4 ? 0 : (max_len + kPickPart - 1) / kPickPart;
}
// Lengths and cuts, before the parts' memory.
static size_t evict_head_bytes(size_t bh) { return (bh * 12 + 255) / 256 * 256; }

}  // namespace q4nx

using namespace q4nx;

extern "C" {

size_t q4nx_kv_evict_ws_bytes(int batch, int n_kv_heads, int max_len) {
  if (!evict_shape_ok(batch, n_kv_heads, 64, max_len, 1, 0)) return 0;
  const size_t bh = (size_t)batch * n_kv_heads;
  return (size_t)Q4NX_WS_COUNTER_BYTES + evict_head_bytes(bh) +
         bh * evict_parts(bh, max_len) * (kPickPart * 4 + kPickBins * 2 + 16);
}

int q4nx_kv_evict(const uint16_t* k_cache, const uint16_t* v_cache, int64_t kv_b_stride, int64_t kv_h_stride,
                  const float* weights, int64_t w_b_stride, int64_t w_h_stride, const int32_t* lens, int max_len,
                  int budget, int recent, const float* rope_tab, int max_pos, uint16_t* k_out, uint16_t* v_out,
                  int64_t out_b_stride, int64_t out_h_stride, float* weights_out, int64_t wout_b_stride,
                  int64_t wout_h_stride, int room, int32_t* lens_out, int32_t* kept, int batch, int n_kv_heads,
                  int head_dim, void* ws, size_t ws_bytes, void* stream) {
  const char* what = "q4nx_kv_evict";
  Q4NX_REQUIRE(evict_shape_ok(batch, n_kv_heads, head_dim, max_len, budget, recent), Q4NX_ERR_SHAPE,
               "%s: batch=%d Hkv=%d head_dim=%d (64, 128) max_len=%d (below 2^24) budget=%d (positive) recent=%d "
               "(0..budget)",
               what, batch, n_kv_heads, head_dim, max_len, budget, recent);
  Q4NX_REQUIRE(k_cache && v_cache && weights && lens && k_out && v_out && weights_out && lens_out && kept,
               Q4NX_ERR_ARG, "%s: caches, weights, lens, their outputs and kept are required", what);
  Q4NX_REQUIRE(Q4NX_ALIGNED(k_cache, 16) && Q4NX_ALIGNED(v_cache, 16) && Q4NX_ALIGNED(k_out, 16) &&
                   Q4NX_ALIGNED(v_out, 16) && Q4NX_ALIGNED(rope_tab, 16),
               Q4NX_ERR_ARG, "%s: caches and table must be 16-byte aligned", what);
  const bool in_place = k_out == k_cache;
  Q4NX_REQUIRE(in_place ? v_out == v_cache && weights_out == weights && out_b_stride == kv_b_stride &&
                              out_h_stride == kv_h_stride && wout_b_stride == w_b_stride &&
                              wout_h_stride == w_h_stride
                        : v_out != v_cache && weights_out != weights,
               Q4NX_ERR_ARG, "%s: K, V and weights are cut down in place together, or none of them", what);
  Q4NX_REQUIRE(kv_h_stride >= (int64_t)max_len * head_dim && kv_h_stride % 8 == 0 &&
                   kv_b_stride >= (int64_t)n_kv_heads * kv_h_stride && kv_b_stride % 8 == 0,
               Q4NX_ERR_SHAPE, "%s: cache strides do not hold [Hkv][max_len][head_dim]", what);
  Q4NX_REQUIRE(w_h_stride >= max_len && w_b_stride >= (int64_t)n_kv_heads * w_h_stride, Q4NX_ERR_SHAPE,
               "%s: strides of weights do not hold [Hkv][max_len]", what);
  const int most = budget < max_len ? budget : max_len;   // rows that may be kept
  Q4NX_REQUIRE(in_place || (room >= most && out_h_stride >= (int64_t)room * head_dim && out_h_stride % 8 == 0 &&
                            out_b_stride >= (int64_t)n_kv_heads * out_h_stride && out_b_stride % 8 == 0 &&
                            wout_h_stride >= room && wout_b_stride >= (int64_t)n_kv_heads * wout_h_stride),
               Q4NX_ERR_SHAPE, "%s: the outputs' room of %d does not hold the %d positions kept", what, room, most);
  Q4NX_REQUIRE(rope_tab == nullptr || max_pos >= max_len, Q4NX_ERR_SHAPE,
               "%s: the table's %d positions are fewer than max_len=%d", what, max_pos, max_len);
  const size_t need = q4nx_kv_evict_ws_bytes(batch, n_kv_heads, max_len);
  Q4NX_REQUIRE(ws != nullptr && ws_bytes >= need && Q4NX_ALIGNED(ws, 256), Q4NX_ERR_WS,
               "%s: workspace of %zu bytes (256-aligned) needed, %zu given", what, need, ws_bytes);
  EvictArgs a{};
  a.k = k_cache;
  a.v = v_cache;
  a.weights = weights;
  a.lens = lens;
  a.tab = rope_tab;
  a.k_out = k_out;
  a.v_out = v_out;
  a.weights_out = weights_out;
  a.lens_out = lens_out;
  a.kept = kept;
  const int bh = batch * n_kv_heads, parts = evict_parts(bh, max_len);
  a.parts = parts;
  a.counters = (unsigned*)ws;
  a.n_old = (int32_t*)((uint8_t*)ws + Q4NX_WS_COUNTER_BYTES);
  a.cut = (uint32_t*)(a.n_old + bh);
  a.cand = (uint32_t*)((uint8_t*)a.n_old + evict_head_bytes(bh));
  a.hist = (uint16_t*)(a.cand + (size_t)bh * parts * kPickPart);
  a.part_info = (int32_t*)(a.hist + (size_t)bh * parts * kPickBins);
  a.b_stride = kv_b_stride;
  a.h_stride = kv_h_stride;
  a.w_b_stride = w_b_stride;
  a.w_h_stride = w_h_stride;
  a.ob_stride = out_b_stride;
  a.oh_stride = out_h_stride;
  a.ow_b_stride = wout_b_stride;
  a.ow_h_stride = wout_h_stride;
  a.batch = batch;
  a.hkv = n_kv_heads;
  a.max_len = max_len;
  a.budget = budget;
  a.recent = recent;
  a.room = room;
  hipStream_t s = (hipStream_t)stream;
  // 1 x 1000 to 512 in one launch: 13.3 us a pass, 16.2 in two; more rows go faster by more workgroups than one
  if (max_len <= kPickHeld && most <= kWholeRows && batch <= Q4NX_WS_COUNTER_BYTES / 4) {
    if (head_dim == 64 && in_place) whole_launch<64, true>(a, s);
    else if (head_dim == 64) whole_launch<64, false>(a, s);
    else if (in_place) whole_launch<128, true>(a, s);
    else whole_launch<128, false>(a, s);
    return check_launch(what);
  }
  const int step = kMoveThreads / (head_dim / 16);
  a.blocks = in_place ? 1 : (most + step - 1) / step;
  if (a.blocks > 4096) a.blocks = 4096;
  Q4NX_REQUIRE(2ll * bh * a.blocks < (1ll << 31) && (long long)bh * parts < (1ll << 31), Q4NX_ERR_SHAPE,
               "%s: more than 2^31 workgroups", what);
  if (parts > 0) {
    const dim3 all((unsigned)(bh * parts)), threads(kPartThreads);
    hipLaunchKernelGGL(evict_hist_kernel, all, threads, 0, s, a);
    hipLaunchKernelGGL(evict_cut_kernel, all, threads, 0, s, a);
    hipLaunchKernelGGL(evict_list_kernel, all, threads, 0, s, a);
  } else if (max_len <= kPickFew) {
    hipLaunchKernelGGL((evict_pick_kernel<4, true>), dim3((unsigned)bh), dim3(kPickThreads), 0, s, a);
  } else if (max_len <= kPickHeld) {
    hipLaunchKernelGGL((evict_pick_kernel<16, true>), dim3((unsigned)bh), dim3(kPickThreads), 0, s, a);
  } else {
    hipLaunchKernelGGL((evict_pick_kernel<16, false>), dim3((unsigned)bh), dim3(kPickThreads), 0, s, a);
  }
  const dim3 grid((unsigned)(2 * bh * a.blocks));
  const dim3 threads(kMoveThreads);
  if (head_dim == 64 && in_place) hipLaunchKernelGGL((evict_move_kernel<64, true>), grid, threads, 0, s, a);
  else if (head_dim == 64) hipLaunchKernelGGL((evict_move_kernel<64, false>), grid, threads, 0, s, a);
  else if (in_place) hipLaunchKernelGGL((evict_move_kernel<128, true>), grid, threads, 0, s, a);
  else hipLaunchKernelGGL((evict_move_kernel<128, false>), grid, threads, 0, s, a);
  return check_launch(what);
}

}  // extern "C"
