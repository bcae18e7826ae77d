// Caches cut down to the positions that were given the most attention and the newest ones. No reference
// counterpart (its cache never shrinks).
//
// Per (sequence, kv head) with n = lens[b] > budget positions: of the first n - recent those budget - recent
// of the greatest weights (ties to the lowest position), then the `recent` last, in the order of their
// positions. Two launches: which ones (a radix selection by one workgroup), then the rows. With n <= budget
// all are kept.
//
// Rows move towards the front. Into other memory they move all at once. In place, row i comes from a
// position >= i, so a workgroup that takes rows in order, a block at a time, only overwrites rows that it
// has read: a block's sources lie at or behind the block's own first row, and every later block's behind it.
// K and V have a workgroup each.
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
  int32_t* n_old;          // [batch * hkv]: lengths, for the second launch
  int64_t b_stride, h_stride, w_b_stride, w_h_stride;
  int64_t ob_stride, oh_stride, ow_b_stride, ow_h_stride;
  int batch, hkv, max_len, budget, recent, room;
  int in_place, blocks;    // blocks: workgroups for a (sequence, kv head)'s rows
};

// Greater weights have greater keys; a NaN's is the greatest; -0 and 0 are one value.
__device__ __forceinline__ uint32_t weight_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

constexpr int kPickThreads = 1024;
constexpr int kPickWaves = kPickThreads / 64;
constexpr int kPickBins = 2048;    // 11 bits a pass: 32 bits in three

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

// A wave takes KPT * 64 positions in a row (of every KPT * 1024). HELD: that is all of them, and their keys
// stay in registers; otherwise each pass reads the weights again.
template <int KPT, bool HELD>
__global__ __launch_bounds__(kPickThreads) void evict_pick_kernel(EvictArgs a) {
  __shared__ int s_hist[kPickBins];
  __shared__ int s_sum[kPickWaves], s_gt[kPickWaves], s_eq[kPickWaves];
  __shared__ uint32_t s_key;
  __shared__ int s_left;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int bk = blockIdx.x, b = bk / a.hkv, h = bk - b * a.hkv;
  const int n = min(max(a.lens[b], 0), a.max_len);
  int32_t* kept = a.kept + (size_t)bk * a.budget;
  if (tid == 0) a.n_old[bk] = n;
  if (n <= a.budget) {
    for (int i = tid; i < a.budget; i += kPickThreads) kept[i] = i < n ? i : -1;
    return;
  }
  const int old = n - a.recent, want = a.budget - a.recent;   // want < old
  for (int i = tid; i < a.recent; i += kPickThreads) kept[want + i] = old + i;
  if (want == 0) return;
  const float* w = a.weights + (size_t)b * a.w_b_stride + (size_t)h * a.w_h_stride;

  uint32_t key[KPT];
  auto load = [&](int p0) {   // key 0 (below that of every weight) past the end
    float x[KPT];
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
      const int p = p0 + 64 * i + lane;
      x[i] = p < old ? w[p] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < KPT; ++i) key[i] = p0 + 64 * i + lane < old ? weight_key(x[i]) : 0u;
  };
  const int first = wave * KPT * 64;
  auto each = [&](auto f) {
    if constexpr (HELD) {
      f(first);
    } else {
      for (int p0 = first; p0 < old; p0 += KPT * kPickThreads) {
        load(p0);
        f(p0);
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
    for (int i = tid; i < kPickBins; i += kPickThreads) s_hist[i] = 0;
    __syncthreads();
    each([&](int) {
#pragma unroll
      for (int i = 0; i < KPT; ++i)
        if (key[i] != 0 && (key[i] & known) == found) atomicAdd(&s_hist[(key[i] >> shift) & mask], 1);
    });
    __syncthreads();
    // the bin where the sum from the greatest on reaches `left`: two bins a thread, the greatest first
    const int hi = kPickBins - 1 - 2 * tid;
    const int c0 = s_hist[hi], c1 = s_hist[hi - 1];
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
  for (int p0 = 0; p0 < old; p0 += KPT * kPickThreads) {
    if constexpr (!HELD) load(p0 + first);
    int gt = 0, eq = 0;
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
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
      const uint64_t same = __ballot(key[i] == found);
      const bool take = key[i] > found || (key[i] == found && seen + __popcll(same & below) < left);
      const uint64_t who = __ballot(take);
      if (take) kept[at + __popcll(who & below)] = p0 + first + 64 * i + lane;
      at += __popcll(who);
      seen += __popcll(same);
    }
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

// kMoveThreads / (D / 16) rows of K (`which` 0) or V (1) a step: two 16-byte pieces a thread.
template <int D>
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictArgs a) {
  constexpr int L = D / 16, STEP = kMoveThreads / L;   // threads of a row, rows of a step
  const int tid = threadIdx.x, c = tid % L, sub = tid / L;
  int blk = blockIdx.x;
  const int which = blk & 1;
  blk >>= 1;
  const int bk = blk / a.blocks, block = blk % a.blocks;
  const int b = bk / a.hkv, h = bk - b * a.hkv;
  const int n = a.n_old[bk], m = min(n, a.budget);
  const int32_t* kept = a.kept + (size_t)bk * a.budget;
  if (which == 1) {
    // the weights go with V's rows, by the first wave's threads ... of the same blocks
    if (block == 0 && h == 0 && tid == 0) a.lens_out[b] = m;
  }
  if (a.in_place && n <= a.budget) return;
  const uint16_t* from = (which ? a.v : a.k) + (size_t)b * a.b_stride + (size_t)h * a.h_stride;
  uint16_t* to = (which ? a.v_out : a.k_out) + (size_t)b * a.ob_stride + (size_t)h * a.oh_stride;
  const float* w = a.weights + (size_t)b * a.w_b_stride + (size_t)h * a.w_h_stride;
  float* w_to = a.weights_out + (size_t)b * a.ow_b_stride + (size_t)h * a.ow_h_stride;
  const bool turn = which == 0 && a.tab != nullptr;
  // K's second piece is half a row on (its partner of a rotation), V's the next sixteen bytes
  const int e0 = which ? 16 * c : 8 * c, e1 = which ? 16 * c + 8 : D / 2 + 8 * c;

  uint4 x[2], y[2];
  float ws = 0.f, ws2 = 0.f;
  int src = 0;
  auto load = [&](int i0, int& s_, uint4 (&r)[2], float& wv) {
    const int i = i0 + sub;
    s_ = i < m ? kept[i] : -1;
    if (s_ >= 0) {
      r[0] = *(const uint4*)(from + (size_t)s_ * D + e0);
      r[1] = *(const uint4*)(from + (size_t)s_ * D + e1);
      if (which && c == 0) wv = w[s_];
    }
  };
  auto store = [&](int i0, int s_, uint4 (&r)[2], float wv) {
    const int i = i0 + sub;
    if (s_ < 0) return;
    if (turn && s_ != i) turn_back(r[0], r[1], a.tab + (size_t)(s_ - i) * D, D / 2, c);
    *(uint4*)(to + (size_t)i * D + e0) = r[0];
    *(uint4*)(to + (size_t)i * D + e1) = r[1];
    if (which && c == 0) w_to[i] = wv;
  };
  if (!a.in_place) {
    for (int i0 = block * STEP; i0 < m; i0 += a.blocks * STEP) {
      load(i0, src, x, ws);
      store(i0, src, x, ws);
    }
    if (which)
      for (int i = m + block * kMoveThreads + tid; i < a.room; i += a.blocks * kMoveThreads) w_to[i] = 0.f;
    return;
  }
  // in place, one workgroup for all rows: the next step's rows are read before this step's are written
  int src2 = 0;
  load(0, src, x, ws);
  for (int i0 = 0; i0 < m; i0 += STEP) {
    if (i0 + STEP < m) load(i0 + STEP, src2, y, ws2);
    wait_vm();          // this step's rows have been read by every thread before any is written
    __syncthreads();
    store(i0, src, x, ws);
    src = src2;
    x[0] = y[0];
    x[1] = y[1];
    ws = ws2;
  }
  if (which) {
    wait_vm();
    __syncthreads();
    for (int i = m + tid; i < n; i += kMoveThreads) w_to[i] = 0.f;
  }
}

static bool evict_shape_ok(int batch, int hkv, int d, int max_len, int budget, int recent) {
  return batch >= 1 && hkv >= 1 && (long long)batch * hkv <= (1 << 24) && (d == 64 || d == 128) && max_len >= 1 &&
         max_len < (1 << 24) && budget >= 1 && recent >= 0 && recent <= budget;
}

}  // namespace q4nx

using namespace q4nx;

extern "C" {

size_t q4nx_kv_evict_ws_bytes(int batch, int n_kv_heads) {
  if (batch < 1 || n_kv_heads < 1 || (long long)batch * n_kv_heads > (1 << 24)) return 0;
  return (size_t)Q4NX_WS_COUNTER_BYTES + (size_t)batch * n_kv_heads * 4;
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
  const size_t need = q4nx_kv_evict_ws_bytes(batch, n_kv_heads);
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
  a.n_old = (int32_t*)((uint8_t*)ws + Q4NX_WS_COUNTER_BYTES);
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
  a.in_place = in_place;
  const int bh = batch * n_kv_heads;
  const int step = kMoveThreads / (head_dim / 16);
  a.blocks = in_place ? 1 : (most + step - 1) / step;
  if (a.blocks > 4096) a.blocks = 4096;
  Q4NX_REQUIRE(2ll * bh * a.blocks < (1ll << 31), Q4NX_ERR_SHAPE, "%s: more than 2^31 workgroups", what);
  hipStream_t s = (hipStream_t)stream;
  const dim3 heads((unsigned)bh), threads(kPickThreads);
  if (max_len <= 4 * kPickThreads) hipLaunchKernelGGL((evict_pick_kernel<4, true>), heads, threads, 0, s, a);
  else if (max_len <= 16 * kPickThreads) hipLaunchKernelGGL((evict_pick_kernel<16, true>), heads, threads, 0, s, a);
  else if (max_len <= 48 * kPickThreads) hipLaunchKernelGGL((evict_pick_kernel<48, true>), heads, threads, 0, s, a);
  else hipLaunchKernelGGL((evict_pick_kernel<16, false>), heads, threads, 0, s, a);
  const dim3 grid((unsigned)(2 * bh * a.blocks));
  if (head_dim == 64) hipLaunchKernelGGL(evict_move_kernel<64>, grid, dim3(kMoveThreads), 0, s, a);
  else hipLaunchKernelGGL(evict_move_kernel<128>, grid, dim3(kMoveThreads), 0, s, a);
  return check_launch(what);
}

}  // extern "C"
