// Which pages of the 4-bit K/V cache a query reads: an upper bound of q . k over a page's rows, from
// the least and greatest value of each channel of K,
//   score = sum over the group's heads and channels of max(q lo, q hi) = sum_c Q+_c hi_c + Q-_c lo_c
// with Q+ and Q- the sums over the heads of q's positive and negative parts: one product per bound,
// however many heads share the pages. Products and sums are fp64, so that which pages are chosen does
// not hang on the order of a sum. Bounds are 4 D bytes per page and kv head, read once.
// Bound by a chain of loads: a head's row of q is waited for before the next one's, then the four table
// entries of a lane likewise; only the bounds are in flight together. With 2048 pages, one sequence and five
// heads a kv head the waves wait 0.68 of their time, and the VALU is active in 0.25 of the busy cycles.
#include <math.h>

#include "kv4.h"

namespace q4nx {

struct Kv4SelArgs {
  Kv4 c;
  const uint16_t* q;
  int64_t q_stride;
  const int32_t* lens;
  int32_t* sel;
  int n_sel, n_first, n_last, group, max_len, max_pages, parts;
  unsigned long long* keys;   // [n_seqs * hkv][max_pages]
  unsigned* counters;
};

// Pages scored by a workgroup, and its threads, all of which work on the list in the last one to arrive.
// 2048 pages, one sequence (8 kv heads): 14.1 us; 64 pages and 256 threads 16.6, 64 and 512 14.7, 128 and
// 1024 15.6. Eight sequences of up to 938 pages: 15.4, against 15.4, 17.5 and 20.0 us. 64 pages in all take
// 6.3 us.
constexpr int kSelPages = 128;
constexpr int kSelThreads = 512;
constexpr int kSelWaves = kSelThreads / 64;

// Keys from here on: a NaN score (its page is read, so that it shows), above it the pages always read.
constexpr unsigned long long kSpecial = ~1ull;
__device__ __forceinline__ unsigned long long f64_key(double x) {
  if (x != x) return kSpecial;
  const unsigned long long u = (unsigned long long)__double_as_longlong(x);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

__device__ __forceinline__ unsigned long long load_sys64(const unsigned long long* p) {
  return __hip_atomic_load(const_cast<unsigned long long*>(p), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_SYSTEM);
}

template <int NG>
__global__ __launch_bounds__(kSelThreads) void kv4_select_kernel(Kv4SelArgs a) {
  constexpr int D = 32 * NG, L = D / 4, PW = 64 / L;   // lanes per page, pages per wave step
  extern __shared__ unsigned long long s_key[];
  __shared__ int s_hist[256], s_pick[3], s_count[kSelWaves][2], s_special[kSelWaves];
  __shared__ unsigned long long s_range[kSelWaves][2], s_out[kSelPages];
  __shared__ int s_last;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int part = blockIdx.x % a.parts, bk = blockIdx.x / a.parts;
  const int h = bk % a.c.hkv, b = bk / a.c.hkv;
  const int len = max(0, min(a.lens[b], min(a.c.cap, a.max_len)));
  const int np = (len + a.c.page_len - 1) / a.c.page_len;
  unsigned long long* keys = a.keys + (size_t)bk * a.max_pages;

  // ---- this part's scores
  const int sub = lane % L;
  const bool high = sub >= L / 2;
  const int ch = (sub % (L / 2)) * 8;
  if (part * kSelPages < np) {
    double w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    constexpr int HEADS = 8;   // to a round
    for (int g0 = 0; g0 < a.group; g0 += HEADS) {
      u32x4_t y[HEADS];
#pragma unroll
      for (int g = 0; g < HEADS; ++g)
        y[g] = *(const u32x4_t*)(a.q + (int64_t)b * a.q_stride +
                                 (h * a.group + min(g0 + g, a.group - 1)) * D + ch);
#pragma unroll
      for (int g = 0; g < HEADS; ++g) {
        if (g0 + g >= a.group) break;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float f = (i & 1) ? bf16hi(y[g][i >> 1]) : bf16lo(y[g][i >> 1]);
          if (f != f || (f > 0.f) == high) w[i] += (double)f;   // a zero adds nothing to either
        }
      }
    }
    constexpr int STEPS = kSelPages / (kSelWaves * PW);
    const int p0 = part * kSelPages + wave * PW + lane / L;
    int id[STEPS];
    u32x4_t x[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int p = p0 + kSelWaves * PW * i;
      id[i] = p < np ? kv4_page(a.c, b, p) : -1;
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
      x[i] = *(const u32x4_t*)(a.c.pages + (int64_t)max(id[i], 0) * a.c.page_stride +
                               (int64_t)h * kv4_head_bytes(a.c.page_len, D) +
                               a.c.tiles * kv4_tile_bytes(D) + sub * 16);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int p = p0 + kSelWaves * PW * i;
      double s = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        s = fma(w[j], (double)((j & 1) ? bf16hi(x[i][j >> 1]) : bf16lo(x[i][j >> 1])), s);
#pragma unroll
      for (int o = 1; o < L; o <<= 1) s += __shfl_xor(s, o);
      if (sub == 0) {
        const bool always = p < a.n_first || p >= np - a.n_last;
        s_out[p - part * kSelPages] = always ? ~0ull : id[i] < 0 ? kSpecial : f64_key(s);
      }
    }
  }
  // published together: single keys written through cost more than the scores
  __syncthreads();
  for (int e = tid; e < kSelPages && part * kSelPages + e < np; e += kSelThreads)
    __hip_atomic_store(keys + part * kSelPages + e, s_out[e], __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_SYSTEM);
  wait_vm();
  __syncthreads();
  if (tid == 0) s_last = ticket(&a.counters[bk], a.parts) ? 1 : 0;
  __syncthreads();
  if (!s_last) return;

  // ---- the last part to arrive: the n_sel greatest keys, the lowest page first among equals
  int32_t* out = a.sel + (size_t)bk * a.n_sel;
  for (int e = min(np, a.n_sel) + tid; e < a.n_sel; e += kSelThreads) out[e] = -1;
  if (np <= a.n_sel) {
    for (int e = tid; e < np; e += kSelThreads) out[e] = e;
    return;
  }
  // the keys, their range and how many are always read or NaN (those lie above every score)
  unsigned long long lo = kSpecial, hi = 0;
  int special = 0;
  constexpr int kBatch = 4;   // loads in flight: they go past the caches
  for (int e0 = tid; e0 < np; e0 += kSelThreads * kBatch) {
    unsigned long long k[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) k[i] = load_sys64(keys + min(e0 + kSelThreads * i, np - 1));
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (e0 + kSelThreads * i >= np) break;
      s_key[e0 + kSelThreads * i] = k[i];
      if (k[i] >= kSpecial) ++special;
      else {
        lo = k[i] < lo ? k[i] : lo;
        hi = k[i] > hi ? k[i] : hi;
      }
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned long long l2 = __shfl_xor(lo, o), h2 = __shfl_xor(hi, o);
    lo = l2 < lo ? l2 : lo;
    hi = h2 > hi ? h2 : hi;
    special += __shfl_xor(special, o);
  }
  if (lane == 0) {
    s_range[wave][0] = lo;
    s_range[wave][1] = hi;
    s_special[wave] = special;
  }
  if (tid < 256) s_hist[tid] = 0;
  __syncthreads();
  special = 0;
#pragma unroll
  for (int w = 0; w < kSelWaves; ++w) {
    lo = s_range[w][0] < lo ? s_range[w][0] : lo;
    hi = s_range[w][1] > hi ? s_range[w][1] : hi;
    special += s_special[w];
  }
  // Digit by digit from the first bit in which the scores differ: the digit at which the n_sel-th key
  // lies, until a whole bucket fits (two or three digits as a rule). Where the special keys alone are
  // too many, from the top over all of them.
  const bool all = special >= a.n_sel;
  int shift = all ? 64 : lo == hi ? 0 : 64 - __builtin_clzll(lo ^ hi);
  unsigned long long prefix = shift == 64 ? 0 : lo >> shift;
  int want = all ? a.n_sel : a.n_sel - special;
  bool whole = false;
  while (shift > 0 && !whole) {
    const int next = shift > 8 ? shift - 8 : 0, digits = (1 << (shift - next)) - 1;
    for (int e = tid; e < np; e += kSelThreads) {
      const unsigned long long k = s_key[e];
      if ((all || k < kSpecial) && (shift == 64 || (k >> shift) == prefix))
        atomicAdd(&s_hist[(int)(k >> next) & digits], 1);
    }
    __syncthreads();
    if (wave == 0) {   // lane l: digits 255 - 4 l .. 252 - 4 l, the greater first
      int c[4], sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c[i] = s_hist[255 - 4 * lane - i];
        sum += c[i];
      }
      int before = sum;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(before, o);
        if (lane >= o) before += y;
      }
      before -= sum;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (before < want && before + c[i] >= want) {
          s_pick[0] = 255 - 4 * lane - i;
          s_pick[1] = before;
          s_pick[2] = c[i];
        }
        before += c[i];
      }
    }
    __syncthreads();
    prefix = (prefix << (shift - next)) | (unsigned)s_pick[0];
    want -= s_pick[1];
    whole = s_pick[2] == want;
    shift = next;
    if (tid < 256) s_hist[tid] = 0;
    __syncthreads();
  }
  // the pages in order: a wave's stretch of them, 64 at a time; special keys lie above every score, also
  // where a score of +inf has their leading digits
  const int span = (np + kSelThreads - 1) / kSelThreads * 64, e0 = wave * span, e1 = min(np, e0 + span);
  auto above = [&](unsigned long long k) { return !all && k >= kSpecial; };
  auto is_gt = [&](int e) { return e < e1 && (above(s_key[e]) || (s_key[e] >> shift) > prefix); };
  auto is_eq = [&](int e) { return e < e1 && !above(s_key[e]) && (s_key[e] >> shift) == prefix; };
  int gt = 0, eq = 0;
  for (int e = e0; e < e1; e += 64) {
    gt += __popcll(__ballot(is_gt(e + lane)));
    eq += __popcll(__ballot(is_eq(e + lane)));
  }
  if (lane == 0) {
    s_count[wave][0] = gt;
    s_count[wave][1] = eq;
  }
  __syncthreads();
  int g0 = 0, q0 = 0;
  for (int w = 0; w < wave; ++w) {
    g0 += s_count[w][0];
    q0 += s_count[w][1];
  }
  const unsigned long long below = (1ull << lane) - 1;
  for (int e = e0; e < e1; e += 64) {
    const bool g = is_gt(e + lane), q = is_eq(e + lane);
    const unsigned long long bg = __ballot(g), bq = __ballot(q);
    const int gi = g0 + __popcll(bg & below), qi = q0 + __popcll(bq & below);
    if (g || (q && qi < want)) out[gi + min(qi, want)] = e + lane;
    g0 += __popcll(bg);
    q0 += __popcll(bq);
  }
}

}  // namespace q4nx

using namespace q4nx;

extern "C" {

// Pages a sequence may have under max_len.
static int64_t kv4_max_pages(const q4nx_kv4* c, int max_len) {
  const int64_t by_len = ((int64_t)max_len + c->page_len - 1) / c->page_len;
  return by_len < c->table_len ? by_len : c->table_len;
}

size_t q4nx_kv4_select_ws_bytes(const q4nx_kv4* cache, int max_len) {
  Kv4 c;
  if (kv4_resolve(cache, &c, "q4nx_kv4_select_ws_bytes") != Q4NX_OK || max_len < 1) return 0;
  return (size_t)Q4NX_WS_COUNTER_BYTES +
         (size_t)c.n_seqs * c.hkv * (size_t)kv4_max_pages(cache, max_len) * 8;
}

int q4nx_kv4_select(const q4nx_kv4* cache, const uint16_t* q, int64_t q_stride, int n_q_heads,
                    const int32_t* lens, int max_len, int n_sel, int n_first, int n_last, int32_t* sel,
                    void* ws, size_t ws_bytes, void* stream) {
  const char* what = "q4nx_kv4_select";
  Kv4SelArgs a{};
  if (int rc = kv4_resolve(cache, &a.c, what)) return rc;
  Q4NX_REQUIRE(q && lens && sel && Q4NX_ALIGNED(q, 16), Q4NX_ERR_ARG,
               "%s: q (16-byte aligned), lens and sel are required", what);
  Q4NX_REQUIRE(n_q_heads >= 1 && n_q_heads % cache->n_kv_heads == 0 &&
                   n_q_heads / cache->n_kv_heads <= 16 && max_len >= 1,
               Q4NX_ERR_SHAPE, "%s: Hq=%d must be a multiple (<= 16x) of Hkv=%d; max_len=%d", what,
               n_q_heads, cache->n_kv_heads, max_len);
  Q4NX_REQUIRE(n_first >= 0 && n_last >= 0 && n_sel >= 1 && n_sel <= 1 << 20 &&
                   (int64_t)n_first + n_last <= n_sel,
               Q4NX_ERR_ARG, "%s: n_sel=%d must hold the first %d and last %d pages", what, n_sel,
               n_first, n_last);
  Q4NX_REQUIRE(q_stride >= (int64_t)n_q_heads * cache->head_dim && q_stride % 8 == 0, Q4NX_ERR_SHAPE,
               "%s: q_stride=%lld must hold Hq * D and be a multiple of 8", what, (long long)q_stride);
  const int64_t mp = kv4_max_pages(cache, max_len);
  Q4NX_REQUIRE(mp <= 16384, Q4NX_ERR_SHAPE, "%s: %lld pages per sequence, at most 16384", what,
               (long long)mp);
  const int64_t items = (int64_t)a.c.n_seqs * a.c.hkv;
  Q4NX_REQUIRE(items * 4 <= Q4NX_WS_COUNTER_BYTES, Q4NX_ERR_SHAPE,
               "%s: batch*Hkv exceeds the workspace counter region", what);
  const size_t need = q4nx_kv4_select_ws_bytes(cache, max_len);
  Q4NX_REQUIRE(ws != nullptr && ws_bytes >= need && Q4NX_ALIGNED(ws, 256), Q4NX_ERR_WS,
               "%s: workspace of %zu bytes (256-aligned) needed, %zu given", what, need, ws_bytes);
  a.q = q;
  a.q_stride = q_stride;
  a.lens = lens;
  a.sel = sel;
  a.n_sel = n_sel;
  a.n_first = n_first;
  a.n_last = n_last;
  a.group = n_q_heads / cache->n_kv_heads;
  a.max_len = max_len;
  a.max_pages = (int)mp;
  a.parts = (int)((mp + kSelPages - 1) / kSelPages);
  a.counters = (unsigned*)ws;
  a.keys = (unsigned long long*)((uint8_t*)ws + Q4NX_WS_COUNTER_BYTES);
  const dim3 grid((unsigned)(items * a.parts));
  const size_t lds = (size_t)mp * 8;
  if (cache->head_dim == 64)
    hipLaunchKernelGGL(kv4_select_kernel<2>, grid, dim3(kSelThreads), lds, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(kv4_select_kernel<4>, grid, dim3(kSelThreads), lds, (hipStream_t)stream, a);
  return check_launch(what);
}

}  // extern "C"
