// Which pages of the 4-bit K/V cache a query reads: an upper bound of q . k over a page's rows, from
// the least and greatest value of each channel of K,
//   score = sum over the group's heads and channels of max(q lo, q hi) = sum_c Q+_c hi_c + Q-_c lo_c
// with Q+ and Q- the sums over the heads of q's positive and negative parts: one product per bound,
// however many heads share the pages. Products and sums are fp64, so that which pages are chosen does
// not hang on the order of a sum. Bounds are 4 D bytes per page and kv head, read once.
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

constexpr int kSelPages = 64;   // pages scored by a workgroup

__device__ __forceinline__ unsigned long long f64_key(double x) {
  if (x != x) return ~1ull;   // a NaN's page is read, so that it shows; those always read are ~0
  const unsigned long long u = (unsigned long long)__double_as_longlong(x);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

__device__ __forceinline__ unsigned long long load_sys64(const unsigned long long* p) {
  return __hip_atomic_load(const_cast<unsigned long long*>(p), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_SYSTEM);
}

// Sum over the 256 threads of the values before this one's, and of all.
__device__ __forceinline__ int scan256(int v, int* s_scan, int* total) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63) s_scan[wave] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) before += s_scan[w];
    all += s_scan[w];
  }
  *total = all;
  return before + x - v;
}

template <int NG>
__global__ __launch_bounds__(256) void kv4_select_kernel(Kv4SelArgs a) {
  constexpr int D = 32 * NG, L = D / 4, PW = 64 / L;   // lanes per page, pages per wave step
  extern __shared__ unsigned long long s_key[];
  __shared__ int s_hist[256], s_scan[4], s_pick[2];
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
    for (int g = 0; g < a.group; ++g) {
      const u32x4_t x = *(const u32x4_t*)(a.q + (int64_t)b * a.q_stride + (h * a.group + g) * D + ch);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float f = (i & 1) ? bf16hi(x[i >> 1]) : bf16lo(x[i >> 1]);
        if (f != f || (f > 0.f) == high) w[i] += (double)f;   // a zero adds nothing to either
      }
    }
    for (int p = part * kSelPages + wave * PW + lane / L; p < (part + 1) * kSelPages; p += 4 * PW) {
      double s = 0;
      const int id = p < np ? kv4_page(a.c, b, p) : -1;
      if (id >= 0) {
        const uint8_t* at = a.c.pages + (int64_t)id * a.c.page_stride +
                            (int64_t)h * kv4_head_bytes(a.c.page_len, D) +
                            a.c.tiles * kv4_tile_bytes(D) + sub * 16;
        const u32x4_t x = *(const u32x4_t*)at;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          s = fma(w[i], (double)((i & 1) ? bf16hi(x[i >> 1]) : bf16lo(x[i >> 1])), s);
      }
#pragma unroll
      for (int o = 1; o < L; o <<= 1) s += __shfl_xor(s, o);
      if (sub == 0 && p < np) {
        const bool always = p < a.n_first || p >= np - a.n_last || id < 0;
        __hip_atomic_store(keys + p, always ? ~0ull : f64_key(s), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_SYSTEM);
      }
    }
  }
  wait_vm();
  __syncthreads();
  if (tid == 0) s_last = ticket(&a.counters[bk], a.parts) ? 1 : 0;
  __syncthreads();
  if (!s_last) return;

  // ---- the last part to arrive: the n_sel greatest keys, the lowest page first among equals
  int32_t* out = a.sel + (size_t)bk * a.n_sel;
  for (int e = min(np, a.n_sel) + tid; e < a.n_sel; e += 256) out[e] = -1;
  if (np <= a.n_sel) {
    for (int e = tid; e < np; e += 256) out[e] = e;
    return;
  }
  for (int e = tid; e < np; e += 256) s_key[e] = load_sys64(keys + e);
  // digit by digit from the top: the digit at which the n_sel-th key lies, until a whole bucket fits
  unsigned long long prefix = 0;
  int want = a.n_sel, shift = 64;
  bool whole = false;
  while (shift > 0 && !whole) {
    shift -= 8;
    s_hist[tid] = 0;
    __syncthreads();
    for (int e = tid; e < np; e += 256) {
      const unsigned long long k = s_key[e];
      if (shift == 56 || (k >> (shift + 8)) == prefix) atomicAdd(&s_hist[(int)(k >> shift) & 255], 1);
    }
    __syncthreads();
    int all;
    const int mine = s_hist[255 - tid];
    const int above = scan256(mine, s_scan, &all);   // keys of greater digits
    if (above < want && above + mine >= want) {
      s_pick[0] = 255 - tid;
      s_pick[1] = above;
    }
    __syncthreads();
    prefix = (prefix << 8) | (unsigned)s_pick[0];
    want -= s_pick[1];
    whole = s_hist[s_pick[0]] == want;
    __syncthreads();
  }
  // pages in order: a thread's run of them, what lies before it by a sum over the threads
  const int seg = (np + 255) / 256, e0 = tid * seg, e1 = min(np, e0 + seg);
  int gt = 0, eq = 0, all;
  for (int e = e0; e < e1; ++e) {
    const unsigned long long k = s_key[e] >> shift;
    gt += k > prefix;
    eq += k == prefix;
  }
  int g0 = scan256(gt, s_scan, &all);
  int q0 = scan256(eq, s_scan, &all);
  for (int e = e0; e < e1; ++e) {
    const unsigned long long k = s_key[e] >> shift;
    if (k > prefix || (k == prefix && q0 < want)) out[g0 + min(q0, want)] = e;
    g0 += k > prefix;
    q0 += k == prefix;
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
    hipLaunchKernelGGL(kv4_select_kernel<2>, grid, dim3(256), lds, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(kv4_select_kernel<4>, grid, dim3(256), lds, (hipStream_t)stream, a);
  return check_launch(what);
}

}  // extern "C"
