// Pages of the 4-bit K/V cache: taking free ones, sharing and copying them when a sequence goes on
// from another's prefix, giving them back, and moving the live ones together.
//
// refs[p] is how many table entries name page p; a page is free when it is 0. A sequence's row holds
// its pages from the front and -1 behind them. Which page goes where is decided by one workgroup (the
// k-th free page for the k-th that is wanted, a prefix sum over refs), so results do not hang on the
// order of atomics; the second launch moves bytes and rewrites tables over the whole chip, 16 bytes a
// lane, and is bound by memory. Fork of 8 sequences of up to 1000 positions in 40 layers: 5.5 us to decide,
// 7.1 to copy 13.8 MB; compact: 3.5 to decide, 45 to move 103 MB (4.5 TB/s read and written). reserve and free
// together: all 8 x 1024 pages 18.5 us, 256 x 64 29, 2000 x 16 62; a reserve that finds nothing to do 4 to 8.
#include "kv4.h"

namespace q4nx {

constexpr int kPlan = 1024;       // threads of the deciding workgroup
constexpr int kMoveBytes = 16384; // bytes of a page that a workgroup copies at a time

struct Kv4PoolArgs {
  Kv4 c;
  int64_t layer_stride;
  int n_layers, page_bytes;
  int32_t* lens;
  int32_t* refs;
  const int32_t* src;
  const int32_t* dst;
  const int32_t* want;
  int n;
  int32_t* live;     // compact: pages in use
  int32_t* status;
  int32_t* list;     // workspace: see each kernel
};

// Values of the threads before this one, and of all; s_w: kPlan / 64 words.
__device__ __forceinline__ int plan_scan(int v, int* s_w, int* total) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63) s_w[wave] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlan / 64; ++w) {
    const int y = s_w[w];
    if (w < wave) before += y;
    all += y;
  }
  *total = all;
  return before + x - v;
}

// f(page, rank) for the first `need` free pages; how many there are of them.
template <typename F>
__device__ __forceinline__ int free_pages(const Kv4PoolArgs& a, int need, int* s_w, F&& f) {
  int have = 0;
  for (int p0 = 0; p0 < a.c.n_pages && have < need; p0 += 4 * kPlan) {
    const int p = p0 + 4 * (int)threadIdx.x;
    int r[4], mine = 0, all;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r[i] = p + i < a.c.n_pages ? a.refs[p + i] : 1;
      mine += r[i] == 0;
    }
    int at = have + plan_scan(mine, s_w, &all);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (r[i] == 0) {
        if (at < need) f(p + i, at);
        ++at;
      }
    have += all;
  }
  return have < need ? have : need;
}

// fork, first launch: which pairs hold, and the page that takes the copy of each one's last.
// list: [n] pages, -1 without one, -2 for a pair that is not done; then [n] free pages.
__global__ __launch_bounds__(kPlan) void kv4_fork_plan(Kv4PoolArgs a) {
  __shared__ int s_owner[8192];
  __shared__ unsigned s_src[8192 / 32];
  __shared__ int s_w[kPlan / 64], s_bad;
  const int tid = threadIdx.x;
  for (int e = tid; e < a.c.n_seqs; e += kPlan) s_owner[e] = 0x7FFFFFFF;
  for (int e = tid; e < 8192 / 32; e += kPlan) s_src[e] = 0;
  if (tid == 0) s_bad = 0;
  __syncthreads();
  for (int i = tid; i < a.n; i += kPlan) {
    const int s = a.src[i], d = a.dst[i];
    if (s < 0 || s >= a.c.n_seqs || d < 0 || d >= a.c.n_seqs) continue;
    atomicMin(&s_owner[d], i);
    atomicOr(&s_src[s >> 5], 1u << (s & 31));
  }
  __syncthreads();
  int need = 0, bad = 0;
  for (int i0 = 0; i0 < a.n; i0 += kPlan) {   // a pair's rank among those that need a page
    const int i = i0 + tid;
    int state = -2;
    if (i < a.n) {
      const int s = a.src[i], d = a.dst[i];
      if (s >= 0 && s < a.c.n_seqs && d >= 0 && d < a.c.n_seqs && s_owner[d] == i &&
          !((s_src[d >> 5] >> (d & 31)) & 1) && a.c.table[(int64_t)d * a.c.table_stride] < 0) {
        // rows hold their pages from the front: with its last one a source has all that its length needs
        const int len = max(0, min(a.lens[s], a.c.cap));
        if (len == 0 || kv4_page(a.c, s, (len - 1) / a.c.page_len) >= 0)
          state = len % a.c.page_len == 0 ? -1 : 0;
      }
      bad += state == -2;
    }
    int all;
    const int rank = need + plan_scan(state == 0, s_w, &all);
    if (i < a.n) a.list[i] = state == 0 ? rank : state;
    need += all;
  }
  int32_t* fresh = a.list + a.n;
  const int have = free_pages(a, need, s_w, [&](int page, int rank) { fresh[rank] = page; });
  __threadfence_block();
  __syncthreads();
  for (int i = tid; i < a.n; i += kPlan) {
    const int rank = a.list[i];
    if (rank < 0) continue;
    if (rank < have) a.list[i] = fresh[rank];
    else {
      a.list[i] = -2;
      ++bad;
    }
  }
  if (bad) atomicAdd(&s_bad, bad);
  __syncthreads();
  if (tid == 0 && a.status) *a.status = s_bad;
}

// Copies one kMoveBytes piece of a page of one layer.
__device__ __forceinline__ void move_piece(const Kv4PoolArgs& a, int from, int to, int layer,
                                           int piece) {
  const uint8_t* s = a.c.pages + layer * a.layer_stride + (int64_t)from * a.c.page_stride;
  uint8_t* d = a.c.pages + layer * a.layer_stride + (int64_t)to * a.c.page_stride;
  const int o0 = piece * kMoveBytes + (int)threadIdx.x * 16;
  u32x4_t x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (o0 + i * 4096 < a.page_bytes) x[i] = *(const u32x4_t*)(s + o0 + i * 4096);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (o0 + i * 4096 < a.page_bytes) *(u32x4_t*)(d + o0 + i * 4096) = x[i];
}
static int move_pieces(int page_bytes) { return (page_bytes + kMoveBytes - 1) / kMoveBytes; }

// fork, second launch: workgroups [0, n) a pair's table row, the others a piece of its last page.
__global__ __launch_bounds__(256) void kv4_fork_move(Kv4PoolArgs a, int pieces) {
  const int tid = threadIdx.x;
  if ((int)blockIdx.x < a.n) {
    const int i = blockIdx.x, fresh = a.list[i];
    if (fresh == -2) return;
    const int s = a.src[i], d = a.dst[i];
    const int len = max(0, min(a.lens[s], a.c.cap)), full = len / a.c.page_len;
    const int32_t* from = a.c.table + (int64_t)s * a.c.table_stride;
    int32_t* to = a.c.table + (int64_t)d * a.c.table_stride;
    for (int j = tid; j < a.c.table_len; j += 256) {
      int id = -1;
      if (j < full) {
        id = from[j];
        if (id >= 0 && id < a.c.n_pages) atomicAdd(&a.refs[id], 1);
      } else if (j == full) {
        id = fresh;
        if (fresh >= 0) a.refs[fresh] = 1;
      }
      to[j] = id;
    }
    if (tid == 0) a.lens[d] = len;
    return;
  }
  const int w = blockIdx.x - a.n, piece = w % pieces, layer = w / pieces % a.n_layers;
  const int i = w / pieces / a.n_layers, fresh = a.list[i];
  if (fresh < 0) return;
  const int s = a.src[i];
  const int full = max(0, min(a.lens[s], a.c.cap)) / a.c.page_len;
  const int id = kv4_page(a.c, s, full);
  if (id >= 0) move_piece(a, id, fresh, layer, piece);
}

// free: a sequence's entries given back; whoever takes an entry out counts it down, so a sequence
// named twice is freed once.
__global__ __launch_bounds__(256) void kv4_free_kernel(Kv4PoolArgs a) {
  const int tid = threadIdx.x;
  if (blockIdx.x == 0 && blockIdx.y == 0 && a.status) {
    __shared__ int s_bad;
    if (tid == 0) s_bad = 0;
    __syncthreads();
    int bad = 0;
    for (int i = tid; i < a.n; i += 256) bad += a.src[i] < 0 || a.src[i] >= a.c.n_seqs;
    if (bad) atomicAdd(&s_bad, bad);
    __syncthreads();
    if (tid == 0) *a.status = s_bad;
  }
  const int s = a.src[blockIdx.x];
  if (s < 0 || s >= a.c.n_seqs) return;
  int32_t* row = a.c.table + (int64_t)s * a.c.table_stride;
  for (int j = blockIdx.y * 256 + tid; j < a.c.table_len; j += gridDim.y * 256) {
    if (row[j] < 0) continue;
    const int id = atomicExch(&row[j], -1);
    if (id >= 0 && id < a.c.n_pages) atomicSub(&a.refs[id], 1);
  }
  if (blockIdx.y == 0 && tid == 0) a.lens[s] = 0;
}

// reserve: pages for want[b] positions of every sequence. list: [table entries] free pages.
__global__ __launch_bounds__(kPlan) void kv4_reserve_kernel(Kv4PoolArgs a) {
  __shared__ int s_at[8192];      // pages wanted by the sequences up to and with b
  __shared__ int s_have[8192];    // pages b has
  __shared__ int s_w[kPlan / 64], s_bad;
  const int tid = threadIdx.x;
  if (tid == 0) s_bad = 0;
  __syncthreads();   // before any wave counts
  int need = 0;
  for (int b0 = 0; b0 < a.c.n_seqs; b0 += kPlan) {
    const int b = b0 + tid;
    int wants = 0, have = 0;
    if (b < a.c.n_seqs) {
      const int32_t* row = a.c.table + (int64_t)b * a.c.table_stride;
      int hi = a.c.table_len;   // the first entry without a page lies in [have, hi]
      while (have < hi) {
        const int mid = (have + hi) >> 1;
        if (row[mid] >= 0) have = mid + 1;
        else hi = mid;
      }
      const int64_t w = max(0, a.want[b]);
      const int64_t pages = (w + a.c.page_len - 1) / a.c.page_len;
      // more than the row holds: counted as not done, nothing is taken
      wants = pages > a.c.table_len ? 0 : max(0, (int)pages - have);
      if (pages > a.c.table_len) atomicAdd(&s_bad, 1);
    }
    int all;
    const int before = need + plan_scan(wants, s_w, &all);
    if (b < a.c.n_seqs) {
      s_at[b] = before + wants;
      s_have[b] = have;
    }
    need += all;
  }
  __syncthreads();
  const int limit = min(need, a.c.n_pages);
  const int have = free_pages(a, limit, s_w, [&](int page, int rank) { a.list[rank] = page; });
  __threadfence_block();
  __syncthreads();
  // a sequence gets all its pages or none
  for (int b = tid; b < a.c.n_seqs; b += kPlan) {
    const int from = b ? s_at[b - 1] : 0;
    if (s_at[b] > from && s_at[b] > have) atomicAdd(&s_bad, 1);
  }
  for (int r = tid; r < have; r += kPlan) {
    int lo = 0, hi = a.c.n_seqs - 1;   // the first sequence with s_at > r
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (s_at[mid] > r) hi = mid;
      else lo = mid + 1;
    }
    if (s_at[lo] > have) continue;
    const int page = a.list[r];
    a.c.table[(int64_t)lo * a.c.table_stride + s_have[lo] + r - (lo ? s_at[lo - 1] : 0)] = page;
    a.refs[page] = 1;
  }
  __syncthreads();
  if (tid == 0 && a.status) *a.status = s_bad;
}

// compact, first launch: the i-th free page below the count of live ones takes the i-th live page at
// or behind it. list: [0] moves; then [n_pages] from, [n_pages] to, [n_pages] where a page goes.
__global__ __launch_bounds__(kPlan) void kv4_compact_plan(Kv4PoolArgs a) {
  __shared__ int s_w[kPlan / 64];
  const int tid = threadIdx.x, np = a.c.n_pages;
  int mine = 0, live;
  for (int p = tid; p < np; p += kPlan) mine += a.refs[p] > 0;
  plan_scan(mine, s_w, &live);
  int32_t* from = a.list + 1;
  int32_t* to = from + np;
  int32_t* map = to + np;
  int holes = 0, movers = 0;
  for (int p0 = 0; p0 < np; p0 += kPlan) {
    const int p = p0 + tid;
    const bool used = p < np && a.refs[p] > 0;
    int all;
    if (p0 < live) {
      const int hole = p < live && !used;
      const int at = holes + plan_scan(hole, s_w, &all);
      if (hole) to[at] = p;
      holes += all;
    }
    if (p0 + kPlan > live) {
      const int mover = p >= live && used;
      const int at = movers + plan_scan(mover, s_w, &all);
      if (mover) from[at] = p;
      if (p < np) map[p] = p;   // an entry that names a page nothing counts stays as it is
      movers += all;
    }
  }
  __threadfence_block();
  __syncthreads();
  for (int i = tid; i < movers; i += kPlan) map[from[i]] = to[i];
  if (tid == 0) {
    a.list[0] = movers;
    if (a.live) *a.live = live;
  }
}

// compact, second launch: pages, counts and table entries, each over the whole grid.
__global__ __launch_bounds__(256) void kv4_compact_move(Kv4PoolArgs a, int pieces) {
  const int np = a.c.n_pages, moves = a.list[0], tid = threadIdx.x;
  const int32_t* from = a.list + 1;
  const int32_t* to = from + np;
  const int32_t* map = to + np;
  const int64_t work = (int64_t)moves * a.n_layers * pieces;
  for (int64_t w = blockIdx.x; w < work; w += gridDim.x) {
    const int piece = (int)(w % pieces), layer = (int)(w / pieces % a.n_layers);
    const int i = (int)(w / pieces / a.n_layers);
    move_piece(a, from[i], to[i], layer, piece);
  }
  for (int i = blockIdx.x * 256 + tid; i < moves; i += gridDim.x * 256) {
    a.refs[to[i]] = a.refs[from[i]];
    a.refs[from[i]] = 0;
  }
  if (moves == 0) return;
  // entries behind the live pages are the ones that moved: those that name a page before the first
  // mover stay
  const int64_t entries = (int64_t)a.c.n_seqs * a.c.table_len;
  const int first = from[0];
  for (int64_t e = (int64_t)blockIdx.x * 256 + tid; e < entries; e += (int64_t)gridDim.x * 256) {
    int32_t* x = a.c.table + e / a.c.table_len * a.c.table_stride + e % a.c.table_len;
    const int id = *x;
    if (id >= first && id < np) *x = map[id];
  }
}

__global__ __launch_bounds__(256) void kv4_copy_kernel(Kv4PoolArgs a, int pieces) {
  const int w = blockIdx.x, piece = w % pieces, layer = w / pieces % a.n_layers;
  const int i = w / pieces / a.n_layers;
  const int s = a.src[i], d = a.dst[i];
  if (s < 0 || s >= a.c.n_pages || d < 0 || d >= a.c.n_pages || s == d) return;
  move_piece(a, s, d, layer, piece);
}

static int kv4_pool_resolve(const q4nx_kv4* cache, int64_t layer_stride, int n_layers,
                            Kv4PoolArgs* a, const char* what) {
  if (int rc = kv4_resolve(cache, &a->c, what)) return rc;
  a->page_bytes = cache->n_kv_heads * kv4_head_bytes(cache->page_len, cache->head_dim);
  Q4NX_REQUIRE(n_layers >= 1 && n_layers <= 65536 && layer_stride % 16 == 0 &&
                   (n_layers == 1 || layer_stride >= a->page_bytes ||
                    layer_stride <= -(int64_t)a->page_bytes),
               Q4NX_ERR_SHAPE, "%s: n_layers=%d, layer_stride=%lld", what, n_layers,
               (long long)layer_stride);
  a->layer_stride = layer_stride;
  a->n_layers = n_layers;
  return Q4NX_OK;
}

static int kv4_need_ws(const char* what, const void* ws, size_t ws_bytes, size_t need) {
  Q4NX_REQUIRE(ws != nullptr && ws_bytes >= need && Q4NX_ALIGNED(ws, 256), Q4NX_ERR_WS,
               "%s: workspace of %zu bytes (256-aligned) needed, %zu given", what, need, ws_bytes);
  return Q4NX_OK;
}

}  // namespace q4nx

using namespace q4nx;

extern "C" {

size_t q4nx_kv4_pages_ws_bytes(const q4nx_kv4* cache, int n) {
  Kv4 c;
  if (kv4_resolve(cache, &c, "q4nx_kv4_pages_ws_bytes") != Q4NX_OK || n < 0) return 0;
  const size_t by_pages = (size_t)c.n_pages * 3 + 1, by_pairs = (size_t)n * 2;
  return Q4NX_WS_COUNTER_BYTES + 4 * (by_pages > by_pairs ? by_pages : by_pairs);
}

int q4nx_kv4_reserve(const q4nx_kv4* cache, int32_t* refs, const int32_t* want, int32_t* status,
                     void* ws, size_t ws_bytes, void* stream) {
  const char* what = "q4nx_kv4_reserve";
  Kv4PoolArgs a{};
  if (int rc = kv4_pool_resolve(cache, 0, 1, &a, what)) return rc;
  Q4NX_REQUIRE(refs && want, Q4NX_ERR_ARG, "%s: refs and want are required", what);
  Q4NX_REQUIRE((int64_t)cache->n_seqs * ((int64_t)cache->n_pages + 1) < (int64_t)1 << 31 &&
                   (int64_t)cache->n_seqs * cache->table_len < (int64_t)1 << 31,
               Q4NX_ERR_SHAPE, "%s: %d sequences of %d pages", what, cache->n_seqs, cache->n_pages);
  if (int rc = kv4_need_ws(what, ws, ws_bytes, q4nx_kv4_pages_ws_bytes(cache, 0))) return rc;
  a.refs = refs;
  a.want = want;
  a.status = status;
  a.list = (int32_t*)((uint8_t*)ws + Q4NX_WS_COUNTER_BYTES);
  hipLaunchKernelGGL(kv4_reserve_kernel, dim3(1), dim3(kPlan), 0, (hipStream_t)stream, a);
  return check_launch(what);
}

int q4nx_kv4_fork(const q4nx_kv4* cache, int64_t layer_stride, int n_layers, int32_t* lens,
                  int32_t* refs, const int32_t* src, const int32_t* dst, int n, int32_t* status,
                  void* ws, size_t ws_bytes, void* stream) {
  const char* what = "q4nx_kv4_fork";
  Kv4PoolArgs a{};
  if (int rc = kv4_pool_resolve(cache, layer_stride, n_layers, &a, what)) return rc;
  Q4NX_REQUIRE(lens && refs && src && dst, Q4NX_ERR_ARG, "%s: lens, refs, src and dst are required",
               what);
  Q4NX_REQUIRE(n >= 1 && n <= cache->n_seqs, Q4NX_ERR_SHAPE, "%s: n=%d pairs of %d sequences", what, n,
               cache->n_seqs);
  if (int rc = kv4_need_ws(what, ws, ws_bytes, q4nx_kv4_pages_ws_bytes(cache, n))) return rc;
  const int pieces = move_pieces(a.page_bytes);
  const int64_t grid = n + (int64_t)n * n_layers * pieces;
  Q4NX_REQUIRE(grid <= (int64_t)1 << 30, Q4NX_ERR_SHAPE, "%s: %lld workgroups", what, (long long)grid);
  a.lens = lens;
  a.refs = refs;
  a.src = src;
  a.dst = dst;
  a.n = n;
  a.status = status;
  a.list = (int32_t*)((uint8_t*)ws + Q4NX_WS_COUNTER_BYTES);
  hipLaunchKernelGGL(kv4_fork_plan, dim3(1), dim3(kPlan), 0, (hipStream_t)stream, a);
  hipLaunchKernelGGL(kv4_fork_move, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, a, pieces);
  return check_launch(what);
}

int q4nx_kv4_free(const q4nx_kv4* cache, int32_t* lens, int32_t* refs, const int32_t* seqs, int n,
                  int32_t* status, void* stream) {
  const char* what = "q4nx_kv4_free";
  Kv4PoolArgs a{};
  if (int rc = kv4_pool_resolve(cache, 0, 1, &a, what)) return rc;
  Q4NX_REQUIRE(lens && refs && seqs, Q4NX_ERR_ARG, "%s: lens, refs and seqs are required", what);
  Q4NX_REQUIRE(n >= 1 && n <= cache->n_seqs, Q4NX_ERR_SHAPE, "%s: n=%d of %d sequences", what, n,
               cache->n_seqs);
  a.lens = lens;
  a.refs = refs;
  a.src = seqs;
  a.n = n;
  a.status = status;
  const unsigned parts = (unsigned)((cache->table_len + 1023) / 1024);
  hipLaunchKernelGGL(kv4_free_kernel, dim3((unsigned)n, parts > 64 ? 64 : parts), dim3(256), 0,
                     (hipStream_t)stream, a);
  return check_launch(what);
}

int q4nx_kv4_compact(const q4nx_kv4* cache, int64_t layer_stride, int n_layers, int32_t* refs,
                     int32_t* live, void* ws, size_t ws_bytes, void* stream) {
  const char* what = "q4nx_kv4_compact";
  Kv4PoolArgs a{};
  if (int rc = kv4_pool_resolve(cache, layer_stride, n_layers, &a, what)) return rc;
  Q4NX_REQUIRE(refs, Q4NX_ERR_ARG, "%s: refs are required", what);
  if (int rc = kv4_need_ws(what, ws, ws_bytes, q4nx_kv4_pages_ws_bytes(cache, 0))) return rc;
  a.refs = refs;
  a.live = live;
  a.list = (int32_t*)((uint8_t*)ws + Q4NX_WS_COUNTER_BYTES);
  const int pieces = move_pieces(a.page_bytes);
  const int64_t most = (int64_t)(cache->n_pages + 1) / 2 * n_layers * pieces;
  const unsigned grid = (unsigned)(most < 2048 ? most : 2048);
  hipLaunchKernelGGL(kv4_compact_plan, dim3(1), dim3(kPlan), 0, (hipStream_t)stream, a);
  hipLaunchKernelGGL(kv4_compact_move, dim3(grid), dim3(256), 0, (hipStream_t)stream, a, pieces);
  return check_launch(what);
}

int q4nx_kv4_copy_pages(const q4nx_kv4* cache, int64_t layer_stride, int n_layers,
                        const int32_t* src_pages, const int32_t* dst_pages, int n, void* stream) {
  const char* what = "q4nx_kv4_copy_pages";
  Kv4PoolArgs a{};
  if (int rc = kv4_pool_resolve(cache, layer_stride, n_layers, &a, what)) return rc;
  Q4NX_REQUIRE(src_pages && dst_pages, Q4NX_ERR_ARG, "%s: src_pages and dst_pages are required", what);
  const int pieces = move_pieces(a.page_bytes);
  Q4NX_REQUIRE(n >= 1 && (int64_t)n * n_layers * pieces <= (int64_t)1 << 30, Q4NX_ERR_SHAPE,
               "%s: n=%d pages of %d layers", what, n, n_layers);
  a.src = src_pages;
  a.dst = dst_pages;
  a.n = n;
  hipLaunchKernelGGL(kv4_copy_kernel, dim3((unsigned)(n * n_layers * pieces)), dim3(256), 0,
                     (hipStream_t)stream, a, pieces);
  return check_launch(what);
}

}  // extern "C"
