// Rows into and out of the paged 4-bit K/V cache.
//
// One workgroup is one page of one (sequence, kv head), one wave a tile of 32 positions; nothing
// outside its tile is written by a wave, so the nibbles that old and new positions share in a
// dword of V are merged by one lane. Lane (n, kg) holds channels 8 kg .. 8 kg + 7 of every group of
// 32 at positions n and 16 + n: a group's least and greatest value are eight values in the lane and
// two lane swaps (16, 32), and K's dword is made where it is stored. V's dwords run along
// positions: its codes go through LDS as bytes.
#include <math.h>

#include "kv4.h"

namespace q4nx {

struct Kv4RowArgs {
  Kv4 c;
  const uint16_t* k;
  const uint16_t* v;
  void* k_out;
  void* v_out;
  int64_t row_stride, head_stride, seq_stride, src_rows;
  int by_position, out_f32;
  const int32_t* pos;
  const int32_t* cu;
};

__device__ __forceinline__ uint32_t xor16_u(uint32_t v, bool mx) {
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return mx ? max(r[0], r[1]) : min(r[0], r[1]);
}
__device__ __forceinline__ uint32_t xor32_u(uint32_t v, bool mx) {
  const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return mx ? max(r[0], r[1]) : min(r[0], r[1]);
}

// What a (sequence, page) of a call covers: its new positions are [first, last).
struct Kv4Span {
  int page, b, h, first, last;
  int64_t src0;   // the source row of position p is src0 + p
};
__device__ __forceinline__ bool kv4_span(const Kv4RowArgs& a, Kv4Span* s) {
  s->h = blockIdx.x % a.c.hkv;
  s->b = blockIdx.x / a.c.hkv;
  const int64_t p0 = a.pos[s->b];
  int64_t c0 = s->b, n = 1;
  if (a.cu) {
    c0 = a.cu[s->b];
    n = (int64_t)a.cu[s->b + 1] - c0;
  }
  int64_t lo = p0, hi = p0 + n;
  s->src0 = a.by_position ? 0 : c0 - p0;
  // rows that the other side does not have; positions that the table does not have are not written
  // (and read as NaN)
  if (lo < -s->src0) lo = -s->src0;
  if (hi > a.src_rows - s->src0) hi = a.src_rows - s->src0;
  const int64_t floor = a.k_out ? -(int64_t)0x7FFFFF00 : 0, ceil = a.k_out ? 0x7FFFFF00 : a.c.cap;
  if (lo < floor) lo = floor;
  if (hi > ceil) hi = ceil;
  if (hi <= lo) return false;
  const int64_t lp0 = (lo - (lo < 0 ? a.c.page_len - 1 : 0)) / a.c.page_len;
  const int64_t lp = lp0 + blockIdx.y, base = lp * a.c.page_len;
  if (base >= hi) return false;
  s->first = (int)(lo > base ? lo : base);
  s->last = (int)(hi < base + a.c.page_len ? hi : base + a.c.page_len);
  s->page = (int)lp;
  return true;
}

struct Kv4Group {   // one group of one row: this lane's eight codes, a nibble each, and (d, m)
  uint32_t lo, hi;  // codes of channels 0..3 and 4..7, a byte each
  uint32_t dm;
  bool bad;
};

// Quantises the group of 32 channels whose eight values (packed bf16) are in lanes kg = 0..3.
__device__ __forceinline__ Kv4Group kv4_quant(const u32x4_t& x) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = bf16lo(x[i]);
    f[2 * i + 1] = bf16hi(x[i]);
  }
  float lo = f[0], hi = f[0];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, f[i]);
    hi = fmaxf(hi, f[i]);
    top = max(top, __float_as_uint(f[i]) & 0x7FFFFFFFu);
  }
  lo = -xor32_max(xor16_max(-lo));
  hi = xor32_max(xor16_max(hi));
  top = xor32_u(xor16_u(top, true), true);
  const float d = round_bf16_op((hi - lo) / 15.0f);
  Kv4Group r;
  r.bad = top >= 0x7F800000u || !(d < INFINITY);
  r.lo = r.hi = 0;
  if (d > 0.f && !r.bad) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float q = fminf(rintf((f[i] - lo) / d), 15.0f);
      (i < 4 ? r.lo : r.hi) |= (uint32_t)q << (8 * (i & 3));
    }
  }
  r.dm = r.bad ? kKv4NaN : (__float_as_uint(d) >> 16) | (__float_as_uint(lo) & 0xFFFF0000u);
  return r;
}

// bytes b0..b7 (codes of channels 0..7) -> K's dword: nibbles 0, 2, 4, 6, 1, 3, 5, 7
__device__ __forceinline__ uint32_t kv4_kdword(uint32_t lo, uint32_t hi) {
  const uint32_t even = (lo & 0xFu) | ((lo >> 12) & 0xF0u) | ((hi & 0xFu) << 8) | ((hi >> 4) & 0xF000u);
  const uint32_t l1 = lo >> 8, h1 = hi >> 8;
  const uint32_t odd = (l1 & 0xFu) | ((l1 >> 12) & 0xF0u) | ((h1 & 0xFu) << 8) | ((h1 >> 4) & 0xF000u);
  return even | (odd << 16);
}

__device__ __forceinline__ float bound_min(float a, float b) {
  return a != a ? a : (b != b ? b : fminf(a, b));
}
__device__ __forceinline__ float bound_max(float a, float b) {
  return a != a ? a : (b != b ? b : fmaxf(a, b));
}

template <int NG>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4RowArgs a) {
  constexpr int D = 32 * NG, C = D / 64;
  __shared__ __attribute__((aligned(16))) uint8_t s_v[4][32][D + 8];
  __shared__ float s_b[4][2][D];
  Kv4Span s;
  if (!kv4_span(a, &s)) return;   // uniform over the workgroup
  const int id = kv4_page(a.c, s.b, s.page);
  if (id < 0) return;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, kg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int base = s.page * a.c.page_len + wave * kKv4Tile;
  uint8_t* head = a.c.pages + (int64_t)id * a.c.page_stride +
                  (int64_t)s.h * kv4_head_bytes(a.c.page_len, D);
  uint8_t* tile = head + wave * kv4_tile_bytes(D);
  const int t0 = max(s.first - base, 0), t1 = min(s.last - base, kKv4Tile);   // new: [t0, t1)
  const int64_t src = (a.by_position ? s.b * a.seq_stride : 0) + s.h * a.head_stride;

  // ---- K: codes, scales, and the bounds of each channel over the tile's new positions
  float lo[NG][8], hi[NG][8];
  uint32_t bad = 0;
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lo[g][i] = INFINITY;
      hi[g][i] = -INFINITY;
    }
  u32x4_t kx[2][NG], vx[2][NG];
#pragma unroll
  for (int tt = 0; tt < 2; ++tt) {
    const int t = 16 * tt + n;
    const bool now = t >= t0 && t < t1;
    // a row of the span for the lanes that have none: its values are not used
    const int64_t row = src + (s.src0 + (now ? base + t : s.first)) * a.row_stride;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      kx[tt][g] = *(const u32x4_t*)(a.k + row + 32 * g + 8 * kg);
      vx[tt][g] = *(const u32x4_t*)(a.v + row + 32 * g + 8 * kg);
    }
  }
  if (t0 < t1) {
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      const int t = 16 * tt + n;
      const bool now = t >= t0 && t < t1;
      uint32_t w[NG];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const Kv4Group q = kv4_quant(kx[tt][g]);
        w[g] = kv4_kdword(q.lo, q.hi);
        if (now) {
          if (kg == (g & 3))
            *(uint32_t*)(tile + 32 * D + (t * NG + g) * 4) = q.dm;
          if (q.bad) bad |= 1u << g;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            lo[g][2 * i] = fminf(lo[g][2 * i], bf16lo(kx[tt][g][i]));
            hi[g][2 * i] = fmaxf(hi[g][2 * i], bf16lo(kx[tt][g][i]));
            lo[g][2 * i + 1] = fminf(lo[g][2 * i + 1], bf16hi(kx[tt][g][i]));
            hi[g][2 * i + 1] = fmaxf(hi[g][2 * i + 1], bf16hi(kx[tt][g][i]));
          }
        }
      }
      if (now) {
#pragma unroll
        for (int c = 0; c < C; ++c)
          *(uint2*)(tile + (c * 64 + lane) * 16 + 8 * tt) = make_uint2(w[2 * c], w[2 * c + 1]);
      }
    }
    // ---- V: codes as bytes through LDS, then a dword per channel and eight positions
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      const int t = 16 * tt + n;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const Kv4Group q = kv4_quant(vx[tt][g]);
        if (t >= t0 && t < t1 && kg == (g & 3))
          *(uint32_t*)(tile + 32 * D + (32 * NG + t * NG + g) * 4) = q.dm;
        *(uint2*)&s_v[wave][t][32 * g + 8 * kg] = make_uint2(q.lo, q.hi);
      }
    }
  }
  // the channel bounds over the 16 positions of a row of lanes, one lane's word per channel
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const bool any_bad = __any((bad >> g) & 1);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float l = -group16_max(-lo[g][i]), h = group16_max(hi[g][i]);
      if (n == i) {
        s_b[wave][0][32 * g + 8 * kg + i] = any_bad ? NAN : l;
        s_b[wave][1][32 * g + 8 * kg + i] = any_bad ? NAN : h;
      }
    }
  }
  __syncthreads();
  if (t0 < t1) {
    uint32_t keep = 0;   // nibbles of positions that are not new
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int t = 16 * (e >> 2) + 4 * kg + (e & 3);
      if (t < t0 || t >= t1) keep |= 0xFu << (4 * e);
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      u32x4_t* dst = (u32x4_t*)(tile + 16 * D + (c * 64 + lane) * 16);
      u32x4_t w;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        uint32_t x = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          x |= (uint32_t)s_v[wave][16 * (e >> 2) + 4 * kg + (e & 3)][64 * c + 16 * t + n] << (4 * e);
        w[t] = x;
      }
      if (keep == 0xFFFFFFFFu) continue;
      if (keep) {
        const u32x4_t old = *dst;
#pragma unroll
        for (int t = 0; t < 4; ++t) w[t] = (w[t] & ~keep) | (old[t] & keep);
      }
      *dst = w;
    }
  }
  // ---- the page's bounds: of this call's rows, with the older ones' unless the page begins here
  uint16_t* bounds = (uint16_t*)(head + a.c.tiles * kv4_tile_bytes(D));
  const bool begins = s.first == s.page * a.c.page_len;
  for (int e = tid; e < 2 * D; e += (int)blockDim.x) {
    const int side = e / D, ch = e % D;
    float x = begins ? s_b[0][side][ch] : bf16_to_f32(bounds[e]);
    for (int w = begins ? 1 : 0; w < a.c.tiles; ++w)
      x = side ? bound_max(x, s_b[w][side][ch]) : bound_min(x, s_b[w][side][ch]);
    // a bf16 value: nothing is rounded
    bounds[e] = x != x ? (uint16_t)0x7FC0 : (uint16_t)(__float_as_uint(x) >> 16);
  }
}

__device__ __forceinline__ void kv4_put(void* out, int f32, int64_t at, const float (&y)[8]) {
  if (f32) {
    float4* p = (float4*)((float*)out + at);
    p[0] = make_float4(y[0], y[1], y[2], y[3]);
    p[1] = make_float4(y[4], y[5], y[6], y[7]);
  } else {
    uint4* p = (uint4*)((uint16_t*)out + at);
    *p = make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]),
                    pack_bf16x2(y[6], y[7]));
  }
}

template <int NG>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4RowArgs a) {
  constexpr int D = 32 * NG, C = D / 64;
  __shared__ __attribute__((aligned(16))) uint8_t s_v[4][32][D + 8];
  Kv4Span s;
  if (!kv4_span(a, &s)) return;
  const int id = kv4_page(a.c, s.b, s.page);   // none: the rows read as NaN
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, kg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int base = s.page * a.c.page_len + wave * kKv4Tile;
  const uint8_t* tile = a.c.pages + (int64_t)max(id, 0) * a.c.page_stride +
                        (int64_t)s.h * kv4_head_bytes(a.c.page_len, D) +
                        wave * kv4_tile_bytes(D);
  const int t0 = max(s.first - base, 0), t1 = min(s.last - base, kKv4Tile);
  u32x4_t kw[C];
  if (t0 < t1) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      kw[c] = *(const u32x4_t*)(tile + (c * 64 + lane) * 16);
      const u32x4_t vw = *(const u32x4_t*)(tile + 16 * D + (c * 64 + lane) * 16);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          s_v[wave][16 * (e >> 2) + 4 * kg + (e & 3)][64 * c + 16 * t + n] = (vw[t] >> (4 * e)) & 15;
    }
  }
  __syncthreads();
  if (t0 >= t1) return;
#pragma unroll
  for (int tt = 0; tt < 2; ++tt) {
    const int t = 16 * tt + n;
    if (t < t0 || t >= t1) continue;
    const int64_t out = ((s.src0 + base + t) * a.c.hkv + s.h) * D + 8 * kg;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      uint32_t dk = *(const uint32_t*)(tile + 32 * D + (t * NG + g) * 4);
      uint32_t dv = *(const uint32_t*)(tile + 32 * D + (32 * NG + t * NG + g) * 4);
      if (id < 0) dk = dv = kKv4NaN;
      const uint32_t w = kw[g >> 1][2 * tt + (g & 1)];
      const uint2 vb = *(const uint2*)&s_v[wave][t][32 * g + 8 * kg];
      float y[8], z[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t kc = (w >> (4 * (i >> 1) + 16 * (i & 1))) & 15u;
        const uint32_t vc = ((i < 4 ? vb.x : vb.y) >> (8 * (i & 3))) & 15u;
        y[i] = fmaf((float)kc, bf16lo(dk), bf16hi(dk));
        z[i] = fmaf((float)vc, bf16lo(dv), bf16hi(dv));
      }
      kv4_put(a.k_out, a.out_f32, out + 32 * g, y);
      kv4_put(a.v_out, a.out_f32, out + 32 * g, z);
    }
  }
}

int kv4_resolve(const q4nx_kv4* c, Kv4* out, const char* what) {
  Q4NX_REQUIRE(c != nullptr && c->pages != nullptr && c->table != nullptr, Q4NX_ERR_ARG,
               "%s: a cache with pages and a table is required", what);
  Q4NX_REQUIRE(c->head_dim == 64 || c->head_dim == 128, Q4NX_ERR_SHAPE,
               "%s: head_dim=%d, 64 and 128 are built", what, c->head_dim);
  Q4NX_REQUIRE(c->page_len == 32 || c->page_len == 64 || c->page_len == 128, Q4NX_ERR_SHAPE,
               "%s: page_len=%d, not 32, 64 or 128", what, c->page_len);
  Q4NX_REQUIRE(c->n_kv_heads >= 1 && c->n_kv_heads <= 1024 && c->n_pages >= 1 &&
                   c->n_pages <= 1 << 28,
               Q4NX_ERR_SHAPE,
               "%s: n_kv_heads=%d (1..1024), n_pages=%d (1..2^28)", what, c->n_kv_heads, c->n_pages);
  Q4NX_REQUIRE(c->n_seqs >= 1 && c->n_seqs <= 8192 && c->table_len >= 1 &&
                   c->table_stride >= c->table_len &&
                   (int64_t)c->table_len * c->page_len <= (int64_t)1 << 30,
               Q4NX_ERR_SHAPE,
               "%s: a table of %d sequences (1..8192) x %d pages (up to 2^30 positions), stride %lld",
               what, c->n_seqs, c->table_len, (long long)c->table_stride);
  const int64_t bytes = (int64_t)c->n_kv_heads * kv4_head_bytes(c->page_len, c->head_dim);
  Q4NX_REQUIRE(c->page_stride >= bytes && c->page_stride % 16 == 0 && Q4NX_ALIGNED(c->pages, 16),
               Q4NX_ERR_SHAPE,
               "%s: pages must be 16-byte aligned, page_stride=%lld a multiple of 16 of at least %lld",
               what, (long long)c->page_stride, (long long)bytes);
  *out = Kv4{c->pages, c->page_stride, c->table, c->table_stride, c->n_pages, c->page_len,
             c->page_len / kKv4Tile, c->n_kv_heads, c->n_seqs, c->table_len,
             c->table_len * c->page_len};
  return Q4NX_OK;
}

// Pages that max_new consecutive positions can touch.
static unsigned kv4_span_pages(int max_new, int page_len) {
  return (unsigned)(((int64_t)max_new + page_len - 2) / page_len + 1);
}

}  // namespace q4nx

using namespace q4nx;

extern "C" {

size_t q4nx_kv4_page_bytes(int page_len, int n_kv_heads, int head_dim) {
  if ((page_len != 32 && page_len != 64 && page_len != 128) || n_kv_heads < 1 ||
      n_kv_heads > 1024 || (head_dim != 64 && head_dim != 128))
    return 0;
  return (size_t)n_kv_heads * kv4_head_bytes(page_len, head_dim);
}

int q4nx_kv4_append(const q4nx_kv4* cache, const uint16_t* k, const uint16_t* v, int by_position,
                    int64_t src_rows, int64_t row_stride, int64_t head_stride, int64_t seq_stride,
                    const int32_t* pos, const int32_t* cu, int max_new, void* stream) {
  const char* what = "q4nx_kv4_append";
  Kv4RowArgs a{};
  if (int rc = kv4_resolve(cache, &a.c, what)) return rc;
  Q4NX_REQUIRE(k && v && pos && Q4NX_ALIGNED(k, 16) && Q4NX_ALIGNED(v, 16), Q4NX_ERR_ARG,
               "%s: k, v (16-byte aligned) and pos are required", what);
  Q4NX_REQUIRE((by_position == 0 || by_position == 1) && src_rows >= 1 && row_stride >= 0 &&
                   head_stride >= 0 && seq_stride >= 0 && row_stride % 8 == 0 &&
                   head_stride % 8 == 0 && seq_stride % 8 == 0,
               Q4NX_ERR_SHAPE,
               "%s: src_rows=%lld must be positive, strides %lld, %lld, %lld multiples of 8", what,
               (long long)src_rows, (long long)row_stride, (long long)head_stride,
               (long long)seq_stride);
  Q4NX_REQUIRE(max_new >= 1 && (cu != nullptr || max_new == 1), Q4NX_ERR_ARG,
               "%s: max_new=%d (1 where cu is NULL)", what, max_new);
  a.k = k;
  a.v = v;
  a.by_position = by_position;
  a.src_rows = src_rows;
  a.row_stride = row_stride;
  a.head_stride = head_stride;
  a.seq_stride = seq_stride;
  a.pos = pos;
  a.cu = cu;
  const dim3 grid((unsigned)(a.c.n_seqs * a.c.hkv), kv4_span_pages(max_new, a.c.page_len));
  Q4NX_REQUIRE(grid.y <= 65535, Q4NX_ERR_SHAPE, "%s: max_new=%d spans more than 65535 pages", what,
               max_new);
  const dim3 block(64 * a.c.tiles);
  if (cache->head_dim == 64)
    hipLaunchKernelGGL(kv4_append_kernel<2>, grid, block, 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(kv4_append_kernel<4>, grid, block, 0, (hipStream_t)stream, a);
  return check_launch(what);
}

int q4nx_kv4_read(const q4nx_kv4* cache, void* k_out, void* v_out, int out_f32, int64_t out_rows,
                  const int32_t* pos, const int32_t* cu, int max_new, void* stream) {
  const char* what = "q4nx_kv4_read";
  Kv4RowArgs a{};
  if (int rc = kv4_resolve(cache, &a.c, what)) return rc;
  Q4NX_REQUIRE(k_out && v_out && pos && Q4NX_ALIGNED(k_out, 16) && Q4NX_ALIGNED(v_out, 16),
               Q4NX_ERR_ARG, "%s: outputs (16-byte aligned) and pos are required", what);
  Q4NX_REQUIRE(out_rows >= 1, Q4NX_ERR_SHAPE, "%s: out_rows=%lld must be positive", what,
               (long long)out_rows);
  Q4NX_REQUIRE(max_new >= 1 && (cu != nullptr || max_new == 1), Q4NX_ERR_ARG,
               "%s: max_new=%d (1 where cu is NULL)", what, max_new);
  a.k_out = k_out;
  a.v_out = v_out;
  a.out_f32 = out_f32 != 0;
  a.src_rows = out_rows;
  a.pos = pos;
  a.cu = cu;
  const dim3 grid((unsigned)(a.c.n_seqs * a.c.hkv), kv4_span_pages(max_new, a.c.page_len));
  Q4NX_REQUIRE(grid.y <= 65535, Q4NX_ERR_SHAPE, "%s: max_new=%d spans more than 65535 pages", what,
               max_new);
  const dim3 block(64 * a.c.tiles);
  if (cache->head_dim == 64)
    hipLaunchKernelGGL(kv4_read_kernel<2>, grid, block, 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(kv4_read_kernel<4>, grid, block, 0, (hipStream_t)stream, a);
  return check_launch(what);
}

}  // extern "C"
