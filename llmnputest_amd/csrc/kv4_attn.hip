// Attention over the paged 4-bit K/V cache, on the matrix cores.
//
// A query row is (new token i, query head of the group); 16 rows are the columns of every tile.
// With x = d_g c + m_g per group g of 32 channels,
//   S^T[pos][row]  = sum_g d_g[pos] (c . q)_g + m_g[pos] (sum of q)_g
//   O^T[dim][row] += sum_pos (p d_g(dim))[pos] c[pos][dim] + sum_pos p m_g(dim)
// so the codes enter the matrix cores as they are stored, as the bf16 numbers 128 + c (exact), and
// the scales stay in fp32. The 128 is taken out exactly where it can be: the score's accumulator
// starts at -128 (sum of q)_g, and the values' sum is joined by an operand of -128s. p d_g enters as
// two bf16 terms, which carry it to 2^-17.
#include <math.h>

#include "kv4.h"

namespace q4nx {

struct Kv4AttnArgs {
  Kv4 c;
  const uint16_t* q;
  int64_t q_stride;
  uint16_t* out;
  float* out_f32;
  const int32_t* cu;
  const int32_t* lens;
  const int32_t* sel;
  int n_sel, hq, group, total, row_tiles, n_split;
  float scale_l2;
  float* partial;
  uint32_t partial_bytes;
  unsigned* counters;
};

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

constexpr int kWaves = 4;

template <int NG>
__global__ __launch_bounds__(256) void kv4_attn_kernel(Kv4AttnArgs a) {
  constexpr int D = 32 * NG, C = D / 64, NT = D / 16, REC = D + 4;
  __shared__ __attribute__((aligned(16))) float s_o[kWaves][16][REC];
  __shared__ __attribute__((aligned(16))) float s_fin[16][REC];
  __shared__ int s_last;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, kg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int split = blockIdx.x % a.n_split;
  const int bk = blockIdx.x / a.n_split;        // (b * hkv + h) * row_tiles + rt
  const int rt = bk % a.row_tiles;
  const int h = (bk / a.row_tiles) % a.c.hkv;
  const int b = bk / a.row_tiles / a.c.hkv;
  int c0 = b, nq = 1;
  if (a.cu) {
    c0 = a.cu[b];
    nq = a.cu[b + 1] - c0;
    if (c0 < 0 || nq < 0) nq = 0;
    nq = min(nq, a.total - c0);
  }
  const int rows = nq * a.group;
  if (rt * 16 >= rows) return;   // uniform, and in every split of it
  const int row = rt * 16 + n;
  const bool live = row < rows;
  const int tok = live ? row / a.group : 0, qh = live ? row % a.group : 0;
  const int end = live ? max(0, min(a.lens[b] - nq + tok + 1, a.c.cap)) : 0;   // positions this row sees
  const int top = max(0, min(a.lens[b] - nq + min(rt * 16 + 15, rows - 1) / a.group + 1, a.c.cap));

  // q, and its sums by group
  u32x4_t q[NG];
  float qs[NG];
  {
    const uint16_t* p = a.q + (int64_t)(c0 + tok) * a.q_stride + (h * a.group + qh) * D + 8 * kg;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      q[g] = live ? *(const u32x4_t*)(p + 32 * g) : u32x4_t{0, 0, 0, 0};
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) s += bf16lo(q[g][i]) + bf16hi(q[g][i]);
      qs[g] = xor32_sum(xor16_sum(s));
    }
  }
  f32x4_t o[NT], off[NG];
  float ms[NG], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int u = 0; u < NT; ++u) o[u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    off[g] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    ms[g] = 0.f;
  }
  const u32x4_t minus = {0xC300C300u, 0xC300C300u, 0xC300C300u, 0xC300C300u};

  const int tpp = a.c.tiles;
  const int nt = a.sel ? a.n_sel * tpp : (top + kKv4Tile - 1) / kKv4Tile;
  const int chunk = (nt + a.n_split - 1) / a.n_split;
  const int t_end = min(nt, (split + 1) * chunk);
  for (int t = split * chunk + wave; t < t_end; t += kWaves) {
    const int e = t / tpp, sub = t % tpp;
    int lp = e;
    if (a.sel) lp = a.sel[((int64_t)b * a.c.hkv + h) * a.n_sel + e];
    if (lp < 0 || (int64_t)lp * a.c.page_len + sub * kKv4Tile >= top) continue;
    const int base = lp * a.c.page_len + sub * kKv4Tile;
    const int id = kv4_page(a.c, b, lp);
    const uint8_t* tile = a.c.pages + (int64_t)max(id, 0) * a.c.page_stride +
                          (int64_t)h * kv4_head_bytes(a.c.page_len, D) + sub * kv4_tile_bytes(D);
    u32x4_t kc[C], vc[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      kc[c] = *(const u32x4_t*)(tile + (c * 64 + lane) * 16);
      vc[c] = *(const u32x4_t*)(tile + 16 * D + (c * 64 + lane) * 16);
    }
    uint32_t ks[2][4][NG], vs[2][4][NG];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const int at = ((16 * tt + 4 * kg + i) * NG + g) * 4;
          ks[tt][i][g] = *(const uint32_t*)(tile + 32 * D + at);
          vs[tt][i][g] = *(const uint32_t*)(tile + 32 * D + 128 * NG + at);
          if (id < 0) ks[tt][i][g] = kKv4NaN;
        }
    float s[2][4];
    bool ok[2][4];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[tt][i] = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float z = -128.f * qs[g];
        const f32x4_t r = mfma_bf16(kv4_operand(kc[g >> 1][2 * tt + (g & 1)]), q[g], f32x4_t{z, z, z, z});
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s[tt][i] += bf16lo(ks[tt][i][g]) * r[i] + bf16hi(ks[tt][i][g]) * qs[g];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ok[tt][i] = base + 16 * tt + 4 * kg + i < end;
        s[tt][i] = ok[tt][i] ? s[tt][i] * a.scale_l2 : -INFINITY;
      }
    }
    float mr = s[0][0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mr = fmaxf(mr, s[i >> 2][i & 3]);
    mr = xor32_max(xor16_max(mr));
    const float mn = fmaxf(m, mr);
    const float mb = mn == -INFINITY ? 0.f : mn;
    const float corr = ex2(m - mb);
    m = mn;
    l *= corr;
#pragma unroll
    for (int u = 0; u < NT; ++u) o[u] *= corr;
    float p[2][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i >> 2][i & 3] = ex2(s[i >> 2][i & 3] - mb);
      l += p[i >> 2][i & 3];
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      ms[g] *= corr;
      off[g] *= corr;
      u32x4_t hi, lo;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // a masked position's scale may be anything (the page's older bytes): not 0 * NaN
        const float x0 = ok[0][i] ? p[0][i] * bf16lo(vs[0][i][g]) : 0.f;
        const float x1 = ok[1][i] ? p[1][i] * bf16lo(vs[1][i][g]) : 0.f;
        ms[g] += ok[0][i] ? p[0][i] * bf16hi(vs[0][i][g]) : 0.f;
        ms[g] += ok[1][i] ? p[1][i] * bf16hi(vs[1][i][g]) : 0.f;
        hi[i] = pack_bf16x2_op(x0, x1);
        lo[i] = pack_bf16x2_op(x0 - bf16lo(hi[i]), x1 - bf16hi(hi[i]));
      }
      off[g] = mfma_bf16(minus, hi, off[g]);
      off[g] = mfma_bf16(minus, lo, off[g]);
#pragma unroll
      for (int u = 2 * g; u < 2 * g + 2; ++u) {
        const u32x4_t v = kv4_operand(vc[u >> 2][u & 3]);
        o[u] = mfma_bf16(v, hi, o[u]);
        o[u] = mfma_bf16(v, lo, o[u]);
      }
    }
  }

  // ---- the waves' states through LDS: s_o[wave][row][dim], m and l behind the dims
  l = xor32_sum(xor16_sum(l));
#pragma unroll
  for (int g = 0; g < NG; ++g) ms[g] = xor32_sum(xor16_sum(ms[g]));
#pragma unroll
  for (int u = 0; u < NT; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      s_o[wave][n][16 * u + 4 * kg + i] = o[u][i] + off[u >> 1][i] + ms[u >> 1];
  if (kg == 0) {
    s_o[wave][n][D] = m;
    s_o[wave][n][D + 1] = l;
  }
  __syncthreads();
  const int used = min(16, rows - rt * 16);
  for (int e = tid; e < used * D; e += 256) {
    const int r = e / D, d = e % D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, s_o[w][r][D]);
    const float Mb = M == -INFINITY ? 0.f : M;
    float L = 0.f, A = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = ex2(s_o[w][r][D] - Mb);
      L = fmaf(s_o[w][r][D + 1], f, L);
      A = fmaf(s_o[w][r][d], f, A);
    }
    s_fin[r][d] = A;
    if (d < 4) s_fin[r][D + d] = d == 0 ? M : (d == 1 ? L : 0.f);
  }
  __syncthreads();
  if (a.n_split > 1) {
    const __amdgpu_buffer_rsrc_t pr = make_rsrc(a.partial, a.partial_bytes);
    const uint32_t rec = ((uint32_t)bk * a.n_split + split) * (16 * REC * 4);
    for (int e = tid; e < used * REC / 4; e += 256)
      st16_sys(pr, rec + e * 16, ((const uint4*)&s_fin[0][0])[e]);
    wait_vm();
    __syncthreads();
    if (tid == 0) s_last = ticket(&a.counters[bk], a.n_split) ? 1 : 0;
    __syncthreads();
    if (!s_last) return;
    const float* recs = a.partial + (size_t)bk * a.n_split * 16 * REC;
    for (int e = tid; e < used * D; e += 256) {
      const int r = e / D, d = e % D;
      float M = -INFINITY, L = 0.f, A = 0.f;
      for (int sp = 0; sp < a.n_split; ++sp) {
        const float* p = recs + ((size_t)sp * 16 + r) * REC;
        const float mi = load_sys(p + D), li = load_sys(p + D + 1), ai = load_sys(p + d);
        const float Mn = fmaxf(M, mi), Mb = Mn == -INFINITY ? 0.f : Mn;
        const float f0 = ex2(M - Mb), f1 = ex2(mi - Mb);
        L = L * f0 + li * f1;
        A = A * f0 + ai * f1;
        M = Mn;
      }
      s_fin[r][d] = A;
      if (d == 0) s_fin[r][D + 1] = L;
    }
    __syncthreads();
  }
  for (int e = tid; e < used * D; e += 256) {
    const int r = e / D, d = e % D;
    const float L = s_fin[r][D + 1];
    const float y = L == 0.f ? 0.f : attn_div(s_fin[r][d], L);   // nothing seen: 0; a NaN stays
    const int row_ = rt * 16 + r;
    const int64_t at = ((int64_t)(c0 + row_ / a.group) * a.hq + h * a.group + row_ % a.group) * D + d;
    if (a.out) a.out[at] = f32_to_bf16(y);
    if (a.out_f32) a.out_f32[at] = y;
  }
}

static size_t kv4_partial_bytes(int64_t items, int n_split, int d) {
  return (size_t)items * n_split * 16 * (d + 4) * 4;
}

static int kv4_row_tiles(int max_new, int group) { return (int)(((int64_t)max_new * group + 15) / 16); }

// Splits per row tile, by the positions a sequence may have.
static int kv4_auto_split(int64_t items, int tiles) {
  int64_t s = 1024 / (items < 1 ? 1 : items);
  const int64_t by_len = (tiles + 2 * kWaves - 1) / (2 * kWaves);
  s = s < by_len ? s : by_len;
  return (int)(s < 1 ? 1 : (s > 64 ? 64 : s));
}

struct Kv4Plan {
  int64_t items;
  int n_split;
  size_t bytes;
};
static Kv4Plan kv4_plan(const q4nx_kv4* c, int n_q_heads, int max_new, int max_len, int n_sel,
                        int n_split) {
  Kv4Plan p;
  const int rt = kv4_row_tiles(max_new, n_q_heads / c->n_kv_heads);
  p.items = (int64_t)c->n_seqs * c->n_kv_heads * rt;
  const int64_t cap = (int64_t)c->table_len * c->page_len;
  const int64_t len = n_sel ? (int64_t)n_sel * c->page_len : (max_len < cap ? max_len : cap);
  p.n_split = n_split > 0 ? n_split : kv4_auto_split(p.items, (int)((len + kKv4Tile - 1) / kKv4Tile));
  p.bytes = p.n_split > 1 ? (size_t)Q4NX_WS_COUNTER_BYTES +
                                kv4_partial_bytes(p.items, p.n_split, c->head_dim)
                          : 0;
  return p;
}

static bool kv4_attn_shape(const q4nx_kv4* c, int n_q_heads, int max_new, int max_len, int n_sel) {
  return n_q_heads >= 1 && n_q_heads % c->n_kv_heads == 0 && n_q_heads / c->n_kv_heads <= 16 &&
         max_new >= 1 && max_new <= 1 << 20 && max_len >= 1 && n_sel >= 0 &&
         (int64_t)n_sel * c->page_len <= (int64_t)1 << 30;
}

}  // namespace q4nx

using namespace q4nx;

extern "C" {

size_t q4nx_kv4_attn_ws_bytes(const q4nx_kv4* cache, int n_q_heads, int max_new, int max_len,
                              int n_sel, int n_split) {
  Kv4 c;
  if (kv4_resolve(cache, &c, "q4nx_kv4_attn_ws_bytes") != Q4NX_OK ||
      !kv4_attn_shape(cache, n_q_heads, max_new, max_len, n_sel) || n_split < 0 || n_split > 1024)
    return 0;
  return kv4_plan(cache, n_q_heads, max_new, max_len, n_sel, n_split).bytes;
}

int q4nx_kv4_attn(const q4nx_kv4* cache, const uint16_t* q, int64_t q_stride, uint16_t* out,
                  float* out_f32, int n_q_heads, const int32_t* cu, int total, int max_new,
                  const int32_t* lens, int max_len, float scale, const int32_t* sel, int n_sel,
                  int n_split, void* ws, size_t ws_bytes, void* stream) {
  const char* what = "q4nx_kv4_attn";
  Kv4AttnArgs a{};
  if (int rc = kv4_resolve(cache, &a.c, what)) return rc;
  Q4NX_REQUIRE(q && lens && (out || out_f32) && Q4NX_ALIGNED(q, 16), Q4NX_ERR_ARG,
               "%s: q (16-byte aligned), lens and an output are required", what);
  Q4NX_REQUIRE((sel != nullptr) == (n_sel > 0) && n_split >= 0 && n_split <= 1024, Q4NX_ERR_ARG,
               "%s: sel and n_sel=%d go together; n_split=%d outside 0..1024", what, n_sel, n_split);
  Q4NX_REQUIRE(kv4_attn_shape(cache, n_q_heads, max_new, max_len, n_sel), Q4NX_ERR_SHAPE,
               "%s: Hq=%d must be a multiple (<= 16x) of Hkv=%d; max_new=%d max_len=%d n_sel=%d", what,
               n_q_heads, cache->n_kv_heads, max_new, max_len, n_sel);
  Q4NX_REQUIRE(cu ? total >= 1 : (max_new == 1 && total == cache->n_seqs), Q4NX_ERR_SHAPE,
               "%s: total=%d, max_new=%d (without cu one token for each of %d sequences)", what, total,
               max_new, cache->n_seqs);
  Q4NX_REQUIRE(n_sel == 0 || max_new == 1, Q4NX_ERR_SHAPE,
               "%s: a page list is for one token per sequence, max_new=%d", what, max_new);
  Q4NX_REQUIRE(q_stride >= (int64_t)n_q_heads * cache->head_dim && q_stride % 8 == 0, Q4NX_ERR_SHAPE,
               "%s: q_stride=%lld must hold Hq * D and be a multiple of 8", what, (long long)q_stride);
  const Kv4Plan p = kv4_plan(cache, n_q_heads, max_new, max_len, n_sel, n_split);
  Q4NX_REQUIRE(p.items * p.n_split <= (int64_t)1 << 30, Q4NX_ERR_SHAPE,
               "%s: %lld workgroups", what, (long long)(p.items * p.n_split));
  if (p.n_split > 1) {
    Q4NX_REQUIRE(p.bytes - Q4NX_WS_COUNTER_BYTES < (size_t)1 << 31 &&
                     p.items * 4 <= Q4NX_WS_COUNTER_BYTES,
                 Q4NX_ERR_SHAPE, "%s: too many rows for %d splits", what, p.n_split);
    Q4NX_REQUIRE(ws != nullptr && ws_bytes >= p.bytes && Q4NX_ALIGNED(ws, 256), Q4NX_ERR_WS,
                 "%s: workspace of %zu bytes (256-aligned) needed, %zu given", what, p.bytes, ws_bytes);
    a.counters = (unsigned*)ws;
    a.partial = (float*)((uint8_t*)ws + Q4NX_WS_COUNTER_BYTES);
    a.partial_bytes = (uint32_t)(p.bytes - Q4NX_WS_COUNTER_BYTES);
  }
  a.q = q;
  a.q_stride = q_stride;
  a.out = out;
  a.out_f32 = out_f32;
  a.cu = cu;
  a.lens = lens;
  a.sel = sel;
  a.n_sel = n_sel;
  a.hq = n_q_heads;
  a.group = n_q_heads / cache->n_kv_heads;
  a.total = total;
  a.row_tiles = kv4_row_tiles(max_new, a.group);
  a.n_split = p.n_split;
  if (max_len < a.c.cap) a.c.cap = max_len;
  a.scale_l2 = (float)((double)scale * 1.4426950408889634);
  const dim3 grid((unsigned)(p.items * p.n_split));
  if (cache->head_dim == 64)
    hipLaunchKernelGGL(kv4_attn_kernel<2>, grid, dim3(256), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(kv4_attn_kernel<4>, grid, dim3(256), 0, (hipStream_t)stream, a);
  return check_launch(what);
}

}  // extern "C"
