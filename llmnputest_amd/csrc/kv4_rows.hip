// Rows into and out of the paged 4-bit K/V cache.
//
// One workgroup is one page of one (sequence, kv head), a pair of waves a tile of 32 positions, one for
// K and one for V; nothing outside its tile is written by a wave, so the nibbles that old and new
// positions share in a dword of V are merged by one lane. Lane (n, kg) holds channels 8 kg .. 8 kg + 7
// of every group of 32 at positions n and 16 + n: a group's least and greatest value are eight values in
// the lane and two lane swaps (16, 32), and K's dword is made where it is stored. V's dwords run along
// positions: its codes go through LDS as words of four bytes, channels n, 16 + n, 32 + n and 48 + n of
// a position, made by a lane swap and a 4 x 4 transpose of bytes in registers on either side.
// Bound by instructions (26 of the VALU a value in all to append, 13 to read) and one tile's chain of latencies:
// 9k rows of 8 kv heads x 64 append in 16 us (21.5 MB, 1.3 TB/s), the VALU active in 0.68 of the busy cycles
// and the waves waiting 0.40 of their time, and read in 11 (2.0 TB/s), 0.54 and 0.43; one row of each of 8
// sequences in 5.5 and 3.6. With one wave for K and V in turn, and V's bytes through LDS one by one, the
// appends took 27.
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

// bf16 bits as signed 16-bit words of the same order, two to a register (its own inverse): least and
// greatest values then take packed integer instructions. -0 lies below +0; a positive NaN or infinity is
// 0x7F80 or above, a negative one 0x807F or below.
typedef short s16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ s16x2 order(uint32_t x) {
  const s16x2 v = __builtin_bit_cast(s16x2, x);
  return v ^ ((v >> 15) & (short)0x7FFF);
}
__device__ __forceinline__ s16x2 least(s16x2 a, s16x2 b) { return __builtin_elementwise_min(a, b); }
__device__ __forceinline__ s16x2 most(s16x2 a, s16x2 b) { return __builtin_elementwise_max(a, b); }
__device__ __forceinline__ s16x2 as_s16(uint32_t x) { return __builtin_bit_cast(s16x2, x); }
__device__ __forceinline__ uint32_t as_u32(s16x2 x) { return __builtin_bit_cast(uint32_t, x); }
// over the lanes 16 and 32 away
__device__ __forceinline__ s16x2 kg_least(s16x2 x) {
  auto r = __builtin_amdgcn_permlane16_swap(as_u32(x), as_u32(x), false, false);
  x = least(as_s16(r[0]), as_s16(r[1]));
  r = __builtin_amdgcn_permlane32_swap(as_u32(x), as_u32(x), false, false);
  return least(as_s16(r[0]), as_s16(r[1]));
}
__device__ __forceinline__ s16x2 kg_most(s16x2 x) {
  auto r = __builtin_amdgcn_permlane16_swap(as_u32(x), as_u32(x), false, false);
  x = most(as_s16(r[0]), as_s16(r[1]));
  r = __builtin_amdgcn_permlane32_swap(as_u32(x), as_u32(x), false, false);
  return most(as_s16(r[0]), as_s16(r[1]));
}
template <int CTRL>
__device__ __forceinline__ s16x2 dpp16(s16x2 x) {
  return as_s16((uint32_t)__builtin_amdgcn_mov_dpp((int)as_u32(x), CTRL, 0xf, 0xf, false));
}
// over a row of 16 lanes
__device__ __forceinline__ s16x2 row_least(s16x2 x) {
  x = least(x, dpp16<kDppXor1>(x));
  x = least(x, dpp16<kDppXor2>(x));
  x = least(x, dpp16<kDppHalfMirror>(x));
  return least(x, dpp16<kDppRor8>(x));
}
__device__ __forceinline__ s16x2 row_most(s16x2 x) {
  x = most(x, dpp16<kDppXor1>(x));
  x = most(x, dpp16<kDppXor2>(x));
  x = most(x, dpp16<kDppHalfMirror>(x));
  return most(x, dpp16<kDppRor8>(x));
}

// What a (sequence, page) of a call covers: its new positions are [first, last).
struct Kv4Span {
  int page, b, h, first, last;
  int64_t src0;   // the source row of position p is src0 + p
};
__device__ __forceinline__ bool kv4_span(const Kv4RowArgs& a, Kv4Span* s) {
  s->h = blockIdx.x % a.c.hkv;
  s->b = blockIdx.x / a.c.hkv;
  // a position past either of these is as far outside the cache as they are: a table holds at most 2^30, and
  // a launch covers fewer rows of a sequence
  const int64_t p0 = max(-(1 << 30), min(a.pos[s->b], 1 << 30));
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

// y[i] byte t = x[t] byte i
__device__ __forceinline__ void transpose4(uint32_t (&x)[4]) {
  const uint32_t p0 = perm(x[1], x[0], 0x05010400u), p1 = perm(x[1], x[0], 0x07030602u);
  const uint32_t p2 = perm(x[3], x[2], 0x05010400u), p3 = perm(x[3], x[2], 0x07030602u);
  x[0] = perm(p2, p0, 0x05040100u);
  x[1] = perm(p2, p0, 0x07060302u);
  x[2] = perm(p3, p1, 0x05040100u);
  x[3] = perm(p3, p1, 0x07060302u);
}
// Codes of V in LDS: [position][channel n of 16][channels n, 16 + n, 32 + n, 48 + n] bytes, 20 words a
// position so that neither side meets in a bank. A lane's words of a row lie from here on.
constexpr int kVRow = 20;
__device__ __forceinline__ int v_col(int kg) { return 8 * (kg & 1) + 4 * (kg >> 1); }
// This lane's codes of its position, channels 8 kg .. + 7 of groups 0 and 1 (bytes), <-> the four words
// from v_col(kg): lanes 32 apart hold channels 16 apart and exchange halves.
__device__ __forceinline__ u32x4_t v_words(uint2 g0, uint2 g1) {
  const auto a = __builtin_amdgcn_permlane32_swap(g0.x, g0.y, false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(g1.x, g1.y, false, false);
  uint32_t x[4] = {a[0], a[1], b[0], b[1]};
  transpose4(x);
  return u32x4_t{x[0], x[1], x[2], x[3]};
}
__device__ __forceinline__ void v_bytes(const u32x4_t& w, uint2* g0, uint2* g1) {
  uint32_t x[4] = {w[0], w[1], w[2], w[3]};
  transpose4(x);
  const auto a = __builtin_amdgcn_permlane32_swap(x[0], x[1], false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(x[2], x[3], false, false);
  *g0 = make_uint2(a[0], a[1]);
  *g1 = make_uint2(b[0], b[1]);
}

struct Kv4Group {   // one group of one row: this lane's eight codes, a nibble each, and (d, m)
  uint32_t lo, hi;  // codes of channels 0..3 and 4..7, a byte each
  uint32_t dm;
  bool bad;
};

// Quantises the group of 32 channels whose eight values (packed bf16) are in lanes kg = 0..3.
__device__ __forceinline__ Kv4Group kv4_quant(const u32x4_t& x, const s16x2 (&key)[4]) {
  const s16x2 l2 = kg_least(least(least(key[0], key[1]), least(key[2], key[3])));
  const s16x2 h2 = kg_most(most(most(key[0], key[1]), most(key[2], key[3])));
  const short lk = l2[0] < l2[1] ? l2[0] : l2[1], hk = h2[0] > h2[1] ? h2[0] : h2[1];
  const s16x2 lh = {lk, hk};
  const uint32_t lohi = as_u32(order(as_u32(lh)));
  const float lo = bf16lo(lohi), hi = bf16hi(lohi);
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = bf16lo(x[i]);
    f[2 * i + 1] = bf16hi(x[i]);
  }
  const float d = round_bf16_op((hi - lo) / 15.0f);
  Kv4Group r;
  r.bad = hk >= (short)0x7F80 || lk <= (short)0x807F || !(d < INFINITY);
  r.lo = r.hi = 0;
  // (x - m) / d correctly rounded, as the format has it: with the rounded reciprocal of d, one step on the
  // quotient's exact remainder gives it (Markstein); groups so small or large that the reciprocal leaves
  // the normal range divide
  float q[8];
  const bool far = d > 0.f && !(d > 0x1p-100f && d < 0x1p100f);
  const float r0 = __builtin_amdgcn_rcpf(d), y = fmaf(fmaf(-d, r0, 1.0f), r0, r0);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = f[i] - lo, q0 = t * y;
    q[i] = fmaf(fmaf(-q0, d, t), y, q0);
  }
  if (__any(far)) {
    asm volatile("");
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (far) q[i] = fminf((f[i] - lo) / d, 15.0f);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint32_t& w = i < 4 ? r.lo : r.hi;
    // at most 15 / (1 - 2^-9) where d has its eight bits: rounds to 15
    w = __builtin_amdgcn_cvt_pk_u8_f32(rintf(q[i]), i & 3, w);
  }
  const uint32_t mask = d > 0.f && !r.bad ? 0x0F0F0F0Fu : 0u;
  r.lo &= mask;
  r.hi &= mask;
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

// The bound of two parts as ordered words, 0x7FC0 (NaN) where either is.
__device__ __forceinline__ short bound_of(short a, short b, bool greatest) {
  if (a == 0x7FC0 || b == 0x7FC0) return 0x7FC0;
  return (a < b) == greatest ? b : a;
}

template <int NG>
__global__ __launch_bounds__(512) void kv4_append_kernel(Kv4RowArgs a) {
  constexpr int D = 32 * NG, C = D / 64;
  __shared__ __attribute__((aligned(16))) uint32_t s_v[4][C][32][kVRow];
  __shared__ __attribute__((aligned(16))) short s_b[4][2][D];
  Kv4Span s;
  if (!kv4_span(a, &s)) return;   // uniform over the workgroup
  const int id = kv4_page(a.c, s.b, s.page);
  if (id < 0) return;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, kg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 7);   // the tile
  const bool is_v = __builtin_amdgcn_readfirstlane(tid >> 6) & 1;
  const int base = s.page * a.c.page_len + wave * kKv4Tile;
  uint8_t* head = a.c.pages + (int64_t)id * a.c.page_stride +
                  (int64_t)s.h * kv4_head_bytes(a.c.page_len, D);
  uint8_t* tile = head + wave * kv4_tile_bytes(D);
  const int t0 = max(s.first - base, 0), t1 = min(s.last - base, kKv4Tile);   // new: [t0, t1)
  const int64_t src = (a.by_position ? s.b * a.seq_stride : 0) + s.h * a.head_stride;
  const uint16_t* rows = is_v ? a.v : a.k;
  const bool any = t0 < t1;
  // the page's bounds so far, on their way while rows are quantised: with 128 threads and more, two of the
  // 2 D for each
  uint16_t* bounds = (uint16_t*)(head + a.c.tiles * kv4_tile_bytes(D));
  const bool begins = s.first == s.page * a.c.page_len;
  uint32_t bound0[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) bound0[i] = bounds[min(tid + i * (int)blockDim.x, 2 * D - 1)];

  u32x4_t x[2][NG], old[C];
  uint32_t keep = 0;   // nibbles of V's dwords whose positions are not new
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int t = 16 * (e >> 2) + 4 * kg + (e & 3);
    if (t < t0 || t >= t1) keep |= 0xFu << (4 * e);
  }
  if (any) {
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      const int t = 16 * tt + n;
      const bool now = t >= t0 && t < t1;
      // a row of the span for the lanes that have none: its values are not used
      const int64_t row = src + (s.src0 + (now ? base + t : s.first)) * a.row_stride;
#pragma unroll
      for (int g = 0; g < NG; ++g) x[tt][g] = *(const u32x4_t*)(rows + row + 32 * g + 8 * kg);
    }
    if (is_v && keep) {
#pragma unroll
      for (int c = 0; c < C; ++c) old[c] = *(const u32x4_t*)(tile + 16 * D + (c * 64 + lane) * 16);
    }
  }
  uint8_t* scales = tile + 32 * D + (is_v ? 128 * NG : 0);
  if (is_v) {
    // ---- V: codes as bytes through LDS, then a dword per channel and eight positions
    if (any) {
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        const int t = 16 * tt + n;
        uint2 codes[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          s16x2 key[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) key[i] = order(x[tt][g][i]);
          const Kv4Group q = kv4_quant(x[tt][g], key);
          codes[g] = make_uint2(q.lo, q.hi);
          if (t >= t0 && t < t1 && kg == (g & 3)) *(uint32_t*)(scales + (t * NG + g) * 4) = q.dm;
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
          *(u32x4_t*)&s_v[wave][c][t][v_col(kg)] = v_words(codes[2 * c], codes[2 * c + 1]);
      }
      __builtin_amdgcn_wave_barrier();   // the wave's own words
#pragma unroll
      for (int c = 0; c < C; ++c) {
        u32x4_t* dst = (u32x4_t*)(tile + 16 * D + (c * 64 + lane) * 16);
        uint32_t y[4];   // byte j of dword t: positions 2 j and 2 j + 1 of the eight
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int p = 16 * (j >> 1) + 4 * kg + 2 * (j & 1);
          y[j] = s_v[wave][c][p][n] | s_v[wave][c][p + 1][n] << 4;
        }
        transpose4(y);
        u32x4_t w = {y[0], y[1], y[2], y[3]};
        if (keep == 0xFFFFFFFFu) continue;
        if (keep) {
#pragma unroll
          for (int t = 0; t < 4; ++t) w[t] = (w[t] & ~keep) | (old[c][t] & keep);
        }
        *dst = w;
      }
    }
  } else {
    // ---- K: codes, scales, and the bounds of each channel over the tile's new positions
    s16x2 lo[NG][4], hi[NG][4];
    uint32_t bad = 0;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        lo[g][i] = s16x2{0x7FFF, 0x7FFF};
        hi[g][i] = s16x2{(short)0x8000, (short)0x8000};
      }
    if (any) {
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        const int t = 16 * tt + n;
        const bool now = t >= t0 && t < t1;
        uint32_t w[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          s16x2 key[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) key[i] = order(x[tt][g][i]);
          const Kv4Group q = kv4_quant(x[tt][g], key);
          w[g] = kv4_kdword(q.lo, q.hi);
          if (now && kg == (g & 3)) *(uint32_t*)(scales + (t * NG + g) * 4) = q.dm;
          bad |= now && q.bad ? 1u << g : 0u;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            lo[g][i] = least(lo[g][i], now ? key[i] : lo[g][i]);
            hi[g][i] = most(hi[g][i], now ? key[i] : hi[g][i]);
          }
        }
        if (now) {
#pragma unroll
          for (int c = 0; c < C; ++c)
            *(uint2*)(tile + (c * 64 + lane) * 16 + 8 * tt) = make_uint2(w[2 * c], w[2 * c + 1]);
        }
      }
    }
    // the channel bounds over the 16 positions of a row of lanes, as ordered words; NaN is above any
    // value and below any, so a group that has one shows in both
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const bool any_bad = __any((bad >> g) & 1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const s16x2 l = row_least(lo[g][i]), h = row_most(hi[g][i]);
        if (n == i) {
          const s16x2 nan = {0x7FC0, 0x7FC0};
          *(s16x2*)&s_b[wave][0][32 * g + 8 * kg + 2 * i] = any_bad ? nan : l;
          *(s16x2*)&s_b[wave][1][32 * g + 8 * kg + 2 * i] = any_bad ? nan : h;
        }
      }
    }
  }
  __syncthreads();
  // ---- the page's bounds: of this call's rows, with the older ones' unless the page begins here
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = tid + i * (int)blockDim.x;
    if (e >= 2 * D) break;
    const int side = e / D, ch = e % D;
    short x = s_b[0][side][ch];
    for (int w = 1; w < a.c.tiles; ++w) x = bound_of(x, s_b[w][side][ch], side);
    if (!begins) {
      const bool nan = (bound0[i] & 0x7FFFu) > 0x7F80u;
      x = bound_of(x, nan ? (short)0x7FC0 : order(bound0[i])[0], side);
    }
    bounds[e] = x == 0x7FC0 ? (uint16_t)0x7FC0 : (uint16_t)as_u32(order((uint32_t)(uint16_t)x));
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
__global__ __launch_bounds__(512) void kv4_read_kernel(Kv4RowArgs a) {
  constexpr int D = 32 * NG, C = D / 64;
  __shared__ __attribute__((aligned(16))) uint32_t s_v[4][C][32][kVRow];
  Kv4Span s;
  if (!kv4_span(a, &s)) return;
  const int id = kv4_page(a.c, s.b, s.page);   // none: the rows read as NaN
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, kg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 7);
  const bool is_v = __builtin_amdgcn_readfirstlane(tid >> 6) & 1;
  const int base = s.page * a.c.page_len + wave * kKv4Tile;
  const uint8_t* tile = a.c.pages + (int64_t)max(id, 0) * a.c.page_stride +
                        (int64_t)s.h * kv4_head_bytes(a.c.page_len, D) +
                        wave * kv4_tile_bytes(D);
  const int t0 = max(s.first - base, 0), t1 = min(s.last - base, kKv4Tile);
  if (t0 >= t1) return;   // no barrier below
  u32x4_t w[C];
  uint32_t dm[2][NG];
#pragma unroll
  for (int c = 0; c < C; ++c) w[c] = *(const u32x4_t*)(tile + (is_v ? 16 * D : 0) + (c * 64 + lane) * 16);
#pragma unroll
  for (int tt = 0; tt < 2; ++tt)
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      dm[tt][g] = *(const uint32_t*)(tile + 32 * D + (is_v ? 128 * NG : 0) + ((16 * tt + n) * NG + g) * 4);
      if (id < 0) dm[tt][g] = kKv4NaN;
    }
  uint2 code[2][NG];   // this lane's channels of positions n and 16 + n, a byte each
  if (is_v) {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int odd = 0; odd < 2; ++odd) {   // positions 2 j + odd of the eight
        uint32_t x[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t] = (w[c][t] >> (4 * odd)) & 0x0F0F0F0Fu;
        transpose4(x);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          s_v[wave][c][16 * (j >> 1) + 4 * kg + 2 * (j & 1) + odd][n] = x[j];
      }
    __builtin_amdgcn_wave_barrier();   // the wave's own words
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
      for (int c = 0; c < C; ++c)
        v_bytes(*(const u32x4_t*)&s_v[wave][c][16 * tt + n][v_col(kg)], &code[tt][2 * c],
                &code[tt][2 * c + 1]);
  } else {
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        // nibbles 0, 2, 4, 6 in the low half, 1, 3, 5, 7 in the high one -> bytes in order
        const uint32_t x = w[g >> 1][2 * tt + (g & 1)], e = x & 0x0F0F0F0Fu, o = (x >> 4) & 0x0F0F0F0Fu;
        // e: channels 0, 4, 1, 5; o: 2, 6, 3, 7
        code[tt][g] = make_uint2(perm(o, e, 0x06040200u), perm(o, e, 0x07050301u));
      }
  }
  void* dst = is_v ? a.v_out : a.k_out;
#pragma unroll
  for (int tt = 0; tt < 2; ++tt) {
    const int t = 16 * tt + n;
    if (t < t0 || t >= t1) continue;
    const int64_t out = ((s.src0 + base + t) * a.c.hkv + s.h) * D + 8 * kg;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t c = ((i < 4 ? code[tt][g].x : code[tt][g].y) >> (8 * (i & 3))) & 255u;
        y[i] = fmaf((float)c, bf16lo(dm[tt][g]), bf16hi(dm[tt][g]));
      }
      kv4_put(dst, a.out_f32, out + 32 * g, y);
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
             c->page_len == 128 ? 2 : c->page_len == 64 ? 1 : 0, c->table_len * c->page_len};
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
  const dim3 block(128 * a.c.tiles);
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
  const dim3 block(128 * a.c.tiles);
  if (cache->head_dim == 64)
    hipLaunchKernelGGL(kv4_read_kernel<2>, grid, block, 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(kv4_read_kernel<4>, grid, block, 0, (hipStream_t)stream, a);
  return check_launch(what);
}

}  // extern "C"
