// Attention over the paged 4-bit K/V cache, on the matrix cores: single tokens (codes enter the products
// as they are stored), and blocks of new tokens (tiles taken apart once for 128 rows). Scores, their maxima
// and sums, and the outputs are fp32 until they are written.
//
// With x = d_g c + m_g per group g of 32 channels,
//   score = sum_g d_g (c . q)_g + m_g (sum of q)_g,    out = sum_pos p d_g c + sum_pos p m_g
// so a code is an operand as it is, the bf16 number 128 + c for K and 16 + c for V (exact), and the scales
// stay in fp32. The offsets are taken out again: a score's accumulator starts at -128 (sum of q)_g, and
// m_g - 16 d_g takes m_g's place in the values. p d_g enters as two bf16 terms, which carry it to 2^-18,
// so that a value is off by at most 31 2^-18 of its step.
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
  int n_sel, hq, group, total;
  int n_split, chunk;   // blocks: workgroups per row tile, tiles for each of them
  int unit;             // one token: tiles per part of a (sequence, kv head), 0: by what there is
  bool whole;           // one token: every (sequence, kv head) is one part
  float scale_l2;
  u32x4_t* ops;         // blocks: tiles taken apart beforehand, [seq * hkv][ops_tiles][4 NG][2][64]
  uint32_t* bad;        // their V's NaN groups, [..][ops_tiles][NG]: a bit per position
  int ops_tiles;
  float* partial;
  uint32_t partial_bytes;
  unsigned* counters;
};

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

constexpr int kWaves = 4;
// Tiles of a call above which its workgroups share one line of them, and how many there have to be for
// each (sequence, kv head) as a mean.
constexpr int kLineTiles = 16384;
constexpr int kMostTiles = 128, kMostParts = 32;   // of a part and of an item (a mean) that are not on a line
// A (sequence, kv head) is one part where it has at most kShortTiles, and from kWholeItems of them of at
// most kWholeTiles on.
constexpr int kShortTiles = 32, kWholeItems = 512, kWholeTiles = 64;
__host__ __device__ constexpr int kv4_line_mean(int d) { return d == 64 ? 256 : 64; }
// Those workgroups: what the chip holds at once (three waves per SIMD at D = 64, two at 128).
__host__ __device__ constexpr int kv4_line(int d) { return d == 64 ? 768 : 512; }
constexpr int kMergeParts = 64;   // records of an item merged per pass
constexpr int kMergeBatch = 8;    // of them in flight per thread

// x - bf16 (the lo or hi half of pair) in one instruction; the difference of a number and its bf16
// rounding is exact. The pair (-1, 0) comes from a register: as an inline constant -1.0 the
// instruction takes it for (0, -1).
typedef short s16x2_t __attribute__((ext_vector_type(2)));
struct Kv4Minus {
  uint32_t lo = 0x0000BF80u, hi = 0xBF800000u;
  __device__ Kv4Minus() { asm volatile("" : "+v"(lo), "+v"(hi)); }
  static __device__ __forceinline__ float dot(float x, uint32_t pair, uint32_t one) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(s16x2_t, pair),
                                           __builtin_bit_cast(s16x2_t, one), x, false);
  }
  // a pair as two bf16 terms each: 2^-18 of a value is left out
  __device__ __forceinline__ void split(float x0, float x1, uint32_t& hi_, uint32_t& lo_) const {
    hi_ = pack_bf16x2_op(x0, x1);
    lo_ = pack_bf16x2_op(dot(x0, hi_, lo), dot(x1, hi_, hi));
  }
};

template <int NG>
struct Kv4TileRegs {
  u32x4_t k[NG / 2], v[NG / 2];
  uint32_t s[NG];
};

// The waves' states of `used` rows in s_o ([wave][row][dims, m, l]) -> s_fin, then the records of the
// item's parts in their order by whichever workgroup arrives last, and the rows out.
template <int D, int TH, int NW, int ROWS, typename Rec>
__device__ __forceinline__ void kv4_finish(const Kv4AttnArgs& a, float (*s_o)[ROWS][D + 4],
                                           float (*s_fin)[D + 4], int* s_last, int item, int part,
                                           int parts, Rec&& rec_of, int used, int c0, int row0, int h) {
  constexpr int REC = D + 4;
  const int tid = threadIdx.x;
  __syncthreads();
  for (int e = tid; e < used * D; e += TH) {
    const int r = e / D, d = e % D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, s_o[w][r][D]);
    const float Mb = M == -INFINITY ? 0.f : M;
    float L = 0.f, A = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = ex2(s_o[w][r][D] - Mb);
      L = fmaf(s_o[w][r][D + 1], f, L);
      A = fmaf(s_o[w][r][d], f, A);
    }
    s_fin[r][d] = A;
    if (d < 4) s_fin[r][D + d] = d == 0 ? M : (d == 1 ? L : 0.f);
  }
  __syncthreads();
  if (parts > 1) {
    const __amdgpu_buffer_rsrc_t pr = make_rsrc(a.partial, a.partial_bytes);
    const uint32_t rec = (uint32_t)rec_of(part) * (ROWS * REC * 4);
    for (int e = tid; e < used * REC / 4; e += TH)
      st16_sys(pr, rec + e * 16, ((const uint4*)s_fin)[e]);
    wait_vm();
    __syncthreads();
    if (tid == 0) *s_last = ticket(&a.counters[item], parts) ? 1 : 0;
    __syncthreads();
    if (!*s_last) return;
    // 16 lanes of a row find the parts' weights; a thread sums four channels over every ng-th part, its
    // first records on their way meanwhile; ng sums meet in LDS
    constexpr int KC = (ROWS * D / 4 + TH - 1) / TH;
    __shared__ float s_f[kMergeParts][ROWS], s_c[ROWS];
    const int cols = used * D / 4, ng = max(1, min(NW, TH / cols));
    const int grp = cols < TH ? tid / cols : 0, c0_ = tid - grp * cols;
    float4 A[KC];
    float M = -INFINITY, L = 0.f;   // of row tid / 16, in its 16 lanes
#pragma unroll
    for (int k = 0; k < KC; ++k) A[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p0 = 0; p0 < parts; p0 += kMergeParts) {
      const int cnt = min(kMergeParts, parts - p0);
      uint4 x[KC][kMergeBatch];
      auto fetch = [&](int k0) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < KC; ++k) {
          const int c = min(c0_ + k * TH, cols - 1);
#pragma unroll
          for (int i = 0; i < kMergeBatch; ++i)
            x[k][i] = ld16_sys(pr, (uint32_t)rec_of(p0 + min(grp + ng * (k0 + i), cnt - 1)) *
                                           (ROWS * REC * 4) +
                                       (c / (D / 4)) * (REC * 4) + (c % (D / 4)) * 16);
        }
      };
      if (grp < ng) fetch(0);
      const int r = tid >> 4, j = tid & 15;
      if (r < used) {
        float mi[4], li[4], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = j + 16 * i < cnt;
          const float* p = a.partial + ((size_t)rec_of(p0 + (in ? j + 16 * i : 0)) * ROWS + r) * REC + D;
          mi[i] = in ? load_sys(p) : -INFINITY;
          li[i] = in ? load_sys(p + 1) : 0.f;
          top = fmaxf(top, mi[i]);
        }
        const float Mn = fmaxf(M, group16_max(top)), Mb = Mn == -INFINITY ? 0.f : Mn;
        const float f = ex2(M - Mb);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float g = ex2(mi[i] - Mb);
          s_f[j + 16 * i][r] = g;
          sum = fmaf(li[i], g, sum);
        }
        L = fmaf(L, f, group16_sum(sum));
        M = Mn;
        if (j == 0) s_c[r] = f;
      }
      __syncthreads();
      if (grp < ng) {
#pragma unroll
        for (int k = 0; k < KC; ++k) {
          const float f = s_c[min(c0_ + k * TH, cols - 1) / (D / 4)];
          A[k].x *= f;
          A[k].y *= f;
          A[k].z *= f;
          A[k].w *= f;
        }
        for (int k0 = 0; grp + ng * k0 < cnt; k0 += kMergeBatch) {
          if (k0) fetch(k0);
#pragma unroll
          for (int k = 0; k < KC; ++k) {
            const int row = min(c0_ + k * TH, cols - 1) / (D / 4);
#pragma unroll
            for (int i = 0; i < kMergeBatch; ++i) {
              const int p = grp + ng * (k0 + i);
              if (p < cnt) {
                const float g = s_f[p][row];
                A[k].x = fmaf(__uint_as_float(x[k][i].x), g, A[k].x);
                A[k].y = fmaf(__uint_as_float(x[k][i].y), g, A[k].y);
                A[k].z = fmaf(__uint_as_float(x[k][i].z), g, A[k].z);
                A[k].w = fmaf(__uint_as_float(x[k][i].w), g, A[k].w);
              }
            }
          }
        }
      }
      __syncthreads();
    }
    if (tid < 16 * used && (tid & 15) == 0) s_fin[tid >> 4][D + 1] = L;
#pragma unroll
    for (int k = 0; k < KC; ++k) {
      const int c = c0_ + k * TH;
      if (grp < ng && c < cols) *(float4*)&s_o[grp][c / (D / 4)][c % (D / 4) * 4] = A[k];
    }
    __syncthreads();
    for (int e = tid; e < used * D; e += TH) {
      float y = 0.f;
      for (int g = 0; g < ng; ++g) y += s_o[g][e / D][e % D];
      s_fin[e / D][e % D] = y;
    }
    __syncthreads();
  }
  for (int e = tid; e < used * D; e += TH) {
    const int r = e / D, d = e % D;
    const float L = s_fin[r][D + 1];
    const float y = L == 0.f ? 0.f : attn_div(s_fin[r][d], L);   // nothing seen: 0; a NaN stays
    const int row = row0 + r;
    const int64_t at = ((int64_t)(c0 + row / a.group) * a.hq + h * a.group + row % a.group) * D + d;
    if (a.out) a.out[at] = f32_to_bf16(y);
    if (a.out_f32) a.out_f32[at] = y;
  }
}

// One token per sequence. The group's heads are the rows of a score tile, spread so that a lane holds
// R = ceil(heads / 4) of them for one position (head 4 i + kg in register i), and all that belongs to a
// position, its scales and the exponentials, is done once per head and position:
//   S[head][pos] = d_g (c . q)_g + m_g (sum of q)_g, summed over g;   C starts at -128 (sum of q)_g
//   O^T[dim][head] += c^T[dim][pos] . (p d_g)^T[pos][head];  sum p (m_g - 16 d_g) apart, per lane
// p d_g goes through LDS from rows to columns: a lane's pair (position n, 16 + n) is an operand
// register as it is, so the writes are consecutive dwords and an operand one 16-byte read. The scales
// are one load of 4 NG bytes a lane (K's positions in lanes 0..31, V's in 32..63), spread by lane swaps.
// A tile is 169 instructions of the VALU and 12 of the matrix cores (315 and 24 at D = 128), a third of them to
// take the codes apart. 8 sequences of up to 65536 positions, 180 MB, take 43 to 46 us, 4.0 to 4.2 TB/s of the
// 6.5 that a plain read reaches: the VALU is active in 0.77 of the busy cycles (what is found before the tiles
// and merged behind them makes it 222 instructions a tile), the matrix cores in 0.16, and the 2.4 waves a SIMD
// wait 0.30 of their time. 16 of up to 5003 at D = 128, 52 MB, take 20 us: VALU 0.50, matrix cores 0.10; 1.8 waves
// a SIMD, which wait half of their time, are too few. Short calls are a chain of latencies: 1 x 513 takes 8.0.
// A wave takes every fourth tile of its part; a lane finds the page of one of the wave's next 64
// tiles, so table and list are read ahead, and two tiles are in flight while one is computed.
//
// Who does what is decided here, from the lengths as they are. Of W tiles in all a part has W / 768 (D = 64;
// 512 at 128: what the chip holds at once, less half a part for each item) of one (sequence, kv head), at
// least 8 (W < 1024) or 16, at most 128 and no more than 32 parts an item as a mean; from 16384 tiles on, if
// that is more than 256 (64 at 128) for each item, the W tiles are one line that 768 (512) workgroups cut
// evenly, so that lengths however unlike load the chip alike, and a workgroup's stretch may end one item
// and begin the next. Times in us with 40 heads of 8 kv heads, line / parts: b8 x 65536 45.6 / 50.2,
// b1 x 131072 34 / 38, b32 x 8192 38 / 28, b64 x 4096 48 / 32; 64 heads of D = 128, b32 x 8192 56 / 63. In
// parts of 32 tiles as against W / 512, 32 heads of D = 128, b16 x 5003: 22.3 / 20.4.
// Known from the call's sizes, items of at most 32 tiles are one part each, and from 512 items on of at
// most 64, and nothing is looked for: b1 x 513 8.0 (9.0 in three parts), b1 x 640 8.1 (9.0), b64 x 1024 12.0
// (15.8), b64 x 2048 19.2 (21.6), b2040 x 128 107 (292); but b1 x 1300 11.9 (9.3 in parts), b16 x 2048 15.6
// (12.4). Near the line few items lose a little: b1 x 770 9.3 (9.0 in four parts), x 1024 10.0 (9.1), b8 alike.

// x / y for quotients below 2^20 or so: the reciprocal is off by less than one in them.
__device__ __forceinline__ int div_few(int x, int y) {
  int q = (int)((float)x * __builtin_amdgcn_rcpf((float)y));
  q -= q * y > x;
  q += (q + 1) * y <= x;
  return q;
}

// Inclusive sum over the lanes of a wave.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);   // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);   // lane 15 to the next row
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);   // lane 31 to the upper half
  return x;
}

template <int NG, int R>
__global__ __launch_bounds__(256) void kv4_decode_kernel(Kv4AttnArgs a) {
  constexpr int D = 32 * NG, C = D / 64, NT = D / 16, PF = 2, H = 4 * R;
  constexpr int kLine = kv4_line(D);
  __shared__ __attribute__((aligned(16))) float s_o[kWaves][H][D + 4];
  __shared__ __attribute__((aligned(16))) float s_fin[H][D + 4];
  __shared__ __attribute__((aligned(16))) uint32_t s_p[kWaves][NG][2][H * 16];
  __shared__ float s_x[kWaves][NG + 1][H];   // sums of p (m - 16 d), and a move of the reference
  __shared__ int s_last;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, kg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tpp = a.c.tiles, nb = a.c.n_seqs, hkv = a.c.hkv;
  auto len_of = [&](int b) { return b < nb ? max(0, min(a.lens[b], a.c.cap)) : 0; };
  auto tiles_of = [&](int len) {
    return a.sel ? a.n_sel * tpp : max(1, (len + kKv4Tile - 1) / kKv4Tile);
  };
  const int len0 = len_of(lane);   // of the first 64 sequences, the only ones as a rule
  // x(tiles) summed over the sequences up to the one whose hkv shares hold `target`: that sequence,
  // what lies before it, its x and length (no such one: all sequences)
  struct Where {
    int b, before, x, len;
  };
  auto find = [&](int target, auto&& x) {
    Where r{nb, 0, 0, 0};
    if (nb <= 64) {
      const int mine = lane < nb ? x(tiles_of(len0)) : 0, sum = wave_scan(mine);
      const unsigned long long hit = __ballot(lane < nb && sum * hkv > target);
      if (hit) {
        r.b = __builtin_ctzll(hit);
        r.x = __builtin_amdgcn_readlane(mine, r.b);
        r.len = __builtin_amdgcn_readlane(len0, r.b);
        r.before = __builtin_amdgcn_readlane(sum, r.b) - r.x;
      } else {
        r.before = __builtin_amdgcn_readlane(sum, 63);
      }
      return r;
    }
    for (int c = 0; c < nb; c += 256) {   // four sequences a lane
      int len[4], mine[4], all = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) len[j] = len_of(c + 4 * lane + j);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        mine[j] = c + 4 * lane + j < nb ? x(tiles_of(len[j])) : 0;
        all += mine[j];
      }
      const int sum = wave_scan(all);
      const unsigned long long hit = __ballot((r.before + sum) * hkv > target);
      if (hit) {   // the first lane that passes the target does so at one of its sequences
        const int l0 = __builtin_ctzll(hit);
        r.before += __builtin_amdgcn_readlane(sum - all, l0);
        r.b = c + 4 * l0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          r.x = __builtin_amdgcn_readlane(mine[j], l0);
          r.len = __builtin_amdgcn_readlane(len[j], l0);
          if ((r.before + r.x) * hkv > target) break;
          r.before += r.x;
          ++r.b;
        }
        return r;
      }
      r.before += __builtin_amdgcn_readlane(sum, 63);
    }
    return r;
  };
  const int W = a.unit ? 0 : find(0x7FFFFFFF, [](int x) { return x; }).before * hkv;
  const bool line = a.unit == 0 && W > kLineTiles && W > (int64_t)kv4_line_mean(D) * nb * hkv;
  if (line && (int)blockIdx.x >= kLine) return;
  // parts of their own: as many as the chip holds at once (half of an item's last part is empty as a mean)
  const int room = max(kLine - nb * hkv / 2, kLine / 2);
  const int unit = a.unit ? a.unit
                   : line ? (W + kLine - 1) / kLine
                          : min(max(max((W + room - 1) / room, W / (kMostParts * nb * hkv)),
                                    W < 1024 ? 8 : 16), kMostTiles);
  auto share = [&](int x) { return line ? x : div_few(x + unit - 1, unit); };

  for (int at = blockIdx.x * (line ? unit : 1), left = line ? unit : 1;;) {
  Where f{at / hkv, at / hkv, 1, 0};
  if (a.whole) f.len = len_of(f.b);
  else f = find(at, share);
  if (f.b >= nb) return;
  const int b = f.b, end = f.len, nt = tiles_of(f.len);
  const int rem = at - f.before * hkv;
  const int h = div_few(rem, f.x), in = rem - h * f.x;
  const int take = line ? min(left, f.x - in) : 1;
  // the item's parts, this one, its tiles, the workgroup of its first part
  const int off = at - in, rec0 = line ? off / unit : off;
  const int part = line ? (int)blockIdx.x - rec0 : in;
  const int parts = line ? (off + f.x - 1) / unit - rec0 + 1 : f.x;
  const int first = line ? in : in * unit, stop = line ? in + take : min(nt, (in + 1) * unit);
  const int item = b * hkv + h;

  // q (of the negative scale's sign) as the rows of a tile: row 4 kg + i is head 4 i + kg
  u32x4_t q[NG];
  f32x4_t z[NG];
  float qs[NG][R];
  {
    const int head = 4 * (n & 3) + (n >> 2);
    const bool live = (n & 3) < R && head < a.group;
    const uint16_t* p = a.q + (int64_t)b * a.q_stride + (h * a.group + (live ? head : 0)) * D + 8 * kg;
    const uint32_t sign = a.scale_l2 < 0.f ? 0x80008000u : 0u;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      q[g] = *(const u32x4_t*)(p + 32 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) q[g][i] = live ? q[g][i] ^ sign : 0u;
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) s += bf16lo(q[g][i]) + bf16hi(q[g][i]);
      s = xor32_sum(xor16_sum(s));
      z[g] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < R; ++i) {
        qs[g][i] = __shfl(s, 4 * kg + i);
        z[g][i] = -128.f * qs[g][i];
      }
    }
  }
  const float scale = fabsf(a.scale_l2);
  f32x4_t o[NT];
  float ms[NG][R], m[R], mb[R], lim[R], l[R];
#pragma unroll
  for (int u = 0; u < NT; ++u) o[u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < R; ++i) {
    m[i] = lim[i] = -INFINITY;
    mb[i] = l[i] = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) ms[g][i] = 0.f;
  }
  const Kv4Minus neg;
  const int t0 = first + wave, t1 = stop;
  const int64_t head_off = (int64_t)h * kv4_head_bytes(a.c.page_len, D);
  // the operand this lane reads: row n of s_p (rows past H again the first ones)
  const uint32_t p_at = (uint32_t)((n % H) * 16 + 4 * kg);

  for (int i0 = 0; t0 + kWaves * i0 < t1; i0 += 64) {
    const int count = min(64, (t1 - t0 - kWaves * i0 + kWaves - 1) / kWaves);
    // this lane's tile: its page, and its first position (past every length when there is none)
    int id = 0, pos = 1 << 30;
    if (lane < count) {
      const int t = t0 + kWaves * (i0 + lane);
      const int e = t >> a.c.shift, sub = t & (tpp - 1);
      const int lp = a.sel ? a.sel[(int64_t)item * a.n_sel + e] : e;
      if (lp >= 0 && lp < a.c.table_len) {
        id = kv4_page(a.c, b, lp) * 4 + sub;   // negative: no page
        pos = lp * a.c.page_len + sub * kKv4Tile;
      }
    }
    Kv4TileRegs<NG> buf[PF];
    auto load = [&](Kv4TileRegs<NG>& r, int i) __attribute__((always_inline)) {
      const int x = __builtin_amdgcn_readlane(id, i);
      const uint8_t* tile = a.c.pages + (int64_t)(x < 0 ? 0 : x >> 2) * a.c.page_stride + head_off +
                            (x < 0 ? 0 : x & 3) * kv4_tile_bytes(D);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        r.k[c] = *(const u32x4_t*)(tile + (c * 64 + lane) * 16);
        r.v[c] = *(const u32x4_t*)(tile + 16 * D + (c * 64 + lane) * 16);
      }
      if constexpr (NG == 2) {
        const uint2 s = *(const uint2*)(tile + 32 * D + lane * 8);
        r.s[0] = s.x;
        r.s[1] = s.y;
      } else {
        const u32x4_t s = *(const u32x4_t*)(tile + 32 * D + lane * 16);
#pragma unroll
        for (int g = 0; g < 4; ++g) r.s[g] = s[g];
      }
    };
    auto compute = [&](const Kv4TileRegs<NG>& r, int i0_) __attribute__((always_inline)) {
      const int base = __builtin_amdgcn_readlane(pos, i0_);
      const bool none = __builtin_amdgcn_readlane(id, i0_) < 0;
      const bool part = base + kKv4Tile > end || none;
      uint32_t w[NG], sc[2][2][NG];   // [K, V][tt]: this lane's position's scales
#pragma unroll
      for (int g = 0; g < NG; ++g) w[g] = r.s[g];
      if (part) {
        // masked positions' scales may be anything (the page's older bytes)
        const bool seen = base + (lane & 31) < end;
#pragma unroll
        for (int g = 0; g < NG; ++g) w[g] = seen ? (none ? kKv4NaN : w[g]) : 0u;
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const auto x = __builtin_amdgcn_permlane16_swap(w[g], w[g], false, false);
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
          const auto y = __builtin_amdgcn_permlane32_swap(x[tt], x[tt], false, false);
          sc[0][tt][g] = y[0];
          sc[1][tt][g] = y[1];
        }
      }
      float s[2][R];
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
        for (int i = 0; i < R; ++i) s[tt][i] = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const f32x4_t y = mfma_bf16(q[g], kv4_operand(r.k[g >> 1][2 * tt + (g & 1)]), z[g]);
          const float d = bf16lo(sc[0][tt][g]), mm = bf16hi(sc[0][tt][g]);
#pragma unroll
          for (int i = 0; i < R; ++i) s[tt][i] = fmaf(d, y[i], fmaf(mm, qs[g][i], s[tt][i]));
        }
      }
      if (part) {
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
          if (base + 16 * tt + n >= end)
#pragma unroll
            for (int i = 0; i < R; ++i) s[tt][i] = -INFINITY;
      }
      // a head's reference moves only when a score has passed it by 2^8: sums stay far from overflow
      float top[R];
      bool move = false;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        top[i] = fmaxf(s[0][i], s[1][i]) * scale;
        move |= top[i] > lim[i];
      }
      if (__any(move)) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const float mn = fmaxf(m[i], group16_max(top[i]));
          const float nb_ = mn == -INFINITY ? 0.f : mn;
          const float f_ = ex2(m[i] - nb_);
          m[i] = mn;
          mb[i] = nb_;
          lim[i] = mn + 8.f;
          l[i] *= f_;
#pragma unroll
          for (int g = 0; g < NG; ++g) ms[g][i] *= f_;
          if (n == 0) s_x[wave][NG][4 * i + kg] = f_;
        }
        __builtin_amdgcn_wave_barrier();
        const float f_ = s_x[wave][NG][n % H];
#pragma unroll
        for (int u = 0; u < NT; ++u) o[u] *= f_;
        __builtin_amdgcn_wave_barrier();
      }
      float p[2][R];
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int i = 0; i < R; ++i) p[tt][i] = ex2(fmaf(s[tt][i], scale, -mb[i]));
      if (part) {
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
          if (base + 16 * tt + n >= end)
#pragma unroll
            for (int i = 0; i < R; ++i) p[tt][i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < R; ++i) l[i] += p[0][i] + p[1][i];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float d0 = bf16lo(sc[1][0][g]), d1 = bf16lo(sc[1][1][g]);
        const float m0 = fmaf(-16.f, d0, bf16hi(sc[1][0][g]));
        const float m1 = fmaf(-16.f, d1, bf16hi(sc[1][1][g]));
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const float x0 = p[0][i] * d0, x1 = p[1][i] * d1;
          ms[g][i] = fmaf(p[0][i], m0, fmaf(p[1][i], m1, ms[g][i]));
          const uint32_t hi = pack_bf16x2_op(x0, x1);
          s_p[wave][g][0][64 * i + lane] = hi;
          s_p[wave][g][1][64 * i + lane] =
              pack_bf16x2_op(Kv4Minus::dot(x0, hi, neg.lo), Kv4Minus::dot(x1, hi, neg.hi));
        }
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const u32x4_t hi = *(const u32x4_t*)&s_p[wave][g][0][p_at];
        const u32x4_t lo = *(const u32x4_t*)&s_p[wave][g][1][p_at];
#pragma unroll
        for (int u = 2 * g; u < 2 * g + 2; ++u) {
          const u32x4_t v = kv4_operand16(r.v[u >> 2][u & 3]);
          o[u] = mfma_bf16(v, hi, o[u]);
          o[u] = mfma_bf16(v, lo, o[u]);
        }
      }
      __builtin_amdgcn_wave_barrier();
    };
    // loads stand outside every branch (the last tile again behind the end): the wait for a tile then
    // leaves the younger loads in flight
#pragma unroll
    for (int j = 0; j < PF; ++j) load(buf[j], min(j, count - 1));
    for (int i = 0; i < count; i += PF) {
#pragma unroll
      for (int j = 0; j < PF; ++j) {
        if (i + j < count) compute(buf[j], i + j);
        load(buf[j], min(i + j + PF, count - 1));
      }
    }
  }

#pragma unroll
  for (int i = 0; i < R; ++i) {
    l[i] = group16_sum(l[i]);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      ms[g][i] = group16_sum(ms[g][i]);
      if (n == 0) s_x[wave][g][4 * i + kg] = ms[g][i];
    }
    if (n == 0) {
      s_o[wave][4 * i + kg][D] = m[i];
      s_o[wave][4 * i + kg][D + 1] = l[i];
    }
  }
  __builtin_amdgcn_wave_barrier();
  if (n < H) {
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const float y = s_x[wave][u >> 1][n];
      *(float4*)&s_o[wave][n][16 * u + 4 * kg] =
          make_float4(o[u][0] + y, o[u][1] + y, o[u][2] + y, o[u][3] + y);
    }
  }
  // a workgroup has at most one part that another began and one that another goes on with
  auto rec_of = [&](int p) { return line ? 2 * (rec0 + p) + (p == 0) : rec0 + p; };
  kv4_finish<D, 256, kWaves, H>(a, s_o, s_fin, &s_last, item, part, parts, rec_of, a.group, b, 0, h);
  at += take;
  left -= take;
  if (left <= 0) return;
  __syncthreads();
  }
}

// Blocks of new tokens. A workgroup has RB = 16 CT NW query rows (token, head of the group) of one
// (sequence, kv head), a wave CT tiles of 16; all of them share each tile of the cache, which the waves
// take apart together, once, into operands in LDS:
//   K = (d c + m) scale log2(e) and V = d c + m, each as two bf16 terms (2^-18 of the value)
//   S^T[pos][row] = K . Q^T - reference,  O^T[dim][row] += V^T . P^T with P as two terms (hi hi, lo hi,
//   hi lo: 20 products of 16 x 16 x 32 for 32 positions, 16 rows and D = 64)
// The reference is the accumulator's start, so an exponential is one instruction a score. A score tile's
// lanes hold rows as columns and positions 4 kg + e and 16 + 4 kg + e, the order of V's operand, so P
// goes from registers to registers. While a tile is computed the next one's bytes are on their way, and
// its operands are written to the other buffer: one barrier a tile.
// A wave's tile is 640 cycles of the matrix cores and 650 of the VALU (exponentials, P's terms). 8192 tokens,
// 40 heads of 8 kv heads: 720 us, 478 TFLOP/s of the attention's own and 1.2 PFLOP/s of products, the matrix
// cores busy in 0.57 of the busy cycles and the VALU in 0.59 at three waves a SIMD (a library's bf16 product
// reaches 1.24 to 1.28); 32 heads of D = 128 1056 us, 520 TFLOP/s, 0.58 and 0.39 at two waves.
// 2048 tokens: 87 us, 0.34, bound by the longest row block's 64 tiles of 1.3 us.
// Poison: in tiles that some rows do not see, V's groups of NaN are left out of the product (0 times
// NaN) and given to the rows that see them.
template <int D>
constexpr int kv4_block_waves() { return 4; }
constexpr int kBlockCt = 2;   // at 4 long prompts take 2 % less, short ones 40 % more
template <int D>
constexpr int kv4_block_rows() { return 16 * kBlockCt * kv4_block_waves<D>(); }

// A tile taken apart: a wave's dword of every lane's four of K and of V (C chunks of 64 channels).
template <int NG>
struct Kv4Apart {
  static constexpr int D = 32 * NG, C = NG / 2, KJ = 2 * NG;
  uint32_t kc[C], ks[C], vc[C], vs[C][8];

  __device__ __forceinline__ void fetch(const uint8_t* tile, int wave, int lane) {
    const int n = lane & 15, kg = lane >> 4, ktt = wave >> 1, kgg = wave & 1;
    const uint8_t* pc = tile + lane * 16 + wave * 4;
    const uint8_t* pk = tile + 32 * D + ((16 * ktt + n) * NG + kgg) * 4;
    const uint8_t* pv = tile + 32 * D + 128 * NG + kg * 16 * NG + (wave >> 1) * 4;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      kc[c] = *(const uint32_t*)(pc + c * 1024);
      vc[c] = *(const uint32_t*)(pc + 16 * D + c * 1024);
      ks[c] = *(const uint32_t*)(pk + c * 8);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        vs[c][e] = *(const uint32_t*)(pv + c * 8 + (16 * (e >> 2) + (e & 3)) * NG * 4);
    }
  }
  __device__ __forceinline__ void poison() {   // an entry that names no page
#pragma unroll
    for (int c = 0; c < C; ++c) {
      ks[c] = kKv4NaN;
#pragma unroll
      for (int e = 0; e < 8; ++e) vs[c][e] = kKv4NaN;
    }
  }
  // V without its NaN groups, and without positions from `seen` (of this tile's 32) on, which may hold
  // anything (the page's older bytes); f(group, NaN positions) once for each group
  template <typename F>
  __device__ __forceinline__ void clean(int seen, int wave, int lane, F&& f) {
    const int kg = lane >> 4;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      uint32_t bad = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int p = 16 * (e >> 2) + 4 * kg + (e & 3);
        const bool out = p >= seen, nan = !(fabsf(bf16lo(vs[c][e]) + bf16hi(vs[c][e])) < INFINITY);
        if (!out && nan) bad |= 1u << p;
        if (out || nan) vs[c][e] = 0u;
      }
      bad |= (uint32_t)__shfl_xor((int)bad, 16);
      bad |= (uint32_t)__shfl_xor((int)bad, 32);
      if (lane == 0 && (wave & 1) == 0) f(2 * c + (wave >> 1), bad);
    }
  }
  // out(dword, high terms, low terms): K's 2 NG, then V's
  template <typename F>
  __device__ __forceinline__ void spread(float scale, int wave, const Kv4Minus& neg, F&& out) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const float d = bf16lo(ks[c]) * scale, m = bf16hi(ks[c]) * scale;
      u32x4_t hi, lo;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        uint32_t y0, y1;
        neg.split(fmaf((float)((kc[c] >> (4 * r)) & 15u), d, m),
                  fmaf((float)((kc[c] >> (4 * r + 16)) & 15u), d, m), y0, y1);
        hi[r] = y0;
        lo[r] = y1;
      }
      out(4 * c + wave, hi, lo);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        uint32_t y0, y1;
        neg.split(fmaf((float)((vc[c] >> (4 * r)) & 15u), bf16lo(vs[c][r]), bf16hi(vs[c][r])),
                  fmaf((float)((vc[c] >> (4 * r + 16)) & 15u), bf16lo(vs[c][4 + r]), bf16hi(vs[c][4 + r])),
                  y0, y1);
        hi[r] = y0;
        lo[r] = y1;
      }
      out(KJ + 4 * c + wave, hi, lo);
    }
  }
};

// Tiles taken apart beforehand, one per workgroup, for calls in which many row blocks read each: 16 KB
// (D = 64) written once in place of some 110 instructions a wave and row block. 8192 tokens: 908 us without,
// 720 with, 16 of them here (1537 and 1056 at D = 128, 32 heads); 2048 tokens 101 and 87; 3 x up to 509 over
// 8191 208 and 163; 512 tokens 27.6 and 26.1.
template <int NG>
__global__ __launch_bounds__(256) void kv4_apart_kernel(Kv4AttnArgs a) {
  constexpr int D = 32 * NG;
  const int t = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int end = max(0, min(a.lens[b], a.c.cap)), lane = threadIdx.x & 63;
  if (t * kKv4Tile >= end) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int id = kv4_page(a.c, b, t >> a.c.shift);
  Kv4Apart<NG> x;
  x.fetch(a.c.pages + (int64_t)max(id, 0) * a.c.page_stride +
              (int64_t)h * kv4_head_bytes(a.c.page_len, D) + (t & (a.c.tiles - 1)) * kv4_tile_bytes(D),
          wave, lane);
  if (id < 0) x.poison();
  const int64_t at = ((int64_t)b * a.c.hkv + h) * a.ops_tiles + t;
  x.clean(end - t * kKv4Tile, wave, lane, [&](int g, uint32_t bad) { a.bad[at * NG + g] = bad; });
  u32x4_t* out = a.ops + at * (4 * NG * 128) + lane;
  const Kv4Minus neg;
  x.spread(a.scale_l2, wave, neg, [&](int j, const u32x4_t& hi, const u32x4_t& lo) {
    out[j * 128] = hi;
    out[j * 128 + 64] = lo;
  });
}

// PRE: the tiles come from kv4_apart_kernel, straight into LDS.
template <int NG, bool PRE>
__global__ __launch_bounds__(64 * kv4_block_waves<32 * NG>()) void kv4_block_kernel(Kv4AttnArgs a) {
  constexpr int D = 32 * NG, NT = D / 16, CT = kBlockCt, NW = kv4_block_waves<D>();
  constexpr int RB = 16 * CT * NW, REC = D + 4, KJ = 2 * NG;
  static_assert(NW == 4 && CT == 2, "a wave takes one dword of four; its row tiles are 2, 1 or 0");
  __shared__ __attribute__((aligned(16))) u32x4_t s_op[2][4 * NG][2][64];   // [buffer][K, V dwords][term][lane]
  __shared__ uint32_t s_bad[2][NG];
  __shared__ int s_last;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, kg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // the row block: of the sequences' blocks in order, in each the rows that see most first
  const int item = blockIdx.x / a.n_split, split = blockIdx.x - item * a.n_split;
  const int h = item % a.c.hkv, index = item / a.c.hkv;
  auto tokens_of = [&](int b) {
    const int from = a.cu[b], n = a.cu[b + 1] - from;
    return from < 0 || n < 0 ? 0 : min(n, a.total - from);
  };
  int b = -1, rb = 0;
  for (int s0 = 0, before = 0; s0 < a.c.n_seqs && b < 0; s0 += 64) {
    const bool in = s0 + lane < a.c.n_seqs;
    const int mine = in ? (max(0, tokens_of(s0 + lane)) * a.group + RB - 1) / RB : 0;
    const int sum = before + wave_scan(mine);
    const unsigned long long hit = __ballot(in && sum > index && sum - mine <= index);
    if (hit) {
      const int l0 = __builtin_ctzll(hit);
      b = s0 + l0;
      rb = __builtin_amdgcn_readlane(sum, l0) - 1 - index;
    }
    before = __builtin_amdgcn_readlane(sum, 63);
  }
  if (b < 0) return;
  const int c0 = a.cu[b], nq = tokens_of(b);
  const int rows = nq * a.group, row0 = rb * RB;
  const int first_tok = row0 / a.group, last_tok = (min(row0 + RB, rows) - 1) / a.group;
  auto sees = [&](int tok) { return max(0, min(max(a.lens[b], 0) - nq + tok + 1, a.c.cap)); };
  const int top = sees(last_tok), all_see = sees(first_tok);
  const int nt = (top + kKv4Tile - 1) / kKv4Tile;
  const int parts = max(1, (nt + a.chunk - 1) / a.chunk);
  if (split >= parts) return;
  const int t_begin = split * a.chunk, t_end = min(nt, (split + 1) * a.chunk);

  u32x4_t q[CT][NG];
  int end[CT], tiles_w = 0;   // positions a row sees; this wave's tiles of rows
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int r0 = row0 + (c * NW + wave) * 16, row = r0 + n;
    if (r0 < rows) tiles_w = c + 1;
    const bool live = row < rows;
    const int tok = live ? row / a.group : 0, qh = live ? row % a.group : 0;
    end[c] = live ? sees(tok) : 0;
    const uint16_t* p = a.q + (int64_t)(c0 + tok) * a.q_stride + (h * a.group + qh) * D + 8 * kg;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      q[c][g] = *(const u32x4_t*)(p + 32 * g);
      if (!live) q[c][g] = u32x4_t{0, 0, 0, 0};
    }
  }
  f32x4_t o[CT][NT], nref[CT];   // the negative reference, four times; 0 while there is none
  int lim[CT];                   // the word of 8, what a score may pass it by; while there is none, the least
  float l[CT];
  constexpr int kLimit = 0x41000000;
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    nref[c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    lim[c] = INT32_MIN;
    l[c] = 0.f;
#pragma unroll
    for (int u = 0; u < NT; ++u) o[c][u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  const Kv4Minus neg;

  // ---- a tile's operands into a buffer: taken apart here, or copied
  Kv4Apart<NG> x_;
  int id_now = 0, id_next = 0;
  uint32_t bad_now[NG], bad_next[NG];
  const int64_t ops0 = ((int64_t)b * a.c.hkv + h) * a.ops_tiles;
  auto page = [&](int t) __attribute__((always_inline)) { return kv4_page(a.c, b, t >> a.c.shift); };
  auto fetch = [&](int t, int id) __attribute__((always_inline)) {
    x_.fetch(a.c.pages + (int64_t)max(id, 0) * a.c.page_stride +
                 (int64_t)h * kv4_head_bytes(a.c.page_len, D) +
                 (t & (a.c.tiles - 1)) * kv4_tile_bytes(D),
             wave, lane);
  };
  auto spread = [&](int t, int id, int buf) __attribute__((always_inline)) {
    if (id < 0) x_.poison();
    if ((t + 1) * kKv4Tile > all_see)
      x_.clean(top - t * kKv4Tile, wave, lane, [&](int g, uint32_t bad) { s_bad[buf][g] = bad; });
    x_.spread(a.scale_l2, wave, neg, [&](int j, const u32x4_t& hi, const u32x4_t& lo) {
      s_op[buf][j][0][lane] = hi;
      s_op[buf][j][1][lane] = lo;
    });
  };
  auto copy = [&](int t, int buf) __attribute__((always_inline)) {
    const u32x4_t* from = a.ops + (ops0 + t) * (4 * NG * 128) + wave * (2 * NG * 64) + lane;
    u32x4_t* to = &s_op[buf][wave * NG][0][0];
#pragma unroll
    for (int i = 0; i < 2 * NG; ++i)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + 64 * i),
                                       (__attribute__((address_space(3))) void*)(to + 64 * i), 16, 0, 0);
#pragma unroll
    for (int g = 0; g < NG; ++g) bad_next[g] = a.bad[(ops0 + t) * NG + g];
  };
  // one tile for the first N of this wave's row tiles; part: some rows do not see all of it (the empty
  // asm keeps what follows from being done for every tile and selected)
  auto compute = [&](auto n_tiles, int t, int buf) __attribute__((always_inline)) {
    constexpr int N = decltype(n_tiles)::value;
    const int base = t * kKv4Tile;
    const bool part = base + kKv4Tile > all_see;
    f32x4_t s[N][2];
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        const int j = 4 * (g >> 1) + 2 * tt + (g & 1);
        const u32x4_t hi = s_op[buf][j][0][lane], lo = s_op[buf][j][1][lane];
#pragma unroll
        for (int c = 0; c < N; ++c) s[c][tt] = mfma_bf16(hi, q[c][g], g == 0 ? nref[c] : s[c][tt]);
#pragma unroll
        for (int c = 0; c < N; ++c) s[c][tt] = mfma_bf16(lo, q[c][g], s[c][tt]);
      }
    if (part) {
      asm volatile("");
#pragma unroll
      for (int c = 0; c < N; ++c)
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (base + 16 * tt + 4 * kg + e >= end[c]) s[c][tt][e] = -INFINITY;
    }
    // The reference moves only when a score has passed it by 2^8: sums stay far from overflow. As signed
    // words, floats compare alike where one is positive, which is all that is asked here (a NaN's word is
    // greater than any), and take no canonicalising step.
    bool move = false;
#pragma unroll
    for (int c = 0; c < N; ++c) {
      int y = __float_as_int(s[c][0][0]);
#pragma unroll
      for (int e = 1; e < 8; ++e) y = max(y, __float_as_int(s[c][e >> 2][e & 3]));
      move |= y > lim[c];
    }
    if (__any(move)) {
#pragma unroll
      for (int c = 0; c < N; ++c) {
        float y = s[c][0][0];
#pragma unroll
        for (int e = 1; e < 8; ++e) y = fmaxf(y, s[c][e >> 2][e & 3]);
        y = xor32_max(xor16_max(y));
        const bool first = lim[c] != kLimit, now = y > (first ? -INFINITY : 0.f);
        const float by = now ? y : 0.f, f = now && first ? 0.f : ex2(-by);
        if (now) lim[c] = kLimit;
        l[c] *= f;
#pragma unroll
        for (int u = 0; u < NT; ++u) o[c][u] *= f;
        nref[c] -= by;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) s[c][tt] -= by;
      }
    }
    u32x4_t ph[N], pl[N];
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p0 = ex2(s[c][0][e]), p1 = ex2(s[c][1][e]);
        l[c] += p0 + p1;
        uint32_t y0, y1;
        neg.split(p0, p1, y0, y1);
        ph[c][e] = y0;
        pl[c][e] = y1;
      }
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const u32x4_t hi = s_op[buf][KJ + u][0][lane], lo = s_op[buf][KJ + u][1][lane];
#pragma unroll
      for (int c = 0; c < N; ++c) o[c][u] = mfma_bf16(hi, ph[c], o[c][u]);
#pragma unroll
      for (int c = 0; c < N; ++c) o[c][u] = mfma_bf16(hi, pl[c], o[c][u]);
#pragma unroll
      for (int c = 0; c < N; ++c) o[c][u] = mfma_bf16(lo, ph[c], o[c][u]);
    }
    if (PRE || part) {
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t bad = PRE ? bad_now[g] : s_bad[buf][g];
        if (bad == 0) continue;
#pragma unroll
        for (int c = 0; c < N; ++c) {
          // the row's positions of this tile are the first end - base
          const int k = end[c] - base;
          const uint32_t mine = k >= 32 ? bad : k <= 0 ? 0u : bad & ((1u << k) - 1u);
          if (mine) {
#pragma unroll
            for (int u = 2 * g; u < 2 * g + 2; ++u) o[c][u] += NAN;
          }
        }
      }
    }
  };

  if (t_begin < t_end) {
    if constexpr (PRE) {
      copy(t_begin, 0);
      wait_vm();
    } else {
      id_now = page(t_begin);
      fetch(t_begin, id_now);
      id_next = page(min(t_begin + 1, t_end - 1));
      spread(t_begin, id_now, 0);
    }
  }
  __syncthreads();
  auto run = [&](auto n_tiles) __attribute__((always_inline)) {
    for (int t = t_begin; t < t_end; ++t) {
      const int buf = (t - t_begin) & 1;
      if constexpr (PRE) {
#pragma unroll
        for (int g = 0; g < NG; ++g) bad_now[g] = bad_next[g];
        if (t + 1 < t_end) copy(t + 1, buf ^ 1);
        if constexpr (decltype(n_tiles)::value > 0) compute(n_tiles, t, buf);
        wait_vm();
      } else {
        id_now = id_next;
        fetch(min(t + 1, t_end - 1), id_now);
        id_next = page(min(t + 2, t_end - 1));
        if constexpr (decltype(n_tiles)::value > 0) compute(n_tiles, t, buf);
        if (t + 1 < t_end) spread(t + 1, id_now, buf ^ 1);
      }
      __syncthreads();
    }
  };
  if (tiles_w == 2) run(std::integral_constant<int, 2>{});
  else if (tiles_w == 1) run(std::integral_constant<int, 1>{});
  else run(std::integral_constant<int, 0>{});

  // ---- rows out: a lane has four channels of its row in each o[u]
#pragma unroll
  for (int c = 0; c < CT; ++c) l[c] = xor32_sum(xor16_sum(l[c]));
  if (parts == 1) {
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const int row = row0 + (c * NW + wave) * 16 + n;
      if (row >= rows) continue;
      const int64_t at = ((int64_t)(c0 + row / a.group) * a.hq + h * a.group + row % a.group) * D + 4 * kg;
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = l[c] == 0.f ? 0.f : attn_div(o[c][u][e], l[c]);
        if (a.out)
          *(uint2*)(a.out + at + 16 * u) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
        if (a.out_f32) *(float4*)(a.out_f32 + at + 16 * u) = make_float4(y[0], y[1], y[2], y[3]);
      }
    }
    return;
  }
  const __amdgpu_buffer_rsrc_t pr = make_rsrc(a.partial, a.partial_bytes);
  const uint32_t rec0 = (uint32_t)item * a.n_split * (RB * REC * 4);
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int r = (c * NW + wave) * 16 + n;
    if (row0 + r >= rows) continue;
    const uint32_t at = rec0 + (uint32_t)(split * RB + r) * (REC * 4);
#pragma unroll
    for (int u = 0; u < NT; ++u)
      st16_sys(pr, at + (16 * u + 4 * kg) * 4,
               make_uint4(__float_as_uint(o[c][u][0]), __float_as_uint(o[c][u][1]),
                          __float_as_uint(o[c][u][2]), __float_as_uint(o[c][u][3])));
    if (kg == 0)
      st16_sys(pr, at + D * 4, make_uint4(__float_as_uint(lim[c] != kLimit ? -INFINITY : -nref[c][0]),
                                          __float_as_uint(l[c]), 0u, 0u));
  }
  wait_vm();
  __syncthreads();
  if (tid == 0) s_last = ticket(&a.counters[item], parts) ? 1 : 0;
  __syncthreads();
  if (!s_last) return;
  // Two threads a row find the parts' weights, then a thread sums four channels of eight rows at a time,
  // sixteen records in flight. The operands' buffers hold the weights.
  constexpr int PB = 32, RT = 64 * NW * 4 / D, E = 8;   // parts per pass, rows per step, steps
  static_assert(RB % (RT * E) == 0 && sizeof(s_op) >= PB * RB * 4, "the weights fit, rows come out even");
  float(*s_w)[RB] = (float(*)[RB])s_op;
  const int used = min(RB, rows - row0), mine = min(tid >> 1, used - 1);
  float M = -INFINITY, L = 0.f;
  for (int p0 = 0; p0 < parts; p0 += 16) {
    uint4 ml[8];
    float Mn = M;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int p = p0 + 2 * i + (tid & 1);
      ml[i] = ld16_sys(pr, rec0 + (uint32_t)(min(p, parts - 1) * RB + mine) * (REC * 4) + D * 4);
      if (p >= parts) ml[i].x = __float_as_uint(-INFINITY);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) Mn = fmaxf(Mn, __uint_as_float(ml[i].x));
    Mn = fmaxf(Mn, __shfl_xor(Mn, 1));
    const float Mb = Mn == -INFINITY ? 0.f : Mn;
    L *= ex2(M - Mb);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int p = p0 + 2 * i + (tid & 1);
      if (p < parts) L = fmaf(__uint_as_float(ml[i].y), ex2(__uint_as_float(ml[i].x) - Mb), L);
      if (p < min(parts, PB)) s_w[p][tid >> 1] = __uint_as_float(ml[i].x);
    }
    M = Mn;
  }
  L += __shfl_xor(L, 1);
  const float Mb = M == -INFINITY ? 0.f : M;
  __shared__ float s_l[RB];
  if ((tid & 1) == 0) s_l[tid >> 1] = L;
  const int r0 = tid / (D / 4), d = tid % (D / 4) * 4;
  for (int k0 = 0; k0 < used; k0 += RT * E) {   // once at D = 64, twice at 128
    float4 A[E];
#pragma unroll
    for (int k = 0; k < E; ++k) A[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int g0 = 0; g0 < parts; g0 += PB) {
      const int cnt = min(PB, parts - g0);
      __syncthreads();
      if (k0 == 0 || parts > PB) {   // the first ones' references lie there already
        const bool have = k0 == 0 && g0 == 0;
        for (int i = tid & 1; i < cnt; i += 2) {
          const float m = have ? s_w[i][tid >> 1]
                               : __uint_as_float(ld16_sys(pr, rec0 + (uint32_t)((g0 + i) * RB + mine) *
                                                                         (REC * 4) + D * 4).x);
          s_w[i][tid >> 1] = ex2(m - Mb);
        }
      }
      __syncthreads();
      for (int p0 = 0; p0 < cnt; p0 += 2) {
        uint4 v[2][E];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int k = 0; k < E; ++k)
            v[i][k] = ld16_sys(pr, rec0 + (uint32_t)((g0 + min(p0 + i, cnt - 1)) * RB +
                                                     min(k0 + RT * k + r0, used - 1)) * (REC * 4) + d * 4);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (p0 + i < cnt)
#pragma unroll
            for (int k = 0; k < E; ++k) {
              const float g = s_w[p0 + i][k0 + RT * k + r0];
              A[k].x = fmaf(__uint_as_float(v[i][k].x), g, A[k].x);
              A[k].y = fmaf(__uint_as_float(v[i][k].y), g, A[k].y);
              A[k].z = fmaf(__uint_as_float(v[i][k].z), g, A[k].z);
              A[k].w = fmaf(__uint_as_float(v[i][k].w), g, A[k].w);
            }
      }
    }
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const int r = k0 + RT * k + r0, row = row0 + r;
      if (r >= used) continue;
      const float sum = s_l[r];
      float y[4] = {A[k].x, A[k].y, A[k].z, A[k].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = sum == 0.f ? 0.f : attn_div(y[i], sum);
      const int64_t at = ((int64_t)(c0 + row / a.group) * a.hq + h * a.group + row % a.group) * D + d;
      if (a.out) *(uint2*)(a.out + at) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
      if (a.out_f32) *(float4*)(a.out_f32 + at) = make_float4(y[0], y[1], y[2], y[3]);
    }
  }
}

// Row blocks of a call, at most.
static int64_t kv4_row_blocks(int n_seqs, int total, int group, int rows) {
  return n_seqs + (int64_t)total * group / rows;
}
// Workgroups that share a row block's tiles: the number that takes least by what was measured (us at
// D = 64; both terms are twice as long at 128). A tile takes 1.3 where a CU has one workgroup, 1.8 with two
// and 2.2 with the three it can hold; merging 3, 0.5 for each part, and 0.0175 for each record. 64 tokens over
// 8000 positions, 40 heads of 8 kv heads: 49 us in 15 parts, 59 in 8, 65 in 32; 256 tokens 90 in 9,
// 101 in 10 (a second round of workgroups), 311 in one; 4 tokens over 1000 15 in 8, 20 in 3.
static int kv4_block_split(int64_t blocks, int tiles) {
  int best = 1;
  float least = 0.f;
  for (int s = 1; s <= 32 && s <= tiles && (s == 1 || blocks * s <= 768); ++s) {
    const float tile = blocks * s <= 256 ? 1.3f : blocks * s <= 512 ? 1.8f : 2.2f;
    const float merge = s == 1 ? 0.f : 3.f + s * (0.5f + 0.0175f * (float)blocks);
    const float cost = (float)((tiles + s - 1) / s) * tile + merge;
    if (s == 1 || cost < 0.97f * least) {
      best = s;
      least = cost;
    }
  }
  return best;
}

// Bytes that a choice made here asks for, at most: within a default workspace.
constexpr int64_t kMostBytes = 192 << 20;
// Tiles are taken apart beforehand from so many row blocks per sequence (as a mean) on.
constexpr int kApartBlocks = 4;

struct Kv4Plan {
  int64_t items, grid;
  int n_split, chunk, unit;
  bool shared;   // whether an item may be of several parts
  bool whole;    // every item is one part
  size_t bytes;  // workspace, `ops` of it before the tiles taken apart beforehand (0: none are)
  size_t ops;
  int ops_tiles;
};
static Kv4Plan kv4_plan(const q4nx_kv4* c, int n_q_heads, int total, int max_len, int n_sel,
                        int n_split) {
  const bool block = total > 0;   // the rows of blocks, 0: one token per sequence
  Kv4Plan p{};
  const int group = n_q_heads / c->n_kv_heads;
  const int64_t cap = (int64_t)c->table_len * c->page_len;
  const int64_t len = n_sel ? (int64_t)n_sel * c->page_len : (max_len < cap ? max_len : cap);
  const int tiles = (int)((len + kKv4Tile - 1) / kKv4Tile);
  int64_t recs;
  int rows = 16;
  if (block) {
    rows = c->head_dim == 64 ? kv4_block_rows<64>() : kv4_block_rows<128>();
    p.items = c->n_kv_heads * kv4_row_blocks(c->n_seqs, total, group, rows);
    int64_t blocks = ((int64_t)total * group + rows - 1) / rows;   // as a rule: full blocks
    blocks = c->n_kv_heads * (blocks > c->n_seqs ? blocks : c->n_seqs);
    const int want = n_split > 0 ? n_split
                     : p.items * 4 > Q4NX_WS_COUNTER_BYTES ? 1 : kv4_block_split(blocks, tiles);
    p.chunk = (tiles + want - 1) / want;
    p.n_split = (tiles + p.chunk - 1) / p.chunk;   // every split has work at the longest length
    p.grid = recs = p.items * p.n_split;
    p.shared = p.n_split > 1;
  } else {
    p.items = (int64_t)c->n_seqs * c->n_kv_heads;
    rows = (group + 3) / 4 * 4;
    if (n_split > 0) p.unit = (tiles + n_split - 1) / n_split;
    // no counter for each, or short ones (so many of them that they fill the chip and end together)
    else if (p.items * 4 > Q4NX_WS_COUNTER_BYTES || tiles <= kShortTiles ||
             (p.items >= kWholeItems && tiles <= kWholeTiles))
      p.unit = tiles;
    // by what there is: parts of 8 tiles and more, as many as there is room for besides one for each item
    // (or of kMostTiles), or one line
    const int line = kv4_line(c->head_dim);
    const int64_t all = p.items * tiles, room = all / 8 < line ? all / 8 : line;
    const int64_t few = kv4_line_mean(c->head_dim) * p.items, most = (all < few ? all : few) / kMostTiles;
    p.grid = p.unit ? p.items * ((tiles + p.unit - 1) / p.unit)
                    : p.items + (room > most ? room : most);
    if (!p.unit && p.items * ((tiles + 7) / 8) < p.grid) p.grid = p.items * ((tiles + 7) / 8);
    if (!p.unit && all > kLineTiles && p.grid < line) p.grid = line;
    recs = p.grid > 2 * line ? p.grid : 2 * line;
    // cut by the lengths as they are, any item may be of several parts
    p.shared = p.unit < tiles;
  }
  p.bytes = p.shared ? (size_t)Q4NX_WS_COUNTER_BYTES + (size_t)recs * rows * (c->head_dim + 4) * 4 : 0;
  if (!block && n_split == 0 && (int64_t)p.bytes > kMostBytes) {   // thousands of items: one part each
    p.unit = tiles;
    p.grid = p.items;
    p.shared = false;
    p.bytes = 0;
  }
  p.whole = p.unit >= tiles;
  const int64_t heads = (int64_t)c->n_seqs * c->n_kv_heads;
  const int64_t ops = heads * tiles * (256 * c->head_dim + c->head_dim / 8);
  if (block && (int64_t)total * group >= (int64_t)kApartBlocks * rows * c->n_seqs && ops <= kMostBytes) {
    p.ops = (p.bytes ? p.bytes + 255 : Q4NX_WS_COUNTER_BYTES) & ~(size_t)255;
    p.ops_tiles = tiles;
    p.bytes = p.ops + (size_t)ops;
  }
  return p;
}

static bool kv4_attn_shape(const q4nx_kv4* c, int n_q_heads, int max_new, int max_len, int n_sel) {
  return n_q_heads >= 1 && n_q_heads % c->n_kv_heads == 0 && n_q_heads / c->n_kv_heads <= 16 &&
         max_new >= 1 && max_len >= 1 && n_sel >= 0 &&
         (int64_t)n_sel * c->page_len <= (int64_t)1 << 30;
}

}  // namespace q4nx

using namespace q4nx;

extern "C" {

size_t q4nx_kv4_attn_ws_bytes(const q4nx_kv4* cache, int n_q_heads, int total, int max_new,
                              int max_len, int n_sel, int n_split) {
  Kv4 c;
  if (kv4_resolve(cache, &c, "q4nx_kv4_attn_ws_bytes") != Q4NX_OK ||
      !kv4_attn_shape(cache, n_q_heads, max_new, max_len, n_sel) || n_split < 0 || n_split > 1024 ||
      total < 0)
    return 0;
  return kv4_plan(cache, n_q_heads, total, max_len, n_sel, n_split).bytes;
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
  Q4NX_REQUIRE(Q4NX_ALIGNED(out, 8) && Q4NX_ALIGNED(out_f32, 16), Q4NX_ERR_ARG,
               "%s: out must be 8-byte, out_f32 16-byte aligned", what);
  Q4NX_REQUIRE((sel != nullptr) == (n_sel > 0) && n_split >= 0 && n_split <= 1024, Q4NX_ERR_ARG,
               "%s: sel and n_sel=%d go together; n_split=%d outside 0..1024", what, n_sel, n_split);
  Q4NX_REQUIRE(kv4_attn_shape(cache, n_q_heads, max_new, max_len, n_sel), Q4NX_ERR_SHAPE,
               "%s: Hq=%d must be a multiple (<= 16x) of Hkv=%d; max_new=%d max_len=%d n_sel=%d", what,
               n_q_heads, cache->n_kv_heads, max_new, max_len, n_sel);
  Q4NX_REQUIRE(cu ? total >= 1 : (max_new == 1 && total == cache->n_seqs), Q4NX_ERR_SHAPE,
               "%s: total=%d, max_new=%d (without cu one token for each of %d sequences)", what, total,
               max_new, cache->n_seqs);
  Q4NX_REQUIRE(n_sel == 0 || cu == nullptr, Q4NX_ERR_SHAPE,
               "%s: a page list is for one token per sequence, without cu", what);
  Q4NX_REQUIRE(q_stride >= (int64_t)n_q_heads * cache->head_dim && q_stride % 8 == 0, Q4NX_ERR_SHAPE,
               "%s: q_stride=%lld must hold Hq * D and be a multiple of 8", what, (long long)q_stride);
  Q4NX_REQUIRE((int64_t)total * n_q_heads < (int64_t)1 << 30, Q4NX_ERR_SHAPE,
               "%s: total=%d rows of %d heads, fewer than 2^30 in all", what, total, n_q_heads);
  const Kv4Plan p = kv4_plan(cache, n_q_heads, cu ? total : 0, max_len, n_sel, n_split);
  const int64_t longest = n_sel ? (int64_t)n_sel * cache->page_len : max_len;
  Q4NX_REQUIRE(p.grid <= (int64_t)1 << 30 &&
                   (cu != nullptr || p.items * (longest / kKv4Tile + 1) < (int64_t)1 << 31),
               Q4NX_ERR_SHAPE, "%s: %lld rows of up to %lld positions", what, (long long)p.items,
               (long long)longest);
  if (p.bytes)
    Q4NX_REQUIRE(ws != nullptr && ws_bytes >= p.bytes && Q4NX_ALIGNED(ws, 256), Q4NX_ERR_WS,
                 "%s: workspace of %zu bytes (256-aligned) needed, %zu given", what, p.bytes, ws_bytes);
  if (p.shared) {
    const size_t recs = (p.ops ? p.ops : p.bytes) - Q4NX_WS_COUNTER_BYTES;
    Q4NX_REQUIRE(recs < (size_t)1 << 31 && p.items * 4 <= Q4NX_WS_COUNTER_BYTES, Q4NX_ERR_SHAPE,
                 "%s: %lld rows to be shared by several workgroups", what, (long long)p.items);
    a.counters = (unsigned*)ws;
    a.partial = (float*)((uint8_t*)ws + Q4NX_WS_COUNTER_BYTES);
    a.partial_bytes = (uint32_t)recs;
  }
  if (p.ops) {
    const int64_t tiles = (int64_t)a.c.n_seqs * a.c.hkv * p.ops_tiles;
    a.ops = (u32x4_t*)((uint8_t*)ws + p.ops);
    a.bad = (uint32_t*)((uint8_t*)a.ops + tiles * 256 * cache->head_dim);
    a.ops_tiles = p.ops_tiles;
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
  a.n_split = p.n_split;
  a.chunk = p.chunk;
  a.unit = p.unit;
  a.whole = p.whole;
  if (max_len < a.c.cap) a.c.cap = max_len;
  a.scale_l2 = (float)((double)scale * 1.4426950408889634);
  const dim3 grid((unsigned)p.grid);
  const bool d64 = cache->head_dim == 64;
  hipStream_t s = (hipStream_t)stream;
  if (cu == nullptr) {
    auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a); };
    switch ((a.group + 3) / 4) {   // heads per lane
      case 1: d64 ? run(kv4_decode_kernel<2, 1>) : run(kv4_decode_kernel<4, 1>); break;
      case 2: d64 ? run(kv4_decode_kernel<2, 2>) : run(kv4_decode_kernel<4, 2>); break;
      case 3: d64 ? run(kv4_decode_kernel<2, 3>) : run(kv4_decode_kernel<4, 3>); break;
      default: d64 ? run(kv4_decode_kernel<2, 4>) : run(kv4_decode_kernel<4, 4>); break;
    }
  }
  else {
    auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a); };
    if (p.ops) {
      const dim3 tiles((unsigned)p.ops_tiles, (unsigned)a.c.hkv, (unsigned)a.c.n_seqs);
      if (d64) hipLaunchKernelGGL(kv4_apart_kernel<2>, tiles, dim3(256), 0, s, a);
      else hipLaunchKernelGGL(kv4_apart_kernel<4>, tiles, dim3(256), 0, s, a);
      d64 ? run(kv4_block_kernel<2, true>) : run(kv4_block_kernel<4, true>);
    } else {
      d64 ? run(kv4_block_kernel<2, false>) : run(kv4_block_kernel<4, false>);
    }
  }
  return check_launch(what);
}

}  // extern "C"
