// Attention of few query rows over a part of a cache, on the matrix cores: what the shared-prefix
// attention (attn_prefix.hip) and the attention that sums its weights (attn_weights.hip) are made of.
#pragma once

#include <math.h>

#include "common.h"

namespace q4nx {

constexpr int kPartWaves = 4;
constexpr int kPartRound = kPartWaves * 32;   // positions of a workgroup's round
// Records of a (sequence, head): a lane of the merge each, at most 32 of a prefix and 32 of an own cache.
constexpr int kMaxParts = 32;
// A part's rows are read with 32-bit byte offsets.
constexpr int kMaxChunk = 1 << 22;

// A record: acc[D], then m (scale * log2 e units) and l, two pad words.
template <int D>
constexpr int kRec = D + 4;

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// A workgroup of 4 waves takes R <= 16 query rows over rows of a cache. Each wave scores 32 positions a round
// for all of them:
//   S^T[pos][row]  = K[pos][:] . q[row][:]      A = 16 K rows as stored, B = q^T
//   O^T[dim][row] += V^T[dim][pos] . P^T[pos][row]
// Lane j + 16 g of a score tile holds row j at positions 4 g .. 4 g + 3; P.V takes its 32 positions in
// that order (slot 8 g + e <-> position 16 (e / 4) + 4 g + e % 4), so P^T is in place, and V^T is
// gathered to match: a lane loads channels 4 j .. 4 j + 3 of its 8 positions and v_perm makes operands
// u = 0 .. 3 of the channels 4 i + u. This kind of work waits for memory, so P enters as two bf16 terms
// (2^-17 of it is lost) and two rounds are in flight beside the one that is computed (D = 64; one for
// D = 128, where three buffers would not fit the registers).
template <int D>
struct Narrow {
  static constexpr int KC = D / 32, VH = D / 64, NB = D == 64 ? 3 : 2;
  u32x4_t q[KC];
  f32x4_t o[4 * VH];
  float m, l;   // of this wave's positions; l of this lane's

  __device__ __forceinline__ void init(const uint16_t* qrow, int R) {
    const int lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
#pragma unroll
    for (int c = 0; c < KC; ++c)
      q[c] = j < R ? *(const u32x4_t*)(qrow + 32 * c + 8 * g) : u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
    for (int u = 0; u < 4 * VH; ++u) o[u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.f;
  }

  // Cache rows [0, end) of kbase, vbase (rows of D, packed). SCORES: the scaled scores also go to
  // scores[row * score_stride + pos], up to the end of the last round.
  template <bool SCORES>
  __device__ __forceinline__ void run(const uint16_t* kbase, const uint16_t* vbase, int end, float scale_l2,
                                      int R, float* scores, int64_t score_stride) {
    const int lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
    const int w0 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 32;
    const __amdgpu_buffer_rsrc_t kr = make_rsrc(kbase, (uint32_t)end * (2 * D));
    const __amdgpu_buffer_rsrc_t vr = make_rsrc(vbase, (uint32_t)end * (2 * D));
    struct Buf {
      u32x4_t k[2][KC];
      uint2 v[8][VH];
    } buf[NB];
    auto load = [&](Buf& x, int p0) {   // rows past the end read zeros
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          const v4i_t v = __builtin_amdgcn_raw_buffer_load_b128(
              kr, (int)((uint32_t)(p0 + 16 * t + j) * (2 * D) + 16u * g + 64u * c), 0, 0);
          x.k[t][c] = u32x4_t{(uint32_t)v.x, (uint32_t)v.y, (uint32_t)v.z, (uint32_t)v.w};
        }
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int h = 0; h < VH; ++h) {
          const auto v = __builtin_amdgcn_raw_buffer_load_b64(
              vr, (int)((uint32_t)(p0 + 16 * (e >> 2) + 4 * g + (e & 3)) * (2 * D) + 8u * j + 128u * h), 0, 0);
          x.v[e][h] = make_uint2((uint32_t)v[0], (uint32_t)v[1]);
        }
    };
    auto round = [&](const Buf& x, int p0) {
      f32x4_t s[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        s[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < KC; ++c) s[t] = mfma_bf16(x.k[t][c], q[c], s[t]);
      }
      float sc[8], mr = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool ok = p0 + 16 * (e >> 2) + 4 * g + (e & 3) < end;
        sc[e] = ok ? s[e >> 2][e & 3] * scale_l2 : -INFINITY;
        mr = fmaxf(mr, sc[e]);
      }
      if constexpr (SCORES) {
        if (j < R) {
          float* to = scores + j * score_stride + p0 + 4 * g;
          *(float4*)to = make_float4(sc[0], sc[1], sc[2], sc[3]);
          *(float4*)(to + 16) = make_float4(sc[4], sc[5], sc[6], sc[7]);
        }
      }
      mr = xor32_max(xor16_max(mr));
      const float mn = fmaxf(m, mr);
      const float mb = mn == -INFINITY ? 0.f : mn;   // nothing seen yet: every p and the rescale are 0
      const float corr = exp2_hw(m - mb);
      float p[8], ls = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = exp2_hw(sc[e] - mb);
        ls += p[e];
      }
      l = fmaf(l, corr, ls);
      m = mn;
#pragma unroll
      for (int u = 0; u < 4 * VH; ++u) o[u] *= corr;
      u32x4_t pp[2];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        pp[0][w] = pack_bf16x2_op(p[2 * w], p[2 * w + 1]);
        pp[1][w] = pack_bf16x2_op(p[2 * w] - bf16lo(pp[0][w]), p[2 * w + 1] - bf16hi(pp[0][w]));
      }
#pragma unroll
      for (int h = 0; h < VH; ++h)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          u32x4_t av;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t lo = u < 2 ? x.v[2 * w][h].x : x.v[2 * w][h].y;
            const uint32_t hi = u < 2 ? x.v[2 * w + 1][h].x : x.v[2 * w + 1][h].y;
            av[w] = perm(hi, lo, (u & 1) ? 0x07060302u : 0x05040100u);
          }
          o[4 * h + u] = mfma_bf16(av, pp[0], o[4 * h + u]);
          o[4 * h + u] = mfma_bf16(av, pp[1], o[4 * h + u]);
        }
    };
    const int n = end > 0 ? (end + kPartRound - 1) / kPartRound : 0;
    static_for<0, NB - 1>([&](auto i) {
      if ((int)i < n) load(buf[i], (int)i * kPartRound + w0);
    });
    for (int r = 0; r < n; r += NB)
      static_for<0, NB>([&](auto i) {
        if (r + (int)i + NB - 1 < n) load(buf[((int)i + NB - 1) % NB], (r + (int)i + NB - 1) * kPartRound + w0);
        if (r + (int)i < n) round(buf[i], (r + (int)i) * kPartRound + w0);
      });
  }

  // The waves' states meet in `lds` (4 (D + 2) R floats); emit(row, d, acc of channels d .. d + 3, m, l).
  template <typename Emit>
  __device__ __forceinline__ void finish(int R, float* lds, Emit emit) {
    const int tid = threadIdx.x, lane = tid & 63, j = lane & 15, g = lane >> 4, wave = tid >> 6;
    float* s_o = lds;                       // [wave][row][D]
    float* s_m = lds + kPartWaves * R * D;  // [wave][row]
    float* s_l = s_m + kPartWaves * R;
    l = xor32_sum(xor16_sum(l));
    if (j < R) {
      if (g == 0) {
        s_m[wave * R + j] = m;
        s_l[wave * R + j] = l;
      }
#pragma unroll
      for (int h = 0; h < VH; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *(float4*)(s_o + (wave * R + j) * D + 64 * h + 16 * g + 4 * e) =
              make_float4(o[4 * h][e], o[4 * h + 1][e], o[4 * h + 2][e], o[4 * h + 3][e]);
    }
    __syncthreads();
    for (int i = tid; i < R * (D / 4); i += kPartWaves * 64) {
      const int row = i / (D / 4), d = i % (D / 4) * 4;
      float M = s_m[row];
#pragma unroll
      for (int w = 1; w < kPartWaves; ++w) M = fmaxf(M, s_m[w * R + row]);
      const float Mb = M == -INFINITY ? 0.f : M;
      float L = 0.f;
      float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kPartWaves; ++w) {
        const float f = exp2_hw(s_m[w * R + row] - Mb);
        const float4 x = *(const float4*)(s_o + (w * R + row) * D + d);
        L = fmaf(s_l[w * R + row], f, L);
        A.x = fmaf(x.x, f, A.x);
        A.y = fmaf(x.y, f, A.y);
        A.z = fmaf(x.z, f, A.z);
        A.w = fmaf(x.w, f, A.w);
      }
      emit(row, d, A, M, L);
    }
  }
};

// A record of a part, where it is kept.
template <int D>
__device__ __forceinline__ void put_record(float* to, int d, const float4& A, float m, float l) {
  *(float4*)(to + d) = A;
  if (d == 0) *(float2*)(to + D) = make_float2(m, l);
}

// acc / l of four channels; 0 where nothing was seen
__device__ __forceinline__ float4 whole(const float4& A, float l) {
  return l == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                  : make_float4(attn_div(A.x, l), attn_div(A.y, l), attn_div(A.z, l), attn_div(A.w, l));
}

// The merge of a (sequence, query head)'s records by one wave: record r < slots at rec + r * stride, those
// with valid(r) count. Groups of D/4 lanes take a record each, four channels a lane; nothing is waited for
// before all records are on their way (valid() may wait for lengths), stale ones of earlier launches among
// them. Channels 4 c .. 4 c + 3 (c = lane % (D/4)) of the answer in every group; 0 where nothing was seen.
template <int D, typename Valid>
__device__ __forceinline__ float4 merge_records(const float* rec, size_t stride, int slots, int lane, Valid valid) {
  constexpr int LR = D / 4, GR = 64 / LR, U = 4;   // lanes of a record, records at once, and in flight
  const int q = lane / LR, c = lane % LR;
  const float2 head = *(const float2*)(rec + (size_t)min(lane, slots - 1) * stride + D);
  float4 x[U];
#pragma unroll
  for (int i = 0; i < U; ++i) x[i] = *(const float4*)(rec + (size_t)min(GR * i + q, slots - 1) * stride + 4 * c);
  const bool counts = valid(lane);   // by all lanes: it may vote
  const bool ok = lane < slots && counts;
  const uint64_t who = __ballot(ok);
  const float m = ok ? head.x : -INFINITY, l = ok ? head.y : 0.f;
  const float M = wave_max(m);
  const float f = m == -INFINITY ? 0.f : exp2_hw(m - M);
  const float L = wave_sum(m == -INFINITY ? l : f * l);   // a NaN of any record reaches L
  float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int r0 = 0; r0 < slots; r0 += U * GR) {
    if (r0 > 0) {
#pragma unroll
      for (int i = 0; i < U; ++i)
        x[i] = *(const float4*)(rec + (size_t)min(r0 + GR * i + q, slots - 1) * stride + 4 * c);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int r = r0 + GR * i + q;
      const float w = __shfl(f, r & 63);
      if (r < slots && (who >> (r & 63) & 1)) {
        A.x = fmaf(x[i].x, w, A.x);
        A.y = fmaf(x[i].y, w, A.y);
        A.z = fmaf(x[i].z, w, A.z);
        A.w = fmaf(x[i].w, w, A.w);
      }
    }
  }
  float* const a = (float*)&A;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (GR == 4) a[i] = xor16_sum(a[i]);
    a[i] = xor32_sum(a[i]);
  }
  return whole(A, L);
}

// Its four channels of the answer at `at` of the outputs that are wanted.
__device__ __forceinline__ void put_channels(uint16_t* out, float* out_f32, size_t at, const float4& A) {
  if (out) *(uint2*)(out + at) = make_uint2(pack_bf16x2(A.x, A.y), pack_bf16x2(A.z, A.w));
  if (out_f32) *(float4*)(out_f32 + at) = A;
}

// Parts of at least `unit` positions that len (< 2^24) is cut in, about `want` of them, and the positions of
// one, a multiple of `step`.
static inline void cut_parts(int len, long long want, int unit, int step, int* ns, int* chunk) {
  int n = want < 1 ? 1 : want > kMaxParts ? kMaxParts : (int)want;
  if (n > (len + unit - 1) / unit) n = (len + unit - 1) / unit;
  if (n < (len + kMaxChunk - 1) / kMaxChunk) n = (len + kMaxChunk - 1) / kMaxChunk;
  *chunk = ((len + n - 1) / n + step - 1) / step * step;
  *ns = (len + *chunk - 1) / *chunk;
}

}  // namespace q4nx
