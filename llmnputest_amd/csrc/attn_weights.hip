// Attention of one token per sequence that also sums, per kv head, the weights that its query heads gave
// each position: what kv_evict.hip decides by. No reference counterpart (its cache never shrinks).
//
//   p[h][l]       = softmax over l < len of scale q[h] . K[l]
//   out[h]        = sum_l p[h][l] V[l]
//   weights[l]   += sum over the group's heads of p[h][l]      (the newest position's is set)
//
// A weight needs the maximum and the sum of the whole row, which a part of it does not know. The parts
// (Narrow) therefore also leave their scores, 4 Hq bytes a position beside the 4 D Hkv of K and V, and
// the second launch turns them into weights once every part's (m, l) is there; its last workgroup of a
// (sequence, kv head) merges the outputs. Short rows, and those of
// many sequences whose scores LDS holds, are one launch.

#include "attn_parts.h"

namespace q4nx {

struct WeightArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const int32_t* lens;
  uint16_t* out;
  float* out_f32;
  float* weights;      // [batch][hkv] rows of w_b_stride, w_h_stride
  float* rec;          // [batch * hkv][ns][G][kRec<D>]
  float* scores;       // [batch * hkv][G][score_stride]
  int64_t b_stride, h_stride, w_b_stride, w_h_stride, score_stride;
  int batch, hq, hkv, G, max_len, ns, chunk, start;
  float scale_l2;
};

template <int D>
__global__ __launch_bounds__(256) void weight_parts_kernel(WeightArgs a) {
  __shared__ __attribute__((aligned(16))) float lds[kPartWaves * 16 * D + 8 * 16];
  int blk = blockIdx.x;
  const int bk = blk % (a.batch * a.hkv), part = blk / (a.batch * a.hkv);
  const int b = bk / a.hkv, kvh = bk - b * a.hkv;
  const int len = min(max(a.lens[b], 0), a.max_len);
  const int start = part * a.chunk;
  if (start >= len) return;
  const int end = min(a.chunk, len - start);
  const size_t at = (size_t)b * a.b_stride + (size_t)kvh * a.h_stride + (size_t)start * D;
  const size_t rec = ((size_t)bk * a.ns + part) * (size_t)(a.G * kRec<D>);
  Narrow<D> st;
  st.init(a.q + ((size_t)b * a.hq + kvh * a.G + min((int)(threadIdx.x & 15), a.G - 1)) * D, a.G);
  st.template run<true>(a.k + at, a.v + at, end, a.scale_l2, a.G,
                        a.scores + (size_t)bk * a.G * a.score_stride + start, a.score_stride);
  st.finish(a.G, lds, [&](int r, int d, const float4& A, float m, float l) {
    put_record<D>(a.rec + rec + (size_t)r * kRec<D>, d, A, m, l);
  });
}

// One workgroup per (sequence, kv head): everything, the scores in LDS.
template <int D>
__global__ __launch_bounds__(kPartWaves * 64) void weight_whole_kernel(WeightArgs a, int score_stride) {
  extern __shared__ __attribute__((aligned(16))) float lds[];   // scores [G][score_stride], then states
  __shared__ float s_m[16], s_l[16];
  const int tid = threadIdx.x;
  const int b = blockIdx.x / a.hkv, kvh = blockIdx.x - b * a.hkv;
  const int len = min(max(a.lens[b], 0), a.max_len);
  const size_t at = (size_t)b * a.b_stride + (size_t)kvh * a.h_stride;
  const size_t row = (size_t)b * a.hq + kvh * a.G;
  float* const scores = lds;
  float* const to = a.weights + (size_t)b * a.w_b_stride + (size_t)kvh * a.w_h_stride;
  Narrow<D> st;
  st.init(a.q + (row + min(tid & 15, a.G - 1)) * D, a.G);
  st.template run<true>(a.k + at, a.v + at, len, a.scale_l2, a.G, scores, score_stride);
  st.finish(a.G, lds + a.G * score_stride, [&](int r, int d, const float4& A, float m, float l) {
    put_channels(a.out, a.out_f32, (row + r) * D + d, whole(A, l));
    if (d == 0) {
      s_m[r] = m == -INFINITY ? 0.f : m;
      s_l[r] = l == 0.f ? 0.f : 1.f / l;
    }
  });
  __syncthreads();
  for (int p = tid; p < len; p += kPartWaves * 64) {
    const float old = a.start || p == len - 1 ? 0.f : to[p];
    float w = 0.f;
    for (int h = 0; h < a.G; ++h) w = fmaf(exp2_hw(scores[h * score_stride + p] - s_m[h]), s_l[h], w);
    to[p] = old + w;
  }
}

constexpr int kWeightSpan = 1024;   // positions of a workgroup of the second launch

template <int D>
__global__ __launch_bounds__(256) void weight_sum_kernel(WeightArgs a, int spans) {
  constexpr int GH = 8, P = kWeightSpan / 256;   // heads in flight, positions a thread
  __shared__ float s_m[16], s_l[16];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int bk = blockIdx.x / (spans + 1), span = blockIdx.x % (spans + 1);
  const int b = bk / a.hkv, kvh = bk - b * a.hkv;
  const int len = min(max(a.lens[b], 0), a.max_len);
  const float* rec = a.rec + (size_t)bk * a.ns * (size_t)(a.G * kRec<D>);
  if (span == spans) {
    for (int h = wave; h < a.G; h += 4) {
      const float4 A = merge_records<D>(rec + (size_t)h * kRec<D>, (size_t)a.G * kRec<D>, a.ns, lane,
                                        [&](int r) { return r * a.chunk < len; });
      if (lane < D / 4) put_channels(a.out, a.out_f32, ((size_t)b * a.hq + kvh * a.G + h) * D + 4 * lane, A);
    }
    return;
  }
  const int p0 = span * kWeightSpan + tid;
  // scores and old weights are on their way before the length is known (within the buffers; those behind
  // it are left out)
  const __amdgpu_buffer_rsrc_t scores =
      make_rsrc(a.scores + (size_t)bk * a.G * a.score_stride, (uint32_t)(a.G * a.score_stride * 4));
  float* to = a.weights + (size_t)b * a.w_b_stride + (size_t)kvh * a.w_h_stride;
  float s[GH][P], w[P], old[P];
  auto load = [&](int h0) {   // heads that are none read zeros, outside the buffer
#pragma unroll
    for (int g = 0; g < GH; ++g)
#pragma unroll
      for (int i = 0; i < P; ++i)
        s[g][i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(
                                                scores, ((h0 + g) * (int)a.score_stride + p0 + 256 * i) * 4, 0, 0));
  };
  load(0);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    w[i] = 0.f;
    old[i] = a.start ? 0.f : to[min(p0 + 256 * i, a.max_len - 1)];
  }
  for (int h = wave; h < a.G; h += 4) {
    const float2 head = *(const float2*)(rec + ((size_t)min(lane, a.ns - 1) * a.G + h) * kRec<D> + D);
    const bool ok = lane < a.ns && lane * a.chunk < len;
    const float m = ok ? head.x : -INFINITY, l = ok ? head.y : 0.f;
    const float M = wave_max(m);
    const float L = wave_sum(m == -INFINITY ? l : exp2_hw(m - M) * l);
    if (lane == 0) {
      s_m[h] = M == -INFINITY ? 0.f : M;
      s_l[h] = L == 0.f ? 0.f : 1.f / L;
    }
  }
  __syncthreads();
  for (int h0 = 0; h0 < a.G; h0 += GH) {
    if (h0 > 0) load(h0);
#pragma unroll
    for (int g = 0; g < GH; ++g) {
      if (h0 + g >= a.G) break;
      const float m = s_m[h0 + g], li = s_l[h0 + g];
#pragma unroll
      for (int i = 0; i < P; ++i) w[i] = fmaf(exp2_hw(s[g][i] - m), li, w[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int p = p0 + 256 * i;
    if (p < len) to[p] = p == len - 1 ? w[i] : old[i] + w[i];
  }
}

struct WeightPlan {
  int ns, chunk;         // ns 0: one launch
  int64_t score_stride;
};

// Bytes of LDS that a workgroup with a whole row takes.
static size_t whole_lds(int G, int d, int64_t score_stride) {
  return (size_t)G * (score_stride + kPartWaves * (d + 2)) * 4;
}

static WeightPlan weight_plan(int batch, int hq, int hkv, int d, int max_len) {
  WeightPlan p{};
  // One launch, as far as LDS holds a row's scores: for any length where rows fill most of the chip (64 x 1024,
  // 40 q / 8 kv heads: 26.1 us, 35.2 in two launches; 64 x 2100 51.6, 66.4; 20 x 2100 19.1, 22.5; 16 x 2100 18.3,
  // 18.9), else up to 256 KB of K and V for a compute unit (12 x 1024 10.5, 12.4; D = 128, 1 x 900 14.7, 12.3)
  const int round = 32 * kPartWaves;
  p.score_stride = (max_len + round - 1) / round * round;
  const bool fits = whole_lds(hq / hkv, d, p.score_stride) <= 65024;
  if (fits && ((long long)batch * hkv >= 160 || max_len <= 65536 / d)) return p;
  cut_parts(max_len, 1024 / ((long long)hkv * batch), 256, kPartRound, &p.ns, &p.chunk);
  p.score_stride = (int64_t)p.ns * p.chunk;
  return p;
}

static bool weight_shape_ok(int batch, int hq, int hkv, int d, int max_len) {
  return batch >= 1 && batch <= (1 << 20) && hkv >= 1 && hkv <= 1024 && hq >= hkv && hq % hkv == 0 && hq / hkv <= 16 &&
         (d == 64 || d == 128) && max_len >= 1 && max_len < (1 << 24) && (long long)batch * hq < (1 << 28);
}

static size_t weight_rec_bytes(const WeightPlan& p, int batch, int hq, int d) {
  return (size_t)batch * hq * p.ns * (d + 4) * 4;
}

static size_t weight_ws(const WeightPlan& p, int batch, int hq, int d) {
  return (size_t)Q4NX_WS_COUNTER_BYTES +
         (p.ns == 0 ? 0 : weight_rec_bytes(p, batch, hq, d) + (size_t)batch * hq * p.score_stride * 4);
}

template <int D>
static void weight_launch(const WeightArgs& a, hipStream_t s) {
  if (a.ns == 0) {
    hipLaunchKernelGGL(weight_whole_kernel<D>, dim3((unsigned)(a.batch * a.hkv)), dim3(kPartWaves * 64),
                       whole_lds(a.G, D, a.score_stride), s, a, (int)a.score_stride);
    return;
  }
  const int spans = (a.max_len + kWeightSpan - 1) / kWeightSpan;
  hipLaunchKernelGGL(weight_parts_kernel<D>, dim3((unsigned)(a.batch * a.hkv * a.ns)), dim3(256), 0, s, a);
  hipLaunchKernelGGL(weight_sum_kernel<D>, dim3((unsigned)(a.batch * a.hkv * (spans + 1))), dim3(256), 0, s, a, spans);
}

}  // namespace q4nx

using namespace q4nx;

extern "C" {

size_t q4nx_gqa_decode_weights_ws_bytes(int batch, int n_q_heads, int n_kv_heads, int head_dim, int max_len) {
  if (!weight_shape_ok(batch, n_q_heads, n_kv_heads, head_dim, max_len)) return 0;
  return weight_ws(weight_plan(batch, n_q_heads, n_kv_heads, head_dim, max_len), batch, n_q_heads, head_dim);
}

int q4nx_gqa_decode_weights(const uint16_t* q, const uint16_t* k_cache, const uint16_t* v_cache,
                            int64_t kv_b_stride, int64_t kv_h_stride, const int32_t* lens, int max_len,
                            float* weights, int64_t w_b_stride, int64_t w_h_stride, int start, uint16_t* out,
                            float* out_f32, int batch, int n_q_heads, int n_kv_heads, int head_dim, float scale,
                            void* ws, size_t ws_bytes, void* stream) {
  const char* what = "q4nx_gqa_decode_weights";
  Q4NX_REQUIRE(weight_shape_ok(batch, n_q_heads, n_kv_heads, head_dim, max_len), Q4NX_ERR_SHAPE,
               "%s: batch=%d Hq=%d (a multiple of Hkv, at most 16 times) Hkv=%d head_dim=%d (64, 128) "
               "max_len=%d (below 2^24)",
               what, batch, n_q_heads, n_kv_heads, head_dim, max_len);
  Q4NX_REQUIRE(q && k_cache && v_cache && lens && weights && (out || out_f32), Q4NX_ERR_ARG,
               "%s: q, caches, lens, weights and an output are required", what);
  Q4NX_REQUIRE(Q4NX_ALIGNED(q, 16) && Q4NX_ALIGNED(k_cache, 16) && Q4NX_ALIGNED(v_cache, 16), Q4NX_ERR_ARG,
               "%s: q and caches must be 16-byte aligned", what);
  Q4NX_REQUIRE(Q4NX_ALIGNED(out, 8) && Q4NX_ALIGNED(out_f32, 16), Q4NX_ERR_ARG,
               "%s: out must be 8-byte, out_f32 16-byte aligned", what);
  Q4NX_REQUIRE(kv_h_stride >= (int64_t)max_len * head_dim && kv_h_stride % 8 == 0 &&
                   kv_b_stride >= (int64_t)n_kv_heads * kv_h_stride && kv_b_stride % 8 == 0,
               Q4NX_ERR_SHAPE, "%s: cache strides do not hold [Hkv][max_len][head_dim]", what);
  Q4NX_REQUIRE(w_h_stride >= max_len && w_b_stride >= (int64_t)n_kv_heads * w_h_stride, Q4NX_ERR_SHAPE,
               "%s: strides of weights do not hold [Hkv][max_len]", what);
  Q4NX_REQUIRE(scale >= 0.f, Q4NX_ERR_ARG, "%s: scale must not be negative", what);
  const WeightPlan p = weight_plan(batch, n_q_heads, n_kv_heads, head_dim, max_len);
  Q4NX_REQUIRE((long long)n_kv_heads * batch * (max_len / kWeightSpan + 2) < (1ll << 31), Q4NX_ERR_SHAPE,
               "%s: more than 2^31 workgroups", what);
  const size_t need = weight_ws(p, batch, n_q_heads, head_dim);
  Q4NX_REQUIRE(ws != nullptr && ws_bytes >= need && Q4NX_ALIGNED(ws, 256), Q4NX_ERR_WS,
               "%s: workspace of %zu bytes (256-aligned) needed, %zu given", what, need, ws_bytes);
  WeightArgs a{};
  a.q = q;
  a.k = k_cache;
  a.v = v_cache;
  a.lens = lens;
  a.out = out;
  a.out_f32 = out_f32;
  a.weights = weights;
  a.scores = (float*)((uint8_t*)ws + Q4NX_WS_COUNTER_BYTES);   // rows of whole rounds: 16-byte aligned
  a.rec = a.scores + (size_t)batch * n_q_heads * p.score_stride;
  a.b_stride = kv_b_stride;
  a.h_stride = kv_h_stride;
  a.w_b_stride = w_b_stride;
  a.w_h_stride = w_h_stride;
  a.score_stride = p.score_stride;
  a.batch = batch;
  a.hq = n_q_heads;
  a.hkv = n_kv_heads;
  a.G = n_q_heads / n_kv_heads;
  a.max_len = max_len;
  a.ns = p.ns;
  a.chunk = p.chunk;
  a.start = start != 0;
  a.scale_l2 = (float)((double)scale * 1.4426950408889634);
  hipStream_t s = (hipStream_t)stream;
  if (head_dim == 64) weight_launch<64>(a, s);
  else weight_launch<128>(a, s);
  return check_launch(what);
}

}  // extern "C"
