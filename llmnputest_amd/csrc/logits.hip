// Rules for the next token on logits: penalties for tokens that were seen, biases, masks of allowed tokens,
// and the greatest of what remains. No reference counterpart (its token choice is transformers' generate,
// chat.py:74-78).
//
// Per token, in fp32, each step rounded (no fused multiply-add, so the values are those of the steps as
// written):
//   seen (count word not 0):  x = x > 0 ? x / repetition : x * repetition
//   x -= frequency * count;   count > 0: x -= presence;   x += bias;   not allowed: x = -inf
// (a token that is listed several times: the sum of its biases, in the order of the list)
// A count word holds how often a token was generated and, in the sign bit, whether the prompt has it.
// Bound by memory: logits, counts and masks are read once, what comes of the logits is written once.

#include <math.h>

#include "common.h"

namespace q4nx {

struct LogitArgs {
  const void* logits;
  void* out;
  const int32_t* counts;
  const float *repetition, *presence, *frequency;
  const int32_t* bias_ids;
  const float* bias_values;
  const int32_t* bias_cu;
  const uint32_t* mask;
  const int32_t* mask_rows;
  int32_t* tokens;
  unsigned long long* keys;
  unsigned* slots;          // a row's arrivals, an unused word, its greatest key
  int64_t stride, out_stride, count_stride, mask_stride;
  int vocab, batch, n_mask, n_bias, parts, slot_words;
};

constexpr int kLogitThreads = 256;

// Product and difference rounded apart.
__device__ __forceinline__ float penalised(float x, float repetition, float frequency, float presence, int said) {
#pragma clang fp contract(off)
  x = x > 0.f ? x / repetition : x * repetition;
  const float often = frequency * (float)said;
  x = x - often;
  return said > 0 ? x - presence : x;
}

// Rows need no alignment beyond their type's: 16-byte accesses of any address are single instructions here.
typedef uint32_t u32x4_any_t __attribute__((ext_vector_type(4), aligned(2)));

// Long calls (U = 4) stream past the caches (64 x 100353: 21.1 to 18.9 us).
template <bool STREAM>
__device__ __forceinline__ u32x4_any_t logit_load(const u32x4_any_t* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load(p);
  else return *p;
}

// VEC values a load (16 bytes), U loads a thread, in flight together.
template <typename T, int U>
__global__ __launch_bounds__(kLogitThreads) void adjust_logits_kernel(LogitArgs a) {
  constexpr int VEC = 16 / sizeof(T), SPAN = kLogitThreads * VEC * U;
  __shared__ float s_bias[SPAN];
  __shared__ unsigned long long s_key[kLogitThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.x / a.parts, v0 = (blockIdx.x % a.parts) * SPAN;
  const T* const in = (const T*)a.logits + (int64_t)b * a.stride;
  T* const to = (T*)a.out + (int64_t)b * a.out_stride;
  const int32_t* const cnt = a.counts == nullptr ? nullptr : a.counts + (int64_t)b * a.count_stride;

  union Piece {
    u32x4_any_t v;
    T e[VEC];
  } x[U];
  int32_t n[U][VEC];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int v = v0 + (u * kLogitThreads + tid) * VEC;
    if (v + VEC <= a.vocab) {
      x[u].v = logit_load<U == 4>((const u32x4_any_t*)(in + v));
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[u].e[i] = v + i < a.vocab ? in[v + i] : (T)0;
    }
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      if (cnt != nullptr && v + i + 4 <= a.vocab) {
        const u32x4_any_t c = logit_load<U == 4>((const u32x4_any_t*)(cnt + v + i));
#pragma unroll
        for (int k = 0; k < 4; ++k) n[u][i + k] = (int32_t)c[k];
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) n[u][i + k] = cnt != nullptr && v + i + k < a.vocab ? cnt[v + i + k] : 0;
      }
    }
  }
  uint32_t may[U];   // the word of the VEC tokens (they lie in one)
  const int row = a.mask == nullptr ? -1 : a.mask_rows == nullptr ? b : a.mask_rows[b];
  if (row >= 0) {
    const uint32_t* const words = a.mask + (int64_t)row * a.mask_stride;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = v0 + (u * kLogitThreads + tid) * VEC;
      may[u] = row < a.n_mask && v < a.vocab ? words[v >> 5] >> (v & 31) : 0u;
    }
  }
  const float rep = a.repetition == nullptr ? 1.f : a.repetition[b];
  const float pres = a.presence == nullptr ? 0.f : a.presence[b];
  const float freq = a.frequency == nullptr ? 0.f : a.frequency[b];

  // ---- the biases that fall here, summed in the order of the list
  int bias_from = 0, bias_to = 0;
  if (a.bias_cu != nullptr) {
    bias_from = max(a.bias_cu[b], 0);
    bias_to = min(a.bias_cu[b + 1], a.n_bias);
  }
  const bool biased = bias_from < bias_to;
  if (biased) {
    for (int i = tid; i < SPAN; i += kLogitThreads) s_bias[i] = 0.f;
    __syncthreads();
    if (wave == 0)
      for (int i0 = bias_from; i0 < bias_to; i0 += 64) {
        const int i = i0 + lane;
        const int id = i < bias_to ? a.bias_ids[i] : -1;
        const bool here = id >= v0 && id < v0 + SPAN && id < a.vocab;
        const float val = here ? a.bias_values[i] : 0.f;
        // one lane at a time: a wave's LDS operations keep their order
        for (uint64_t who = __ballot(here); who != 0; who &= who - 1)
          if (lane == __builtin_ctzll(who)) s_bias[id - v0] += val;
      }
    __syncthreads();
  }

  unsigned long long best = 0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int at = (u * kLogitThreads + tid) * VEC, v = v0 + at;
    float f[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if constexpr (sizeof(T) == 2) f[i] = bf16_to_f32(x[u].e[i]);
      else f[i] = x[u].e[i];
      const int32_t c = n[u][i];
      if (c != 0) f[i] = penalised(f[i], rep, freq, pres, c & 0x7fffffff);
      if (biased) f[i] += s_bias[at + i];
      if (row >= 0 && !(may[u] >> i & 1u)) f[i] = -INFINITY;
      if (v + i < a.vocab) {
        const unsigned long long k = argmax_key(f[i], (uint32_t)(v + i));
        best = k > best ? k : best;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2) x[u].v[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
      else x[u].v[i] = __float_as_uint(f[i]);
    }
    if (v + VEC <= a.vocab) {
      if constexpr (U == 4) __builtin_nontemporal_store(x[u].v, (u32x4_any_t*)(to + v));
      else *(u32x4_any_t*)(to + v) = x[u].v;
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (v + i < a.vocab) to[v + i] = x[u].e[i];
    }
  }
  if (a.tokens == nullptr && a.keys == nullptr) return;

  // ---- the greatest: the workgroups' keys meet in one word (whose order of arrival does not matter), the
  // last one takes it
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    const unsigned long long k = __shfl_xor(best, d);
    best = k > best ? k : best;
  }
  if (lane == 0) s_key[wave] = best;
  __syncthreads();
  if (tid != 0) return;
#pragma unroll
  for (int w = 1; w < kLogitThreads / 64; ++w) best = s_key[w] > best ? s_key[w] : best;
  if (a.parts > 1) {
    unsigned* const slot = a.slots + (size_t)b * a.slot_words;
    unsigned long long* const top = (unsigned long long*)(slot + 2);
    atomicMax(top, best);
    wait_vm();
    if (!ticket(slot, a.parts)) return;
    best = atomicExch(top, 0ull);
  }
  if (a.tokens != nullptr) a.tokens[b] = (int32_t)(0xffffffffu - (uint32_t)best);
  if (a.keys != nullptr) a.keys[b] = best;
}

// Counts of a list of tokens added to a row: one token a thread.
__global__ __launch_bounds__(256) void count_tokens_kernel(int32_t* counts, int64_t stride, const int32_t* tokens,
                                                           const int32_t* cu, int n_tokens, int vocab,
                                                           int prompt) {
  const int b = blockIdx.y;
  const int from = cu == nullptr ? b : max(cu[b], 0), to = cu == nullptr ? b + 1 : min(cu[b + 1], n_tokens);
  int32_t* const row = counts + (int64_t)b * stride;
  for (int i = from + (int)(blockIdx.x * 256 + threadIdx.x); i < to; i += (int)gridDim.x * 256) {
    const int t = tokens[i];
    if (t < 0 || t >= vocab) continue;
    if (prompt) atomicOr((unsigned*)row + t, 0x80000000u);
    else atomicAdd(row + t, 1);
  }
}

// Counts from nothing: a workgroup counts the tokens of its span of the vocabulary in LDS and writes the span.
constexpr int kCountSpan = 8192;
constexpr int kCountThreads = 512;
__global__ __launch_bounds__(kCountThreads) void count_fresh_kernel(int32_t* counts, int64_t stride,
                                                                    const int32_t* tokens, const int32_t* cu,
                                                                    int n_tokens, int vocab, int prompt) {
  __shared__ int32_t s[kCountSpan];
  const int b = blockIdx.y, v0 = blockIdx.x * kCountSpan;
  const int from = cu == nullptr ? b : max(cu[b], 0), to = cu == nullptr ? b + 1 : min(cu[b + 1], n_tokens);
  const int span = min(kCountSpan, vocab - v0);
  for (int i = threadIdx.x; i < kCountSpan; i += kCountThreads) s[i] = 0;
  __syncthreads();
  constexpr int U = 8;   // in flight (one at a time, 8 lists of 4096 took 8.1 us of 6.9)
  for (int i0 = from + (int)threadIdx.x; i0 < to; i0 += U * kCountThreads) {
    int t[U];
#pragma unroll
    for (int u = 0; u < U; ++u) t[u] = i0 + u * kCountThreads < to ? tokens[i0 + u * kCountThreads] : -1;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (t[u] < v0 || t[u] - v0 >= span) continue;
      if (prompt) atomicOr((unsigned*)s + (t[u] - v0), 0x80000000u);
      else atomicAdd(s + (t[u] - v0), 1);
    }
  }
  __syncthreads();
  int32_t* const row = counts + (int64_t)b * stride + v0;
  for (int i = threadIdx.x; i < span; i += kCountThreads) row[i] = s[i];
}

static int logit_span(int bf16, int u) { return kLogitThreads * (bf16 ? 8 : 4) * u; }

}  // namespace q4nx

using namespace q4nx;

extern "C" {

int q4nx_count_tokens(int32_t* counts, int64_t count_stride, int vocab, int batch, const int32_t* tokens,
                      int n_tokens, const int32_t* cu, int prompt, int start, void* stream) {
  const char* what = "q4nx_count_tokens";
  Q4NX_REQUIRE(counts && (tokens || n_tokens == 0), Q4NX_ERR_ARG, "%s: counts and tokens are required", what);
  Q4NX_REQUIRE(vocab >= 1 && vocab <= (1 << 28) && batch >= 1 && batch <= 65535 && n_tokens >= 0 &&
                   count_stride >= vocab && (cu || n_tokens == batch),
               Q4NX_ERR_SHAPE, "%s: vocab=%d batch=%d n_tokens=%d (one per sequence without cu)", what, vocab, batch,
               n_tokens);
  hipStream_t s = (hipStream_t)stream;
  if (start) {
    const dim3 grid((unsigned)((vocab + kCountSpan - 1) / kCountSpan), (unsigned)batch);
    hipLaunchKernelGGL(count_fresh_kernel, grid, dim3(kCountThreads), 0, s, counts, count_stride, tokens, cu,
                       n_tokens, vocab, prompt);
  } else if (n_tokens > 0) {
    const int wgs = (n_tokens + 255) / 256;
    const dim3 grid(cu == nullptr ? 1u : (unsigned)(wgs < 64 ? wgs : 64), (unsigned)batch);
    hipLaunchKernelGGL(count_tokens_kernel, grid, dim3(256), 0, s, counts, count_stride, tokens, cu, n_tokens,
                       vocab, prompt);
  }
  return check_launch(what);
}

int q4nx_adjust_logits(const void* logits, int bf16, int64_t stride, void* out, int64_t out_stride, int vocab,
                       int batch, const int32_t* counts, int64_t count_stride, const float* repetition,
                       const float* presence, const float* frequency, const int32_t* bias_ids,
                       const float* bias_values, int n_biases, const int32_t* bias_cu, const uint32_t* mask,
                       int64_t mask_stride, int n_mask, const int32_t* mask_rows, int32_t* tokens,
                       uint64_t* keys, void* ws, size_t ws_bytes, void* stream) {
  const char* what = "q4nx_adjust_logits";
  Q4NX_REQUIRE(logits && out, Q4NX_ERR_ARG, "%s: logits and out are required", what);
  Q4NX_REQUIRE(vocab >= 1 && vocab <= (1 << 28) && batch >= 1 && batch <= Q4NX_WS_COUNTER_BYTES / 16 &&
                   stride >= vocab && out_stride >= vocab && (!counts || count_stride >= vocab),
               Q4NX_ERR_SHAPE, "%s: vocab=%d batch=%d (at most %d), strides of at least vocab", what, vocab, batch,
               Q4NX_WS_COUNTER_BYTES / 16);
  Q4NX_REQUIRE(counts || (!repetition && !presence && !frequency), Q4NX_ERR_ARG, "%s: penalties need counts", what);
  Q4NX_REQUIRE((bias_ids != nullptr) == (bias_cu != nullptr) && (bias_values != nullptr) == (bias_cu != nullptr) &&
                   n_biases >= 0,
               Q4NX_ERR_ARG, "%s: biases are ids, values and cu", what);
  Q4NX_REQUIRE(mask ? (n_mask >= 1 && mask_stride >= (vocab + 31) / 32 && (mask_rows || n_mask >= batch))
                    : !mask_rows,
               Q4NX_ERR_SHAPE, "%s: mask needs (vocab + 31) / 32 words a row, a row per sequence or mask_rows", what);
  Q4NX_REQUIRE(ws != nullptr && ws_bytes >= Q4NX_WS_COUNTER_BYTES && Q4NX_ALIGNED(ws, 256), Q4NX_ERR_WS,
               "%s: workspace of %d bytes (256-aligned) needed, %zu given", what, Q4NX_WS_COUNTER_BYTES, ws_bytes);
  LogitArgs a{};
  a.logits = logits;
  a.out = out;
  a.counts = counts;
  a.repetition = repetition;
  a.presence = presence;
  a.frequency = frequency;
  a.bias_ids = bias_ids;
  a.bias_values = bias_values;
  a.bias_cu = bias_cu;
  a.mask = mask;
  a.mask_rows = mask_rows;
  a.tokens = tokens;
  a.keys = (unsigned long long*)keys;
  a.slots = (unsigned*)ws;
  a.stride = stride;
  a.out_stride = out_stride;
  a.count_stride = count_stride;
  a.mask_stride = mask_stride;
  a.vocab = vocab;
  a.batch = batch;
  a.n_mask = n_mask;
  a.n_bias = n_biases;
  // rows' words on lines of their own as far as the counters go: with all of 8 rows' on one line, 122
  // workgroups a row took 19 us, most of them for the atomics
  a.slot_words = Q4NX_WS_COUNTER_BYTES / 4 / batch / 4 * 4;
  if (a.slot_words > 64) a.slot_words = 64;
  // 16-byte loads a thread: more of them, and fewer workgroups that meet at a row's word, as soon as about
  // 512 workgroups remain
  int u = 4;
  while (u > 1 && (long long)batch * ((vocab + logit_span(bf16, u) - 1) / logit_span(bf16, u)) < 512) u /= 2;
  const int span = logit_span(bf16, u);
  a.parts = (vocab + span - 1) / span;
  Q4NX_REQUIRE((long long)a.parts * batch < (1ll << 31), Q4NX_ERR_SHAPE, "%s: more than 2^31 workgroups", what);
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)(a.parts * batch)), threads(kLogitThreads);
  switch (u + (bf16 ? 8 : 0)) {
    case 1: hipLaunchKernelGGL((adjust_logits_kernel<float, 1>), grid, threads, 0, s, a); break;
    case 2: hipLaunchKernelGGL((adjust_logits_kernel<float, 2>), grid, threads, 0, s, a); break;
    case 4: hipLaunchKernelGGL((adjust_logits_kernel<float, 4>), grid, threads, 0, s, a); break;
    case 9: hipLaunchKernelGGL((adjust_logits_kernel<uint16_t, 1>), grid, threads, 0, s, a); break;
    case 10: hipLaunchKernelGGL((adjust_logits_kernel<uint16_t, 2>), grid, threads, 0, s, a); break;
    default: hipLaunchKernelGGL((adjust_logits_kernel<uint16_t, 4>), grid, threads, 0, s, a); break;
  }
  return check_launch(what);
}

}  // extern "C"
