// Attention of one token per sequence over a prefix that many sequences share and over each one's own
// cache. No reference counterpart: its attention reads one sequence's cache per query head
// (designs/granite_gemv/granite_attention.h:221-237).
//
//   out[b][h] = softmax(scale q[b][h] . [Kpre; Kown]^T) [Vpre; Vown]
//
// The rows of a prefix are read once for all members of its group: per kv head the members' query heads
// of the group are the rows of one product, R = members * Hq/Hkv of them, and the exact (m, l, acc) merge
// joins what the prefix's parts and the own cache's parts give. Two launches: the parts, and the merge.
//
// Parts, all in one grid (the prefix's first, which take longest; the own cache's, which wait for memory,
// run beside them):
//   own caches      (sequence, kv head, part): Narrow
//   prefix, R > 16  (kv head, 64 NR rows, part): part_wide below
//   prefix, R <= 16 (kv head, part): Narrow over the members' rows
// Short calls are one launch: a workgroup a (sequence, kv head) takes the prefix's rows, then
// its own.

#include "attn_parts.h"

namespace q4nx {

struct PrefixArgs {
  const uint16_t* q;
  const uint16_t* k;      // own rows, [batch][hkv][..][D]
  const uint16_t* v;
  const uint16_t* kp;     // the prefixes', [n_prefixes][hkv][..][D]
  const uint16_t* vp;
  const int32_t* lens;
  const int32_t* plens;
  const int32_t* cu;      // nullptr: one prefix, all sequences
  uint16_t* out;
  float* out_f32;
  float* rec;             // [batch * hkv][slots][G][kRec<D>], own parts first
  int64_t b_stride, h_stride, pp_stride, ph_stride;
  int batch, hq, hkv, G, n_prefixes, max_prefix, max_len;
  int ns_pre, chunk_pre, tiles, ns_own, chunk_own;
  float scale_l2;
};

// The group of prefix p: sequences [first, first + members).
struct Group {
  int p, first, members;
};
__device__ __forceinline__ int cu_at(const PrefixArgs& a, int p) {
  return a.cu == nullptr ? (p > 0 ? a.batch : 0) : min(max(a.cu[p], 0), a.batch);
}
// Tiles of RT rows (64 or 128) of a prefix with so many members.
__device__ __forceinline__ int tiles_of(int members, int G, int RT) { return (members * G + RT - 1) / RT; }

// Which prefix row tile t belongs to, 64 prefixes at a time; t becomes its index there. p = -1: none.
__device__ __forceinline__ Group find_tile(const PrefixArgs& a, int RT, int lane, int& t) {
  for (int p0 = 0; p0 < a.n_prefixes; p0 += 64) {
    const int p = p0 + lane;
    int first = 0, members = 0;
    if (p < a.n_prefixes) {
      first = cu_at(a, p);
      members = max(cu_at(a, p + 1) - first, 0);
    }
    const int n = tiles_of(members, a.G, RT);
    int upto = n;   // inclusive scan
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int x = __shfl_up(upto, d);
      if (lane >= d) upto += x;
    }
    const uint64_t past = __ballot(upto > t);
    if (past != 0) {
      const int w = __builtin_ctzll(past);
      t -= __builtin_amdgcn_readlane(upto - n, w);
      return {p0 + w, __builtin_amdgcn_readlane(first, w), __builtin_amdgcn_readlane(members, w)};
    }
    t -= __builtin_amdgcn_readlane(upto, 63);
  }
  return {-1, 0, 0};
}

// 64 NR query rows (16 NR a wave) over cache rows [0, end): tiles of 64 positions of K and V go through
// LDS, loaded ahead, read by all four waves; a tile's scores are computed beside the previous tile's
// exponentials. V^T comes out of the transposing LDS read. P enters
// as two bf16 terms, its upper half and what that leaves (2^-15 of it is lost); l is their sum, by a product
// with ones. The running maximum is the first tile's and moves only when a weight against it
// exceeds 2^8, which leaves out nearly every search for it and every rescaling of the accumulators.
// 16-byte pieces of a row are swizzled by the row, so that 16 rows' pieces lie in different banks.
template <int D>
__device__ __forceinline__ int swz_k(int row, int c) {
  return row * (D / 8) + (c ^ (D == 64 ? (row >> 1) & 7 : row & 15));
}
template <int D>
__device__ __forceinline__ int swz_v(int row, int c) {
  return row * (D / 8) + (c ^ (D == 64 ? row & 7 : (row & 7) * 2));
}

// 16 bytes a lane from base + voff to LDS at lds + 16 lane. No register receives them; who reads them waits
// for the count of loads first. (The builtin makes the compiler wait before every later read of LDS.) m0 is a
// register that the compiler reserves, and warns about as one that is changed; it has no other use of it here.
__device__ __forceinline__ void lds16(const void* base, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :: "s"(lds), "v"(voff), "s"(base) : "memory");
}

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;

template <int D, int NR, typename RowAt, typename RecOf>
__device__ __forceinline__ void part_wide(const PrefixArgs& a, const uint16_t* kbase, const uint16_t* vbase,
                                          int end, int row0, int R, uint4* lds, RowAt row_at, RecOf rec_of) {
  constexpr int KC = D / 32, C = D / 8, LD = 64 * C / 256;
  uint4* const sk = lds;                  // [2][64 * C]
  uint4* const sv = lds + 2 * 64 * C;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = lane & 15, g = lane >> 4;
  const int r0 = row0 + wave * 16 * NR;

  u32x4_t q[NR][KC];
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const int r = r0 + 16 * n + j;
      q[n][c] = r < R ? *(const u32x4_t*)(row_at(r) + 32 * c + 8 * g) : u32x4_t{0u, 0u, 0u, 0u};
    }
  f32x4_t o[NR][D / 16], l[NR];
  float m[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    m[n] = -INFINITY;
    l[n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < D / 16; ++u) o[n][u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  // Tile t of K or V straight into its LDS buffer, 16 bytes a lane; a lane fetches what the swizzle puts in
  // its place. Rows past the end: the last one again, which moves no maximum, with a weight of 0 (`weigh`).
  const uint32_t k0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint4*)sk;
  const uint32_t v0 = k0 + 2 * 64 * C * 16;
  const int nt = (end + 63) / 64;
  const int row_of = tid / C;   // of this lane's first piece; the others are 256 / C rows on each
  const uint32_t ck = (uint32_t)((swz_k<D>(row_of, tid % C) % C) * 16);
  const uint32_t cv = (uint32_t)((swz_v<D>(row_of, tid % C) % C) * 16);
  auto fetch = [&](const uint16_t* base, uint32_t lds0, uint32_t c, int t) {
    if (t >= nt) return;
    const uint16_t* const from = base + (size_t)t * 64 * D;
    const int lim = min(63, end - 1 - t * 64);
#pragma unroll
    for (int i = 0; i < LD; ++i)
      lds16(from, (uint32_t)min(row_of + i * (256 / C), lim) * (2 * D) + c,
            lds0 + (uint32_t)((t & 1) * 64 * C + wave * 64 + 256 * i) * 16);
  };
  const bool busy = r0 < R;   // waves without rows only load
  const uint32_t one2 = 0x3F803F80u;
  const u32x4_t ones = {one2, one2, one2, one2};

  f32x4_t s[NR][4];   // the tile's scores
  // operands read from LDS a step ahead of their products (left to the compiler, every pair of products
  // waited for its own reads); only arithmetic is moved across
  u32x4_t kf[2][KC], vf[D / 16];
  auto hold = [] { __builtin_amdgcn_sched_barrier(0xE); };
  auto read_k = [&](int t, int x) {
#pragma unroll
    for (int c = 0; c < KC; ++c)
      kf[x & 1][c] = *(const u32x4_t*)(sk + (t & 1) * 64 * C + swz_k<D>(16 * x + j, 4 * c + g));
    hold();
  };
  auto read_v = [&](int t, int x2) {
#pragma unroll
    for (int u = 0; u < D / 16; ++u) {
      uint2 h[2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int row = 32 * x2 + 16 * y + 4 * g + (j >> 2);
        const char* p = (const char*)(sv + (t & 1) * 64 * C + swz_v<D>(row, 2 * u + ((j & 3) >> 1))) + 8 * (j & 1);
        h[y] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)p));
      }
      vf[u] = u32x4_t{h[0].x, h[0].y, h[1].x, h[1].y};
    }
    hold();
  };
  auto score = [&](int x) {
#pragma unroll
    for (int n = 0; n < NR; ++n) s[n][x] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
      for (int n = 0; n < NR; ++n) s[n][x] = mfma_bf16(kf[x & 1][c], q[n][c], s[n][x]);
  };
  // The greatest scaled score of subtiles x0 .. x1 - 1, per row.
  auto greatest = [&](int n, int x0, int x1) {
    float v = -INFINITY;
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (x >= x0 && x < x1)
#pragma unroll
        for (int e = 0; e < 4; ++e) v = fmaxf(v, s[n][x][e]);
    return xor32_max(xor16_max(v)) * a.scale_l2;
  };
  // Weights of half a tile against the maximum as it stands, and whether one is above 2^8 (or a NaN; positive
  // floats and NaNs, compared as whole numbers) or there is no maximum yet (every score so far was -inf).
  // `last`: some positions may lie past the end; theirs are 0, whatever the scale (scores of -inf would be NaN
  // with a scale of 0). Apart from the other tiles: as selects in every one, this made 120 us of 90 with
  // 256 x 16384.
  float w[NR][8];
  auto weigh = [&](int x2, auto last) {
    uint32_t top = 0;
    bool none = false;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      none |= m[n] == -INFINITY;
      const float mb = m[n] == -INFINITY ? 0.f : m[n];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[n][i] = exp2_hw(fmaf(s[n][2 * x2 + (i >> 2)][i & 3], a.scale_l2, -mb));
        if constexpr (last)
          if ((nt - 1) * 64 + 32 * x2 + 16 * (i >> 2) + 4 * g + (i & 3) >= end) w[n][i] = 0.f;
        top = max(top, __float_as_uint(w[n][i]));
      }
    }
    return __any(top > 0x43800000u || none);
  };
  // one tile's weights and their product; as its scores are used up, the next tile's take their place
  auto tile = [&](int t, auto more) {
    constexpr std::integral_constant<bool, !more> last{};
    if constexpr (more) {
      // K of tile t + 2 takes the place of tile t's, V of t + 1 that of t - 1's: both were last read
      // before the barrier that began this tile (the first tile's K, in front of the loop)
      fetch(kbase, k0, ck, t + 2);
      fetch(vbase, v0, cv, t + 1);
    }
    if (busy) {
      if constexpr (more) read_k(t + 1, 0);
#pragma unroll
      for (int x2 = 0; x2 < 2; ++x2) {
        if (weigh(x2, last)) {   // the maximum moves, and what was summed against it
#pragma unroll
          for (int n = 0; n < NR; ++n) {
            const float mn = fmaxf(m[n], greatest(n, 2 * x2, 2 * x2 + 2));
            const float corr = mn == -INFINITY ? 0.f : exp2_hw(m[n] - mn);
            m[n] = mn;
            l[n] *= corr;
#pragma unroll
            for (int u = 0; u < D / 16; ++u) o[n][u] *= corr;
          }
          weigh(x2, last);
        }
        if constexpr (more) read_k(t + 1, 2 * x2 + 1);
        read_v(t, x2);
        u32x4_t pp[NR], pr[NR];
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const uint32_t hi = perm(__float_as_uint(w[n][2 * y + 1]), __float_as_uint(w[n][2 * y]), 0x07060302u);
            pp[n][y] = hi;
            pr[n][y] = pack_bf16x2_op(w[n][2 * y] - bf16lo(hi), w[n][2 * y + 1] - bf16hi(hi));
          }
        if constexpr (more) {
          score(2 * x2);
          if (x2 == 0) read_k(t + 1, 2);
          score(2 * x2 + 1);
        }
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          l[n] = mfma_bf16(ones, pp[n], l[n]);
          l[n] = mfma_bf16(ones, pr[n], l[n]);
        }
#pragma unroll
        for (int u = 0; u < D / 16; ++u)
#pragma unroll
          for (int n = 0; n < NR; ++n) {
            o[n][u] = mfma_bf16(vf[u], pp[n], o[n][u]);
            o[n][u] = mfma_bf16(vf[u], pr[n], o[n][u]);
          }
      }
    }
    if constexpr (more) {
      wait_vm();
      __syncthreads();
    }
  };
  fetch(kbase, k0, ck, 0);
  fetch(vbase, v0, cv, 0);
  fetch(kbase, k0, ck, 1);
  wait_vm();
  __syncthreads();
  if (busy) {
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      read_k(0, x);
      score(x);
    }
#pragma unroll
    for (int n = 0; n < NR; ++n) m[n] = greatest(n, 0, 4);
  }
  // every wave has read the first tile of K before any fetches the third into its place (waves without rows
  // read nothing and would be far ahead)
  if (nt > 2) __syncthreads();
  for (int t = 0; t + 1 < nt; ++t) tile(t, std::true_type{});
  tile(nt - 1, std::false_type{});
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int r = r0 + 16 * n + j;
    if (r >= R) continue;
    float* to = a.rec + rec_of(r);
#pragma unroll
    for (int u = 0; u < D / 16; ++u)
      *(float4*)(to + 16 * u + 4 * g) = make_float4(o[n][u][0], o[n][u][1], o[n][u][2], o[n][u][3]);
    if (g == 0) *(float2*)(to + D) = make_float2(m[n], l[n][0]);
  }
}

template <int D, int NR>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void prefix_parts_kernel(PrefixArgs a) {
  constexpr int kNarrow = (kPartWaves * 16 * D + 8 * 16) * 4;
  constexpr int kWide = 4 * 64 * D * 2;
  __shared__ __attribute__((aligned(16))) uint4 lds[(kNarrow > kWide ? kNarrow : kWide) / 16];
  const int lane = threadIdx.x & 63;
  const int slots = a.ns_own + a.ns_pre;
  int blk = blockIdx.x;
  const int n_pre = a.hkv * a.tiles * a.ns_pre;
  if (blk < n_pre) {
    // the kv head fastest: with 8 of them an XCD's L2 holds one head's rows for all of its row tiles
    const int kvh = blk % a.hkv;
    blk /= a.hkv;
    int t = blk % a.tiles;
    const int part = blk / a.tiles;
    const Group gr = find_tile(a, 64 * NR, lane, t);
    if (gr.p < 0) return;
    const int len = min(max(a.plens[gr.p], 0), a.max_prefix);
    const int start = part * a.chunk_pre;
    if (start >= len) return;
    const int end = min(a.chunk_pre, len - start);
    const int R = gr.members * a.G;
    const size_t at = (size_t)gr.p * a.pp_stride + (size_t)kvh * a.ph_stride + (size_t)start * D;
    auto row_at = [&](int r) {
      const int i = r / a.G;
      return a.q + ((size_t)(gr.first + i) * a.hq + kvh * a.G + (r - i * a.G)) * D;
    };
    auto rec_of = [&](int r) {
      const int i = r / a.G;
      return (((size_t)(gr.first + i) * a.hkv + kvh) * slots + a.ns_own + part) * (size_t)(a.G * kRec<D>) +
             (size_t)(r - i * a.G) * kRec<D>;
    };
    if (R <= 16) {
      Narrow<D> st;
      st.init(row_at(min(lane & 15, R - 1)), R);
      st.template run<false>(a.kp + at, a.vp + at, end, a.scale_l2, R, nullptr, 0);
      st.finish(R, (float*)lds, [&](int r, int d, const float4& A, float m, float l) {
        put_record<D>(a.rec + rec_of(r), d, A, m, l);
      });
    } else
      part_wide<D, NR>(a, a.kp + at, a.vp + at, end, t * 64 * NR, R, lds, row_at, rec_of);
    return;
  }
  blk -= n_pre;
  const int kvh = blk % a.hkv;
  blk /= a.hkv;
  const int b = blk % a.batch, part = blk / a.batch;
  const int len = min(max(a.lens[b], 0), a.max_len);
  const int start = part * a.chunk_own;
  if (start >= len) return;
  const int end = min(a.chunk_own, len - start);
  const size_t at = (size_t)b * a.b_stride + (size_t)kvh * a.h_stride + (size_t)start * D;
  const size_t rec = (((size_t)b * a.hkv + kvh) * slots + part) * (size_t)(a.G * kRec<D>);
  Narrow<D> st;
  st.init(a.q + ((size_t)b * a.hq + kvh * a.G + min(lane & 15, a.G - 1)) * D, a.G);
  st.template run<false>(a.k + at, a.v + at, end, a.scale_l2, a.G, nullptr, 0);
  st.finish(a.G, (float*)lds, [&](int r, int d, const float4& A, float m, float l) {
    put_record<D>(a.rec + rec + (size_t)r * kRec<D>, d, A, m, l);
  });
}

// The prefix of sequence b (-1: none) and its length, by all lanes of a wave; one round of loads for 64
// prefixes.
struct Prefix {
  int p, len;
};
__device__ __forceinline__ Prefix prefix_of(const PrefixArgs& a, int b, int lane) {
  for (int p0 = 0; p0 < a.n_prefixes; p0 += 64) {
    const int p = min(p0 + lane, a.n_prefixes - 1);
    const int n = a.plens[p];
    const uint64_t who = __ballot(p == p0 + lane && cu_at(a, p) <= b && b < cu_at(a, p + 1));
    if (who != 0) {
      const int w = __builtin_ctzll(who);
      return {p0 + w, min(max(__builtin_amdgcn_readlane(n, w), 0), a.max_prefix)};
    }
  }
  return {-1, 0};
}

// One workgroup per (sequence, kv head): everything.
template <int D>
__global__ __launch_bounds__(kPartWaves * 64) void prefix_whole_kernel(PrefixArgs a) {
  extern __shared__ __attribute__((aligned(16))) float lds[];   // kPartWaves * G * (D + 2)
  const int lane = threadIdx.x & 63;
  const int b = blockIdx.x / a.hkv, kvh = blockIdx.x - b * a.hkv;
  const size_t row = (size_t)b * a.hq + kvh * a.G;
  Narrow<D> st;
  st.init(a.q + (row + min(lane & 15, a.G - 1)) * D, a.G);
  const int len = min(max(a.lens[b], 0), a.max_len);
  const Prefix p = prefix_of(a, b, lane);
  if (p.len > 0) {
    const size_t at = (size_t)p.p * a.pp_stride + (size_t)kvh * a.ph_stride;
    st.template run<false>(a.kp + at, a.vp + at, p.len, a.scale_l2, a.G, nullptr, 0);
  }
  const size_t at = (size_t)b * a.b_stride + (size_t)kvh * a.h_stride;
  if (len > 0) st.template run<false>(a.k + at, a.v + at, len, a.scale_l2, a.G, nullptr, 0);
  st.finish(a.G, lds, [&](int r, int d, const float4& A, float, float l) {
    put_channels(a.out, a.out_f32, (row + r) * D + d, whole(A, l));
  });
}

// One wave per (sequence, query head): the records that were written, merged.
template <int D>
__global__ __launch_bounds__(256) void prefix_merge_kernel(PrefixArgs a) {
  const int lane = threadIdx.x & 63;
  const int i = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  if (i >= a.batch * a.hq) return;
  const int b = i / a.hq, h = i - b * a.hq;
  const int kvh = h / a.G, slots = a.ns_own + a.ns_pre;
  const float* rec = a.rec + (((size_t)b * a.hkv + kvh) * slots * a.G + (h - kvh * a.G)) * kRec<D>;
  const float4 A = merge_records<D>(rec, (size_t)a.G * kRec<D>, slots, lane, [&](int r) {
    const int len = min(max(a.lens[b], 0), a.max_len);
    const int pl = prefix_of(a, b, lane).len;
    return r < a.ns_own ? r * a.chunk_own < len : (r - a.ns_own) * a.chunk_pre < pl;
  });
  if (lane < D / 4) put_channels(a.out, a.out_f32, (size_t)i * D + 4 * lane, A);
}

struct PrefixPlan {
  bool whole;   // one launch
  int nr, tiles, ns_pre, chunk_pre, ns_own, chunk_own;
};

// How the work is cut. Only bounds are known here (the lengths are on the device).
static PrefixPlan prefix_plan(int batch, int hq, int hkv, int d, int n_prefixes, int max_prefix, int max_len) {
  const int G = hq / hkv;
  const long long rows = (long long)batch * G;
  PrefixPlan p{};
  if (n_prefixes == 0) max_prefix = 0;
  // One launch up to 256 KB of K and V for each compute unit, which takes 1024 positions of D = 64 in 5 us
  // (eager / in a graph, two launches: 8 x 500 10.6 / 7.1, 13.4 / 9.2; 8 x 900 10.7 / 9.3, 13.3 / 9.3; 64 x 300
  // 10.4 / 8.8, 13.4 / 12.5; 1 x 900 10.5 / 9.1, 13.2 / 7.1; D = 128, 8 x 900 14.5 / 14.7, 13.3 / 10.4)
  const long long each = ((long long)batch * hkv + 255) / 256;   // a compute unit's workgroups
  p.whole = each * (max_prefix + max_len) <= 65536 / d;
  if (p.whole) return p;
  // 32 rows a wave where prefixes have more than 64 of them on average and the registers hold it
  p.nr = d == 64 && rows > 64ll * (n_prefixes > 1 ? n_prefixes : 1) ? 2 : 1;
  const int rt = 64 * p.nr;
  // every prefix may end inside a tile; a tile has a member at least (prefixes may have none)
  const long long most = (rows + rt - 1) / rt + (n_prefixes > 0 ? n_prefixes - 1 : 0);
  p.tiles = (int)(most < batch ? most : batch);
  if (max_prefix == 0) p.tiles = 0;
  if (p.tiles > 0)
    // D = 64: what the chip holds at once, three workgroups a compute unit (256 x 16384: 384 / 512 / 640 / 768 /
    // 1024 took 119 / 94 / 96 / 91 / 95 us). D = 128: less, beside the own caches' parts (48 x 5003: 384 / 512 /
    // 768 / 1024 took 30.4 / 32.0 / 32.3 / 34.2)
    cut_parts(max_prefix, (d == 64 ? 768 : 384) / ((long long)hkv * p.tiles), rows <= 16 ? kPartRound : 256, 64,
              &p.ns_pre, &p.chunk_pre);
  if (max_len > 0)
    cut_parts(max_len, 1024 / ((long long)hkv * batch), 256, kPartRound, &p.ns_own, &p.chunk_own);
  if (p.chunk_pre == 0) p.chunk_pre = 64;
  if (p.chunk_own == 0) p.chunk_own = kPartRound;
  return p;
}

static bool prefix_shape_ok(int batch, int hq, int hkv, int d, int n_prefixes, int max_prefix, int max_len) {
  return batch >= 1 && batch <= (1 << 20) && hkv >= 1 && hkv <= 1024 && hq >= hkv && hq % hkv == 0 && hq / hkv <= 16 &&
         (d == 64 || d == 128) && n_prefixes >= 0 && n_prefixes <= (1 << 20) && max_prefix >= 0 &&
         max_prefix < (1 << 24) && max_len >= 0 && max_len < (1 << 24) && (long long)batch * hq < (1 << 28);
}

static size_t prefix_rec_bytes(const PrefixPlan& p, int batch, int hq, int d) {
  return (size_t)batch * hq * (p.ns_own + p.ns_pre) * (d + 4) * 4;
}

template <int D>
static void prefix_launch(const PrefixArgs& a, const PrefixPlan& p, hipStream_t s) {
  if (p.whole) {
    const size_t lds = (size_t)kPartWaves * a.G * (D + 2) * 4;
    hipLaunchKernelGGL(prefix_whole_kernel<D>, dim3((unsigned)(a.batch * a.hkv)), dim3(kPartWaves * 64), lds, s, a);
    return;
  }
  const unsigned grid = (unsigned)(a.hkv * (p.tiles * p.ns_pre + a.batch * p.ns_own));
  if (D == 64 && p.nr == 2) hipLaunchKernelGGL((prefix_parts_kernel<64, 2>), dim3(grid), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((prefix_parts_kernel<D, 1>), dim3(grid), dim3(256), 0, s, a);
  const unsigned wgs = (unsigned)(((long long)a.batch * a.hq + 3) / 4);
  hipLaunchKernelGGL(prefix_merge_kernel<D>, dim3(wgs), dim3(256), 0, s, a);
}

}  // namespace q4nx

using namespace q4nx;

extern "C" {

size_t q4nx_gqa_prefix_decode_ws_bytes(int batch, int n_q_heads, int n_kv_heads, int head_dim, int n_prefixes,
                                       int max_prefix, int max_len) {
  if (!prefix_shape_ok(batch, n_q_heads, n_kv_heads, head_dim, n_prefixes, max_prefix, max_len)) return 0;
  const PrefixPlan p = prefix_plan(batch, n_q_heads, n_kv_heads, head_dim, n_prefixes, max_prefix, max_len);
  return (size_t)Q4NX_WS_COUNTER_BYTES + prefix_rec_bytes(p, batch, n_q_heads, head_dim);
}

int q4nx_gqa_prefix_decode(const uint16_t* q, const uint16_t* k_prefix, const uint16_t* v_prefix,
                           int64_t prefix_stride, int64_t prefix_h_stride, const int32_t* prefix_lens,
                           const int32_t* cu, int n_prefixes, int max_prefix, const uint16_t* k_cache,
                           const uint16_t* v_cache, int64_t kv_b_stride, int64_t kv_h_stride,
                           const int32_t* lens, int max_len, uint16_t* out, float* out_f32, int batch,
                           int n_q_heads, int n_kv_heads, int head_dim, float scale, void* ws, size_t ws_bytes,
                           void* stream) {
  const char* what = "q4nx_gqa_prefix_decode";
  Q4NX_REQUIRE(prefix_shape_ok(batch, n_q_heads, n_kv_heads, head_dim, n_prefixes, max_prefix, max_len),
               Q4NX_ERR_SHAPE,
               "%s: batch=%d Hq=%d (a multiple of Hkv, at most 16 times) Hkv=%d head_dim=%d (64, 128) "
               "n_prefixes=%d (at most 2^20) max_prefix=%d max_len=%d (below 2^24)",
               what, batch, n_q_heads, n_kv_heads, head_dim, n_prefixes, max_prefix, max_len);
  const bool pre = n_prefixes > 0 && max_prefix > 0, own = max_len > 0;
  Q4NX_REQUIRE(q && lens && (out || out_f32) && (!own || (k_cache && v_cache)) &&
                   (!pre || (k_prefix && v_prefix && prefix_lens)),
               Q4NX_ERR_ARG, "%s: q, the caches, their lengths and an output are required", what);
  Q4NX_REQUIRE(!pre || n_prefixes == 1 || cu, Q4NX_ERR_ARG, "%s: %d prefixes need cu", what, n_prefixes);
  Q4NX_REQUIRE(Q4NX_ALIGNED(q, 16) && Q4NX_ALIGNED(k_cache, 16) && Q4NX_ALIGNED(v_cache, 16) &&
                   Q4NX_ALIGNED(k_prefix, 16) && Q4NX_ALIGNED(v_prefix, 16),
               Q4NX_ERR_ARG, "%s: q and the caches must be 16-byte aligned", what);
  Q4NX_REQUIRE(Q4NX_ALIGNED(out, 8) && Q4NX_ALIGNED(out_f32, 16), Q4NX_ERR_ARG,
               "%s: out must be 8-byte, out_f32 16-byte aligned", what);
  Q4NX_REQUIRE(!own || (kv_h_stride >= (int64_t)max_len * head_dim && kv_h_stride % 8 == 0 &&
                        kv_b_stride >= (int64_t)n_kv_heads * kv_h_stride && kv_b_stride % 8 == 0),
               Q4NX_ERR_SHAPE, "%s: cache strides do not hold [Hkv][max_len][head_dim]", what);
  Q4NX_REQUIRE(!pre || (prefix_h_stride >= (int64_t)max_prefix * head_dim && prefix_h_stride % 8 == 0 &&
                        (n_prefixes == 1 || (prefix_stride >= (int64_t)n_kv_heads * prefix_h_stride &&
                                             prefix_stride % 8 == 0))),
               Q4NX_ERR_SHAPE, "%s: prefix strides do not hold [Hkv][max_prefix][head_dim]", what);
  Q4NX_REQUIRE(scale >= 0.f, Q4NX_ERR_ARG, "%s: scale must not be negative", what);
  const PrefixPlan p = prefix_plan(batch, n_q_heads, n_kv_heads, head_dim, n_prefixes, max_prefix, max_len);
  Q4NX_REQUIRE((long long)n_kv_heads * ((long long)p.tiles * p.ns_pre + (long long)batch * p.ns_own) < (1ll << 31),
               Q4NX_ERR_SHAPE, "%s: more than 2^31 workgroups", what);
  const size_t need = (size_t)Q4NX_WS_COUNTER_BYTES + prefix_rec_bytes(p, batch, n_q_heads, head_dim);
  Q4NX_REQUIRE(ws != nullptr && ws_bytes >= need && Q4NX_ALIGNED(ws, 256), Q4NX_ERR_WS,
               "%s: workspace of %zu bytes (256-aligned) needed, %zu given", what, need, ws_bytes);
  PrefixArgs a{};
  a.q = q;
  a.k = k_cache;
  a.v = v_cache;
  a.kp = k_prefix;
  a.vp = v_prefix;
  a.lens = lens;
  a.plens = prefix_lens;
  a.cu = cu;
  a.out = out;
  a.out_f32 = out_f32;
  a.rec = (float*)((uint8_t*)ws + Q4NX_WS_COUNTER_BYTES);
  a.b_stride = kv_b_stride;
  a.h_stride = kv_h_stride;
  a.pp_stride = n_prefixes > 1 ? prefix_stride : 0;
  a.ph_stride = prefix_h_stride;
  a.batch = batch;
  a.hq = n_q_heads;
  a.hkv = n_kv_heads;
  a.G = n_q_heads / n_kv_heads;
  a.n_prefixes = pre ? n_prefixes : 0;
  a.max_prefix = max_prefix;
  a.max_len = max_len;
  a.ns_pre = p.ns_pre;
  a.chunk_pre = p.chunk_pre;
  a.tiles = p.tiles;
  a.ns_own = p.ns_own;
  a.chunk_own = p.chunk_own;
  a.scale_l2 = (float)((double)scale * 1.4426950408889634);
  hipStream_t s = (hipStream_t)stream;
  if (head_dim == 64) prefix_launch<64>(a, p, s);
  else prefix_launch<128>(a, p, s);
  return check_launch(what);
}

}  // extern "C"
