// The paged 4-bit K/V cache: what its kernels share.
//
// A row's channels are quantised in groups of 32: m the least value, d = bf16((max - m) / 15),
// code = rint((x - m) / d) held to 0..15 (each step rounded to fp32); it stands for d * code + m.
// A page holds page_len positions; per kv head page_len/32 tiles, then the bounds of K's channels.
// A tile is 32 positions in the order the matrix cores take them (D = head_dim, lane = 16 kg + n):
//   K codes  [D/64][64 lanes][4 dwords]: dword 2 tt + g of lane (n, kg) is position 16 tt + n,
//            channels 64 c + 32 g + 8 kg + i, nibbles (lowest first) i = 0, 2, 4, 6, 1, 3, 5, 7
//   V codes  [D/64][64 lanes][4 dwords]: dword t is channel 64 c + 16 t + n, nibbles (lowest first)
//            positions 4 kg .. 4 kg + 3 and 16 + 4 kg .. 16 + 4 kg + 3
//   K scales bf16 (d, m) [32][D/32], V scales the same
// so one 16-byte load per lane is a whole operand set, and (dword >> 4 r) & 0x000f000f are the codes
// of operand elements 2 r and 2 r + 1: or-ed into 0x4300 each is the bf16 number 128 + code
// (three bits higher, into 0x4180: 16 + code).
#pragma once

#include "common.h"

namespace q4nx {

constexpr int kKv4Tile = 32;             // positions per tile
constexpr uint32_t kKv4NaN = 0x7FC07FC0u;   // (d, m) of a group with a NaN or an infinity

struct Kv4 {
  uint8_t* pages;
  int64_t page_stride;
  int32_t* table;
  int64_t table_stride;
  int n_pages, page_len, tiles, hkv, n_seqs, table_len;
  int shift;   // log2 of tiles, the tiles of a page
  int cap;   // positions a sequence can hold: table_len * page_len
};

__host__ __device__ constexpr int kv4_tile_bytes(int d) { return 40 * d; }
__host__ __device__ constexpr int kv4_head_bytes(int page_len, int d) {
  return page_len / kKv4Tile * kv4_tile_bytes(d) + 4 * d;
}

// Checks *c and fills *out; a negative Q4NX_ERR_* with the message set otherwise.
int kv4_resolve(const q4nx_kv4* c, Kv4* out, const char* what);

// The physical page of logical page `lp` of sequence b, -1 when the entry names none.
__device__ __forceinline__ int kv4_page(const Kv4& c, int b, int lp) {
  if (lp < 0 || lp >= c.table_len) return -1;
  const int id = c.table[(int64_t)b * c.table_stride + lp];
  return id >= 0 && id < c.n_pages ? id : -1;
}

// Two codes as the bf16 pair (128 + code, 128 + code): a shift and v_and_or_b32, which takes one
// constant from a scalar register and needs the other in a vector register.
__device__ __forceinline__ uint32_t kv4_pair(uint32_t w, int r) {
  uint32_t mask = 0x000F000Fu, bias = 0x43004300u;
  asm("" : "+s"(mask));
  asm("" : "+v"(bias));
  return ((w >> (4 * r)) & mask) | bias;
}
__device__ __forceinline__ u32x4_t kv4_operand(uint32_t w) {
  return u32x4_t{kv4_pair(w, 0), kv4_pair(w, 1), kv4_pair(w, 2), kv4_pair(w, 3)};
}

// The same as (16 + code, 16 + code): one shift more, and an eighth of what is left of a rounding of the
// other operand when the 16 is taken out of a sum again.
__device__ __forceinline__ u32x4_t kv4_operand16(uint32_t w) {
  uint32_t mask = 0x00780078u, bias = 0x41804180u;
  asm("" : "+s"(mask));
  asm("" : "+v"(bias));
  return u32x4_t{((w << 3) & mask) | bias, ((w >> 1) & mask) | bias, ((w >> 5) & mask) | bias,
                 ((w >> 9) & mask) | bias};
}

}  // namespace q4nx
