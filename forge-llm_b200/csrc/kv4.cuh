// The 4-bit KV cache's layout and addressing, shared by its kernels.
//
// A row is one kv head of one slot: dH values x as codes c in 0..15 on the
// row's own grid, x^ = base + step * c (step, base in bf16).  Element e sits in
// nibble e & 1 of byte e / 2; a row is padded to pad(dH) elements so that
// it is a whole number of 16-byte units.  Row (layer, block, head, slot in
// block) has index ((layer * blocks + block) * nKV + head) * block_size + slot:
// the slots of one head of one block are contiguous, which is what a kernel
// that walks one head's history reads.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace fcu {
namespace kv4 {

constexpr int kMaxDh = 256;
constexpr int kMaxGroup = 16;   // q heads per kv head

// Elements a row of dH values is stored as: the widths that the kernels are built for,
// whole 16-byte pieces.
__host__ __device__ inline int pad(int dH) {
  return dH <= 32 ? 32 : dH <= 64 ? 64 : dH <= 96 ? 96 : dH <= 128 ? 128 : dH <= 192 ? 192 : 256;
}

// One cache as the kernels see it.
struct Cache {
  uint8_t *k, *v;
  uint32_t *kg, *vg;         // bf16 pairs: step low, base high
  float *weight;
  int32_t *pos;
  const int32_t *table;
  int64_t layers, blocks;
  int nKV, dH, rb;           // rb: bytes of a row's codes
  int bs, mb;                // slots per block, blocks per sequence
  int64_t cap;               // slots per sequence
  uint32_t div_mul;          // j / bs = (umulhi(div_mul, j) + j) >> div_shift for j < 2^31
  int div_shift;
};

__device__ __forceinline__ int64_t block_index(const Cache &c, int64_t j) {
  return (__umulhi(c.div_mul, (uint32_t)j) + (uint32_t)j) >> c.div_shift;
}

// Physical block of logical block i of sequence b; -1 if the table names a
// block the cache does not have (its slots are then never touched).
__device__ __forceinline__ int64_t block_of(const Cache &c, int64_t b, int64_t i) {
  if (!c.table) return b * c.mb + i;
  const int64_t p = c.table[b * c.mb + i];
  return p >= 0 && p < c.blocks ? p : -1;
}

// Row index of slot j of head h of sequence b in layer 0; -1 for a bad block.
__device__ __forceinline__ int64_t row_of(const Cache &c, int64_t b, int h, int64_t j) {
  const int64_t i = block_index(c, j);
  const int64_t p = block_of(c, b, i);
  return p < 0 ? -1 : (p * c.nKV + h) * c.bs + (j - i * c.bs);
}

__device__ __forceinline__ float grid_step(uint32_t g) { return __uint_as_float(g << 16); }
__device__ __forceinline__ float grid_base(uint32_t g) { return __uint_as_float(g & 0xffff0000u); }
constexpr uint32_t kNanGrid = 0x7fc07fc0u;   // step and base NaN: every value of the row is NaN

// The host's view checked once for every entry point; 0 or an fcu_status.
int view(const char *who, const fcu_kv4 *in, int64_t B, bool need_values, Cache *out);

}  // namespace kv4
}  // namespace fcu
