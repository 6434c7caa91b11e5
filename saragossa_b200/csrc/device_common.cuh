// Device helpers shared by the kernels: storage conversions (bit-exact with the
// reference's host code), element access through the page layout, and the
// split-K partial merge.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "layout.h"

namespace sgk {

// Device status word values (read back by sgk_state_device_status).
constexpr int DEV_OK = 0;
constexpr int DEV_ERR_WAIT_TIMEOUT = 6;  // a bounded mbarrier wait expired
constexpr int DEV_ERR_BAD_PAGE = 7;      // a block-table entry was out of range

// f32 -> bf16 bits, round to nearest even: bits + 0x7fff + lsb, >> 16, the integer
// form of the reference (src/decode_resident/utils.rs:55-60), NaN not special-cased.
__device__ __forceinline__ uint16_t f32_to_bf16_bits(float v) {
  uint32_t bits = __float_as_uint(v);
  uint32_t lsb = (bits >> 16) & 1u;
  return static_cast<uint16_t>((bits + 0x7fffu + lsb) >> 16);
}
__device__ __forceinline__ float bf16_bits_to_f32(uint16_t b) {
  return __uint_as_float(static_cast<uint32_t>(b) << 16);
}

// f32 bits of a u8 group's scale for the pool's largest one: an infinite scale (a group whose values read back as no numbers)
// counts as none, or every other row of the pool would lose its weights to it from then on.
__device__ __forceinline__ uint32_t u8_scale_for_max(uint32_t scale_bits) {
  return scale_bits < 0x7f80u ? scale_bits << 16 : 0u;
}

// Signed step of (row, group) of a u4 tile as f32. V steps are stored divided by their row's power of two.
__device__ __forceinline__ float u4_step(const uint8_t* tile, int hd, int is_v, int row, int grp) {
  const uint16_t bits = *reinterpret_cast<const uint16_t*>(tile + u4_step_offset(is_v, row, grp, hd));
  if (!is_v) return bf16_bits_to_f32(bits);
  const uint8_t* pow_tile = row < 8 ? tile - tile_bytes(KV_U4G32, hd) : tile;   // the K tile lies before the V tile
  return __half2float(__ushort_as_half(bits)) *
         bf16_bits_to_f32(*reinterpret_cast<const uint16_t*>(pow_tile + u4_pow_offset(row, hd)));
}
__device__ __forceinline__ int u4_code(const uint8_t* tile, int hd, int is_v, int row, int dim) {
  return (tile[is_v ? u4_v_byte(row, dim, hd) : u4_k_byte(row, dim, hd)] >> (4 * u4_nibble(dim))) & 15;
}

// One element (row, dim) of a u4 tile decoded to f32 (the product is exact). A V tile is decoded where it lies, behind
// its K tile.
__device__ __forceinline__ float load_u4_elem(const uint8_t* tile, int hd, int is_v, int row, int dim) {
  return fmaf(static_cast<float>(u4_code(tile, hd, is_v, row, dim)), u4_step(tile, hd, is_v, row, dim / QGROUP),
              bf16_bits_to_f32(*reinterpret_cast<const uint16_t*>(tile + u4_bias_offset(row, dim / QGROUP, hd))));
}

// One stored element (row, dim) of a tile decoded to f32: f32 as is, bf16 upcast,
// u8 q*scale+bias with separate roundings (src/quantization.rs:173-179).
__device__ __forceinline__ float load_tile_elem(const uint8_t* tile, int dtype, int hd, int is_v,
                                                int row, int dim) {
  if (dtype == KV_F32) return reinterpret_cast<const float*>(tile)[row * hd + dim];
  if (dtype == KV_BF16)
    return bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(tile)[bf16_elem_index(row, dim, hd)]);
  int idx = is_v ? u8_v_code_index(row, dim, hd) : u8_k_code_index(row, dim, hd);
  float scale = bf16_bits_to_f32(*reinterpret_cast<const uint16_t*>(tile + u8_scale_offset(row, dim / QGROUP, hd)));
  float bias = bf16_bits_to_f32(*reinterpret_cast<const uint16_t*>(tile + u8_bias_offset(is_v, row, dim / QGROUP, hd)));
  return __fadd_rn(__fmul_rn(static_cast<float>(tile[idx]), scale), bias);
}

// Split-K partials: for every (sequence, q head, split) an un-normalised output
// row, its running maximum (log2 domain) and its sum of weights.
struct Partials {
  float* o;   // [n_seq * q_heads][splits][head_dim]
  float* ml;  // [n_seq * q_heads][splits][2] = {max, sum}
};

// Merges the `splits` partials of q head `qh_global` and writes the normalised
// output. Called by every thread of the block that arrived last.
__device__ __forceinline__ void merge_partials(const Partials& part, int64_t qh_global, int splits,
                                               int hd, float* out_row, int tid, int nthreads) {
  const float* ml = part.ml + qh_global * splits * 2;
  float m = -1.0e30f;
#pragma unroll 8
  for (int s = 0; s < splits; ++s) m = fmaxf(m, __ldcg(ml + 2 * s));
  float denom = 0.0f;
#pragma unroll 8
  for (int s = 0; s < splits; ++s) denom += __ldcg(ml + 2 * s + 1) * exp2f(__ldcg(ml + 2 * s) - m);
  float inv = 1.0f / denom;
  const float* o = part.o + qh_global * splits * hd;
  for (int d = tid; d < hd; d += nthreads) {
    float acc = 0.0f;
#pragma unroll 8
    for (int s = 0; s < splits; ++s)
      acc += __ldcg(o + int64_t(s) * hd + d) * exp2f(__ldcg(ml + 2 * s) - m);
    out_row[d] = acc * inv;
  }
}

}  // namespace sgk
