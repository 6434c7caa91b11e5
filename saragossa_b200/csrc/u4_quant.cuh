// The 4-bit quantiser shared by the append kernels and the fused append of the attention kernel.
//
// A head row is cut into groups of 32 values. Rows at odd positions are quantised negated (y = -x): V
// rows are summed with weights p, and codes that all count up from a minimum would make that sum a
// large number minus a large number; with the sign alternating from row to row neighbouring rows
// cancel inside one matrix instruction and the f32 accumulator keeps its digits.
//   bias = bf16(min y),  step = bf16(max((max y - bias) / 15, 2^-40, 2^(e-16))),
//   2^e = the power of two at or below the largest (max y - bias) / 15 of the head row (at least 2^-40),
//   code = nearest((y - bias) / step), ties to even, kept within 0..15;
//   stored: the codes, (-1)^row * step and (-1)^row * bias.
// The floor 2^(e-16) lets V keep step / 2^e as an fp16 number without loss.
//
// Each rounding is of the exact value, although everything runs in f32: a difference a - b comes with
// its rounding error (Knuth's two-sum, for a difference), multiples of a bf16 step by a number below 16 and of a 9-bit
// midpoint by 15 are exact, and so are the remainders they leave. A division that is rounded to f32
// first and to bf16 afterwards picks the wrong neighbour about once in 2^15 groups.
//
// A group that holds an infinity or a NaN, or whose bias or step is not finite, reads back as NaN.
#pragma once
#include "device_common.cuh"

namespace sgk {

// two f32 operations in one instruction
__device__ __forceinline__ uint64_t pair_of(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ void add2(float& x, float& y, float a, float b) {   // (x, y) += (a, b)
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_of(x, y)), "l"(pair_of(a, b)));
  unpair(r, x, y);
}
__device__ __forceinline__ void fma2(float& x, float& y, float a, float b, float c, float d) {   // (x, y) += (a, b) * (c, d)
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pair_of(a, b)), "l"(pair_of(c, d)), "l"(pair_of(x, y)));
  unpair(r, x, y);
}
__device__ __forceinline__ void mul2(float& x, float& y, float a, float b) {   // (x, y) *= (a, b)
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_of(x, y)), "l"(pair_of(a, b)));
  unpair(r, x, y);
}

constexpr int U4_EXP_MIN = -40;   // smallest step 2^-40

// a - b = d + err exactly
__device__ __forceinline__ float two_diff(float a, float b, float& err) {
  const float d = __fsub_rn(a, b);
  const float z = __fsub_rn(d, a);
  err = __fsub_rn(__fsub_rn(a, __fsub_rn(d, z)), __fadd_rn(b, z));
  return d;
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }   // -126..127

// What the values of one group say of it: bias, width = max y - bias as a pair, exponent of width / 15.
struct U4Range {
  float bias, width, err;
  int exponent;   // U4_EXP_MIN .. 127
  bool finite;
};
__device__ __forceinline__ U4Range u4_range(float lo, float hi) {
  U4Range r;
  r.bias = bf16_bits_to_f32(f32_to_bf16_bits(lo));
  r.width = two_diff(hi, r.bias, r.err);
  r.finite = fabsf(r.bias) < INFINITY && r.width < INFINITY;
  // floor(log2(width / 15)), from a quotient that may be a unit off; anything below the least exponent counts as that
  const int guess = static_cast<int>(__float_as_uint(fmaxf(r.width, 0x1p-40f) * (1.0f / 15.0f)) >> 23);
  const float at = 15.0f * __uint_as_float(static_cast<uint32_t>(guess) << 23);
  int e = guess - 127;
  if (r.width < at || (r.width == at && r.err < 0.0f)) e -= 1;
  if (r.width > 2.0f * at || (r.width == 2.0f * at && r.err >= 0.0f)) e += 1;
  r.exponent = r.finite ? max(e, U4_EXP_MIN) : U4_EXP_MIN;
  return r;
}
// bf16 bits of the (positive) step of a group; row_exponent = the largest exponent of the head row.
__device__ __forceinline__ uint16_t u4_step_bits(const U4Range& r, int row_exponent) {
  const float floor_step = pow2f(max(row_exponent - 16, U4_EXP_MIN));
  const float at = 15.0f * floor_step;
  const uint32_t low = __float_as_uint(r.width * (1.0f / 15.0f)) & 0xffff0000u;
  const float mid = 15.0f * __uint_as_float(low | 0x8000u);   // the border to the next bf16 value, times 15
  const bool up = r.width > mid || (r.width == mid && (r.err > 0.0f || (r.err == 0.0f && (low & 0x10000u))));
  uint32_t bits = (low >> 16) + (up ? 1u : 0u);
  if (r.width < at || (r.width == at && r.err <= 0.0f)) bits = __float_as_uint(floor_step) >> 16;
  return static_cast<uint16_t>(r.finite ? bits : 0x7fc0u);
}
// Code of y; inv ~ 1 / step (an error of a few units in the last place is mended below).
__device__ __forceinline__ uint32_t u4_code_of(float y, float bias, float step, float inv) {
  const float t = __fsub_rn(y, bias);
  const float guess = fminf(fmaxf(t * inv, 0.0f), 15.0f) + 12582912.0f;   // 1.5 * 2^23: rounds to a whole number
  int code = static_cast<int>(__float_as_uint(guess) & 15u);
  const float rest = fmaf(-(guess - 12582912.0f), step, t);   // exact
  const float half = 0.5f * step;
  if (fabsf(rest) >= half) {   // at a border, or past it: rare
    float err;
    two_diff(y, bias, err);
    const bool tie_moves = err == 0.0f && (code & 1);
    if (rest > half || (rest == half && (err > 0.0f || tie_moves))) code += 1;
    else if (rest < -half || (rest == -half && (err < 0.0f || tie_moves))) code -= 1;
    code = min(max(code, 0), 15);
  }
  return static_cast<uint32_t>(code);
}
// The same for eight values sign * v of a group at once: codes of v[0..3] and v[4..7] as the bytes c[j] + 16 c[j + 4]; inv15 ~
// 1 / (15 step). The code is guessed, and right when t is less than half a step from it: t and the distance are rounded
// once each, and a border between two codes is a number that f32 holds, so neither rounding carries a value across it. The
// borders are looked at only when one of the eight lies on one.
__device__ __forceinline__ uint32_t u4_codes8(const float (&v)[8], float sign, float bias, float step, float inv15) {
  float t[8], n[8], d[8], byte[4];
#pragma unroll
  for (int j = 0; j < 8; ++j) t[j] = -bias, n[j] = 12582912.0f;   // 1.5 * 2^23: rounds to a whole number
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    fma2(t[j], t[j + 1], v[j], v[j + 1], sign, sign);
    fma2(n[j], n[j + 1], __saturatef(t[j] * inv15), __saturatef(t[j + 1] * inv15), 15.0f, 15.0f);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) byte[j] = n[j];
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    add2(n[j], n[j + 1], -12582912.0f, -12582912.0f);
    d[j] = t[j], d[j + 1] = t[j + 1];
    fma2(d[j], d[j + 1], n[j], n[j + 1], -step, -step);
  }
  fma2(byte[0], byte[1], n[4], n[5], 16.0f, 16.0f);
  fma2(byte[2], byte[3], n[6], n[7], 16.0f, 16.0f);
  uint32_t word = __byte_perm(__byte_perm(__float_as_uint(byte[0]), __float_as_uint(byte[1]), 0x0040),
                              __byte_perm(__float_as_uint(byte[2]), __float_as_uint(byte[3]), 0x0040), 0x5410);
  float far = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) far = fmaxf(far, fabsf(d[j]));
  if (far >= 0.5f * step) {
    word = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) word |= u4_code_of(sign * v[j], bias, step, 15.0f * inv15) << (8 * (j & 3) + (j >> 2) * 4);
  }
  return word;
}
// fp16 bits of step / 2^row_exponent, with the row's sign: exact (8 significant bits, >= 2^-16).
__device__ __forceinline__ uint16_t u4_v_factor_bits(uint16_t step_bits, int row_exponent, uint32_t odd) {
  if (step_bits == 0x7fc0) return 0x7e00;
  const float f = bf16_bits_to_f32(step_bits) * pow2f(-row_exponent);
  return static_cast<uint16_t>(__half_as_ushort(__float2half_rn(f)) | (odd << 15));
}
__device__ __forceinline__ void warp_min_max(float x, float& lo, float& hi) {
  asm("redux.sync.min.NaN.f32 %0, %1, 0xffffffff;" : "=f"(lo) : "f"(x));
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(hi) : "f"(x));
}

// One head row of G groups held by a warp, lane l with element l of every group.
template <int G>
struct U4Row {
  uint32_t code[G];
  uint16_t step[G], bias[G];   // step positive, bias signed (bf16 bits)
  int exponent;
  __device__ __forceinline__ void quantize(const float (&x)[G], uint32_t odd) {
    const float sign = odd ? -1.0f : 1.0f;
    U4Range r[G];
    exponent = U4_EXP_MIN;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float lo, hi;
      warp_min_max(sign * x[g], lo, hi);
      r[g] = u4_range(lo, hi);
      exponent = max(exponent, r[g].exponent);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      step[g] = u4_step_bits(r[g], exponent);
      const float s = bf16_bits_to_f32(step[g]);
      code[g] = r[g].finite ? u4_code_of(sign * x[g], r[g].bias, s, 1.0f / s) : 0u;
      bias[g] = static_cast<uint16_t>(r[g].finite ? (__float_as_uint(sign * r[g].bias) >> 16) : 0u);
    }
  }
};

// Quantises and stores one head row of `hd` values (xs, shared memory) as row `row` of a u4 tile; one
// whole warp. ktile / vtile: the K tile and the V tile behind it.
__device__ __forceinline__ void u4_store_row(uint8_t* ktile, uint8_t* vtile, int hd, int is_v, int row, const float* xs, int lane) {
  uint8_t* tile = is_v ? vtile : ktile;
  const uint32_t odd = row & 1;
  const float sign = odd ? -1.0f : 1.0f;
  const int groups = hd / QGROUP;
  int row_exponent = U4_EXP_MIN;
  for (int g = 0; g < groups; ++g) {
    float lo, hi;
    warp_min_max(sign * xs[g * QGROUP + lane], lo, hi);
    row_exponent = max(row_exponent, u4_range(lo, hi).exponent);
  }
  for (int g = 0; g < groups; ++g) {
    const float y = sign * xs[g * QGROUP + lane];
    float lo, hi;
    warp_min_max(y, lo, hi);
    const U4Range r = u4_range(lo, hi);
    const uint16_t step_bits = u4_step_bits(r, row_exponent);
    const float step = bf16_bits_to_f32(step_bits);
    const uint32_t code = r.finite ? u4_code_of(y, r.bias, step, 1.0f / step) : 0u;
    const uint32_t high = __shfl_down_sync(0xffffffffu, code, 16);
    const int dim = g * QGROUP + lane;
    if (lane < 16) tile[is_v ? u4_v_byte(row, dim, hd) : u4_k_byte(row, dim, hd)] = static_cast<uint8_t>(code | (high << 4));
    if (lane == 0) {
      *reinterpret_cast<uint16_t*>(tile + u4_step_offset(is_v, row, g, hd)) =
          is_v ? u4_v_factor_bits(step_bits, row_exponent, odd) : static_cast<uint16_t>(step_bits ^ (odd << 15));
      *reinterpret_cast<uint16_t*>(tile + u4_bias_offset(row, g, hd)) =
          static_cast<uint16_t>(r.finite ? (__float_as_uint(sign * r.bias) >> 16) : 0u);
    }
  }
  if (is_v && lane == 0)
    *reinterpret_cast<uint16_t*>((row < 8 ? ktile : vtile) + u4_pow_offset(row, hd)) =
        static_cast<uint16_t>(__float_as_uint(pow2f(row_exponent)) >> 16);
}

// A head row spread over ROW_LANES = hd / 8 neighbouring lanes: four lanes per group, lane q = lane % 4 with dims 4q .. 4q+3
// (v[0..3]) and 16 + 4q .. (v[4..7]) of the group, whose codes are four whole bytes. All lanes of the warp call.
struct U4Lane {
  uint32_t word;            // the four bytes
  uint16_t step, bias;      // step positive, bias signed (bf16 bits)
  int exponent;             // of the row
};
__device__ __forceinline__ float min_nan(float a, float b) {   // NaN when either is
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void min_max8(const float (&v)[8], float& lo, float& hi) {   // NaN when one of the eight is
  lo = hi = v[0];
#pragma unroll
  for (int j = 1; j < 8; ++j) lo = min_nan(lo, v[j]), hi = max_nan(hi, v[j]);
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Range, step and row exponent of one group from its least and largest value; step NaN when the group is not finite.
template <int ROW_LANES>
__device__ __forceinline__ U4Range u4_group(float lo, float hi, uint32_t odd, U4Lane& out) {
  const U4Range r = u4_range(odd ? -hi : lo, odd ? -lo : hi);
  out.exponent = r.exponent;
#pragma unroll
  for (int off = 4; off < ROW_LANES; off <<= 1) out.exponent = max(out.exponent, __shfl_xor_sync(0xffffffffu, out.exponent, off));
  out.step = u4_step_bits(r, out.exponent);
  out.bias = static_cast<uint16_t>(r.finite ? (__float_as_uint(odd ? -r.bias : r.bias) >> 16) : 0u);
  return r;
}
template <int ROW_LANES>
__device__ __forceinline__ U4Lane u4_quantize_lanes(const float (&v)[8], uint32_t odd, int lane) {
  float lo, hi;
  min_max8(v, lo, hi);
#pragma unroll
  for (int off = 1; off < 4; off <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, off));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, off));
  }
  U4Lane out;
  const U4Range r = u4_group<ROW_LANES>(lo, hi, odd, out);
  const float s = bf16_bits_to_f32(out.step);
  const uint32_t word = u4_codes8(v, odd ? -1.0f : 1.0f, r.bias, s, rcp_approx(s) * (1.0f / 15.0f));
  out.word = r.finite ? word : 0u;
  return out;
}
// The same for B (two or four) pieces a lane at once, of rows of the same parity: lane q works out the range and the step of
// piece q % B of its group for all four lanes. word[i]: the codes of piece i; the rest belongs to piece q % B.
template <int ROW_LANES, int B>
__device__ __forceinline__ U4Lane u4_quantize_pieces(const float (&v)[B][8], uint32_t odd, int lane, uint32_t (&word)[B]) {
  static_assert(B == 2 || B == 4, "pieces are shared among four lanes");
  float lo[B], hi[B];
#pragma unroll
  for (int i = 0; i < B; ++i) min_max8(v[i], lo[i], hi[i]);
  const bool b0 = lane & 1, b1 = lane & 2;
  // each exchange halves the pieces a lane has partial minima of
#pragma unroll
  for (int i = 0; i < B; i += 2) {
    const float lo_got = __shfl_xor_sync(0xffffffffu, b0 ? lo[i] : lo[i + 1], 1), hi_got = __shfl_xor_sync(0xffffffffu, b0 ? hi[i] : hi[i + 1], 1);
    lo[i / 2] = min_nan(b0 ? lo[i + 1] : lo[i], lo_got);
    hi[i / 2] = max_nan(b0 ? hi[i + 1] : hi[i], hi_got);
  }
  constexpr int LAST = B / 2 - 1;
  const float lo_got = __shfl_xor_sync(0xffffffffu, b1 ? lo[0] : lo[LAST], 2), hi_got = __shfl_xor_sync(0xffffffffu, b1 ? hi[0] : hi[LAST], 2);
  U4Lane out;
  const U4Range r = u4_group<ROW_LANES>(min_nan(b1 ? lo[LAST] : lo[0], lo_got), max_nan(b1 ? hi[LAST] : hi[0], hi_got), odd, out);
  const float s = bf16_bits_to_f32(out.step), inv15 = rcp_approx(s) * (1.0f / 15.0f);
#pragma unroll
  for (int i = 0; i < B; ++i) {
    const int from = (lane & ~3) | i;
    const float bias_i = __shfl_sync(0xffffffffu, r.bias, from), s_i = __shfl_sync(0xffffffffu, s, from),
                inv_i = __shfl_sync(0xffffffffu, inv15, from);
    const uint32_t w = u4_codes8(v[i], odd ? -1.0f : 1.0f, bias_i, s_i, inv_i);
    word[i] = s_i == s_i ? w : 0u;
  }
  out.word = 0;
  return out;
}
// Stores what became of row `row`, group grp: the codes of lane q of four, and the rest, which one lane stores.
__device__ __forceinline__ void u4_store_codes(uint8_t* tile, int hd, int is_v, int row, int grp, int q, uint32_t word) {
  const int dim = grp * QGROUP + 4 * q;
  if (is_v) {
#pragma unroll
    for (int j = 0; j < 4; ++j) tile[u4_v_byte(row, dim + j, hd)] = static_cast<uint8_t>(word >> (8 * j));
  } else {
    *reinterpret_cast<uint32_t*>(tile + u4_k_byte(row, dim, hd)) = word;
  }
}
__device__ __forceinline__ void u4_store_meta(uint8_t* ktile, uint8_t* vtile, int hd, int is_v, int row, int grp, const U4Lane& x) {
  uint8_t* tile = is_v ? vtile : ktile;
  const uint32_t odd = row & 1;
  *reinterpret_cast<uint16_t*>(tile + u4_step_offset(is_v, row, grp, hd)) =
      is_v ? u4_v_factor_bits(x.step, x.exponent, odd) : static_cast<uint16_t>(x.step ^ (odd << 15));
  *reinterpret_cast<uint16_t*>(tile + u4_bias_offset(row, grp, hd)) = x.bias;
  if (is_v && grp == 0)
    *reinterpret_cast<uint16_t*>((row < 8 ? ktile : vtile) + u4_pow_offset(row, hd)) = static_cast<uint16_t>(__float_as_uint(pow2f(x.exponent)) >> 16);
}

}  // namespace sgk
