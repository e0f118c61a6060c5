// The 8-bit paged key/value cache: its layout, its two formats, and the tables that say where an entry's tokens are.
//
// A block is a page's 16 tokens of one kv head.  Keys [D / 64][16 tokens][64], values [D / 64][4 quads of tokens][64][4 tokens of the quad], one byte a
// value, so that the 16 bytes that lane (n = lane & 15, q = lane >> 4) loads at chunk * 1024 + (keys: n * 64 + q * 16, values: q * 256 + n * 16) are
//   keys    token n, values 64 chunk + 16 q ..+15   two A operands of v_mfma_f32_16x16x32 (token n, reduction index 8 q + i), the query's rows as B
//   values  tokens 4 q .. 4 q + 3 of the values 64 chunk + 4 n ..+3: what the second product wants beside the weights that the first one left in the lane
// and the 64 lanes read one contiguous KiB.  No shuffle, no transposition and no shared memory between memory and the matrix cores.
//
// A block's scale is a power of two: code * scale is then exact in bf16, a rescaled e4m3 code is exact but where it becomes subnormal, and an int8 code that is
// rescaled again and again, one power at a time, is off by half a final step times 1 + 1/2 + 1/4 ...: less than one step.
#pragma once

#include <type_traits>

#include "typed.h"

namespace pk {

constexpr int kKv8Page = 16;
constexpr int kE4m3 = 0, kInt8 = 1;
constexpr int kKv8LeastExp = -100;   // of a block without a finite value but 0; 2^100 times any value it holds is then below fp32's largest

struct Kv8 {
  uint8_t* codes;
  float* scales;
  int64_t code_stride, scale_stride;   // of a page: bytes, values
  const int32_t *indptr, *ids;
  int32_t n_ids, n_pages, kv_heads, entries;

  // page of an entry's block, -1 where it has none: no table, whatever it holds, makes an address outside the cache
  __device__ __forceinline__ int page(int e, int block) const {
    const int first = indptr[e], n = indptr[e + 1] - first, at = first + block;
    if (block < 0 || block >= n || (unsigned)at >= (unsigned)n_ids) return -1;
    const int id = ids[at];
    return (unsigned)id < (unsigned)n_pages ? id : -1;
  }
  // blocks that an entry's table has: no length, whatever its table holds, makes a walk longer than this
  __device__ __forceinline__ int blocks(int e) const { return max(0, min(indptr[e + 1] - indptr[e], n_ids)); }
  // tokens of an entry said to have n
  __device__ __forceinline__ int tokens(int e, int n) const { return (int)max((int64_t)0, min((int64_t)n, (int64_t)blocks(e) * kKv8Page)); }
  __device__ __forceinline__ uint8_t* block(int page, int side, int head, int dim) const {
    return codes + page * code_stride + (int64_t)(side * kv_heads + head) * (kKv8Page * dim);
  }
  __device__ __forceinline__ float* scale(int page, int side, int head) const { return scales + page * scale_stride + side * kv_heads + head; }
};

// rows row0[e] .. row0[e + 1] - 1 within [0, n_rows)
struct RowSpan { int first, n; };
__device__ __forceinline__ RowSpan row_span(const int32_t* row0, int e, int n_rows) {
  const int a = max(row0[e], 0), b = min(row0[e + 1], n_rows);
  return {a, max(b - a, 0)};
}

template <int FMT> constexpr float kv8_top() { return FMT == kE4m3 ? 448.f : 127.f; }
// the largest code * 2^e within fp32, 240 * 2^120 or 127 * 2^121: a value that would be rounded past it, to 2^128, is taken for it
template <int FMT> constexpr float kv8_largest() { return FMT == kE4m3 ? 0x1.ep127f : 0x1.fcp127f; }

// least e with amax <= top 2^e: 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6
template <int FMT>
__device__ __forceinline__ int kv8_exp(float amax) {
  if (!(amax > 0.f)) return kKv8LeastExp;
  int x;
  const float m = frexpf(amax, &x);   // amax = m 2^x, 1/2 <= m < 1
  const int e = FMT == kE4m3 ? x - 9 + (m > 0.875f) : x - 7 + (m > 127.f / 128.f);
  return max(e, kKv8LeastExp);
}

__device__ __forceinline__ float pow2f(int e) { return ldexpf(1.f, e); }

// the exponent that a scale stands for
__device__ __forceinline__ int exp_of(float scale) { return (int)((__builtin_bit_cast(uint32_t, scale) >> 23) & 255) - 127; }

// four codes as numbers
template <int FMT>
__device__ __forceinline__ void kv8_numbers(uint32_t w, float* o) {
  if constexpr (FMT == kE4m3) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    o[0] = a.x; o[1] = a.y; o[2] = b.x; o[3] = b.y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = (float)(int8_t)(w >> (8 * i));
  }
}
// four numbers, already divided by the scale, to the nearest codes (ties to even; beyond the top: the top; NaN: 0)
template <int FMT>
__device__ __forceinline__ uint32_t kv8_codes(const float* x, float top = kv8_top<FMT>()) {
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = x[i] == x[i] ? fminf(fmaxf(x[i], -top), top) : 0.f;
  if constexpr (FMT == kE4m3) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
  } else {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= ((uint32_t)(int)rintf(y[i]) & 255u) << (8 * i);
    return w;
  }
}
// eight codes as a bf16 operand (every code is a bf16 number): e4m3 times a scale for each four, which the conversion multiplies by on its way; int8 as they are
template <int FMT>
__device__ __forceinline__ bf16x8_t kv8_operand2(uint32_t lo, uint32_t hi, float scale_lo, float scale_hi) {
  typedef __attribute__((ext_vector_type(4))) uint32_t w4;
  w4 o;
  if constexpr (FMT == kE4m3) {
    o.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale_lo, false));
    o.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale_lo, true));
    o.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale_hi, false));
    o.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale_hi, true));
  } else {
    // a byte to a float in one instruction each; the compiler's own choice takes the byte out first
    auto at = [](uint32_t w, auto i) {
      float f;
      if constexpr (i() == 0) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0" : "=v"(f) : "v"(w));
      else if constexpr (i() == 1) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(f) : "v"(w));
      else if constexpr (i() == 2) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(f) : "v"(w));
      else asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(f) : "v"(w));
      return f;
    };
    constexpr std::integral_constant<int, 0> i0{};
    constexpr std::integral_constant<int, 1> i1{};
    constexpr std::integral_constant<int, 2> i2{};
    constexpr std::integral_constant<int, 3> i3{};
    const float a[4] = {at(lo, i0), at(lo, i1), at(lo, i2), at(lo, i3)}, b[4] = {at(hi, i0), at(hi, i1), at(hi, i2), at(hi, i3)};
    auto top = [](float l, float h) { return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, h), __builtin_bit_cast(uint32_t, l), 0x07060302u); };
    o.x = top(a[0], a[1]); o.y = top(a[2], a[3]); o.z = top(b[0], b[1]); o.w = top(b[2], b[3]);
  }
  return __builtin_bit_cast(bf16x8_t, o);
}

template <int FMT>
__device__ __forceinline__ bf16x8_t kv8_operand(uint32_t lo, uint32_t hi, float scale = 1.f) { return kv8_operand2<FMT>(lo, hi, scale, scale); }

// A query or a weight as a sum of bf16 operands: itself where it is bf16 (a weight: rounded to it), in three parts where it is fp32 (24 bits: nothing lost)
template <typename T> constexpr int kv8_parts() { return sizeof(T) == 2 ? 1 : 3; }
template <int NP>
__device__ __forceinline__ void kv8_split(const float* x, bf16x8_t* p) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = pack_bf2(r[2 * i], r[2 * i + 1]);
      r[2 * i] -= bf_lo(w[i]);
      r[2 * i + 1] -= bf_hi(w[i]);
    }
    p[k] = __builtin_bit_cast(bf16x8_t, w);
  }
}
__device__ __forceinline__ void kv8_query(const uint16_t* q, bf16x8_t* p) { p[0] = *reinterpret_cast<const bf16x8_t*>(q); }
__device__ __forceinline__ void kv8_query(const float* q, bf16x8_t* p) {
  float x[8];
  Vec8<float>::load(q, x);
  kv8_split<3>(x, p);
}

}  // namespace pk
