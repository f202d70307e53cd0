// The two 16-bit element types of the grouped and paged attention kernels: MFMA
// and conversions, fragments held as four 32-bit words of either type.
#pragma once

#include "common.cuh"

namespace mea {

struct Bf16 {
  static __device__ __forceinline__ f32x16 mma(const u32x4& a, const u32x4& b, const f32x16& c) {
    return mfma32(as_frag(a), as_frag(b), c);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack2(lo, hi); }
  static __device__ __forceinline__ float lo(uint32_t w) { return lo_bf(w); }
  static __device__ __forceinline__ float hi(uint32_t w) { return hi_bf(w); }
  static constexpr uint32_t kInf = 0x7F80u;
  // Adds this lane's weights to l: as rounded for the product with V (p), so that
  // the quotient is a mean of v rows with weights that sum to 1 and the roundings
  // cancel where one key dominates (o's error at normal q, k, v: 2.4e-3 -> 2.1e-3
  // of its norm, at logits of standard deviation 4: 2.6e-3 -> 1.9e-3; rounding the
  // exact o: 1.6e-3). Eight v_dot2_f32_bf16 with ones.
  static __device__ __forceinline__ float add_weights(float l, const f32x16&, const u32x4 (&p)[2]) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 ones = __builtin_bit_cast(bf16x2, 0x3F803F80u);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t pair = p[i >> 2][i & 3];  // (a value: a cast of the element itself takes element 0)
      l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), ones, l, false);
    }
    return l;
  }
  // A weight may grow to this before the running maximum is raised: bf16 has the
  // exponents of fp32, so only the fp32 sums bound it.
  static constexpr float kMaxWeight = 0x1p40f;
};

struct Fp16 {
  typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x16 mma(const u32x4& a, const u32x4& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  // Round to nearest even.
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
  }
  static __device__ __forceinline__ float lo(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[0]; }
  static __device__ __forceinline__ float hi(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[1]; }
  static constexpr uint32_t kInf = 0x7C00u;
  // The weights before their rounding: it is an eighth of bf16's, and small fp16
  // weights lose more of themselves in it.
  static __device__ __forceinline__ float add_weights(float l, const f32x16& w, const u32x4 (&)[2]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) l += w[i];
    return l;
  }
  static constexpr float kMaxWeight = 0x1p14f;  // the largest fp16 number is 65504
};

// Whether a word holds an infinity or a NaN: bit 15 of each half of the result.
template <class E>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  constexpr uint32_t add = (0x8000u - E::kInf) * 0x10001u;
  return ((w & 0x7FFF7FFFu) + add) & 0x80008000u;
}
// 0xFFFF in each half whose bit 15 is set.
__device__ __forceinline__ uint32_t spread(uint32_t bits) { return (bits >> 15) * 0xFFFFu; }

// Largest magnitude seen so far, per half (infinities and NaN are the largest).
__device__ __forceinline__ uint32_t max_magnitude(uint32_t top, const u32x4& v) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int e = 0; e < 4; ++e)
    top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, top),
                                                                 __builtin_bit_cast(u16x2, v[e] & 0x7FFF7FFFu)));
  return top;
}
// The fragment with 0 in the place of every infinity and NaN.
template <class E>
__device__ __forceinline__ u32x4 finite_only(const u32x4& v) {
  u32x4 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = v[e] & ~spread(not_finite<E>(v[e]));
  return r;
}
// One 32-row block of O^T (rows 8 r4 + 4 h + e): adds the infinities and NaN of
// one key's V row where this lane's query sees the key. row: V row + 4 h. Their
// positive weights do not change them.
template <class E>
__device__ __forceinline__ void add_not_finite(f32x16& o, const bf16_bits* row, bool sees) {
#pragma unroll
  for (int r4 = 0; r4 < 4; ++r4) {
    const u32x2 w = *reinterpret_cast<const u32x2*>(row + 8 * r4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t pair = w[e >> 1];
      const float x = e & 1 ? E::hi(pair) : E::lo(pair);
      if (sees && !__builtin_isfinite(x)) o[4 * r4 + e] += x;
    }
  }
}

// Inclusive sum over the wave's lanes, every lane taking part: within rows of sixteen
// lanes by DPP row shifts, then the last lane of a row, and of half a wave, to those behind.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
  return v;
}

}  // namespace mea
