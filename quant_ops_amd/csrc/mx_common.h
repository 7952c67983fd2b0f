// Microscaled (OCP MX) formats on gfx950: 32 consecutive values of a row share
// the scale 2^e, held as the byte e + 127 (255: NaN), and are coded as FP4
// e2m1 (two per byte, the even value in the low bits) or FP8 e4m3. A row of F
// values has B = ceil(F / 32) blocks; the last is padded with zeros, so a row
// of codes has 16 B (FP4) or 32 B (FP8) bytes.
//
// e = floor(log2(largest magnitude of the block)) - emax, clamped to -127 ..;
// emax is 2 (e2m1, largest value 6) or 8 (e4m3, 448). Codes are v / 2^e rounded
// to nearest even and saturated. A block that holds a NaN or an infinity gets
// the byte 255 and zero codes: it reads back as NaN.
#pragma once

#include "common.h"

namespace qo {

typedef float v2f __attribute__((ext_vector_type(2)));
typedef short v2s __attribute__((ext_vector_type(2)));

struct FP4 {
  static constexpr int code = QO_MX_FP4, emax = 2, words = 1;   // words: dwords of 8 codes
};
struct FP8 {
  static constexpr int code = QO_MX_FP8, emax = 8, words = 2;
};

// Maximum over the four lanes of a quad (they hold one block, eight values each).
__device__ inline uint32_t quad_max_u32(uint32_t u) {
  u = max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0xB1, 0xF, 0xF, false));   // quad_perm 1,0,3,2
  return max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0x4E, 0xF, 0xF, false));   // quad_perm 2,3,0,1
}

// Scale byte of a block from the bits of its largest magnitude: with the sign
// cleared, bit patterns order like the values, and infinities and NaN (field
// 255) are above all others. Subnormal maxima (field 0) give the lowest byte.
template <class Q>
__device__ inline uint32_t mx_scale_byte(uint32_t top) {
  const int field = (int)(top >> 23);
  return field == 255 ? 255u : (uint32_t)max(field - Q::emax, 0);
}

// Eight values of a block -> one (FP4) or two (FP8) words of codes. The
// conversion takes 2^e from the exponent field of its scale operand, whose
// field is the scale byte. FP8 overflows to NaN, so its values are clamped
// first: 448 2^e (2^e at least 2^-127: exact).
template <class Q>
__device__ inline void mx_codes8(const float (&v)[8], uint32_t byte, uint32_t (&w)[Q::words]) {
  const float scale = __builtin_bit_cast(float, byte << 23);
  if constexpr (Q::code == QO_MX_FP4) {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], scale, 3);
    w[0] = byte == 255u ? 0u : c;
  } else {
    const float most = ldexpf(448.f, (int)byte - 127);
    float u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = __builtin_amdgcn_fmed3f(v[i], -most, most);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      v2s c = {0, 0};
      c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, u[4 * h], u[4 * h + 1], scale, false);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, u[4 * h + 2], u[4 * h + 3], scale, true);
      w[h] = byte == 255u ? 0u : __builtin_bit_cast(uint32_t, c);
    }
  }
}

// The values of the codes in a word: eight (FP4) or four (FP8).
template <class Q>
__device__ inline void mx_word_values(uint32_t w, uint32_t byte, float (&v)[8 / Q::words]) {
  const float scale = __builtin_bit_cast(float, byte << 23);   // field 255 reads as NaN
  v2f p[4 / Q::words];
  if constexpr (Q::code == QO_MX_FP4) {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3);
  } else {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, false);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, true);
  }
#pragma unroll
  for (int i = 0; i < 8 / Q::words; ++i) v[i] = p[i / 2][i % 2];
}

// Elements 8 c .. of a row of n (the rest 0). Whole pieces are one 16-byte load (two
// for float32) at any alignment, which global loads allow. WHOLE: n is a
// multiple of 8, so a piece is there or not; the load then has no branch (a
// piece past the end reads the row's first and drops it), and loads of several
// pieces are under way together.
template <class D>
struct Raw8 {
  typename D::T t[8];
};
template <class D, bool WHOLE>
__device__ inline Raw8<D> load8(const typename D::T* row, int c, int64_t n) {
  Raw8<D> r;
  if constexpr (WHOLE) {
    __builtin_memcpy(r.t, row + (8 * c < n ? 8 * c : 0), sizeof(r.t));
  } else {
    const typename D::T* p = row + 8 * c;
    if (8 * c + 8 <= n) {
      __builtin_memcpy(r.t, p, sizeof(r.t));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) r.t[i] = 8 * c + i < n ? p[i] : (typename D::T)0.f;
    }
  }
  return r;
}
template <class D, bool WHOLE>
__device__ inline void values8(const Raw8<D>& r, int c, int64_t n, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = !WHOLE || 8 * c < n ? D::to_f(r.t[i]) : 0.f;
}

// N values to the N elements at p, the first n of them; NT: as non-temporal 16-byte stores where p allows.
template <class D, int N, bool NT = false>
__device__ inline void store_row(typename D::T* p, int64_t n, const float (&v)[N]) {
  typename D::T t[N];
#pragma unroll
  for (int i = 0; i < N; ++i) t[i] = D::from_f(v[i]);
  if (n >= N) {
    if constexpr (NT) {
      static_assert(sizeof(t) % 16 == 0, "whole pieces");
#pragma unroll
      for (int h = 0; h < (int)sizeof(t) / 16; ++h) {
        v4i w;
        __builtin_memcpy(&w, reinterpret_cast<const char*>(t) + 16 * h, 16);
        __builtin_nontemporal_store(w, reinterpret_cast<v4i*>(p) + h);
      }
    } else {
      __builtin_memcpy(p, t, sizeof(t));
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) p[i] = t[i];
  }
}

// Codes and scale of the block whose eight values v this lane holds beside the
// other three lanes of its quad (chunk c of a row, c / 4 the block).
template <class Q>
__device__ inline void mx_store8(const float (&v)[8], uint8_t* codes, uint8_t* scales, int64_t scales_ld,
                                 int64_t row, int blocks, int c) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __builtin_bit_cast(uint32_t, v[i]) & 0x7FFFFFFFu);
  const uint32_t byte = mx_scale_byte<Q>(quad_max_u32(top));
  uint32_t w[Q::words];
  mx_codes8<Q>(v, byte, w);
  uint32_t* out = reinterpret_cast<uint32_t*>(codes + (row * blocks * 4 + c) * (4 * Q::words));
#pragma unroll
  for (int i = 0; i < Q::words; ++i) out[i] = w[i];
  if ((c & 3) == 0) scales[row * scales_ld + (c >> 2)] = (uint8_t)byte;
}

}  // namespace qo
