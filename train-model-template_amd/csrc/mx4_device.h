// Device helpers of the 4-bit operators (gfx950 only): E2M1 and E4M3 block scales and codes, operand layouts, loads and
// stores of the three plain element types.
//
// Numeric contract: with amax the largest magnitude of a 32-element block and max the format's largest value (6 or 448),
//   e    = the least exponent with amax <= max * 2^e, held as e + 127 in 8 bits: 0 at the least, 254 for an infinite amax,
//          255 (NaN) if the block holds a NaN
//   code = v * 2^-e rounded to the nearest value of the format, ties to the even code; infinities take the largest value
// 6 = 1.5 * 2^2, so with amax = (1 + m) 2^E the exponent is E - 2 + [m > 0.5], from the bits alone.
//
// Register layouts of v_mfma_scale_f32_32x32x64_f8f6f4 and _16x16x128_f8f6f4 with R rows an operand (R = 32 or 16) and
// K = 64 or 128 (measured on the device, mixed formats too):
//   E2M1 operand: lane l holds row l % R, codes k = 32 (l / R) + 0..31 in 16 bytes, even k in the low halves;
//   E4M3 operand: lane l, byte j holds row l % R, k = (K / 2)(j / 16) + 16 (l / R) + j % 16;
//   scales: of (row r, 32-block b) from lane r + R b, byte op_sel of the scale register, for both formats.
// E2M1 products are exact.  E4M3 ones (with an E2M1 operand) are added in groups of 16 consecutive k, in which every term
// loses what lies below 2^-13 of the largest one's powers of two: 5e-6 of a result (rms) for normally distributed values, 7e-5
// where a block's magnitudes spread over all of the format's, 7e-4 of the largest term at the worst.
// v_cvt_scalef32_pk_fp4_{f32, f16, bf16} round x / scale to nearest even for every scale 2^-127..2^126 (all 16-bit mantissa
// patterns, ties and denormal scales compared with a software rounding).
#pragma once

#include "mx_device.h"

#include "../../include/mxfp4_ops.h"

namespace mx4 {

using namespace mxk;

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// ---- scales
template <int kFmt>
__device__ __forceinline__ uint32_t block_exponent(uint32_t amax_b) {
  if constexpr (kFmt == MXFP4_E4M3) return e8m0_from_amax_bits(amax_b);
  const int E = (int)(amax_b >> 23);
  const uint32_t m = amax_b & 0x7fffffu;
  int e = E - 2 + (m > 0x400000u ? 1 : 0);
  e = e < 0 ? 0 : e;
  if (E == 255) e = m ? 255 : 254;
  return (uint32_t)e;
}

// 2^(e - 127) as a float; e = 0 gives the denormal 2^-127
__device__ __forceinline__ float block_scale(uint32_t e) { return __uint_as_float(e == 0u ? 1u << 22 : e << 23); }

// Codes of eight values that share the block exponent e: E2M1 in r[0], E4M3 in r[0], r[1].
// Values of finite blocks are within the format's range by the choice of e.  Blocks with an infinity clamp, blocks with a
// NaN take code 0 (E2M1) or NaN (E4M3); one branch a wave.
template <int kFmt>
__device__ __forceinline__ void encode8(const float* v, uint32_t e, uint32_t* r) {
  constexpr float kMax = kFmt == MXFP4_E4M3 ? 448.f : 6.f;
  float w[8];
  float sc = block_scale(e);
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = v[i];
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(e >= 254u) != 0, 0)) {
    if (e >= 254u) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float t = __builtin_fminf(__builtin_fmaxf(__builtin_ldexpf(v[i], 127 - (int)e), -kMax), kMax);
        w[i] = e == 255u ? 0.f : t;
      }
      sc = 1.f;
    }
  }
  if constexpr (kFmt == MXFP4_E4M3) {
    s16x2 a = {0, 0}, b = {0, 0};
    a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, w[0], w[1], sc, false);
    a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, w[2], w[3], sc, true);
    b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, w[4], w[5], sc, false);
    b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, w[6], w[7], sc, true);
    r[0] = e == 255u ? 0x7f7f7f7fu : __builtin_bit_cast(uint32_t, a);
    r[1] = e == 255u ? 0x7f7f7f7fu : __builtin_bit_cast(uint32_t, b);
  } else {
    uint32_t a = 0;
    a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, w[0], w[1], sc, 0);
    a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, w[2], w[3], sc, 1);
    a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, w[4], w[5], sc, 2);
    a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, w[6], w[7], sc, 3);
    r[0] = a;
  }
}

__device__ __forceinline__ uint32_t absmax8(const float* v) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, abs_bits(v[i]));
  return m;
}

// ---- groups of eight values as they are loaded: 16-bit types packed in one uint4, fp32 in two
template <int kT>
struct Group {
  uint4 w;
  __device__ __forceinline__ void values(float* v) const {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kT == MXFP4_BF16) {
        v[2 * i] = bf16_lo(u[i]);
        v[2 * i + 1] = bf16_hi(u[i]);
      } else {
        const f16x2 h = __builtin_bit_cast(f16x2, u[i]);
        v[2 * i] = (float)h[0];
        v[2 * i + 1] = (float)h[1];
      }
    }
  }
  // the largest magnitude, as fp32 bits (16-bit patterns without the sign order like magnitudes, NaN on top)
  __device__ __forceinline__ uint32_t absmax() const {
    u16x2 m = {0, 0};
    m = absmax2(absmax2(absmax2(absmax2(m, w.x), w.y), w.z), w.w);
    const uint32_t b = max(m.x, m.y);
    if constexpr (kT == MXFP4_BF16) return b << 16;
    else return abs_bits((float)__builtin_bit_cast(_Float16, (uint16_t)b));
  }
};
template <>
struct Group<MXFP4_F32> {
  uint4 w, x;
  __device__ __forceinline__ void values(float* v) const {
    const uint32_t u[8] = {w.x, w.y, w.z, w.w, x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(u[i]);
  }
  __device__ __forceinline__ uint32_t absmax() const {
    float v[8];
    values(v);
    return absmax8(v);
  }
};

// Codes of a group with the block exponent e, as encode8; 16-bit values convert packed, as they are
template <int kT, int kFmt>
__device__ __forceinline__ void encode_group(const Group<kT>& g, uint32_t e, uint32_t* r) {
  if constexpr (kT == MXFP4_F32) {
    float v[8];
    g.values(v);
    encode8<kFmt>(v, e, r);
  } else {
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(e >= 254u) != 0, 0)) {
      float v[8];
      g.values(v);
      encode8<kFmt>(v, e, r);
      return;
    }
    const float sc = block_scale(e);
    const uint32_t u[4] = {g.w.x, g.w.y, g.w.z, g.w.w};
    if constexpr (kFmt == MXFP4_E4M3) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        s16x2 c = {0, 0};
        if constexpr (kT == MXFP4_BF16) {
          c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, __builtin_bit_cast(bf16x2, u[2 * i]), sc, false);
          c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, __builtin_bit_cast(bf16x2, u[2 * i + 1]), sc, true);
        } else {
          c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(c, __builtin_bit_cast(f16x2, u[2 * i]), sc, false);
          c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(c, __builtin_bit_cast(f16x2, u[2 * i + 1]), sc, true);
        }
        r[i] = __builtin_bit_cast(uint32_t, c);
      }
    } else {
      uint32_t c = 0;
      if constexpr (kT == MXFP4_BF16) {
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, u[0]), sc, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, u[1]), sc, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, u[2]), sc, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, u[3]), sc, 3);
      } else {
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2, u[0]), sc, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2, u[1]), sc, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2, u[2]), sc, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2, u[3]), sc, 3);
      }
      r[0] = c;
    }
  }
}

// A group at p (aligned to 16 bytes), or element by element with zeros past the row's end
template <int kT, class T>
__device__ __forceinline__ Group<kT> load_group(const T* p) {
  Group<kT> g;
  g.w = *reinterpret_cast<const uint4*>(p);
  if constexpr (kT == MXFP4_F32) g.x = *reinterpret_cast<const uint4*>(p + 4);
  return g;
}
template <int kT, class T>
__device__ __forceinline__ Group<kT> load_group_edge(const T* row, int64_t c, int64_t cols) {
  uint32_t u[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const T t = row[min(c + i, cols - 1)];
    uint32_t b;
    if constexpr (kT == MXFP4_F32) b = __builtin_bit_cast(uint32_t, t);
    else b = __builtin_bit_cast(uint16_t, t);
    u[i] = c + i < cols ? b : 0u;
  }
  Group<kT> g;
  if constexpr (kT == MXFP4_F32) {
    g.w = make_uint4(u[0], u[1], u[2], u[3]);
    g.x = make_uint4(u[4], u[5], u[6], u[7]);
  } else {
    g.w = make_uint4(u[0] | u[1] << 16, u[2] | u[3] << 16, u[4] | u[5] << 16, u[6] | u[7] << 16);
  }
  return g;
}

// ---- layouts
// Byte of code (r, c) in an operand with ct column tiles (128 wide): E2M1 (the code's byte; odd c is its high half) or E4M3
template <int kFmt>
__device__ __forceinline__ int64_t code_offset(int64_t r, int64_t c, int64_t ct) {
  if constexpr (kFmt == MXFP4_E4M3) return tiled_offset(r, c, ct * 128);
  return ((r >> 4) * ct + (c >> 7)) * 1024 + ((c >> 6) & 1) * 512 + (r & 15) * 32 +
         ((((c >> 5) & 1) ^ ((r >> 3) & 1)) << 4) + ((c & 31) >> 1);
}

// Position of row r in a row order
__device__ __forceinline__ int64_t order_row(int64_t r, int order) {
  if (order == MXFP4_ROWS_PLAIN) return r;
  const int c = (int)(r & 31), a = ((c >> 2) & 3) * 8 + (c >> 4) * 4 + (c & 3);
  const int64_t blk = r >> 5;
  return (order == MXFP4_ROWS_PI ? blk * 32 : blk * 64 + (order == MXFP4_ROWS_UP ? 32 : 0)) + a;
}

// ---- plain element types
template <int kT>
struct Elem;
template <>
struct Elem<MXFP4_BF16> {
  typedef uint16_t T;
  static __device__ __forceinline__ float get(T v) { return bf16_bits_to_f32(v); }
  static __device__ __forceinline__ T put(float f) { return (T)f32_to_bf16_bits(f); }
};
template <>
struct Elem<MXFP4_F16> {
  typedef _Float16 T;
  static __device__ __forceinline__ float get(T v) { return (float)v; }
  static __device__ __forceinline__ T put(float f) { return (T)f; }
};
template <>
struct Elem<MXFP4_F32> {
  typedef float T;
  static __device__ __forceinline__ float get(T v) { return v; }
  static __device__ __forceinline__ T put(float f) { return f; }
};

// 8 values at p, aligned to 16 bytes
template <int kT>
__device__ __forceinline__ void load8(const typename Elem<kT>::T* p, float* v) {
  if constexpr (kT == MXFP4_F32) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = a[i];
      v[4 + i] = b[i];
    }
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kT == MXFP4_BF16) {
        v[2 * i] = bf16_lo(w[i]);
        v[2 * i + 1] = bf16_hi(w[i]);
      } else {
        const f16x2 h = __builtin_bit_cast(f16x2, w[i]);
        v[2 * i] = (float)h[0];
        v[2 * i + 1] = (float)h[1];
      }
    }
  }
}

// a, b rounded to a 16-bit type, packed; the rounded values stay in a, b
template <int kT>
__device__ __forceinline__ uint32_t round2(float& a, float& b) {
  if constexpr (kT == MXFP4_BF16) {
    return rnd2(a, b);
  } else {
    const f16x2 h = {(_Float16)a, (_Float16)b};
    a = (float)h[0];
    b = (float)h[1];
    return __builtin_bit_cast(uint32_t, h);
  }
}

// n consecutive values (a multiple of 4, at most 16) of row p to columns c.. of a row with `cols` columns; vec: p + c is
// aligned to 16 bytes (f32, or 16-bit values 8 at a time) or to 8 (4 at a time)
template <int kT, int n>
__device__ __forceinline__ void store_run(typename Elem<kT>::T* p, int64_t c, int64_t cols, bool vec, const float* v) {
  if (vec && c + n <= cols) {
    if constexpr (kT == MXFP4_F32) {
#pragma unroll
      for (int i = 0; i < n; i += 4) {
        const f32x4 t = {v[i], v[i + 1], v[i + 2], v[i + 3]};
        *reinterpret_cast<f32x4*>(p + c + i) = t;
      }
    } else {
      uint32_t w[n / 2];
#pragma unroll
      for (int i = 0; i < n / 2; ++i) {
        float a = v[2 * i], b = v[2 * i + 1];
        w[i] = round2<kT>(a, b);
      }
      if constexpr (n % 8 == 0) {
#pragma unroll
        for (int i = 0; i < n / 2; i += 4)
          *reinterpret_cast<uint4*>(p + c + 2 * i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
      } else {
#pragma unroll
        for (int i = 0; i < n / 2; i += 2) *reinterpret_cast<uint2*>(p + c + 2 * i) = make_uint2(w[i], w[i + 1]);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < n; ++i)
    if (c + i < cols) p[c + i] = Elem<kT>::put(v[i]);
}

// Columns c0 .. c0 + 31 of rows r0 .. r0 + 31 from a wave whose lane l holds, of row l % 32, the 16 columns at (l / 32) 16.  In 16
// bits the lanes l and l ^ 16 swap halves first, so that an instruction writes 16 rows of 64 bytes and not 32 of 16 in each of
// two places.  r0, c0 are the same in all lanes, all of which call it.
template <int kT>
__device__ __forceinline__ void store_block(typename Elem<kT>::T* p, int64_t ld, int64_t r0, int64_t rows, int64_t c0,
                                            int64_t cols, bool vec, int lane, const float* v) {
  if constexpr (kT != MXFP4_F32) {
    if (vec && c0 + 32 <= cols) {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float a = v[2 * i], b = v[2 * i + 1];
        w[i] = round2<kT>(a, b);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // now w[0..3] row l % 16, w[4..7] row 16 + l % 16, columns 8 (l / 16 % 2) of the 16
        const auto r = __builtin_amdgcn_permlane16_swap(w[i], w[4 + i], false, false);
        w[i] = r[0];
        w[4 + i] = r[1];
      }
      const int64_t c = c0 + (lane >> 5) * 16 + ((lane >> 4) & 1) * 8, r = r0 + (lane & 15);
      if (r < rows) *reinterpret_cast<uint4*>(p + r * ld + c) = make_uint4(w[0], w[1], w[2], w[3]);
      if (r + 16 < rows) *reinterpret_cast<uint4*>(p + (r + 16) * ld + c) = make_uint4(w[4], w[5], w[6], w[7]);
      return;
    }
  }
  const int64_t r = r0 + (lane & 31);
  if (r < rows) store_run<kT, 16>(p + r * ld, c0 + (lane >> 5) * 16, cols, vec, v);
}

// ---- gate functions: f = fn(g); and its derivative
// silu(g) = g s, s = 1 / (1 + exp(-g)); silu' = s (1 + g (1 - s)).
// gelu(g) = g s(2 c (g + a g^3)) with c = sqrt(2 / pi), a = 0.044715 (0.5 (1 + tanh t) = sigmoid(2 t)), so
// gelu' = s + g s (1 - s) 2 c (1 + 3 a g^2).  Both with the hardware exp2 and reciprocal, 1 ulp each.
// 1 - s is off by 2^-24 where s is near 1, which g (1 - s) + 1 takes as g 2^-24.
// gelu' takes its polynomial at g held to +-16, past which s is 0 or 1 in 32 bits (t is +-317 there) and gelu' with it: the
// powers of a larger g would pass 32 bits and give inf * 0.
template <int kFn>
__device__ __forceinline__ float gate_fn(float g) {
  if constexpr (kFn == MXFP4_SILU) {
    return g * fast_sigmoid(g);
  } else {
    const float t = 1.5957691216057308f * g * __builtin_fmaf(0.044715f * g, g, 1.f);
    return g * fast_sigmoid(t);
  }
}
template <int kFn>
__device__ __forceinline__ float gate_fn(float g, float& df) {
  if constexpr (kFn == MXFP4_SILU) {
    const float s = fast_sigmoid(g);
    df = s * __builtin_fmaf(g, 1.f - s, 1.f);
    return g * s;
  } else {
    const float k = __builtin_amdgcn_fmed3f(g, -16.f, 16.f), q = 0.044715f * k * k;
    const float t = 1.5957691216057308f * g * (1.f + q);  // of g itself: NaN stays
    const float s = fast_sigmoid(t);
    df = s * __builtin_fmaf(k * 1.5957691216057308f * __builtin_fmaf(3.f, q, 1.f), 1.f - s, 1.f);
    return g * s;
  }
}

// Offset of the saved gate of (row r, column c) of the forward pass: 32 x 32 blocks, gate then up (1024 elements each),
// each in the order of the GEMM's epilogue (ft_offset in mx_device.h); the up value lies 1024 elements on.
__device__ __forceinline__ int64_t saved_offset(int64_t r, int64_t c, int64_t nb) {
  return ((r >> 5) * nb + (c >> 5)) * 2048 + ((c >> 3) & 1) * 512 + ((r & 31) + 32 * ((c >> 4) & 1)) * 8 + (c & 7);
}

}  // namespace mx4
