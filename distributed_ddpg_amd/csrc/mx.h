// MXFP4 (OCP microscaling, E2M1 elements, E8M0 scales): the layout of a
// quantised matrix and the device helpers of its kernels (mx.hip).
//
// A row's 32 consecutive values share the scale 2^(s - 127); an element's code
// is sign | index into {0 .5 1 1.5 2 3 4 6}.  s = 255 makes the block NaN.
//
// Layout: what v_mfma_scale_f32_16x16x128_f8f6f4 takes as an operand, lane by
// lane.  Lane l of a wave holds row l % 16 and the 32-block l / 16 of 128
// columns: 16 bytes of codes (element 0 in the low nibble of byte 0) and one
// scale byte.
//   codes  [rows / 16][cols / 128][64 lanes][16 bytes]
//   scales [rows / 64][cols / 128][64 lanes][4 bytes]: byte g is the scale of
//          the lane's block in the g-th 16 rows of the 64 (the instruction
//          picks the byte, so one dword serves four products)
// Rows are padded to 64, columns to 128.  Padding columns hold the code 0 under
// a finite scale and add nothing to a product; padding rows are never read
// into a result and hold anything.
#pragma once
#include "tensor_ops.h"

namespace ddpg {

struct MxMat {
  const uint8_t *codes, *scales;
  int rows, cols;
  __host__ __device__ int kt() const { return (cols + 127) >> 7; }
};

inline size_t mx_code_bytes(long long rows, long long cols) {
  return (size_t)((rows + 63) / 64) * (size_t)((cols + 127) / 128) * 4096;
}
inline size_t mx_scale_bytes(long long rows, long long cols) {
  return (size_t)((rows + 63) / 64) * (size_t)((cols + 127) / 128) * 256;
}

// Byte offsets of (16-row group, column tile) codes and (64-row group, column
// tile) scales.
DDPG_DEV size_t mx_code_at(int g16, int kt, int k) { return ((size_t)g16 * kt + k) * 1024; }
DDPG_DEV size_t mx_scale_at(int g64, int kt, int k) { return ((size_t)g64 * kt + k) * 256; }

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// The bits of the largest magnitude of n values: bits order like magnitudes, an
// infinity and a NaN beyond the rest.
template <int N>
DDPG_DEV unsigned mx_top(const float* x) {
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  return top;
}
// A block's scale byte: E = floor(log2 max) - 2 is the exponent field of the
// largest magnitude less 2 (255 stays: not finite), at least 0: below 2^-125 the
// scale stays 2^-127.
DDPG_DEV unsigned mx_scale_of(unsigned top) {
  const int ef = (int)(top >> 23);
  return ef == 255 ? 255u : (unsigned)max(ef - 2, 0);
}
// 2^(s - 127) (2^-127 is subnormal; 255 gives an infinity)
DDPG_DEV float mx_factor(unsigned s) { return __uint_as_float(s ? s << 23 : 0x00400000u); }

// Eight values to codes.  x / 2^E is exact, so v_cvt_scalef32_pk_fp4_f32 makes the
// one rounding: nearest, ties to the even code, at most 6.
DDPG_DEV unsigned mx_codes8(const float* x, float factor) {
  unsigned v = 0;
  v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, x[0], x[1], factor, 0);
  v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, x[2], x[3], factor, 1);
  v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, x[4], x[5], factor, 2);
  v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, x[6], x[7], factor, 3);
  return v;
}

// One block: 32 values to codes and the scale byte.
DDPG_DEV u32x4 mx_quantize_block(const float (&x)[32], unsigned& scale) {
  scale = mx_scale_of(mx_top<32>(x));
  const float f = mx_factor(scale);
  return u32x4{mx_codes8(x, f), mx_codes8(x + 8, f), mx_codes8(x + 16, f), mx_codes8(x + 24, f)};
}

// The factor of a scale byte as the conversions below take it.
DDPG_DEV float mx_scale(unsigned s) {
  return s == 255 ? __uint_as_float(0x7fc00000u) : mx_factor(s);
}

// Eight codes to the values they stand for (exact; a NaN scale gives NaN).
DDPG_DEV void mx_values(unsigned q, unsigned s, float* x) {
  const float f = mx_scale(s);
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, f, 0);
  const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, f, 1);
  const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, f, 2);
  const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, f, 3);
  x[0] = a[0], x[1] = a[1], x[2] = b[0], x[3] = b[1];
  x[4] = c[0], x[5] = c[1], x[6] = d[0], x[7] = d[1];
  if (s == 255)
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = f;
}

// acc += A B^T of 16 x 128 by 16 x 128 codes; sa's byte OA and sb's byte OB
// are the scales.
template <int OA, int OB>
DDPG_DEV f32x4 mx_mfma(const u32x4& a, const u32x4& b, f32x4 acc, unsigned sa, unsigned sb) {
  const i32x8 A = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8 B = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, acc, 4, 4, OA, (int)sa, OB,
                                                          (int)sb);
}

}  // namespace ddpg
