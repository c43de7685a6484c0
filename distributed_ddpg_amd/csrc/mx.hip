// MXFP4 operators: quantisation and its inverse, the product of two quantised
// matrices (a layer's forward), and that product's gradient.  The format and
// its layout: mx.h.
#include "mx.h"

namespace ddpg {

// ---------------------------------------------------------------- quantise
// A wave makes 64 rows x 128 columns: lane l takes row l % 16 and 32-block
// l / 16 of each 16-row group in turn and keeps the four scale bytes of its
// dword.  Its 32 values are 16-byte loads when the columns are adjacent.
template <int DT>
__global__ __launch_bounds__(256) void mx_quantize_kernel(
    const typename Elem<DT>::type* __restrict__ x, int rows, int cols, long long sr, long long sc,
    uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const int kt = (cols + 127) >> 7, l = threadIdx.x & 63;
  const long long tile = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int g64 = (int)(tile / kt), k = (int)(tile % kt);
  if (g64 * 64 >= rows) return;
  const int c0 = k * 128 + (l >> 4) * 32;
  unsigned packed = 0;
  for (int g = 0; g < 4; ++g) {
    const int r = g64 * 64 + g * 16 + (l & 15);
    if (g64 * 64 + g * 16 >= rows) break;
    float v[32];
    if (r < rows && c0 + 32 <= cols && sc == 1) {
      constexpr int V = Elem<DT>::V;
      const typename Elem<DT>::type* p = x + r * sr + c0;
#pragma unroll
      for (int i = 0; i < 32; i += V)
        Elem<DT>::widen(*reinterpret_cast<const U16B*>(p + i), v + i);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        v[i] = r < rows && c0 + i < cols ? (float)x[r * sr + (c0 + i) * sc] : 0.f;
    }
    unsigned s;
    const u32x4 q = mx_quantize_block(v, s);
    packed |= s << (8 * g);
    *reinterpret_cast<u32x4*>(codes + mx_code_at(g64 * 4 + g, kt, k) + l * 16) = q;
  }
  *reinterpret_cast<unsigned*>(scales + mx_scale_at(g64, kt, k) + l * 4) = packed;
}

template <int DT>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(MxMat q,
                                                            typename Elem<DT>::type* out,
                                                            long long ldo) {
  const int kt = q.kt(), l = threadIdx.x & 63;
  const long long tile = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int g16 = (int)(tile / kt), k = (int)(tile % kt);
  const int r = g16 * 16 + (l & 15), c0 = k * 128 + (l >> 4) * 32;
  if (r >= q.rows || c0 >= q.cols) return;
  const u32x4 w = *reinterpret_cast<const u32x4*>(q.codes + mx_code_at(g16, kt, k) + l * 16);
  const unsigned s = q.scales[mx_scale_at(g16 >> 2, kt, k) + l * 4 + (g16 & 3)];
  typename Elem<DT>::type* p = out + r * ldo + c0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v[8];
    mx_values(w[i], s, v);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c0 + 8 * i + j < q.cols) p[8 * i + j] = (typename Elem<DT>::type)v[j];
  }
}

// ---------------------------------------------------------------- product
// y[m][n] = act(sum_k x[m][k] w[n][k] + b[n]).  W is the instruction's A
// operand and X its B: a lane then holds four consecutive n of one m.
struct MxOut {
  void* y;
  const void* bias;
  long long ldo;
  int M, N, dtype, bias_dtype, act;
};

DDPG_DEV float mx_act(float v, int act) {
  if (act == DDPG_ACT_ELU) return elu_f(v);
  if (act == DDPG_ACT_TANH) return tanhf(v);
  return v;
}

DDPG_DEV void mx_store(const MxOut& o, int m, int n, const f32x4& d) {
  if (m >= o.M) return;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (n + r >= o.N) return;
    const float b = o.bias ? load_elem(o.bias, o.bias_dtype, n + r) : 0.f;
    store_elem(o.y, o.dtype, m * o.ldo + n + r, mx_act(__fadd_rn(d[r], b), o.act));
  }
}

// One wave: 64 n x 64 m, operands straight from memory.
__global__ __launch_bounds__(64) void mx_linear_kernel(MxMat x, MxMat w, MxOut o) {
  const int kt = x.kt(), l = threadIdx.x;
  const int nn = (o.N + 63) >> 6, mg = blockIdx.x / nn, ng = blockIdx.x % nn;
  f32x4 acc[4][4] = {};
  for (int k = 0; k < kt; ++k) {
    u32x4 a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = *reinterpret_cast<const u32x4*>(w.codes + mx_code_at(ng * 4 + i, kt, k) + l * 16);
      b[i] = *reinterpret_cast<const u32x4*>(x.codes + mx_code_at(mg * 4 + i, kt, k) + l * 16);
    }
    const unsigned sa = *reinterpret_cast<const unsigned*>(w.scales + mx_scale_at(ng, kt, k) + l * 4);
    const unsigned sb = *reinterpret_cast<const unsigned*>(x.scales + mx_scale_at(mg, kt, k) + l * 4);
#define MX_ROW(i)                                        \
  acc[i][0] = mx_mfma<i, 0>(a[i], b[0], acc[i][0], sa, sb); \
  acc[i][1] = mx_mfma<i, 1>(a[i], b[1], acc[i][1], sa, sb); \
  acc[i][2] = mx_mfma<i, 2>(a[i], b[2], acc[i][2], sa, sb); \
  acc[i][3] = mx_mfma<i, 3>(a[i], b[3], acc[i][3], sa, sb);
    MX_ROW(0) MX_ROW(1) MX_ROW(2) MX_ROW(3)
#undef MX_ROW
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      mx_store(o, mg * 64 + j * 16 + (l & 15), ng * 64 + i * 16 + (l >> 4) * 4, acc[i][j]);
}

// ---------------------------------------------------------------- gradient
// dX = dY W, dW = dY^T X and db = sum_m dY with the values the quantised
// operands stand for, which bfloat16 holds exactly.  dY goes in as bfloat16
// planes that add up to it exactly: one for bf16, two for fp16 (11 bits), three
// for fp32 (24 bits); every product of a plane is summed in fp32.  Both products
// contract over an index that is not the operands' last, so W, X (and dY for
// dW) are first laid out with it last, padded with zeros to whole 64s.
constexpr int mx_planes(int dtype) { return dtype == T_FP32 ? 3 : dtype == T_FP16 ? 2 : 1; }

// The planes of x by truncation: each takes the next 8 significant bits, so the
// difference is exact and the first plane of a finite value is finite.
template <int P>
DDPG_DEV void plane_split(float x, __bf16 (&p)[P]) {
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const unsigned u = __float_as_uint(x);
    const float h = __uint_as_float(
        (u & 0x7fffffffu) > 0x7f800000u ? 0x7fc00000u : i + 1 < P ? u & 0xffff0000u : u);
    p[i] = (__bf16)h;
    x = (u & 0x7f800000u) == 0x7f800000u ? 0.f : __fsub_rn(x, h);
  }
}

// out[c][r] (ldt columns, rows..ldt zero) of a quantised matrix, a 64 x 128
// tile per block through LDS.
__global__ __launch_bounds__(256) void mx_turn_kernel(MxMat q, __bf16* __restrict__ out, int ldt) {
  __shared__ __bf16 t[128][66];
  const int kt = q.kt(), g64 = blockIdx.x / kt, k = blockIdx.x % kt;
  const int g = threadIdx.x >> 6, l = threadIdx.x & 63;
  const int g16 = g64 * 4 + g;
  {
    float v[32];
    if (g16 * 16 + (l & 15) < q.rows) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(q.codes + mx_code_at(g16, kt, k) + l * 16);
      const unsigned s = q.scales[mx_scale_at(g64, kt, k) + l * 4 + g];
#pragma unroll
      for (int i = 0; i < 4; ++i) mx_values(w[i], s, v + 8 * i);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) t[(l >> 4) * 32 + i][g * 16 + (l & 15)] = (__bf16)v[i];
  }
  __syncthreads();
  for (int c = g; c < 128 && k * 128 + c < q.cols; c += 4)
    if (g64 * 64 + l < ldt) out[(size_t)(k * 128 + c) * ldt + g64 * 64 + l] = t[c][l];
}

// dY's planes as they lie ([P][M][ldn], if flat) and turned ([P][N][ldm], if
// turned), and each 64-row block's column sums, a 64 x 64 tile per block.
template <int DT, int P>
__global__ __launch_bounds__(256) void mx_dy_kernel(const typename Elem<DT>::type* __restrict__ dy,
                                                    long long sr, long long sc, int M, int N,
                                                    __bf16* __restrict__ flat, int ldn,
                                                    __bf16* __restrict__ turned, int ldm,
                                                    float* __restrict__ part) {
  __shared__ float t[64][65];
  const int nn = (N + 63) >> 6, mb = blockIdx.x / nn, m0 = mb * 64, n0 = (blockIdx.x % nn) * 64;
  const int w = threadIdx.x >> 6, l = threadIdx.x & 63;
  for (int i = w; i < 64; i += 4) {
    const float v = m0 + i < M && n0 + l < N ? (float)dy[(m0 + i) * sr + (n0 + l) * sc] : 0.f;
    t[i][l] = v;
    if (flat && m0 + i < M) {
      __bf16 p[P];
      plane_split<P>(v, p);
#pragma unroll
      for (int j = 0; j < P; ++j) flat[((size_t)j * M + m0 + i) * ldn + n0 + l] = p[j];
    }
  }
  __syncthreads();
  if (turned)
    for (int i = w; i < 64 && n0 + i < N; i += 4) {
      __bf16 p[P];
      plane_split<P>(t[l][i], p);
#pragma unroll
      for (int j = 0; j < P; ++j) turned[((size_t)j * N + n0 + i) * ldm + m0 + l] = p[j];
    }
  if (part && w == 0 && n0 + l < N) {
    float s = 0.f;
    for (int i = 0; i < 64; ++i) s += t[i][l];
    part[(size_t)mb * N + n0 + l] = s;
  }
}

__global__ __launch_bounds__(256) void mx_db_kernel(const float* __restrict__ part, int np, int N,
                                                    float* __restrict__ db) {
  const int n = blockIdx.x * 256 + threadIdx.x;
  if (n >= N) return;
  double s = 0;
  for (int i = 0; i < np; ++i) s += part[(size_t)i * N + n];
  db[n] = (float)s;
}

// C[i][j] = sum_p sum_k A[p][i][k] B[j][k]; one wave: 64 x 64, operands straight
// from memory.  ld: the padded contraction length of both.
__global__ __launch_bounds__(64) void mx_plane_gemm_kernel(const __bf16* __restrict__ A,
                                                           const __bf16* __restrict__ B, int I,
                                                           int J, int ld, int planes, void* C,
                                                           int dtype) {
  const int nj = (J + 63) >> 6;
  const int l = threadIdx.x, i0 = blockIdx.x / nj * 64, j0 = blockIdx.x % nj * 64;
  f32x4 acc[4][4] = {};
  for (int p = 0; p < planes; ++p)
    for (int k = 0; k < ld; k += 32) {
      bf16x8 a[4], b[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const size_t i = (size_t)p * I + min(i0 + t * 16 + (l & 15), I - 1);
        const size_t j = min(j0 + t * 16 + (l & 15), J - 1);
        a[t] = *reinterpret_cast<const bf16x8*>(A + i * ld + k + 8 * (l >> 4));
        b[t] = *reinterpret_cast<const bf16x8*>(B + j * ld + k + 8 * (l >> 4));
      }
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y)
          acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[y], a[x], acc[x][y], 0, 0, 0);
    }
#pragma unroll
  for (int x = 0; x < 4; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int i = i0 + x * 16 + (l & 15), j = j0 + y * 16 + (l >> 4) * 4;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (i < I && j + r < J) store_elem(C, dtype, (long long)i * J + j + r, acc[x][y][r]);
    }
}

// ---------------------------------------------------------------- host
static constexpr int64_t kMxMaxDim = 1 << 24;  // rows, columns of a matrix

static void mx_check_dims(const char* what, int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0 || rows > kMxMaxDim || cols > kMxMaxDim)
    throw einval("%s: %lld x %lld is outside [0, %lld]", what, (long long)rows, (long long)cols,
                 (long long)kMxMaxDim);
}

static MxMat mx_mat(const char* what, const void* codes, const void* scales, int64_t rows,
                    int64_t cols) {
  mx_check_dims(what, rows, cols);
  if (rows && cols && (!codes || !scales)) throw einval("%s: null codes or scales", what);
  if (!aligned16(codes) || !aligned16(scales)) throw einval("%s: not 16-byte aligned", what);
  return {static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), (int)rows,
          (int)cols};
}

static unsigned grid_x(long long blocks) {
  if (blocks > INT32_MAX) throw einval("%lld blocks are too many for one launch", blocks);
  return (unsigned)blocks;
}

void mx_quantize_launch(hipStream_t st, int dtype, const void* x, int rows, int cols, long long sr,
                        long long sc, uint8_t* codes, uint8_t* scales) {
  if (!rows || !cols) return;
  const long long tiles = (long long)ceil_div(rows, 64) * ceil_div(cols, 128);
  by_dtype(dtype, [&](auto dt) {
    hipLaunchKernelGGL(mx_quantize_kernel<dt.value>, dim3(grid_x((tiles + 3) / 4)), dim3(256), 0, st,
                       static_cast<const typename Elem<dt.value>::type*>(x), rows, cols, sr, sc,
                       codes, scales);
  });
  HIP_TRY(hipGetLastError());
}

void mx_linear_launch(hipStream_t st, const MxMat& x, const MxMat& w, const MxOut& o) {
  if (!o.M || !o.N) return;
  hipLaunchKernelGGL(mx_linear_kernel, dim3(grid_x((long long)ceil_div(o.N, 64) * ceil_div(o.M, 64))),
                     dim3(64), 0, st,
                     x, w, o);
  HIP_TRY(hipGetLastError());
}

// The gradient's workspace, in order.
struct MxGradWs {
  size_t flat, wt, turned, xt, part, total;
  int ldn, ldm, P;
};
static MxGradWs mx_grad_ws(int dtype, int M, int N, int K, bool dx, bool dw, bool db) {
  MxGradWs w{};
  w.P = mx_planes(dtype);
  w.ldn = rup(N, 64);
  w.ldm = rup(M, 64);
  size_t off = 0;
  auto place = [&](size_t& at, bool need, size_t bytes) {
    at = off;
    if (need) off += (bytes + 255) / 256 * 256;
  };
  place(w.flat, dx, (size_t)w.P * M * w.ldn * 2);
  place(w.wt, dx, (size_t)K * w.ldn * 2);
  place(w.turned, dw, (size_t)w.P * N * w.ldm * 2);
  place(w.xt, dw, (size_t)K * w.ldm * 2);
  place(w.part, db, (size_t)ceil_div(M, 64) * N * 4);
  w.total = off;
  return w;
}

static void mx_plane_gemm(hipStream_t st, const __bf16* A, const __bf16* B, int I, int J, int ld,
                          int planes, void* C, int dtype) {
  if (!I || !J) return;
  hipLaunchKernelGGL(mx_plane_gemm_kernel, dim3(grid_x((long long)ceil_div(J, 64) * ceil_div(I, 64))),
                     dim3(64), 0, st, A, B, I, J, ld, planes, C, dtype);
  HIP_TRY(hipGetLastError());
}

static void mx_turn(hipStream_t st, const MxMat& q, __bf16* out, int ldt) {
  if (!q.rows || !q.cols) return;
  hipLaunchKernelGGL(mx_turn_kernel, dim3(grid_x((long long)q.kt() * ceil_div(q.rows, 64))), dim3(256), 0,
                     st, q, out,
                     ldt);
  HIP_TRY(hipGetLastError());
}

void mx_linear_grad_launch(hipStream_t st, int dtype, const void* dy, long long sr, long long sc,
                           const MxMat& x, const MxMat& w, void* dx, float* dw, float* db,
                           char* ws) {
  const int M = x.rows, N = w.rows, K = x.cols;
  const MxGradWs L = mx_grad_ws(dtype, M, N, K, dx, dw, db);
  __bf16* flat = dx ? reinterpret_cast<__bf16*>(ws + L.flat) : nullptr;
  __bf16* turned = dw ? reinterpret_cast<__bf16*>(ws + L.turned) : nullptr;
  float* part = db ? reinterpret_cast<float*>(ws + L.part) : nullptr;
  if (M && N) {
    by_dtype(dtype, [&](auto dt) {
      hipLaunchKernelGGL((mx_dy_kernel<dt.value, mx_planes(dt.value)>),
                         dim3(grid_x((long long)ceil_div(N, 64) * ceil_div(M, 64))), dim3(256), 0, st,
                         static_cast<const typename Elem<dt.value>::type*>(dy), sr, sc, M, N, flat,
                         L.ldn, turned, L.ldm, part);
    });
    HIP_TRY(hipGetLastError());
  }
  if (db && N) {
    hipLaunchKernelGGL(mx_db_kernel, dim3(ceil_div(N, 256)), dim3(256), 0, st, part,
                       ceil_div(M, 64), N, db);
    HIP_TRY(hipGetLastError());
  }
  if (dx) {
    __bf16* wt = reinterpret_cast<__bf16*>(ws + L.wt);
    mx_turn(st, w, wt, L.ldn);
    mx_plane_gemm(st, flat, wt, M, K, L.ldn, L.P, dx, dtype);
  }
  if (dw) {
    __bf16* xt = reinterpret_cast<__bf16*>(ws + L.xt);
    mx_turn(st, x, xt, L.ldm);
    mx_plane_gemm(st, turned, xt, N, K, L.ldm, L.P, dw, T_FP32);
  }
}

}  // namespace ddpg

extern "C" {

int ddpg_mx_sizes(int64_t rows, int64_t cols, size_t* code_bytes, size_t* scale_bytes) {
  return guard(nullptr, [&] {
    mx_check_dims("mx_sizes", rows, cols);
    if (code_bytes) *code_bytes = mx_code_bytes(rows, cols);
    if (scale_bytes) *scale_bytes = mx_scale_bytes(rows, cols);
  });
}

int ddpg_mx_quantize(int device, void* stream, int dtype, const void* x, int64_t rows,
                     int64_t cols, int64_t row_stride, int64_t col_stride, void* codes,
                     void* scales) {
  return guard(nullptr, [&] {
    check_dtype("mx_quantize", dtype);
    mx_mat("mx_quantize", codes, scales, rows, cols);
    if (rows && cols && !x) throw einval("mx_quantize: null input");
    OnDevice on(device);
    mx_quantize_launch(static_cast<hipStream_t>(stream), dtype, x, (int)rows, (int)cols, row_stride,
                       col_stride, static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales));
  });
}

int ddpg_mx_dequantize(int device, void* stream, const void* codes, const void* scales,
                       int64_t rows, int64_t cols, int dtype, void* out, int64_t row_stride) {
  return guard(nullptr, [&] {
    check_dtype("mx_dequantize", dtype);
    const MxMat q = mx_mat("mx_dequantize", codes, scales, rows, cols);
    if (!rows || !cols) return;
    if (!out) throw einval("mx_dequantize: null output");
    if (row_stride < cols) throw einval("mx_dequantize: rows %lld apart overlap", (long long)row_stride);
    OnDevice on(device);
    const long long tiles = (long long)ceil_div(q.rows, 16) * q.kt();
    by_dtype(dtype, [&](auto dt) {
      hipLaunchKernelGGL(mx_dequantize_kernel<dt.value>, dim3(grid_x((tiles + 3) / 4)), dim3(256), 0,
                         static_cast<hipStream_t>(stream), q,
                         static_cast<typename Elem<dt.value>::type*>(out), (long long)row_stride);
    });
    HIP_TRY(hipGetLastError());
  });
}

int ddpg_mx_linear(int device, void* stream, int x_dtype, const void* x, int64_t x_row_stride,
                   int64_t x_col_stride, void* x_codes, void* x_scales, int64_t M, int64_t K,
                   const void* w_codes, const void* w_scales, int64_t N, int bias_dtype,
                   const void* bias, int act, int dtype, void* y, int64_t y_row_stride) {
  return guard(nullptr, [&] {
    const MxMat xq = mx_mat("mx_linear x", x_codes, x_scales, M, K);
    const MxMat wq = mx_mat("mx_linear w", w_codes, w_scales, N, K);
    check_dtype("mx_linear", dtype);
    if (x) check_dtype("mx_linear x", x_dtype);
    if (bias) check_dtype("mx_linear bias", bias_dtype);
    if (act < DDPG_ACT_NONE || act > DDPG_ACT_TANH) throw einval("mx_linear: act %d", act);
    if (!M || !N) return;
    if (!y) throw einval("mx_linear: null output");
    if (y_row_stride < N) throw einval("mx_linear: rows %lld apart overlap", (long long)y_row_stride);
    OnDevice on(device);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (x)
      mx_quantize_launch(st, x_dtype, x, (int)M, (int)K, x_row_stride, x_col_stride,
                         static_cast<uint8_t*>(x_codes), static_cast<uint8_t*>(x_scales));
    const MxOut o{y, bias, (long long)y_row_stride, (int)M, (int)N, dtype, bias_dtype, act};
    mx_linear_launch(st, xq, wq, o);
  });
}

size_t ddpg_mx_linear_grad_workspace(int dtype, int64_t M, int64_t N, int64_t K, int dx, int dw,
                                     int db) {
  if (M < 0 || N < 0 || K < 0 || M > kMxMaxDim || N > kMxMaxDim || K > kMxMaxDim) return 0;
  return mx_grad_ws(dtype, (int)M, (int)N, (int)K, dx != 0, dw != 0, db != 0).total;
}

int ddpg_mx_linear_grad(int device, void* stream, int dtype, const void* dy, int64_t dy_row_stride,
                        int64_t dy_col_stride, int64_t M, int64_t N, int64_t K,
                        const void* x_codes, const void* x_scales, const void* w_codes,
                        const void* w_scales, void* dx, float* dw, float* db, void* ws,
                        size_t ws_bytes) {
  return guard(nullptr, [&] {
    check_dtype("mx_linear_grad", dtype);
    const MxMat xq = mx_mat("mx_linear_grad x", dw ? x_codes : nullptr, dw ? x_scales : nullptr,
                            M, dw ? K : 0);
    const MxMat wq = mx_mat("mx_linear_grad w", dx ? w_codes : nullptr, dx ? w_scales : nullptr,
                            N, dx ? K : 0);
    mx_check_dims("mx_linear_grad", M, K);
    if (M && N && !dy) throw einval("mx_linear_grad: null dy");
    const size_t need = mx_grad_ws(dtype, (int)M, (int)N, (int)K, dx, dw, db).total;
    if (ws_bytes < need || (need && !ws) || !aligned16(ws))
      throw einval("mx_linear_grad: workspace of %zu bytes, %zu needed", ws_bytes, need);
    OnDevice on(device);
    MxMat xm = xq, wm = wq;
    xm.cols = wm.cols = (int)K;
    mx_linear_grad_launch(static_cast<hipStream_t>(stream), dtype, dy, dy_row_stride, dy_col_stride,
                          xm, wm, dx, dw, db, static_cast<char*>(ws));
  });
}

}  // extern "C"
