// MXFP4 operators: quantisation and its inverse, the product of two quantised
// matrices (a layer's forward), and that product's gradient.  The format and
// its layout: mx.h.
#include "mx_gemm.h"

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

// A quantised matrix turned into bfloat16 fragments (mx_gemm.h): rows are its
// columns, the depth its rows (to whole 64s, the padding 0).  A 64 x 128 tile
// per block, through LDS.
__global__ __launch_bounds__(256) void mx_turn_kernel(MxMat q, uint8_t* __restrict__ out) {
  __shared__ __attribute__((aligned(16))) __bf16 t[128][72];
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
  const int steps = (q.rows + 63) / 64 * 2;
  for (int f = g; f < 16; f += 4) {  // 8 row groups x 2 depth steps
    const int c = (f >> 1) * 16, d = (f & 1) * 32;
    const size_t grp = (size_t)k * 8 + (f >> 1);
    if (k * 128 + c >= q.cols) break;
    *reinterpret_cast<bf16x8*>(out + (grp * steps + g64 * 2 + (f & 1)) * 1024 + l * 16) =
        *reinterpret_cast<const bf16x8*>(&t[c + (l & 15)][d + 8 * (l >> 4)]);
  }
}

// dY's planes as fragments (mx_gemm.h; a row group's planes one after the
// other): flat, rows m and depth n (if not null); turned, rows n and depth m (if
// not null); both depths to whole 64s, the padding 0.  And each 64-row
// block's column sums (part, if not null).  A 64 x 64 tile per block.
template <int DT, int P>
__global__ __launch_bounds__(256) void mx_dy_kernel(const typename Elem<DT>::type* __restrict__ dy,
                                                    long long sr, long long sc, int M, int N,
                                                    uint8_t* __restrict__ flat,
                                                    uint8_t* __restrict__ turned,
                                                    float* __restrict__ part) {
  __shared__ float t[64][65];
  const int nn = (N + 63) >> 6, mb = blockIdx.x / nn, nb = blockIdx.x % nn;
  const int m0 = mb * 64, n0 = nb * 64, nm = (M + 63) >> 6;
  const int w = threadIdx.x >> 6, l = threadIdx.x & 63;
  for (int i = w; i < 64; i += 4)
    t[i][l] = m0 + i < M && n0 + l < N ? (float)dy[(m0 + i) * sr + (n0 + l) * sc] : 0.f;
  __syncthreads();
  // 4 row groups x 2 depth steps: a wave takes row group w
  auto put = [&](uint8_t* out, int grp, int steps, int s0, auto at) {
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      bf16x8 f[P];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        __bf16 p[P];
        plane_split<P>(at(w * 16 + (l & 15), d * 32 + 8 * (l >> 4) + e), p);
#pragma unroll
        for (int j = 0; j < P; ++j) f[j][e] = p[j];
      }
#pragma unroll
      for (int j = 0; j < P; ++j)
        *reinterpret_cast<bf16x8*>(out + (((size_t)grp * P + j) * steps + s0 + d) * 1024 + l * 16) =
            f[j];
    }
  };
  if (flat) put(flat, mb * 4 + w, nn * 2, nb * 2, [&](int r, int c) { return t[r][c]; });
  if (turned) put(turned, nb * 4 + w, nm * 2, mb * 2, [&](int r, int c) { return t[c][r]; });
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

// Which kernel a product of I x J outputs takes: the largest tile that leaves
// most of the 256 CUs one, and with fewer tiles the kernel that splits the depth
// over a block's waves.  fp4, us: 16384 x 8192 x 8192 665 on 256 x 256 tiles, 719
// on 128 x 128; 1001 x 300 x 400 14.0 on 128 x 128 tiles, 6.7 split.  bf16: 8192 x 4096
// x 4096 207 against 268, 1001 x 400 x 3 planes of 300 28.4 against 11.0.
template <bool FP4>
static void mx_gemm_launch(hipStream_t st, MxGemm g) {
  MxOut& o = g.o;
  if (!o.I || !o.J) return;
  const int es = elem_size(o.dtype);
  o.vec = o.ldo * es % 16 == 0 && aligned16(o.y);
  const long long big = (long long)ceil_div(o.I, 256) * ceil_div(o.J, 256);
  const long long mid = (long long)ceil_div(o.I, 128) * ceil_div(o.J, 128);
  if (big >= 200) {
    hipLaunchKernelGGL((mx_tile_kernel<FP4, 2, 4, 8, 4, 4>), dim3(grid_x(big)), dim3(512), 0, st, g);
  } else if (mid >= 128) {
    hipLaunchKernelGGL((mx_tile_kernel<FP4, 2, 2, 4, 4, 4>), dim3(grid_x(mid)), dim3(256), 0, st, g);
  } else if (o.I <= 16) {
    hipLaunchKernelGGL((mx_split_kernel<FP4, 1, 1, 8>), dim3(ceil_div(o.J, 16)), dim3(512), 0, st,
                       g);
  } else {
    const long long small = (long long)ceil_div(o.I, 64) * ceil_div(o.J, 64);
    hipLaunchKernelGGL((mx_split_kernel<FP4, 4, 4, 4>), dim3(grid_x(small)), dim3(256), 0, st, g);
  }
  HIP_TRY(hipGetLastError());
}

static FragOp mx_op(const MxMat& q) {
  return {q.codes, q.scales, ceil_div(q.rows, 64) * 4};
}

void mx_linear_launch(hipStream_t st, const MxMat& x, const MxMat& w, const MxOut& o) {
  mx_gemm_launch<true>(st, MxGemm{mx_op(x), mx_op(w), x.kt(), 1, o});
}

// The gradient's workspace, in order.
struct MxGradWs {
  size_t flat, wt, turned, xt, part, total;
  int sn, sm, P;  // depth steps over N, over M
};
static MxGradWs mx_grad_ws(int dtype, int M, int N, int K, bool dx, bool dw, bool db) {
  MxGradWs w{};
  w.P = mx_planes(dtype);
  w.sn = ceil_div(N, 64) * 2;
  w.sm = ceil_div(M, 64) * 2;
  auto frags = [](int rows, size_t steps) { return (size_t)ceil_div(rows, 64) * 4 * steps * 1024; };
  size_t off = 0;
  auto place = [&](size_t& at, bool need, size_t bytes) {
    at = off;
    if (need) off += (bytes + 255) / 256 * 256;
  };
  place(w.flat, dx, frags(M, (size_t)w.P * w.sn));
  place(w.wt, dx, frags(K, w.sn));
  place(w.turned, dw, frags(N, (size_t)w.P * w.sm));
  place(w.xt, dw, frags(K, w.sm));
  place(w.part, db, (size_t)ceil_div(M, 64) * N * 4);
  w.total = off;
  return w;
}

static void mx_turn(hipStream_t st, const MxMat& q, uint8_t* out) {
  if (!q.rows || !q.cols) return;
  hipLaunchKernelGGL(mx_turn_kernel, dim3(grid_x((long long)q.kt() * ceil_div(q.rows, 64))),
                     dim3(256), 0, st, q, out);
  HIP_TRY(hipGetLastError());
}

static void mx_plane_gemm(hipStream_t st, const uint8_t* A, const uint8_t* B, int I, int J,
                          int steps, int planes, void* C, int dtype) {
  const MxOut o{C, nullptr, J, I, J, dtype, 0, DDPG_ACT_NONE, 0};
  mx_gemm_launch<false>(st, MxGemm{{A, nullptr, ceil_div(I, 64) * 4},
                                   {B, nullptr, ceil_div(J, 64) * 4}, steps, planes, o});
}

void mx_linear_grad_launch(hipStream_t st, int dtype, const void* dy, long long sr, long long sc,
                           const MxMat& x, const MxMat& w, void* dx, float* dw, float* db,
                           uint8_t* ws) {
  const int M = x.rows, N = w.rows, K = x.cols;
  const MxGradWs L = mx_grad_ws(dtype, M, N, K, dx, dw, db);
  uint8_t* flat = dx ? ws + L.flat : nullptr;
  uint8_t* turned = dw ? ws + L.turned : nullptr;
  float* part = db ? reinterpret_cast<float*>(ws + L.part) : nullptr;
  if (M && N && (dx || dw || db)) {
    by_dtype(dtype, [&](auto dt) {
      hipLaunchKernelGGL((mx_dy_kernel<dt.value, mx_planes(dt.value)>),
                         dim3(grid_x((long long)ceil_div(N, 64) * ceil_div(M, 64))), dim3(256), 0,
                         st, static_cast<const typename Elem<dt.value>::type*>(dy), sr, sc, M, N,
                         flat, turned, part);
    });
    HIP_TRY(hipGetLastError());
  }
  if (db && N) {
    hipLaunchKernelGGL(mx_db_kernel, dim3(ceil_div(N, 256)), dim3(256), 0, st, part,
                       ceil_div(M, 64), N, db);
    HIP_TRY(hipGetLastError());
  }
  if (dx) {
    mx_turn(st, w, ws + L.wt);
    mx_plane_gemm(st, flat, ws + L.wt, M, K, L.sn, L.P, dx, dtype);
  }
  if (dw) {
    mx_turn(st, x, ws + L.xt);
    mx_plane_gemm(st, turned, ws + L.xt, N, K, L.sm, L.P, dw, T_FP32);
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
    const MxOut o{y, bias, (long long)y_row_stride, (int)M, (int)N, dtype, bias_dtype, act, 0};
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
                          xm, wm, dx, dw, db, static_cast<uint8_t*>(ws));
  });
}

}  // extern "C"
