// MXFP4 operators: quantisation and its inverse, the product of two quantised
// matrices (a layer's forward), and that product's gradient.  The format and
// its layout: mx.h.
#include "mx_gemm.h"

namespace ddpg {

// ---------------------------------------------------------------- quantise
// A block makes one tile of 64 rows x 128 columns.
//
// ROWS (a row's values adjacent): a wave takes 16 rows, four at a time, 16 lanes
// along a row with 8 values each, so that loads are whole lines; the four lanes of
// a 32-block share its largest magnitude and write its 16 bytes of codes together.
// Input that is used once goes past the caches.
//
// Otherwise a wave takes 32 columns and its lanes 64 rows, so that a load is
// contiguous where rows are (a matrix in checkpoint order seen turned); blocks
// that follow each other take rows that follow each other.
//
// Loads past the matrix are from its last element and count as 0.  Bound: bytes;
// 16384 x 8192 bf16 in 57 us (5.9 TB/s), 8192 x 8192 fp32 turned in 55 us (5.5 TB/s;
// through the caches and with blocks along the columns 87).
template <int DT, bool ROWS>
__global__ __launch_bounds__(256) void mx_quantize_kernel(
    const typename Elem<DT>::type* __restrict__ x, int rows, int cols, long long sr, long long sc,
    uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  __shared__ __attribute__((aligned(4))) uint8_t sb[256];
  const int kt = (cols + 127) >> 7, l = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int n64 = (rows + 63) >> 6;
  const int g64 = ROWS ? blockIdx.x / kt : blockIdx.x % n64;
  const int k = ROWS ? blockIdx.x % kt : blockIdx.x / n64;
  if constexpr (ROWS) {
    constexpr int V = Elem<DT>::V, L = 8 / V;  // loads of 8 values
    const int g16 = g64 * 4 + w, c0 = k * 128 + (l & 15) * 8;
    if (g16 * 16 < rows) {
      float v[4][8];
      if (c0 + 8 <= cols) {
        U16B u[4][L];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < L; ++j)
            u[i][j] = load16<true>(x + min(g16 * 16 + i * 4 + (l >> 4), rows - 1) * sr + c0 + j * V);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < L; ++j) Elem<DT>::widen(u[i][j], v[i] + j * V);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j)
            v[i][j] = (float)x[min(g16 * 16 + i * 4 + (l >> 4), rows - 1) * sr + min(c0 + j, cols - 1)];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] = c0 + j < cols ? v[i][j] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = i * 4 + (l >> 4), kb = (l & 15) >> 2;
        unsigned top = mx_top<8>(v[i]);
        // the largest of the block's four lanes (DPP: lanes ^ 1, then ^ 2)
        top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, true));
        top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, true));
        const unsigned s = mx_scale_of(top);
        *reinterpret_cast<unsigned*>(codes + mx_code_at(g16, kt, k) + (kb * 16 + r) * 16 +
                                     (l & 3) * 4) = mx_codes8(v[i], mx_factor(s));
        if ((l & 3) == 0) sb[(kb * 16 + r) * 4 + w] = (uint8_t)s;
      }
    } else {
      sb[l * 4 + w] = 0;
    }
  } else {
    const int row = g64 * 64 + l, c0 = k * 128 + w * 32;
    unsigned s = 0;
    if (g64 * 64 + (l & ~15) < rows) {
      float v[32];
      mx_load_block<DT, true>(x + min(row, rows - 1) * sr, sc, false, c0, cols, v);
      const u32x4 q = mx_quantize_block(v, s);
      *reinterpret_cast<u32x4*>(codes + mx_code_at(g64 * 4 + (l >> 4), kt, k) +
                                (w * 16 + (l & 15)) * 16) = q;
    }
    sb[(w * 16 + (l & 15)) * 4 + (l >> 4)] = (uint8_t)s;
  }
  __syncthreads();
  if (w == 0)
    reinterpret_cast<unsigned*>(scales + mx_scale_at(g64, kt, k))[l] =
        reinterpret_cast<const unsigned*>(sb)[l];
}

// A wave takes 16 rows x 128 columns: the codes go through LDS, so that its lanes
// write along the rows, 16 bytes each.  Bound: bytes; 8192 x 8192 to fp32 in 49 us
// (6.2 TB/s; 286 us with a thread writing its block's 128 bytes).
template <int DT>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(MxMat q,
                                                            typename Elem<DT>::type* out,
                                                            long long ldo) {
  typedef typename Elem<DT>::type T;
  constexpr int V = Elem<DT>::V, PER = 128 / V;  // 16-byte units of a row
  __shared__ __attribute__((aligned(16))) uint8_t sq[4][1024];
  __shared__ uint8_t ss[4][64];
  const int kt = q.kt(), l = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int g16 = blockIdx.x / kt * 4 + w, k = blockIdx.x % kt;
  if (g16 * 16 < q.rows) {
    *reinterpret_cast<u32x4*>(&sq[w][l * 16]) =
        *reinterpret_cast<const u32x4*>(q.codes + mx_code_at(g16, kt, k) + l * 16);
    ss[w][l] = q.scales[mx_scale_at(g16 >> 2, kt, k) + l * 4 + (g16 & 3)];
  }
  __syncthreads();
#pragma unroll
  for (int u = l; u < 16 * PER; u += 64) {
    const int r = u / PER, c = u % PER * V;  // V columns of row r
    const int row = g16 * 16 + r, col = k * 128 + c;
    if (row >= q.rows || col >= q.cols) continue;
    const int at = (c >> 5) * 16 + r;  // the lane that holds the block
    float v[8];
    if (V == 4) {
      mx_values(*reinterpret_cast<const uint16_t*>(&sq[w][at * 16 + (c & 31) / 2]), ss[w][at], v);
    } else {
      mx_values(*reinterpret_cast<const unsigned*>(&sq[w][at * 16 + (c & 31) / 2]), ss[w][at], v);
    }
    T* p = out + row * ldo + col;
    if (col + V <= q.cols) {
      *reinterpret_cast<U16B*>(p) = Elem<DT>::pack(v);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (col + i < q.cols) p[i] = (T)v[i];
    }
  }
}

// ---------------------------------------------------------------- gradient
// dX = dY W, dW = dY^T X and db = sum_m dY with the values the quantised
// operands stand for, which bfloat16 holds exactly.  dY goes in as bfloat16
// planes that add up to it exactly: one for bf16, two for fp16 (11 bits), three
// for fp32 (24 bits; those below 2^-133, bfloat16's smallest number, are rounded off,
// which |dY| >= 2^-110 has none of); every product of a plane is summed in fp32.  Both products
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

// What the two products need first, one launch: blocks of three kinds, each
// with one tile.  Bound: bytes; 8192 x 4096 x 4096 bf16 moves 329 MB in 56 us (5.9
// TB/s).  Lanes lie along dY's columns: where its rows are the adjacent ones, a load
// touches a line a lane (88 us; fp32 103 and 141).
struct MxPrep {
  const void* dy;
  long long sr, sc;
  int M, N;
  uint8_t *flat, *turned;  // dY's planes for dX, for dW (or null)
  float* part;             // column sums of 64-row blocks (or null)
  MxMat w, x;
  uint8_t *wt, *xt;
  int dy_blocks, w_blocks;
  unsigned* tickets;  // cleared for the products' joins
  int ntickets;
};

// A quantised matrix turned into bfloat16 fragments (mx_gemm.h): rows are its
// columns, the depth its rows (to whole 64s, the padding 0).  64 x 128 tile b,
// through LDS.
DDPG_DEV void mx_turn(const MxMat& q, uint8_t* __restrict__ out, int b, __bf16 (&t)[128][72]) {
  const int kt = q.kt(), g64 = b / kt, k = b % kt;
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

// A 64 x 64 tile of dY as fragments of its planes (a row group's planes one after
// the other): flat, rows m and depth n; turned, rows n and depth m; both depths
// to whole 64s, the padding 0.  And the tile's column sums.
template <int DT, int P>
DDPG_DEV void mx_dy(const MxPrep& a, int b, float (&t)[64][65], float (&red)[4][64]) {
  const typename Elem<DT>::type* dy = static_cast<const typename Elem<DT>::type*>(a.dy);
  const int M = a.M, N = a.N, nn = (N + 63) >> 6, mb = b / nn, nb = b % nn;
  const int m0 = mb * 64, n0 = nb * 64, nm = (M + 63) >> 6;
  const int w = threadIdx.x >> 6, l = threadIdx.x & 63;
  {
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i)
      v[i] = (float)dy[min(m0 + w + 4 * i, M - 1) * a.sr + min(n0 + l, N - 1) * a.sc];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float x = m0 + w + 4 * i < M && n0 + l < N ? v[i] : 0.f;
      t[w + 4 * i][l] = x;
      s += x;
    }
    red[w][l] = s;
  }
  __syncthreads();
  if (a.part && w == 0 && n0 + l < N)
    a.part[(size_t)mb * N + n0 + l] = ((red[0][l] + red[1][l]) + red[2][l]) + red[3][l];
  // 4 row groups x 2 depth steps: a wave takes row group w
  auto put = [&](uint8_t* out, int grp, int steps, int s0, auto at) {
#pragma unroll 1
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
  if (a.flat) put(a.flat, mb * 4 + w, nn * 2, nb * 2, [&](int r, int c) { return t[r][c]; });
  if (a.turned) put(a.turned, nb * 4 + w, nm * 2, mb * 2, [&](int r, int c) { return t[c][r]; });
}

template <int DT>
__global__ __launch_bounds__(256) void mx_prep_kernel(MxPrep a) {
  __shared__ __attribute__((aligned(16))) union {
    __bf16 turn[128][72];
    struct {
      float t[64][65], red[4][64];
    } dy;
  } t;
  const int b = blockIdx.x;
  if (b == 0)
    for (int i = threadIdx.x; i < a.ntickets; i += 256) a.tickets[i] = 0;
  if (b < a.dy_blocks)
    mx_dy<DT, mx_planes(DT)>(a, b, t.dy.t, t.dy.red);
  else if (b < a.dy_blocks + a.w_blocks)
    mx_turn(a.w, a.wt, b - a.dy_blocks, t.turn);
  else
    mx_turn(a.x, a.xt, b - a.dy_blocks - a.w_blocks, t.turn);
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
  const unsigned tiles = grid_x((long long)ceil_div(rows, 64) * ceil_div(cols, 128));
  by_dtype(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    auto k = sc == 1 ? mx_quantize_kernel<DT, true> : mx_quantize_kernel<DT, false>;
    hipLaunchKernelGGL(k, dim3(tiles), dim3(256), 0, st,
                       static_cast<const typename Elem<DT>::type*>(x), rows, cols, sr, sc, codes,
                       scales);
  });
  HIP_TRY(hipGetLastError());
}

// How each of the kernels does: fp4 16384 x 8192 x 8192 487 us (4.5 PFLOP/s) on 256 x
// 256 tiles, bf16 8192 x 4096 x 4096 twice in 385 us (1.43 PFLOP/s, both at the power
// limit, the clock below 2 GHz); fp4 2048 x 2048 x 2048 10.8 us (1.6 PFLOP/s) on 128 x
// 128, 512 x 4096 x 4096 12.3 us on 64 x 64, 256 x 1024 x 1024 4.1 us on 32 x 32.
//
// The kernels of a product: tiles of 256 x 256 and 128 x 128 through LDS, and 64 x 64
// and 32 x 32 with the depth split over a block's 4 and 8 waves.
enum { MX_256, MX_128, MX_64, MX_32 };
static constexpr int kMxTile[] = {256, 128, 64, 32};
static constexpr int kMxSlab[] = {256 * 256 * 4, 128 * 128 * 4, 64 * 64 * 4, 32 * 32 * 4};
static long long mx_tiles(int I, int J, int t) {
  return (long long)ceil_div(I, t) * ceil_div(J, t);
}

template <bool FP4>
static void mx_gemm_launch(hipStream_t st, MxGemms& p, int pick) {
  const int tile = kMxTile[pick];
  auto launch = [&](auto k, int threads) {
    long long n = 0;
    for (int i = 0; i < 2; ++i) {
      const MxOut& o = p.g[i].o;
      if (i < p.n) {
        n += mx_tiles(o.I, o.J, tile) * p.g[i].splits;
      }
      p.end[i] = (int)grid_x(n);
    }
    n += ceil_div(p.db_n, 64);
    if (!n) return;
    hipLaunchKernelGGL(k, dim3(grid_x(n)), dim3(threads), 0, st, p);
    HIP_TRY(hipGetLastError());
  };
  switch (pick) {
    case MX_256: launch(mx_tile_kernel<FP4, 2, 4, 8, 4, 4>, 512); break;
    case MX_128: launch(mx_tile_kernel<FP4, 2, 2, 4, 4, 4>, 256); break;
    case MX_64: launch(mx_split_kernel<FP4, 4, 4, 4, 2>, 256); break;
    default: launch(mx_split_kernel<FP4, 2, 2, 8, 4>, 512);
  }
}

static FragOp mx_op(const MxMat& q) {
  return {q.codes, q.scales, ceil_div(q.rows, 64) * 4};
}

void mx_linear_launch(hipStream_t st, const MxMat& x, const MxMat& w, const MxOut& o) {
  if (!o.I || !o.J) return;
  MxGemms p{};
  p.n = 1;
  p.g[0] = {mx_op(x), mx_op(w), x.kt(), 1, o, 1, nullptr, nullptr};
  // Measured on 60 shapes, us: 640 x 1024 x 1024 5.7 on 32 x 32 tiles, 6.0 on 64; 512 x
  // 4096 x 4096 12.3 on 64 x 64, 18.8 on 32, 13.3 on 128; 4096 x 1024 x 1024 8.8 on 128 x
  // 128, 12.0 on 64, 14.8 on 256; 8192 x 2048 x 2048 24.0 on 256 x 256, 26.7 on 128
  auto tiles = [&](int pick) { return mx_tiles(o.I, o.J, kMxTile[pick]); };
  mx_gemm_launch<true>(st, p, tiles(MX_256) >= 256  ? MX_256
                              : tiles(MX_32) <= 640 ? MX_32
                              : tiles(MX_64) <= 512 ? MX_64
                                                    : MX_128);
}

// Whether the rows of x are quantised by every block of 16 columns of the
// product.  A row of 8192 values: 7.6 us so, 8.8 in two launches; 16 rows of 512 4.7
// and 5.7, of 2048 6.5 and 6.3, of 4096 10.2 and 7.2; 64 of 512 7.4 and 5.8 (a second
// launch costs the host 2.5 us besides).
static bool mx_rows_ok(int64_t M, int64_t K) { return M <= 64 && M * K <= 32768; }
void mx_linear_rows_launch(hipStream_t st, int dtype, const void* x, long long sr, long long sc,
                           int M, int K, const MxMat& w, const MxOut& o) {
  if (!M || !o.J) return;
  const RawX r{x, sr, sc, M, K, sc == 1};
  by_dtype(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    auto k = M <= 16   ? mx_rows_kernel<DT, 1, 8>
             : M <= 32 ? mx_rows_kernel<DT, 2, 8>
                       : mx_rows_kernel<DT, 4, 8>;
    hipLaunchKernelGGL(k, dim3(ceil_div(o.J, 16)), dim3(512), 0, st, r, mx_op(w), w.kt(), o);
  });
  HIP_TRY(hipGetLastError());
}

// The gradient's plan: the kernel, the depth's splits and the workspace, in
// order.  Kernel and splits go by both products, so that a result does not depend
// on which are asked for.
struct MxGradPlan {
  size_t flat, wt, turned, xt, part, tickets, slab[2], total;  // slab: of dX, dW
  int sn, sm, P;  // depth steps over N, over M
  int pick, splits[2];
  int ntickets;
};
static MxGradPlan mx_grad_plan(int dtype, int M, int N, int K, bool dx, bool dw, bool db) {
  MxGradPlan w{};
  w.P = mx_planes(dtype);
  w.sn = ceil_div(N, 64) * 2;
  w.sm = ceil_div(M, 64) * 2;
  const long long steps[2] = {(long long)w.P * w.sn, (long long)w.P * w.sm};
  const int I[2] = {M, N};
  auto tiles = [&](int q, int pick) { return mx_tiles(I[q], K, kMxTile[pick]); };
  auto all = [&](int pick) { return tiles(0, pick) * steps[0] + tiles(1, pick) * steps[1]; };
  // Each kernel up to the work (a tile costs about 16 depth steps besides its own)
  // it is best at; us, bf16: 1362 x 195 x 2659 24.2 on 64 x 64 tiles, 24.9 on 32, 28.2 on 128;
  // 2048 x 2048 x 2048 46.2 on 128 x 128, 62.8 on 64, 61.2 on 256; 8192 x 2048 x 2048 136 on
  // 256 x 256, 141 on 128 (4096 x 2048 x 2048 89 and 80)
  auto cost = [&](int pick) { return all(pick) + 16 * (tiles(0, pick) + tiles(1, pick)); };
  w.pick = cost(MX_256) >= 32000  ? MX_256
           : cost(MX_32) <= 40000 ? MX_32
           : cost(MX_64) <= 40000 ? MX_64
                                  : MX_128;
  // a block's depth: an equal share of a launch that fills the chip, but no less
  // than what makes the join worth it
  const long long least[] = {32, 24, 32, 64}, fill[] = {256, 256, 512, 512};
  const long long share = std::max(least[w.pick], (all(w.pick) + fill[w.pick] - 1) / fill[w.pick]);
  size_t off = 0;
  auto place = [&](size_t& at, bool need, size_t bytes) {
    at = off;
    if (need) off += (bytes + 255) / 256 * 256;
  };
  auto frags = [](int rows, size_t steps) { return (size_t)ceil_div(rows, 64) * 4 * steps * 1024; };
  place(w.flat, dx, frags(M, (size_t)w.P * w.sn));
  place(w.wt, dx, frags(K, w.sn));
  place(w.turned, dw, frags(N, (size_t)w.P * w.sm));
  place(w.xt, dw, frags(K, w.sm));
  place(w.part, db, (size_t)ceil_div(M, 64) * N * 4);
  for (int q = 0; q < 2; ++q) {
    w.splits[q] = (int)std::min<long long>(32, std::max<long long>(1, (steps[q] + share / 2) / share));
    if (w.splits[q] > 1) w.ntickets += (int)tiles(q, w.pick);
  }
  place(w.tickets, w.ntickets, (size_t)w.ntickets * 4);
  for (int q = 0; q < 2; ++q)
    place(w.slab[q], w.splits[q] > 1 && (q ? dw : dx),
          (size_t)tiles(q, w.pick) * w.splits[q] * kMxSlab[w.pick]);
  w.total = off;
  return w;
}

void mx_linear_grad_launch(hipStream_t st, int dtype, const void* dy, long long sr, long long sc,
                           const MxMat& x, const MxMat& w, void* dx, float* dw, float* db,
                           uint8_t* ws) {
  const int M = x.rows, N = w.rows, K = x.cols;
  const MxGradPlan L = mx_grad_plan(dtype, M, N, K, dx, dw, db);
  MxPrep a{};
  a.dy = dy;
  a.sr = sr;
  a.sc = sc;
  a.M = M;
  a.N = N;
  a.w = w;
  a.x = x;
  a.flat = dx ? ws + L.flat : nullptr;
  a.turned = dw ? ws + L.turned : nullptr;
  a.part = db ? reinterpret_cast<float*>(ws + L.part) : nullptr;
  a.wt = ws + L.wt;
  a.xt = ws + L.xt;
  const long long n64 = ceil_div(N, 64), m64 = ceil_div(M, 64), kt = ceil_div(K, 128);
  const long long nd = (dx || dw || db) ? n64 * m64 : 0, nw = dx ? n64 * kt : 0,
                  nx = dw ? m64 * kt : 0;
  a.dy_blocks = (int)grid_x(nd);
  a.w_blocks = (int)grid_x(nw);
  a.tickets = reinterpret_cast<unsigned*>(ws + L.tickets);
  a.ntickets = L.ntickets;
  if (nd + nw + nx)
    by_dtype(dtype, [&](auto dt) {
      hipLaunchKernelGGL(mx_prep_kernel<decltype(dt)::value>, dim3(grid_x(nd + nw + nx)), dim3(256),
                         0, st, a);
    });
  HIP_TRY(hipGetLastError());
  MxGemms p{};
  unsigned* tickets = reinterpret_cast<unsigned*>(ws + L.tickets);
  auto add = [&](int q, const uint8_t* I, const uint8_t* J, int ni, int steps, void* C, int type) {
    if (!ni || !K) return;
    // dX's tickets first, then dW's
    unsigned* t = tickets + (q && L.splits[0] > 1 ? mx_tiles(M, K, kMxTile[L.pick]) : 0);
    p.g[p.n++] = {{I, nullptr, ceil_div(ni, 64) * 4},
                  {J, nullptr, ceil_div(K, 64) * 4},
                  steps,
                  L.P,
                  {C, nullptr, K, ni, K, type, 0, DDPG_ACT_NONE},
                  L.splits[q],
                  reinterpret_cast<float*>(ws + L.slab[q]),
                  t};
  };
  // the deeper product's blocks first: the shorter ones fill in behind them
  const bool dw_first = L.sm > L.sn;
  if (dw && dw_first) add(1, a.turned, a.xt, N, L.sm, dw, T_FP32);
  if (dx) add(0, a.flat, a.wt, M, L.sn, dx, dtype);
  if (dw && !dw_first) add(1, a.turned, a.xt, N, L.sm, dw, T_FP32);
  p.db = db;
  p.db_part = a.part;
  p.db_n = db ? N : 0;
  p.db_parts = (int)m64;
  mx_gemm_launch<false>(st, p, L.pick);
}

// ---------------------------------------------------------------- the learner's
// A quantised matrix in one buffer, the scales behind the codes.
size_t mx_bytes(int rows, int cols) { return mx_code_bytes(rows, cols) + mx_scale_bytes(rows, cols); }
static MxMat mx_in(const uint8_t* q, int rows, int cols) {
  return {q, q + mx_code_bytes(rows, cols), rows, cols};
}
void mx_quantize_f32(hipStream_t st, const float* x, int rows, int cols, long long sr, long long sc,
                     uint8_t* q) {
  mx_quantize_launch(st, T_FP32, x, rows, cols, sr, sc, q, q + mx_code_bytes(rows, cols));
}
void mx_layer_f32(hipStream_t st, const float* x, int ldx, int M, int K, const uint8_t* w, int N,
                  const float* bias, int act, float* y, int ldy, uint8_t* xq, bool keep) {
  const MxOut o{y, bias, ldy, M, N, T_FP32, T_FP32, act};
  if (!keep && mx_rows_ok(M, K)) {
    mx_linear_rows_launch(st, T_FP32, x, ldx, 1, M, K, mx_in(w, N, K), o);
    return;
  }
  mx_quantize_f32(st, x, M, K, ldx, 1, xq);
  mx_linear_launch(st, mx_in(xq, M, K), mx_in(w, N, K), o);
}
size_t mx_layer_grad_ws(int M, int N, int K) {
  return mx_grad_plan(T_FP32, M, N, K, true, true, false).total;
}
void mx_layer_grad_f32(hipStream_t st, const float* dy, int lddy, int M, int N, int K,
                       const uint8_t* xq, const uint8_t* w, float* dx, float* dw, uint8_t* ws) {
  mx_linear_grad_launch(st, T_FP32, dy, lddy, 1, mx_in(xq, M, K), mx_in(w, N, K), dx, dw, nullptr,
                        ws);
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
    const unsigned tiles = grid_x((long long)ceil_div(q.rows, 64) * q.kt());
    by_dtype(dtype, [&](auto dt) {
      constexpr int DT = decltype(dt)::value;
      hipLaunchKernelGGL(mx_dequantize_kernel<DT>, dim3(tiles), dim3(256), 0,
                         static_cast<hipStream_t>(stream), q,
                         static_cast<typename Elem<DT>::type*>(out), (long long)row_stride);
    });
    HIP_TRY(hipGetLastError());
  });
}

size_t ddpg_mx_linear_workspace(int64_t M, int64_t K, int64_t N) {
  if (M < 0 || K < 0 || N < 0 || M > kMxMaxDim || K > kMxMaxDim || N > kMxMaxDim) return 0;
  return mx_rows_ok(M, K) ? 0 : mx_code_bytes(M, K) + mx_scale_bytes(M, K);
}

int ddpg_mx_linear(int device, void* stream, int x_dtype, const void* x, int64_t x_row_stride,
                   int64_t x_col_stride, const void* x_codes, const void* x_scales, int64_t M,
                   int64_t K, const void* w_codes, const void* w_scales, int64_t N, int bias_dtype,
                   const void* bias, int act, int dtype, void* y, int64_t y_row_stride, void* ws,
                   size_t ws_bytes) {
  return guard(nullptr, [&] {
    mx_check_dims("mx_linear x", M, K);
    const MxMat wq = mx_mat("mx_linear w", w_codes, w_scales, N, K);
    MxMat xq{nullptr, nullptr, (int)M, (int)K};
    check_dtype("mx_linear", dtype);
    if (bias) check_dtype("mx_linear bias", bias_dtype);
    if (act < DDPG_ACT_NONE || act > DDPG_ACT_TANH) throw einval("mx_linear: act %d", act);
    const bool rows = x && mx_rows_ok(M, K);
    if (!x) {
      xq = mx_mat("mx_linear x", x_codes, x_scales, M, K);
    } else {
      check_dtype("mx_linear x", x_dtype);
      const size_t need = rows ? 0 : mx_code_bytes(M, K) + mx_scale_bytes(M, K);
      if (ws_bytes < need || (need && !ws) || (need && !aligned16(ws)))
        throw einval("mx_linear: workspace of %zu bytes, %zu needed", ws_bytes, need);
    }
    if (!M || !N) return;
    if (!y) throw einval("mx_linear: null output");
    if (y_row_stride < N) throw einval("mx_linear: rows %lld apart overlap", (long long)y_row_stride);
    OnDevice on(device);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const MxOut o{y, bias, (long long)y_row_stride, (int)M, (int)N, dtype, bias_dtype, act};
    if (rows) {
      mx_linear_rows_launch(st, x_dtype, x, x_row_stride, x_col_stride, (int)M, (int)K, wq, o);
      return;
    }
    if (x) {
      uint8_t* codes = static_cast<uint8_t*>(ws);
      uint8_t* scales = codes + mx_code_bytes(M, K);
      mx_quantize_launch(st, x_dtype, x, (int)M, (int)K, x_row_stride, x_col_stride, codes, scales);
      xq.codes = codes;
      xq.scales = scales;
    }
    mx_linear_launch(st, xq, wq, o);
  });
}

size_t ddpg_mx_linear_grad_workspace(int dtype, int64_t M, int64_t N, int64_t K, int dx, int dw,
                                     int db) {
  if (M < 0 || N < 0 || K < 0 || M > kMxMaxDim || N > kMxMaxDim || K > kMxMaxDim) return 0;
  return mx_grad_plan(dtype, (int)M, (int)N, (int)K, dx != 0, dw != 0, db != 0).total;
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
    const size_t need = mx_grad_plan(dtype, (int)M, (int)N, (int)K, dx, dw, db).total;
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
