// Products of operands laid out in matrix-instruction order (gfx950):
//   C[i][j] = sum_k I[i][k] J[j][k]
// A fragment is 16 rows of one instruction's depth, 1 KiB, lane l's 16 bytes at
// 16 l: 128 MXFP4 columns (mx.h) or 32 bfloat16 columns (lane l: row l % 16,
// columns 8 (l / 16) ..).  An operand is [row groups of 16][depth steps][1 KiB],
// row groups padded to whole fours.  Both kinds take as many cycles per
// fragment pair (v_mfma_scale_f32_16x16x128_f8f6f4 on fp4, 4 times the rate of
// v_mfma_f32_16x16x32_bf16), so one kernel serves both.
//
// J is the instruction's first operand: lane l holds C[i = l % 16] of four
// consecutive j = 4 (l / 16) .. +3, which are adjacent in memory.
#pragma once
#include "gemm_h256.h"
#include "mx.h"

namespace ddpg {

// What becomes of C: y = act(C + bias), rounded once to dtype.
struct MxOut {
  void* y;
  const void* bias;
  long long ldo;
  int I, J, dtype, bias_dtype, act;
};

struct FragOp {
  const uint8_t* p;       // fragments
  const uint8_t* scales;  // mx.h's scales, or null
  int groups;             // 16-row groups held (a multiple of 4)
};

struct MxGemm {
  FragOp I, J;
  int kt;      // depth steps of J
  int planes;  // I holds `planes` times kt steps a row group; J's repeat
  MxOut o;
  // the depth in `splits` blocks a tile, joined in the launch (mx_join)
  int splits;
  float* slab;        // [tile][split][a block's sums]
  unsigned* tickets;  // [tile], zero before and after the launch
};

// One launch: n products (blocks 0 .. end[0] - 1, .. end[1] - 1), then 64 columns
// a block of a bias gradient's last sum.  A launch of fp4 is g[0] alone, so that its
// blocks take all arguments at fixed places, with one wait.
struct MxGemms {
  MxGemm g[2];
  int n, end[2];
  const float* db_part;  // [db_parts][db_n]
  float* db;
  int db_parts, db_n;
};

// g[0] or g[1], field by field: loaded at once from fixed places, then selected (a
// load from a selected address waits a second time for the arguments' memory).
template <bool FP4>
DDPG_DEV MxGemm mx_pick(const MxGemms& p, bool second) {
  if constexpr (FP4) return p.g[0];
  const MxGemm &a = p.g[0], &b = p.g[1];
  auto pick = [&](auto x, auto y) { return second ? y : x; };
  return {{pick(a.I.p, b.I.p), nullptr, pick(a.I.groups, b.I.groups)},
          {pick(a.J.p, b.J.p), nullptr, pick(a.J.groups, b.J.groups)},
          pick(a.kt, b.kt),
          a.planes,
          {pick(a.o.y, b.o.y), nullptr, a.o.ldo, pick(a.o.I, b.o.I), a.o.J,
           pick(a.o.dtype, b.o.dtype), 0, DDPG_ACT_NONE},
          pick(a.splits, b.splits),
          pick(a.slab, b.slab),
          pick(a.tickets, b.tickets)};
}

// tanh x = 1 - 2 / (e^2x + 1), which loses nothing from |x| = 0.5 on (error at most
// 2^-22, mostly the reciprocal's); below it x + x^3 p(x^2), p a cubic through the
// Chebyshev nodes of tanh's own on [0, 1/4] (within 2^-23 of the value).  No branches:
// lanes of both kinds share a wave (1000 x 777 x 1203 fp16: 8.2 us with the library's
// tanhf, 7.5 so).
DDPG_DEV float mx_tanh(float x) {
  const float a = fabsf(x), q = __fmul_rn(x, x);
  const float p =
      fmaf(fmaf(fmaf(0.01799921877f, q, -0.05339105427f), q, 0.1333051324f), q, -0.3333331048f);
  const float e = __builtin_amdgcn_exp2f(__fmul_rn(a, 2.885390082f));
  const float y = fmaf(-2.f, __builtin_amdgcn_rcpf(__fadd_rn(e, 1.f)), 1.f);
  return a < 0.5f ? fmaf(__fmul_rn(x, q), p, x) : copysignf(y, x);
}

// ELU, e^x - 1 below 0, for a float32 result.  The difference loses nothing up to x =
// -0.5 (2^-22 of the value at most, mostly the exponential's); above it cancels, down
// to 0 for |x| < 2^-25, so there x + x^2 p(x), p a quartic through the Chebyshev nodes of
// (e^x - 1 - x) / x^2 on [-0.5, 0] (within 2^-23 of the value).  No branches, as above.
DDPG_DEV float mx_elu(float x) {
  const float p = fmaf(
      fmaf(fmaf(fmaf(0.001164287f, x, 0.0082382215f), x, 0.04164993f), x, 0.16666563f), x, 0.5f);
  const float e = __fsub_rn(__builtin_amdgcn_exp2f(__fmul_rn(x, 1.44269504f)), 1.f);
  const float y = x > -0.5f ? fmaf(__fmul_rn(x, x), p, x) : e;
  return x < 0.f ? y : x;
}
// For a 16-bit result: x <= e^x - 1 <= x + x^2 / 2 below 0, and the upper bound is the
// value to x^2 / 6 of it.  With 2^-23 added the difference exceeds that bound where it
// cancels, |x| < 2^-6.6, and the bound is taken; elsewhere the 2^-23 is as little:
// within 2^-15.6 of the value.  v_minimum3 and v_maximum3 choose, keep a NaN, and 0 and x
// as the last bounds make it x from 0 on.  7 instructions, 13 above (8192 x 2048 x 2048
// bf16: 27.4 us with e^x - 1 alone, 28.9 so, 31.5 with the form above).
DDPG_DEV float mx_elu16(float x) {
  const float e = __fsub_rn(__builtin_amdgcn_exp2f(__fmul_rn(x, 1.44269504f)), 0.99999988f);
  const float u = __fmul_rn(x, fmaf(x, 0.5f, 1.f));
  return __builtin_elementwise_maximum(
      x, __builtin_elementwise_minimum(__builtin_elementwise_minimum(e, u), 0.f));
}

template <int N>
DDPG_DEV void mx_act(float (&v)[N], int act, bool fp32) {
  if (act == DDPG_ACT_ELU && fp32) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = mx_elu(v[k]);
  } else if (act == DDPG_ACT_ELU) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = mx_elu16(v[k]);
  } else if (act == DDPG_ACT_TANH) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = mx_tanh(v[k]);
  }
}

// C[i][j .. j+3] of a lane to the output; b: the four biases
DDPG_DEV void mx_store(const MxOut& o, int i, int j, const f32x4& d, const float* b) {
  if (i >= o.I || j >= o.J) return;
  float v[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = __fadd_rn(d[r], b[r]);
  mx_act(v, o.act, o.dtype == T_FP32);
  const long long at = i * o.ldo + j;
  if (j + 4 <= o.J) {  // one store, whatever the row's alignment
    by_dtype(o.dtype, [&](auto dt) {
      typedef typename Elem<decltype(dt)::value>::type T;
      typedef T any4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
      *reinterpret_cast<any4*>(static_cast<T*>(o.y) + at) =
          any4{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    });
    return;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (j + r < o.J) store_elem(o.y, o.dtype, at + r, v[r]);
}

// The biases of N columns from j on, as their bits: loaded first and converted
// last, so that nothing waits for them before the operands are on their way
// (columns past the last repeat its bias, and are not stored).
template <int N>
DDPG_DEV void mx_bias(const MxOut& o, int j, unsigned (&u)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) u[k] = 0;
  if (!o.bias) return;
  if (o.bias_dtype == T_FP32) {
#pragma unroll
    for (int k = 0; k < N; ++k) u[k] = static_cast<const unsigned*>(o.bias)[min(j + k, o.J - 1)];
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k)
      u[k] = static_cast<const unsigned short*>(o.bias)[min(j + k, o.J - 1)];
  }
}
template <int N>
DDPG_DEV void mx_bias_values(const MxOut& o, const unsigned (&u)[N], float (&b)[N]) {
  by_dtype(o.bias_dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
#pragma unroll
    for (int k = 0; k < N; ++k)
      b[k] = DT == T_FP32   ? __uint_as_float(u[k])
             : DT == T_BF16 ? __uint_as_float(u[k] << 16)
                            : (float)__builtin_bit_cast(_Float16, (unsigned short)u[k]);
  });
}

// A wave's TI x 4 fragments to the output by whole rows: 64 rows at a time go
// through 16 KiB of LDS of its own as the fp32 sums (16-byte units of a row
// swizzled by the row, free of bank conflicts), from where 8 lanes take a row's 64
// outputs, 8 each: bias, activation, one rounding, 16-byte stores.  Straight from
// the registers a store covers 32 bytes of a row (28 us a 256 x 256 tile).  The
// second half is a loop, not unrolled code: with the activations inlined at every
// fragment the code outgrew the instruction cache (fp4 8192 x 4096 x 4096 between other
// kernels: 92 us so, 75 as a loop).
template <int DT, int TI>
DDPG_DEV void mx_store_tile(const MxOut& o, lds_char* strip, int i0, int j0,
                            const f32x4 (&acc)[TI][4], const float (&b)[8]) {
  typedef typename Elem<DT>::type T;
  constexpr int V = Elem<DT>::V;
  typedef __attribute__((address_space(3))) f32x4 lds_v4f;
  const int lane = threadIdx.x & 63, q = lane & 7, col = j0 + 8 * q;
  auto at = [&](int r, int unit) { return (lds_v4f*)(strip + r * 256 + ((unit ^ r) & 15) * 16); };
  static_for<TI / 4>([&](auto h_c) {
    constexpr int h = decltype(h_c)::value;
    static_for<16>([&](auto f_c) {
      constexpr int i = decltype(f_c)::value / 4, j = decltype(f_c)::value % 4;
      *at(i * 16 + (lane & 15), j * 4 + (lane >> 4)) = acc[4 * h + i][j];
    });
    __builtin_amdgcn_wave_barrier();
#pragma unroll 1
    for (int it = 0; it < 8; ++it) {
      const int r = it * 8 + (lane >> 3), row = i0 + h * 64 + r;
      const f32x4 lo = *at(r, 2 * q), hi = *at(r, 2 * q + 1);
      if (row >= o.I || col >= o.J) continue;
      float v[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] = __fadd_rn(lo[k], b[k]);
        v[4 + k] = __fadd_rn(hi[k], b[4 + k]);
      }
      mx_act(v, o.act, DT == T_FP32);
      T* p = static_cast<T*>(o.y) + row * o.ldo + col;
      if (col + 8 <= o.J) {  // whatever the row's alignment
#pragma unroll
        for (int k = 0; k < 8; k += V) *reinterpret_cast<U16B*>(p + k) = Elem<DT>::pack(v + k);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (col + k < o.J) p[k] = (T)v[k];
      }
    }
    __builtin_amdgcn_wave_barrier();
  });
}

// acc[j + r][i] += J fragment x I fragment, with scale bytes BJ of sj, BI of si
template <bool FP4, int BJ, int BI>
DDPG_DEV f32x4 frag_mfma(const u32x4& j, const u32x4& i, f32x4 acc, unsigned sj, unsigned si) {
  if constexpr (FP4)
    return mx_mfma<BJ, BI>(j, i, acc, sj, si);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, j),
                                                   __builtin_bit_cast(bf16x8, i), acc, 0, 0, 0);
}

// db[n] = the sum of the row blocks' column sums, in float64: the launch's last
// blocks, 64 columns each, the waves taking partials in turn.
template <int NW>
DDPG_DEV void mx_db(const MxGemms& p, int b, double (&red)[NW][64]) {
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, n = b * 64 + l;
  double s = 0;
  if (n < p.db_n)
#pragma unroll 4
    for (int i = w; i < p.db_parts; i += NW) s += p.db_part[(size_t)i * p.db_n + n];
  red[w][l] = s;
  __syncthreads();
  if (w || n >= p.db_n) return;
  for (int i = 1; i < NW; ++i) s += red[i][l];
  p.db[n] = (float)s;
}

// Tile `lin` of a product.  The grid is one-dimensional: every XCD (workgroups are
// dealt to the 8 in turn) takes a contiguous run of the order, which walks
// eight rows of tiles down before it steps across, so that the tiles an XCD
// works on at once share their operands in its L2.
DDPG_DEV void tile_of(int lin, int ni, int nj, int& ti, int& tj) {
  const unsigned n = ni * nj;
  const unsigned x = lin & 7, q = n >> 3, r = n & 7;
  const unsigned t = x * q + min(x, r) + ((unsigned)lin >> 3);
  const unsigned band = t / (8u * nj), in = t - band * 8 * nj;
  const unsigned rows = min(8u, ni - band * 8), d = in / rows;
  ti = band * 8 + in - d * rows;
  tj = d;
}

// Which of a product's blocks this is: tile, split and its depth steps.
struct MxPart {
  int ti, tj, tile, split, k0, n;
};
template <bool FP4, int BI, int BJ>
DDPG_DEV MxPart mx_part(const MxGemm& g, unsigned lin) {
  const unsigned ni = (unsigned)(g.o.I + BI - 1) / BI, nj = (unsigned)(g.o.J + BJ - 1) / BJ;
  MxPart p;
  p.split = p.k0 = 0;
  p.n = g.kt * g.planes;
  if (!FP4 && g.splits > 1) {  // at most 32, of at most 3 * 2^19 steps
    const unsigned nk = p.n;
    p.split = lin / (ni * nj);
    lin -= p.split * ni * nj;
    p.k0 = nk * p.split / g.splits;
    p.n = nk * (p.split + 1) / g.splits - p.k0;
  }
  tile_of(lin, ni, nj, p.ti, p.tj);
  p.tile = p.ti * nj + p.tj;
  return p;
}

// The blocks of a tile store their sums (lane after lane, 16 bytes each) past the
// XCDs' separate L2s (sc1), wait for the stores, and one thread takes a ticket;
// the block with the last ticket adds the splits' sums in split order, so the
// result does not depend on which came last, and puts the ticket back to zero.
// True in that block.  NF f32x4 a thread; threads `on` take part.
template <int NF>
DDPG_DEV bool mx_join(const MxGemm& g, const MxPart& p, f32x4* acc, int thread, int threads,
                      bool on) {
  __shared__ unsigned last;
  const unsigned bytes = (unsigned)(NF * threads * 16);  // a block's sums
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(reinterpret_cast<char*>(g.slab) + (size_t)p.tile * g.splits * bytes), 0, 0x7fffffff,
      0x00020000);
  if (on)
#pragma unroll
    for (int f = 0; f < NF; ++f)
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, acc[f]), rs,
                                             p.split * bytes + (f * threads + thread) * 16, 0,
                                             KC_SC1);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's sums have left
  __syncthreads();
  if (threadIdx.x == 0) {
    const unsigned was =
        __hip_atomic_fetch_add(g.tickets + p.tile, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = was == (unsigned)(g.splits - 1);
    if (last)
      __hip_atomic_store(g.tickets + p.tile, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last) return false;
  if (on) {
#pragma unroll
    for (int f = 0; f < NF; ++f) acc[f] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < g.splits; ++s)
#pragma unroll
      for (int f = 0; f < NF; ++f)
        acc[f] += __builtin_bit_cast(
            f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                       rs, s * bytes + (f * threads + thread) * 16, 0, KC_SC1));
  }
  return true;
}

// ---------------------------------------------------------------- LDS tiles
template <int OFF>
DDPG_DEV u32x4 lds_b128(unsigned a) {
  u32x4 r;
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(r) : "v"(a), "n"(OFF));
  return r;
}
template <int OFF>
DDPG_DEV unsigned lds_b32(unsigned a) {
  unsigned r;
  asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(r) : "v"(a), "n"(OFF));
  return r;
}

// 16 (4) bytes a lane from memory to LDS, lane after lane.  A plain function: in
// a kernel template the builtin keeps hipcc from emitting the launch stub.
DDPG_DEV void lds_load16(const uint8_t* p, lds_char* to) {
  __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)p, (lds_void*)to, 16, 0,
                                   0);
}
DDPG_DEV void lds_load4(const uint8_t* p, lds_char* to) {
  __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)p, (lds_void*)to, 4, 0,
                                   0);
}

// WI x WJ waves of TI x TJ fragments each, a ring of NS depth steps in LDS.
template <bool FP4, int WI, int WJ, int TI, int TJ, int NS>
struct RingCfg {
  static constexpr int NW = WI * WJ, NT = 64 * NW;
  static constexpr int GI = WI * TI, GJ = WJ * TJ;  // fragments of a step
  static constexpr int PW = (GI + GJ) / NW;         // of them loaded by a wave
  static constexpr int SP = FP4 ? (GI + GJ) / 4 : 0;  // 256-byte scale pieces
  static constexpr int SW = SP / NW;
  static constexpr int SLOT = (GI + GJ) * 1024 + SP * 256;
  static constexpr int LDS = NS * SLOT;
  static_assert(PW * NW == GI + GJ && SW * NW == SP && TI % 4 == 0 && TJ % 4 == 0, "whole pieces");
  static_assert(GI % PW == 0 && (!FP4 || PW == 4 * SW), "a wave's pieces are of one operand");
  static_assert(TJ == 4 && LDS >= NW * 16384, "mx_store_tile");
  static_assert(LDS <= 160 * 1024, "LDS");
  static_assert((GI + GJ) * 1024 + SP * 256 < 65536, "LDS offsets are immediates");
};

// Depth steps s .. s + NS - 1 are in LDS or on their way (global_load_lds, 16
// bytes a lane) while the wave multiplies step s from registers.  Per step: wait
// for the own loads of s + 1; one barrier (so s + 1 is whole and nobody reads s
// any more); then the products, with the LDS reads of s + 1 and the loads of
// s + NS between them; wait for the reads.  An I fragment's registers are
// refilled after its last use, the J fragments, the last I fragment and the
// scales have two sets.  The LDS reads are inline asm because the compiler would
// drain the loads in flight before reads of its own; the wait that ends the step
// is tied to their registers, so none is touched while a read is under way.
template <bool FP4, int WI, int WJ, int TI, int TJ, int NS>
__global__ __launch_bounds__(64 * WI * WJ) void mx_tile_kernel(MxGemms p) {
  using C = RingCfg<FP4, WI, WJ, TI, TJ, NS>;
  __shared__ __attribute__((aligned(1024))) char smem[C::LDS];
  if (!FP4 && (int)blockIdx.x >= p.end[1]) {
    mx_db<C::NW>(p, blockIdx.x - p.end[1], *reinterpret_cast<double(*)[C::NW][64]>(smem));
    return;
  }
  const bool second = !FP4 && (int)blockIdx.x >= p.end[0];
  const MxGemm g = mx_pick<FP4>(p, second);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave / WJ, wj = wave % WJ;
  const MxPart pt =
      mx_part<FP4, C::GI * 16, C::GJ * 16>(g, blockIdx.x - (second ? p.end[0] : 0));
  const int ti = pt.ti, tj = pt.tj, nk = pt.n;
  // J's depth step of the next load (I's planes go on, J's repeat)
  int jk = FP4 ? 0 : (unsigned)pt.k0 % max((unsigned)g.kt, 1u);

  // this wave's pieces of a step: source of the next step to load, LDS place.
  // The sources are the same for all lanes (scalar registers, scalar adds), a
  // lane's place in a piece is its own.
  // Row groups past the operand's last are read from the last one's place
  // (their results are not stored).
  const bool isj = wave >= C::GI / C::PW;  // a wave's pieces are of one operand
  const FragOp& op = isj ? g.J : g.I;
  const uint8_t* src[C::PW];
  const uint8_t* ssrc[C::SW + 1];
  {
    const int g0 = isj ? tj * C::GJ - C::GI + wave * C::PW : ti * C::GI + wave * C::PW;
    const size_t pitch = (size_t)g.kt * (isj ? 1 : g.planes) * 1024;
    const uint8_t* at = op.p + (size_t)(isj ? jk : pt.k0) * 1024;
#pragma unroll
    for (int p = 0; p < C::PW; ++p) src[p] = at + min(g0 + p, op.groups - 1) * pitch;
    const int s0 = isj ? (tj * C::GJ - C::GI) / 4 + wave * C::SW : ti * (C::GI / 4) + wave * C::SW;
#pragma unroll
    for (int p = 0; p < C::SW; ++p)
      ssrc[p] = op.scales + (size_t)min(s0 + p, op.groups / 4 - 1) * g.kt * 256;
  }
  lds_char* const base = (lds_char*)smem;
  const unsigned l16 = lane * 16, l4 = lane * 4;
  auto load_piece = [&](int slot, auto p_c) {
    constexpr int p = decltype(p_c)::value;
    if constexpr (p < C::PW) {
      lds_load16(src[p] + l16, base + slot * C::SLOT + (wave * C::PW + p) * 1024);
      src[p] += 1024;
      if (!FP4 && isj && jk + 1 == g.kt) src[p] -= (size_t)g.kt * 1024;
    } else {
      constexpr int q = p - C::PW;
      lds_load4(ssrc[q] + l4,
                base + slot * C::SLOT + (C::GI + C::GJ) * 1024 + (wave * C::SW + q) * 256);
      ssrc[q] += 256;
    }
    if constexpr (p == C::PW + C::SW - 1) jk = jk + 1 == g.kt ? 0 : jk + 1;
  };
  constexpr int G = C::PW + C::SW;
  constexpr int NM = TI * TJ;
  static_assert(NM >= TJ + 1 + G && NM >= 2 * TJ, "gaps for the loads and the reads");

  unsigned bias[8] = {};  // of the columns this lane will store (a gradient has none)
  if (FP4) mx_bias(g.o, (tj * C::GJ + wj * TJ) * 16 + 8 * (lane & 7), bias);
  f32x4 acc[TI][TJ];
  static_for<TI * TJ>([&](auto q) {
    acc[decltype(q)::value / TJ][decltype(q)::value % TJ] = f32x4{0.f, 0.f, 0.f, 0.f};
  });

  if (nk > 0) {
    u32x4 fi[TI], fl[2], fj[2][TJ];  // fi[TI - 1] is fl
    unsigned si[2][TI / 4] = {}, sj[2][TJ / 4] = {};
    const unsigned lb = (unsigned)(uintptr_t)base;
    const unsigned bi = lb + lane * 16 + wi * TI * 1024;
    const unsigned bj = lb + lane * 16 + (C::GI + wj * TJ) * 1024;
    const unsigned bs = lb + lane * 4 + (C::GI + C::GJ) * 1024;
    const unsigned bsi = bs + wi * (TI / 4) * 256;
    const unsigned bsj = bs + (C::GI / 4 + wj * (TJ / 4)) * 256;
    auto read_i = [&](auto set_c, auto i_c, unsigned so) {
      constexpr int set = decltype(set_c)::value, i = decltype(i_c)::value;
      (i == TI - 1 ? fl[set] : fi[i]) = lds_b128<i * 1024>(bi + so);
    };
    auto read_j = [&](auto set_c, auto j_c, unsigned so) {
      constexpr int set = decltype(set_c)::value, j = decltype(j_c)::value;
      fj[set][j] = lds_b128<j * 1024>(bj + so);
    };
    auto read_s = [&](auto set_c, unsigned so) {
      constexpr int set = decltype(set_c)::value;
      if constexpr (FP4) {
        static_for<TI / 4>([&](auto c) { si[set][decltype(c)::value] = lds_b32<decltype(c)::value * 256>(bsi + so); });
        static_for<TJ / 4>([&](auto c) { sj[set][decltype(c)::value] = lds_b32<decltype(c)::value * 256>(bsj + so); });
      }
    };
    // the reads issued so far have landed in set `set`
    auto landed = [&](auto set_c) {
      constexpr int set = decltype(set_c)::value;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int i = 0; i < TI - 1; ++i) asm volatile("" : "+v"(fi[i]));
      asm volatile("" : "+v"(fl[set]));
#pragma unroll
      for (int j = 0; j < TJ; ++j) asm volatile("" : "+v"(fj[set][j]));
      if constexpr (FP4) {
#pragma unroll
        for (int i = 0; i < TI / 4; ++i) asm volatile("" : "+v"(si[set][i]));
#pragma unroll
        for (int j = 0; j < TJ / 4; ++j) asm volatile("" : "+v"(sj[set][j]));
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    // one step from register set SET.  RT: near the end, where step s + 1 or
    // s + NS may not exist
    auto step = [&](int s, auto set_c, auto rt_c) {
      constexpr int SET = decltype(set_c)::value;
      constexpr bool RT = decltype(rt_c)::value;
      using Other = std::integral_constant<int, SET ^ 1>;
      const bool next = true, stage = !RT || s + NS < nk;
      if (RT && s + NS > nk)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      else
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 2) * G) : "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      const unsigned so = (unsigned)((s + 1) % NS) * C::SLOT;
      const int slot = s % NS;
      static_for<NM>([&](auto q_c) {
        constexpr int q = decltype(q_c)::value, i = q / TJ, j = q % TJ;
        acc[i][j] = frag_mfma<FP4, j % 4, i % 4>(fj[SET][j], i == TI - 1 ? fl[SET] : fi[i], acc[i][j],
                                                 sj[SET][j / 4], si[SET][i / 4]);
        if (next) {
          if constexpr (q < TJ) read_j(Other{}, q_c, so);
          if constexpr (q == TJ - 1) read_i(Other{}, std::integral_constant<int, TI - 1>{}, so);
          if constexpr (q == TJ) read_s(Other{}, so);
          if constexpr (i >= 1 && j == 0) read_i(Other{}, std::integral_constant<int, i - 1>{}, so);
        }
        constexpr int gap = (NM - TJ - 1) / G;
        if constexpr (q > TJ && (q - TJ - 1) % gap == 0 && (q - TJ - 1) / gap < G)
          if (stage) load_piece(slot, std::integral_constant<int, (q - TJ - 1) / gap>{});
        __builtin_amdgcn_sched_barrier(0);
      });
      landed(Other{});
    };
    // the first NS steps on their way, step 0 landed, its fragments read
    for (int s = 0; s < NS && s < nk; ++s)
      static_for<G>([&](auto p_c) { load_piece(s, p_c); });
    if (nk >= NS)
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 1) * G) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    using S0 = std::integral_constant<int, 0>;
    using S1 = std::integral_constant<int, 1>;
    static_for<TI>([&](auto c) { read_i(S0{}, c, 0u); });
    static_for<TJ>([&](auto c) { read_j(S0{}, c, 0u); });
    read_s(S0{}, 0u);
    landed(S0{});
    int s = 0;
    for (; s + 1 + NS < nk; s += 2) {
      step(s, S0{}, std::false_type{});
      step(s + 1, S1{}, std::false_type{});
    }
    for (; s < nk; s += 2) {
      step(s, S0{}, std::true_type{});
      if (s + 1 < nk) step(s + 1, S1{}, std::true_type{});
    }
  }
  if (!FP4 && g.splits > 1 && !mx_join<TI * TJ>(g, pt, &acc[0][0], threadIdx.x, C::NT, true))
    return;
  float b[8];
  mx_bias_values(g.o, bias, b);
  __syncthreads();  // the ring is done with: it carries the results out
  by_dtype(g.o.dtype, [&](auto dt) {
    mx_store_tile<decltype(dt)::value, TI>(g.o, base + wave * 16384, (ti * C::GI + wi * TI) * 16,
                                           (tj * C::GJ + wj * TJ) * 16, acc, b);
  });
}

// ---------------------------------------------------------------- few tiles
// One block: TI x TJ fragments of C, its NW waves taking every NW-th of the
// block's depth steps with operands straight from memory, PF steps ahead; the
// waves' sums are joined in LDS in wave order.
template <bool FP4, int TI, int TJ, int NW, int PF>
__global__ __launch_bounds__(64 * NW) void mx_split_kernel(MxGemms p) {
  __shared__ f32x4 part[NW][TI * TJ][64];
  static_assert(TI * TJ < NW || TI * TJ % NW == 0, "whole fragments a wave");
  if (!FP4 && (int)blockIdx.x >= p.end[1]) {
    mx_db<NW>(p, blockIdx.x - p.end[1], *reinterpret_cast<double(*)[NW][64]>(part));
    return;
  }
  const bool second = !FP4 && (int)blockIdx.x >= p.end[0];
  const MxGemm g = mx_pick<FP4>(p, second);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const MxPart pt = mx_part<FP4, TI * 16, TJ * 16>(g, blockIdx.x - (second ? p.end[0] : 0));
  const int nk = pt.n;
  f32x4 acc[TI][TJ];
#pragma unroll
  for (int i = 0; i < TI; ++i)
#pragma unroll
    for (int j = 0; j < TJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  // the fragments' scales are adjacent bytes of one dword (TI, TJ: 2 or 4)
  const int gi = pt.ti * TI, gj = pt.tj * TJ;
  // the fragments a wave stores have one column group: its biases, loaded early
  static_assert(NW % TJ == 0, "a wave's fragments share their columns");
  const int jj = (gj + wave % TJ) * 16 + (lane >> 4) * 4;
  unsigned bias[4] = {};
  if (FP4) mx_bias(g.o, jj, bias);
  const uint8_t *pi[TI], *pj[TJ];
#pragma unroll
  for (int i = 0; i < TI; ++i)
    pi[i] = g.I.p + ((size_t)min(gi + i, g.I.groups - 1) * g.kt * g.planes + pt.k0) * 1024 + lane * 16;
#pragma unroll
  for (int j = 0; j < TJ; ++j)
    pj[j] = g.J.p + (size_t)min(gj + j, g.J.groups - 1) * g.kt * 1024 + lane * 16;
  const uint8_t* qi = FP4 ? g.I.scales + (size_t)(gi >> 2) * g.kt * 256 + lane * 4 : nullptr;
  const uint8_t* qj = FP4 ? g.J.scales + (size_t)(gj >> 2) * g.kt * 256 + lane * 4 : nullptr;
  struct Step {
    u32x4 i[TI], j[TJ];
    unsigned si, sj;
  };
  auto load = [&](int s, Step& f) {
    const int k = FP4 ? s : (s + pt.k0) % g.kt;
#pragma unroll
    for (int i = 0; i < TI; ++i) f.i[i] = *reinterpret_cast<const u32x4*>(pi[i] + (size_t)s * 1024);
#pragma unroll
    for (int j = 0; j < TJ; ++j) f.j[j] = *reinterpret_cast<const u32x4*>(pj[j] + (size_t)k * 1024);
    f.si = f.sj = 0;
    if constexpr (FP4) {
      f.si = *reinterpret_cast<const unsigned*>(qi + (size_t)k * 256) >> (8 * (gi & 3));
      f.sj = *reinterpret_cast<const unsigned*>(qj + (size_t)k * 256) >> (8 * (gj & 3));
    }
  };
  {
    Step f[PF];
    static_for<PF>([&](auto u) {
      constexpr int U = decltype(u)::value;
      if (wave + U * NW < nk) load(wave + U * NW, f[U]);
    });
    for (int s = wave; s < nk; s += PF * NW)
      static_for<PF>([&](auto u) {
        constexpr int U = decltype(u)::value;
        if (s + U * NW < nk) {
          static_for<TI * TJ>([&](auto q_c) {
            constexpr int i = decltype(q_c)::value / TJ, j = decltype(q_c)::value % TJ;
            acc[i][j] = frag_mfma<FP4, j, i>(f[U].j[j], f[U].i[i], acc[i][j], f[U].sj, f[U].si);
          });
          if (s + (U + PF) * NW < nk) load(s + (U + PF) * NW, f[U]);
        }
      });
  }
#pragma unroll
  for (int i = 0; i < TI; ++i)
#pragma unroll
    for (int j = 0; j < TJ; ++j) part[wave][i * TJ + j][lane] = acc[i][j];
  __syncthreads();
  // fragments wave, wave + NW ..: at most NF a wave
  constexpr int NF = (TI * TJ + NW - 1) / NW;
  constexpr int ON = TI * TJ < NW ? TI * TJ : NW;  // waves with a fragment
  const bool on = wave < TI * TJ;
  int parts = NW;
  if (!FP4 && g.splits > 1) {  // this block's sums joined with the other splits'
    f32x4 sum[NF];
#pragma unroll
    for (int q = 0; q < NF; ++q) {
      const int f = min(wave + q * NW, TI * TJ - 1);
      sum[q] = part[0][f][lane];
#pragma unroll
      for (int w = 1; w < NW; ++w) sum[q] += part[w][f][lane];
    }
    if (!mx_join<NF>(g, pt, sum, threadIdx.x, ON * 64, on)) return;
    if (on)
#pragma unroll
      for (int q = 0; q < NF; ++q) part[0][wave + q * NW][lane] = sum[q];
    parts = 1;
  }
  float b[4];
  mx_bias_values(g.o, bias, b);
  // a loop: unrolled, the activations' code would not stay in the cache
#pragma unroll 1
  for (int f = wave; f < TI * TJ; f += NW) {
    const int i = f / TJ;
    f32x4 sum = part[0][f][lane];
    for (int w = 1; w < parts; ++w) sum += part[w][f][lane];
    mx_store(g.o, (gi + i) * 16 + (lane & 15), jj, sum, b);
  }
}

// Rows of x as they are: the block's products quantise them on their way to the
// registers (each block again: x is small and stays in the caches, and a launch
// is saved).
struct RawX {
  const void* p;
  long long sr, sc;
  int rows, cols;
  int vec;  // columns adjacent
};

// NT: past the caches
template <int DT, bool NT = false>
DDPG_DEV void mx_load_block(const typename Elem<DT>::type* p, long long sc, bool adjacent, int c0,
                            int cols, float (&v)[32]) {
  if (adjacent && c0 + 32 <= cols) {
    constexpr int V = Elem<DT>::V;
#pragma unroll
    for (int i = 0; i < 32; i += V)
      Elem<DT>::widen(*reinterpret_cast<const U16B*>(p + c0 + i), v + i);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const typename Elem<DT>::type* q = p + min(c0 + i, cols - 1) * sc;
      v[i] = (float)(NT ? __builtin_nontemporal_load(q) : *q);
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = c0 + i < cols ? v[i] : 0.f;
  }
}

// y = act(x w^T + b) for at most 16 TI rows: a block makes 16 columns, its waves
// taking every NW-th depth step, the sums joined in wave order.  Bound: latency
// (one row, 1024 x 1024: 4.0 us with the launch; 7.9 as two launches).
template <int DT, int TI, int NW>
__global__ __launch_bounds__(64 * NW) void mx_rows_kernel(RawX x, FragOp w, int kt, MxOut o) {
  __shared__ f32x4 part[NW][TI][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, gj = blockIdx.x;
  typedef typename Elem<DT>::type T;
  // rows past x's repeat its last one, their results are not stored
  const T* xp[TI];
#pragma unroll
  for (int i = 0; i < TI; ++i)
    xp[i] = static_cast<const T*>(x.p) + min(i * 16 + (lane & 15), x.rows - 1) * x.sr;
  const uint8_t* pj = w.p + (size_t)gj * kt * 1024 + lane * 16;
  const uint8_t* qj = w.scales + (size_t)(gj >> 2) * kt * 256 + lane * 4 + (gj & 3);
  const int jj = gj * 16 + (lane >> 4) * 4;
  unsigned bias[4];
  mx_bias(o, jj, bias);
  f32x4 acc[TI];
#pragma unroll
  for (int i = 0; i < TI; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  // U steps at a time, so that their loads overlap (the last may repeat a step,
  // whose product is left out)
  constexpr int U = TI == 1 ? 2 : 1;
  for (int s0 = wave; s0 < kt; s0 += U * NW) {
    u32x4 j[U];
    unsigned sj[U];
    float v[U][TI][32];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = min(s0 + u * NW, kt - 1);
      j[u] = *reinterpret_cast<const u32x4*>(pj + (size_t)s * 1024);
      sj[u] = qj[(size_t)s * 256];
#pragma unroll
      for (int i = 0; i < TI; ++i)
        mx_load_block<DT>(xp[i], x.sc, x.vec, s * 128 + (lane >> 4) * 32, x.cols, v[u][i]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s0 + u * NW < kt)
#pragma unroll
        for (int i = 0; i < TI; ++i) {
          unsigned si;
          const u32x4 q = mx_quantize_block(v[u][i], si);
          acc[i] = mx_mfma<0, 0>(j[u], q, acc[i], sj[u], si);
        }
  }
#pragma unroll
  for (int i = 0; i < TI; ++i) part[wave][i][lane] = acc[i];
  __syncthreads();
  if (wave >= TI) return;
  f32x4 sum = part[0][wave][lane];
#pragma unroll
  for (int s = 1; s < NW; ++s) sum += part[s][wave][lane];
  float b[4];
  mx_bias_values(o, bias, b);
  mx_store(o, wave * 16 + (lane & 15), jj, sum, b);
}

}  // namespace ddpg
