// The global norm over a list of tensors and the clip by it
// (tf.global_norm / tf.clip_by_global_norm: what stands between
// compute_gradients and apply_gradients in a TF learner).
//   n = sqrt(sum_t sum_i x_t[i]^2),   y = x * s,   s = n <= c ? 1 : c / n
// The sum runs in float64: no square of a float32 leaves its range there, and
// the order of the sum does not show in the rounded result.  Nothing is added
// atomically: a block's partial sum goes to its own workspace slot and the
// slots are summed in order, so equal calls give equal bits.
// Bound: bytes (97 M bf16 values: 31 us, 6.2 TB/s); few or small tensors: launches
// (13 gradients of the default networks 3.6 + 1.7 us).  The tensors' table travels
// in the kernel's arguments.
#include "tensor_ops.h"

namespace ddpg {

constexpr int GN_MAXT = 96;         // tensors per launch (4 KiB of kernel arguments)
constexpr int GN_MAXB = 2048;       // blocks (= partial sums) per launch: 8 per CU
constexpr int GN_T = 256;           // threads of a block
constexpr int GN_CHUNK = GN_T * 64; // bytes of a tensor a block takes at a time

struct GnEntry {
  const void* src;
  void* dst;
  long long n;   // elements
  long long ld;  // strided: elements between rows
  int cols;      // strided: elements of a row; 0: dense
  int chunk0;    // first of the launch's chunks in this tensor
};
struct GnTable {
  GnEntry e[GN_MAXT];
  unsigned char dtype[GN_MAXT];
  int nt, nchunks;
  int keep;  // chunks from here on are read again: left in the caches
};

// element i of a tensor (its rows one after the other)
DDPG_DEV long long gn_at(const GnEntry& e, long long i) {
  if (!e.cols) return i;
  const long long r = i / e.cols;
  return r * e.ld + (i - r * e.cols);
}

DDPG_DEV double block_sum(double v, double* red) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0;
#pragma unroll
  for (int w = 0; w < GN_T / 64; ++w) s += red[w];
  return s;
}

// The launch's chunks dealt to its blocks in turn; f(IntC<dtype>, entry, first
// element, elements) for each.
// REV: from the last chunk down.  The tensor of a chunk is found by all lanes at
// once: as many tensors begin at or before it as lanes vote for.
template <bool REV, class F>
DDPG_DEV void gn_chunks(const GnTable& t, F&& f) {
  const int l = threadIdx.x & 63;
  const int c0 = l < t.nt ? t.e[l].chunk0 : INT32_MAX;
  const int c1 = l + 64 < t.nt ? t.e[min(l + 64, GN_MAXT - 1)].chunk0 : INT32_MAX;
  for (int b = blockIdx.x; b < t.nchunks; b += gridDim.x) {
    const int c = REV ? t.nchunks - 1 - b : b;
    const int e = __popcll(__ballot(c0 <= c)) + __popcll(__ballot(c1 <= c)) - 1;
    by_dtype(t.dtype[e], [&](auto dt) {
      constexpr int per = GN_CHUNK / sizeof(typename Elem<dt.value>::type);
      const long long i0 = (long long)(c - t.e[e].chunk0) * per;
      const long long left = t.e[e].n - i0;
      f(dt, t.e[e], i0, left < per ? (int)left : per, c);
    });
  }
}

__global__ __launch_bounds__(GN_T) void gn_partial_kernel(GnTable t, double* part) {
  __shared__ double red[GN_T / 64];
  double s = 0;
  gn_chunks<false>(t, [&](auto dt, const GnEntry& e, long long i0, int n, int c) {
    typedef Elem<dt.value> E;
    constexpr int V = E::V;
    const typename E::type* src = static_cast<const typename E::type*>(e.src);
    const bool vec = !e.cols || e.cols % V == 0;
    auto whole = [&](auto nt) {
#pragma unroll 4
      for (int i = threadIdx.x * V; i + V <= n; i += GN_T * V) {
        float x[V];
        E::widen(load16<decltype(nt)::value>(src + gn_at(e, i0 + i)), x);
#pragma unroll
        for (int k = 0; k < V; ++k) s = fma((double)x[k], (double)x[k], s);
      }
    };
    if (vec && c < t.keep)
      whole(std::true_type{});
    else if (vec)
      whole(std::false_type{});
    // the elements behind the last whole vector, or all of them
    for (int j = vec ? n / V * V + (int)threadIdx.x : (int)threadIdx.x; j < n; j += GN_T) {
      const double x = (double)(float)src[gn_at(e, i0 + j)];
      s = fma(x, x, s);
    }
  });
  const double b = block_sum(s, red);
  if (threadIdx.x == 0) part[blockIdx.x] = b;
}

// Every block sums all partials, in the same order.
DDPG_DEV double gn_total(const double* part, int np, double* red) {
  double s = 0;
  for (int i = threadIdx.x; i < np; i += GN_T) s += part[i];
  return sqrt(block_sum(s, red));
}

// NaN stays NaN, an infinite norm leaves 0
DDPG_DEV double gn_factor(double n, float clip) {
  return n <= (double)clip ? 1.0 : (double)clip / n;
}

// scale (optional): the clip's factor beside the norm
__global__ __launch_bounds__(GN_T) void gn_norm_kernel(const double* part, int np, float* norm,
                                                       float clip, float* scale) {
  __shared__ double red[GN_T / 64];
  const double n = gn_total(part, np, red);
  if (threadIdx.x == 0) {
    *norm = (float)n;
    if (scale) *scale = (float)gn_factor(n, clip);
  }
}

// y = x * s in float64, rounded to float32 and from there to a 16-bit type: off by
// at most half a step of the type and 2^-24 of the value.  given: the norm to use
// instead of the partial sums' (use_norm).
__global__ __launch_bounds__(GN_T) void gn_scale_kernel(GnTable t, const double* part, int np,
                                                        const float* given, float clip,
                                                        float* norm) {
  __shared__ double red[GN_T / 64];
  const double n = given ? (double)*given : gn_total(part, np, red);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
  const double s = gn_factor(n, clip);
  gn_chunks<true>(t, [&](auto dt, const GnEntry& e, long long i0, int m, int c) {
    typedef Elem<dt.value> E;
    constexpr int V = E::V;
    const typename E::type* src = static_cast<const typename E::type*>(e.src);
    typename E::type* dst = static_cast<typename E::type*>(e.dst);
    // in place the destination has the source's rows, one of its own is dense
    const bool same = src == dst;
    if (same && s == 1.0) return;  // nothing changes
    const bool vec = !e.cols || e.cols % V == 0;
    if (vec)
#pragma unroll 4
      for (int i = threadIdx.x * V; i + V <= m; i += GN_T * V) {
        const long long at = gn_at(e, i0 + i);
        float x[V];
        E::widen(load16<false>(src + at), x);
#pragma unroll
        for (int k = 0; k < V; ++k) x[k] = (float)((double)x[k] * s);
        store16_nt(dst + (same ? at : i0 + i), E::pack(x));
      }
    for (int j = vec ? m / V * V + (int)threadIdx.x : (int)threadIdx.x; j < m; j += GN_T) {
      const long long at = gn_at(e, i0 + j);
      dst[same ? at : i0 + j] = (typename E::type)(float)((double)(float)src[at] * s);
    }
  });
}

struct GnList {
  int n;
  const int* dtype;
  const void* const* src;
  void* const* dst;
  const int64_t *count, *cols, *ld;
};

static void gn_check(const GnList& l) {
  if (l.n < 0) throw einval("tensor list of length %d", l.n);
  if (l.n && (!l.dtype || !l.src || !l.count)) throw einval("tensor list: null array");
  if (!l.cols != !l.ld) throw einval("tensor list: cols and ld go together");
  for (int i = 0; i < l.n; ++i) {
    check_dtype("tensor list", l.dtype[i]);
    if (l.count[i] < 0 || l.count[i] > (1ll << 42))
      throw einval("tensor %d: %lld elements", i, (long long)l.count[i]);
    if (l.count[i] && (!l.src[i] || (l.dst && !l.dst[i]))) throw einval("tensor %d: null", i);
    if (l.cols && l.cols[i]) {
      if (l.cols[i] < 1 || l.cols[i] > INT32_MAX || l.ld[i] < 0 || l.count[i] % l.cols[i] ||
          l.ld[i] > (1ll << 56) / std::max<int64_t>(1, l.count[i] / l.cols[i]))
        throw einval("tensor %d: rows of %lld, %lld apart, %lld elements", i,
                     (long long)l.cols[i], (long long)l.ld[i], (long long)l.count[i]);
    }
  }
}

// In place: no element may belong to two entries (it would be scaled twice, or by
// two blocks at once), nor to one and another's input or output.  Rows of
// different column ranges of one matrix interleave without touching; anything else
// that meets is refused.
static void gn_check_disjoint(const GnList& l, const float* use_norm) {
  struct Range {
    uintptr_t lo, hi;
    int i;
    bool write;
    int64_t row, pitch;  // bytes; row 0: dense
  };
  std::vector<Range> r;
  auto add = [&](const void* at, int i, bool write, bool rows) {
    const int64_t es = elem_size(l.dtype[i]), cols = rows && l.cols ? l.cols[i] : 0;
    const int64_t n = cols ? l.count[i] / cols : 1, ld = cols ? l.ld[i] : 0;
    if (write && n > 1 && ld < cols) throw einval("tensor %d overlaps itself", i);
    const int64_t span = cols ? (n - 1) * ld + cols : l.count[i];
    const uintptr_t p = (uintptr_t)at;
    r.push_back({p, p + (uintptr_t)(span * es), i, write, cols * es, ld * es});
    const uintptr_t u = (uintptr_t)use_norm;  // read while the list is written
    if (write && u && u + sizeof(float) > r.back().lo && u < r.back().hi)
      throw einval("use_norm lies in tensor %d, which is clipped in place", i);
  };
  for (int i = 0; i < l.n; ++i) {
    if (!l.count[i]) continue;
    const bool same = l.src[i] == l.dst[i];
    add(l.dst[i], i, true, same);  // a destination of its own is dense
    if (!same) add(l.src[i], i, false, true);
  }
  std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.lo < b.lo; });
  for (size_t a = 0; a < r.size(); ++a)
    for (size_t b = a + 1; b < r.size() && r[b].lo < r[a].hi; ++b) {
      if (!r[a].write && !r[b].write) continue;
      bool apart = false;
      if (r[a].row && r[b].row && r[a].pitch && r[a].pitch == r[b].pitch) {
        const int64_t at = (int64_t)((r[b].lo - r[a].lo) % (uintptr_t)r[a].pitch);
        apart = at >= r[a].row && at + r[b].row <= r[a].pitch;  // b's row within a's pitch
      }
      const int i = r[a].i, j = r[b].i;
      if (!apart) throw einval("tensors %d and %d overlap", std::min(i, j), std::max(i, j));
    }
}

// The clip reads its input twice, the second time from the end: what the first
// pass read last is then still in the 256 MB cache before memory.  1.38 GB moved
// by the clip of 345 M bf16 values: 462 us from the front, 350 so.  What is read
// only once goes past the caches (5.8 -> 6.6 TB/s of a bare read).
static constexpr long long kKeep = 160 << 20;

// The list in tables of GN_MAXT; f(table, blocks) for each.  again: another pass
// follows.
template <class F>
static void gn_tables(const GnList& l, bool again, F&& f) {
  GnTable t;
  t.nt = t.nchunks = 0;
  auto flush = [&] {
    t.keep = again ? t.nchunks - (int)(kKeep / GN_CHUNK) : t.nchunks;
    if (t.nt) f(t, std::min(t.nchunks, GN_MAXB));
    t.nt = t.nchunks = 0;
  };
  for (int i = 0; i < l.n; ++i) {
    if (!l.count[i]) continue;
    const int64_t per = GN_CHUNK / elem_size(l.dtype[i]);
    const int64_t chunks = (l.count[i] + per - 1) / per;
    if (t.nt == GN_MAXT || t.nchunks + chunks > INT32_MAX) flush();
    GnEntry& e = t.e[t.nt];
    e.src = l.src[i];
    e.dst = l.dst ? l.dst[i] : nullptr;
    e.n = l.count[i];
    e.cols = l.cols ? (int)l.cols[i] : 0;
    e.ld = e.cols ? l.ld[i] : 0;
    if (e.cols && e.ld == e.cols) e.cols = 0;
    e.chunk0 = t.nchunks;
    t.dtype[t.nt++] = (unsigned char)l.dtype[i];
    t.nchunks += (int)chunks;
  }
  flush();
}

static size_t gn_ws(int n) { return sizeof(double) * GN_MAXB * (size_t)std::max(1, ceil_div(n, GN_MAXT)); }

// partial sums of the whole list; returns how many
static int gn_partials(const GnList& l, bool again, hipStream_t st, double* part,
                       size_t ws_bytes) {
  int np = 0;
  gn_tables(l, again, [&](const GnTable& t, int blocks) {
    if ((size_t)(np + blocks) * sizeof(double) > ws_bytes)
      throw einval("workspace of %zu bytes is too small", ws_bytes);
    hipLaunchKernelGGL(gn_partial_kernel, dim3(blocks), dim3(GN_T), 0, st, t, part + np);
    HIP_TRY(hipGetLastError());
    np += blocks;
  });
  return np;
}

}  // namespace ddpg

// A learner's gradient before its Adam pass (step.hip): out[0] = the norm of the
// n values at g, out[1] = the factor that clips it.
void clip_factor_launch(hipStream_t st, const float* g, long long n, float clip, double* part,
                        float* out) {
  const int dtype = T_FP32;
  const void* src = g;
  const int64_t count = n;
  const GnList l{1, &dtype, &src, nullptr, &count, nullptr, nullptr};
  const int np = gn_partials(l, true, st, part, gn_ws(1));
  hipLaunchKernelGGL(gn_norm_kernel, dim3(1), dim3(GN_T), 0, st, part, np, out, clip, out + 1);
  HIP_TRY(hipGetLastError());
}
size_t clip_factor_workspace() { return gn_ws(1); }

extern "C" {

size_t ddpg_global_norm_workspace(int n) { return gn_ws(n); }

int ddpg_global_norm(int device, void* stream, int n, const int* dtype, const void* const* src,
                     const int64_t* count, const int64_t* cols, const int64_t* ld, void* ws,
                     size_t ws_bytes, float* norm) {
  return guard(nullptr, [&] {
    const GnList l{n, dtype, src, nullptr, count, cols, ld};
    gn_check(l);
    if (!norm || !ws) throw einval("global_norm: null argument");
    OnDevice on(device);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    double* part = static_cast<double*>(ws);
    const int np = gn_partials(l, false, st, part, ws_bytes);
    hipLaunchKernelGGL(gn_norm_kernel, dim3(1), dim3(GN_T), 0, st, part, np, norm, 0.f,
                       nullptr);
    HIP_TRY(hipGetLastError());
  });
}

int ddpg_clip_by_global_norm(int device, void* stream, int n, const int* dtype,
                             const void* const* src, void* const* dst, const int64_t* count,
                             const int64_t* cols, const int64_t* ld, float clip_norm,
                             const float* use_norm, void* ws, size_t ws_bytes, float* norm) {
  return guard(nullptr, [&] {
    const GnList l{n, dtype, src, dst, count, cols, ld};
    gn_check(l);
    if (!(clip_norm >= 0.f)) throw einval("clip_norm %g is not a number >= 0", clip_norm);
    if (n && !dst) throw einval("clip_by_global_norm: null argument");
    if (!use_norm && (!ws || !norm)) throw einval("clip_by_global_norm: null argument");
    bool inplace = false;
    for (int i = 0; i < n; ++i) inplace = inplace || (count[i] && src[i] == dst[i]);
    if (inplace) gn_check_disjoint(l, use_norm);
    OnDevice on(device);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    double* part = static_cast<double*>(ws);
    const int np = use_norm ? 0 : gn_partials(l, true, st, part, ws_bytes);
    bool first = true;
    gn_tables(l, false, [&](const GnTable& t, int blocks) {
      hipLaunchKernelGGL(gn_scale_kernel, dim3(blocks), dim3(GN_T), 0, st, t, part, np, use_norm,
                         clip_norm, first ? norm : nullptr);
      HIP_TRY(hipGetLastError());
      first = false;
    });
    if (first && !use_norm) {  // no element anywhere: the norm is 0
      hipLaunchKernelGGL(gn_norm_kernel, dim3(1), dim3(GN_T), 0, st, part, 0, norm, 0.f,
                         nullptr);
      HIP_TRY(hipGetLastError());
    }
  });
}

}  // extern "C"
