// Shared parts of the tensor operators (norm.hip, mx.hip): entry points that
// take device pointers and the caller's stream instead of a ddpg_ctx.  Their
// host code keeps no state: outputs and workspaces are the caller's, so calls
// on different streams, or captured into different graphs, share nothing.
#pragma once
#include "ctx.h"

namespace ddpg {

enum { T_FP32 = DDPG_FP32, T_BF16 = DDPG_BF16, T_FP16 = DDPG_FP16 };

inline int elem_size(int dtype) { return dtype == T_FP32 ? 4 : 2; }

inline void check_dtype(const char* what, int dtype) {
  if (dtype != T_FP32 && dtype != T_BF16 && dtype != T_FP16)
    throw einval("%s: dtype %d is none of fp32, bf16, fp16", what, dtype);
}

// 16 bytes at any address: the compiler emits the unaligned global access
struct __attribute__((packed, aligned(2))) U16B {
  uint32_t v[4];
};

// ... past the caches if NT: for bytes that are used once
typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
template <bool NT>
DDPG_DEV U16B load16(const void* p) {
  const u32x4_any* q = static_cast<const u32x4_any*>(p);
  const u32x4_any v = NT ? __builtin_nontemporal_load(q) : *q;
  return {{v[0], v[1], v[2], v[3]}};
}
DDPG_DEV void store16_nt(void* p, const U16B& u) {
  const u32x4_any v = {u.v[0], u.v[1], u.v[2], u.v[3]};
  __builtin_nontemporal_store(v, static_cast<u32x4_any*>(p));
}

// An element type: its loads widened to fp32 (exact), its stores one rounding
// to nearest even; the 16 / sizeof elements of U16B likewise.
template <int DT>
struct Elem;
template <>
struct Elem<T_FP32> {
  typedef float type;
  static constexpr int V = 4;
  static DDPG_DEV void widen(const U16B& u, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(u.v[i]);
  }
  static DDPG_DEV U16B pack(const float* x) {
    U16B u;
#pragma unroll
    for (int i = 0; i < 4; ++i) u.v[i] = __float_as_uint(x[i]);
    return u;
  }
};
template <class H>
struct Elem16 {
  typedef H type;
  static constexpr int V = 8;
  static DDPG_DEV void widen(const U16B& u, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      H h[2];
      __builtin_memcpy(h, &u.v[i], 4);
      x[2 * i] = (float)h[0];
      x[2 * i + 1] = (float)h[1];
    }
  }
  static DDPG_DEV U16B pack(const float* x) {
    U16B u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const H h[2] = {(H)x[2 * i], (H)x[2 * i + 1]};
      __builtin_memcpy(&u.v[i], h, 4);
    }
    return u;
  }
};
template <>
struct Elem<T_BF16> : Elem16<__bf16> {};
template <>
struct Elem<T_FP16> : Elem16<_Float16> {};

// The same for a type known at run time (epilogues).
DDPG_DEV float load_elem(const void* p, int dtype, long long i) {
  if (dtype == T_FP32) return static_cast<const float*>(p)[i];
  if (dtype == T_BF16) return (float)static_cast<const __bf16*>(p)[i];
  return (float)static_cast<const _Float16*>(p)[i];
}
DDPG_DEV void store_elem(void* p, int dtype, long long i, float v) {
  if (dtype == T_FP32)
    static_cast<float*>(p)[i] = v;
  else if (dtype == T_BF16)
    static_cast<__bf16*>(p)[i] = (__bf16)v;
  else
    static_cast<_Float16*>(p)[i] = (_Float16)v;
}

template <int N>
struct IntC {
  static constexpr int value = N;
};
// f(IntC<dtype>) for a run-time dtype
template <class F>
__host__ __device__ __forceinline__ void by_dtype(int dtype, F&& f) {
  if (dtype == T_FP32)
    f(IntC<T_FP32>{});
  else if (dtype == T_BF16)
    f(IntC<T_BF16>{});
  else
    f(IntC<T_FP16>{});
}

}  // namespace ddpg
