// 16-byte pieces ("chunks") of float32 / bfloat16 / float16 rows, widened to fp32 registers.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>
#include "agents_amd.h"

typedef __bf16 vt_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 vt_f16x2 __attribute__((ext_vector_type(2)));
typedef float vt_f32x2 __attribute__((ext_vector_type(2)));

struct VtF32 {
  typedef float elem;
  static constexpr int C = 4;
  static constexpr unsigned LOWEST_WORD = 0xff800000u;       // -inf in every element of a word
  __device__ static inline float one(elem e) { return e; }
  __device__ static inline elem put(float f) { return f; }
  __device__ static inline void widen(const uint4& q, float (&v)[C]) {
    v[0] = __uint_as_float(q.x); v[1] = __uint_as_float(q.y);
    v[2] = __uint_as_float(q.z); v[3] = __uint_as_float(q.w);
  }
  __device__ static inline uint4 pack(const float (&v)[C]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                      __float_as_uint(v[3]));
  }
};

struct VtBf16 {
  typedef __bf16 elem;
  static constexpr int C = 8;
  static constexpr unsigned LOWEST_WORD = 0xff80ff80u;
  __device__ static inline float one(elem e) { return (float)e; }
  __device__ static inline elem put(float f) { return (__bf16)f; }   // round to nearest even
  __device__ static inline void widen(const uint4& q, float (&v)[C]) {
    const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ static inline uint4 pack(const float (&v)[C]) {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const vt_f32x2 f = {v[2 * i], v[2 * i + 1]};
      w[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(f, vt_bf16x2));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

struct VtF16 {
  typedef _Float16 elem;
  static constexpr int C = 8;
  static constexpr unsigned LOWEST_WORD = 0xfc00fc00u;
  __device__ static inline float one(elem e) { return (float)e; }
  __device__ static inline elem put(float f) { return (_Float16)f; }
  __device__ static inline void widen(const uint4& q, float (&v)[C]) {
    const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const vt_f16x2 h = __builtin_bit_cast(vt_f16x2, w[i]);
      v[2 * i] = (float)h.x;
      v[2 * i + 1] = (float)h.y;
    }
  }
  __device__ static inline uint4 pack(const float (&v)[C]) {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const vt_f16x2 h = {(_Float16)v[2 * i], (_Float16)v[2 * i + 1]};
      w[i] = __builtin_bit_cast(unsigned, h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// 16 bytes at any element's address: global accesses need no more than the element's alignment
// (unaligned access is on for global memory), so rows of odd lengths keep wide loads and stores.
__device__ static inline uint4 vt_load16(const void* p) {
  uint4 q;
  __builtin_memcpy(&q, p, 16);
  return q;
}
__device__ static inline void vt_store16(void* p, const uint4& q) { __builtin_memcpy(p, &q, 16); }

typedef unsigned vt_u32x4 __attribute__((ext_vector_type(4), aligned(2)));
// (streaming: the lines are the first that the caches give up)
__device__ static inline void vt_store16_nt(void* p, const uint4& q) {
  const vt_u32x4 v = {q.x, q.y, q.z, q.w};
  __builtin_nontemporal_store(v, reinterpret_cast<vt_u32x4*>(p));
}

// chunk of which only the first `n` elements exist (n <= 0: none); the others read as `fill`
template <typename T>
__device__ static inline void vt_load_part(const typename T::elem* p, int n, float fill,
                                           float (&v)[T::C]) {
#pragma unroll
  for (int j = 0; j < T::C; ++j) v[j] = j < n ? T::one(p[j]) : fill;
}
template <typename T>
__device__ static inline void vt_store_part(typename T::elem* p, int n, const float (&v)[T::C]) {
#pragma unroll
  for (int j = 0; j < T::C; ++j)
    if (j < n) p[j] = T::put(v[j]);
}

// A [.., n] tensor whose leading axes fold to (outer, inner): row r starts at
// (r / inner) * ld_outer + (r % inner) * ld_inner elements.
__device__ static inline int64_t vt_row(int64_t r, int64_t inner, int64_t ld_outer,
                                        int64_t ld_inner) {
  if (inner == 1) return r * ld_outer;
  // (a quotient of 32 bits where it can be one: a fifth of the instructions)
  const int64_t o = ((r | inner) >> 32) == 0 ? (int64_t)((uint32_t)r / (uint32_t)inner) : r / inner;
  return o * ld_outer + (r - o * inner) * ld_inner;
}

// Grids of one workgroup per row: folded into two axes, so that the lanes of an axis stay below 2^32.
// The last row of the fold may hold workgroups past the end: kernels compare vt_block() themselves.
#define VT_GRID_X (1 << 20)
#define VT_MAX_BLOCKS ((int64_t)VT_GRID_X * 65535)
static inline dim3 vt_grid(int64_t blocks) {
  if (blocks <= VT_GRID_X) return dim3((unsigned)blocks);
  return dim3(VT_GRID_X, (unsigned)((blocks + VT_GRID_X - 1) / VT_GRID_X));
}
__device__ static inline int64_t vt_block() {
  return (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
}
