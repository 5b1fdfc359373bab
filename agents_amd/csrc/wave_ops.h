// Exchanges and reductions across the 64 lanes of a wave without LDS: DPP inside rows of 16 lanes,
// v_permlane16_swap / v_permlane32_swap across them (a step of a few cycles where ds_bpermute takes
// about a hundred).  Every lane of the wave must be active.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

typedef unsigned wv_u32x2 __attribute__((ext_vector_type(2)));

template <int CTRL>
__device__ static inline unsigned wv_dpp(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
}

// a = the even rows' (lower half's) values, b = the odd rows' (upper half's), each in both places
template <int M>
__device__ static inline void wv_pair(unsigned v, unsigned& a, unsigned& b) {
  static_assert(M == 16 || M == 32, "rows of 16 or halves of 32");
  const wv_u32x2 r = M == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false)
                             : __builtin_amdgcn_permlane32_swap(v, v, false, false);
  a = r.x;
  b = r.y;
}

// the value of lane (lane ^ M)
template <int M>
__device__ static inline unsigned wv_xor(unsigned v, int lane) {
  if constexpr (M == 1) return wv_dpp<0xB1>(v);          // quad_perm [1,0,3,2]
  else if constexpr (M == 2) return wv_dpp<0x4E>(v);     // quad_perm [2,3,0,1]
  else if constexpr (M == 4) return wv_dpp<0x1B>(wv_dpp<0x141>(v));   // half mirror, then quads
  else if constexpr (M == 8) return wv_dpp<0x128>(v);    // row_ror:8
  else {
    unsigned a, b;
    wv_pair<M>(v, a, b);
    return (lane & M) ? a : b;
  }
}
template <int M>
__device__ static inline unsigned long long wv_xor(unsigned long long v, int lane) {
  const unsigned lo = wv_xor<M>((unsigned)v, lane), hi = wv_xor<M>((unsigned)(v >> 32), lane);
  return ((unsigned long long)hi << 32) | lo;
}

// One step of an all-lanes reduction with a commutative `op`: after steps 1, 2, 4, 8 the lanes of a
// row agree, so the mirrors of half rows and rows stand for lane ^ 4 and lane ^ 8.
template <int STEP, typename F>
__device__ static inline float wv_step(float v, F op) {
  const unsigned u = __float_as_uint(v);
  if constexpr (STEP == 1) return op(v, __uint_as_float(wv_dpp<0xB1>(u)));
  else if constexpr (STEP == 2) return op(v, __uint_as_float(wv_dpp<0x4E>(u)));
  else if constexpr (STEP == 4) return op(v, __uint_as_float(wv_dpp<0x141>(u)));
  else if constexpr (STEP == 8) return op(v, __uint_as_float(wv_dpp<0x140>(u)));
  else {
    unsigned a, b;
    wv_pair<STEP>(u, a, b);
    return op(__uint_as_float(a), __uint_as_float(b));
  }
}

// over groups of W neighbouring lanes, in each of them the same bits
template <int W, typename F>
__device__ static inline float wv_group(float v, F op) {
  if constexpr (W >= 2) v = wv_step<1>(v, op);
  if constexpr (W >= 4) v = wv_step<2>(v, op);
  if constexpr (W >= 8) v = wv_step<4>(v, op);
  if constexpr (W >= 16) v = wv_step<8>(v, op);
  if constexpr (W >= 32) v = wv_step<16>(v, op);
  if constexpr (W >= 64) v = wv_step<32>(v, op);
  return v;
}
template <int W>
__device__ static inline float wv_group_sum(float v) {
  return wv_group<W>(v, [](float a, float b) { return a + b; });
}
template <int W>
__device__ static inline float wv_group_max(float v) {
  return wv_group<W>(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ static inline float wv_sum(float v) { return wv_group_sum<64>(v); }
__device__ static inline float wv_max(float v) { return wv_group_max<64>(v); }

// ---- descending order of 64 keys, one per lane ---------------------------------------------------
template <int J, typename K>
__device__ static inline K wv_keep(K v, bool larger, int lane) {
  const K o = wv_xor<J>(v, lane);
  return (larger == (v > o)) ? v : o;
}

// bitonic network; `flip` reverses the order
template <typename K>
__device__ static inline K wv_sort_desc(K v, int lane, bool flip = false) {
#define WV_STAGE(KK, J) v = wv_keep<J>(v, (((lane & J) == 0) == ((lane & KK) == 0)) != flip, lane);
  WV_STAGE(2, 1)
  WV_STAGE(4, 2) WV_STAGE(4, 1)
  WV_STAGE(8, 4) WV_STAGE(8, 2) WV_STAGE(8, 1)
  WV_STAGE(16, 8) WV_STAGE(16, 4) WV_STAGE(16, 2) WV_STAGE(16, 1)
  WV_STAGE(32, 16) WV_STAGE(32, 8) WV_STAGE(32, 4) WV_STAGE(32, 2) WV_STAGE(32, 1)
  WV_STAGE(64, 32) WV_STAGE(64, 16) WV_STAGE(64, 8) WV_STAGE(64, 4) WV_STAGE(64, 2) WV_STAGE(64, 1)
#undef WV_STAGE
  return v;
}

// the 64 best, descending, of a descending and an ascending list
template <typename K>
__device__ static inline K wv_merge_desc(K desc, K asc, int lane) {
  K v = desc > asc ? desc : asc;
  v = wv_keep<32>(v, (lane & 32) == 0, lane);
  v = wv_keep<16>(v, (lane & 16) == 0, lane);
  v = wv_keep<8>(v, (lane & 8) == 0, lane);
  v = wv_keep<4>(v, (lane & 4) == 0, lane);
  v = wv_keep<2>(v, (lane & 2) == 0, lane);
  return wv_keep<1>(v, (lane & 1) == 0, lane);
}
