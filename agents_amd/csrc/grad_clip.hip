// Norms of many gradient tensors of their own storage, and the clipped tensors.
//   global (tf.clip_by_global_norm):  n = sqrt(sum over all tensors of g^2),  g' = g clip / max(n, clip)
//   each   (tf.clip_by_norm, eager_utils.clip_gradient_norms): the same with a tensor's own n
// A norm that is not finite makes every value it scales NaN (tf.clip_by_global_norm).
// Bound by HBM: a pass that reads every tensor for the sum and one that reads it again (from the
// 256 MB memory-side cache where it fits) and writes.  The tensors' pointers travel in the kernel
// arguments (no copy to the device, so a captured graph replays them as they are), AA_CLIP_TENSORS
// per launch.  Every workgroup takes one contiguous piece of one tensor and leaves one sum in
// float64 -- a square of the float32 range neither overflows nor vanishes there, and an addition in
// float64 costs no more than one in float32 on this machine --; the pieces' sums are added in a fixed
// order by every workgroup of the second pass itself (at most a few thousand of them, from L2), so
// the join costs no launch.  Past AA_CLIP_JOIN pieces a launch of one workgroup adds them first.
#include <math.h>
#include "common.h"
#include "agents_amd.h"
#include "vec_types.h"

#define CLIP_THREADS 256
#define CLIP_MIN_PIECE 8192        // elements
#define CLIP_PIECES 2048           // workgroups a large list is cut into: 8 per CU
#define CLIP_JOIN 4096

struct ClipList {
  const void* src[AA_CLIP_TENSORS];
  void* dst[AA_CLIP_TENSORS];
  int64_t n[AA_CLIP_TENSORS];
  uint32_t first[AA_CLIP_TENSORS + 1];   // first workgroup of every tensor
  int32_t count;
  int64_t piece;                         // elements per workgroup
};

__device__ static inline int clip_find(const ClipList& L, unsigned b) {
  int lo = 0, hi = L.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (L.first[mid] <= b) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ static inline double clip_block_sum(double v, double* red) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
  for (unsigned w = 0; w < (blockDim.x >> 6); ++w) s += red[w];
  return s;
}

template <typename T>
__global__ void __launch_bounds__(CLIP_THREADS)
aa_clip_sumsq_kernel(ClipList L, double* __restrict__ partial) {
  constexpr int C = T::C;
  __shared__ double red[16];
  const int t = clip_find(L, blockIdx.x);
  const int64_t lo = (int64_t)(blockIdx.x - L.first[t]) * L.piece;
  const int64_t n = L.n[t] - lo < L.piece ? L.n[t] - lo : L.piece;
  const typename T::elem* g = reinterpret_cast<const typename T::elem*>(L.src[t]) + lo;
  double s0 = 0.0, s1 = 0.0;
  int64_t c = (int64_t)threadIdx.x * C;
  for (; c + C <= n; c += CLIP_THREADS * C) {
    float v[C];
    T::widen(vt_load16(g + c), v);
#pragma unroll
    for (int j = 0; j < C; j += 2) {
      s0 = fma((double)v[j], (double)v[j], s0);
      s1 = fma((double)v[j + 1], (double)v[j + 1], s1);
    }
  }
  for (int64_t k = c; k < n && k < c + C; ++k) s0 += (double)T::one(g[k]) * (double)T::one(g[k]);
  const double s = clip_block_sum(s0 + s1, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__global__ void __launch_bounds__(1024)
aa_clip_join_kernel(const double* __restrict__ partial, int64_t count, double* __restrict__ out,
                    float* __restrict__ norm) {
  __shared__ double red[16];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < count; i += 1024) s += partial[i];
  s = clip_block_sum(s, red);
  if (threadIdx.x == 0) {
    *out = s;
    if (norm != nullptr) *norm = (float)sqrt(s);
  }
}

template <typename T>
__global__ void __launch_bounds__(CLIP_THREADS)
aa_clip_scale_kernel(ClipList L, const double* __restrict__ partial, int64_t count, double clip,
                     int each, float* __restrict__ norm) {
  constexpr int C = T::C;
  __shared__ double red[16];
  const int t = clip_find(L, blockIdx.x);
  // `partial` is the list's own in `each` mode, the whole call's otherwise
  const int64_t p0 = each ? L.first[t] : 0, p1 = each ? L.first[t + 1] : count;
  double s = 0.0;
  for (int64_t i = p0 + threadIdx.x; i < p1; i += CLIP_THREADS) s += partial[i];
  const double nrm = sqrt(clip_block_sum(s, red));
  if (threadIdx.x == 0 && norm != nullptr) {
    if (each) {
      if (blockIdx.x == L.first[t]) norm[t] = (float)nrm;
    } else if (blockIdx.x == 0) {
      norm[0] = (float)nrm;
    }
  }
  // the factor is rounded to fp32 once; no clipping gives exactly 1
  const float f = nrm <= clip ? 1.f : isfinite(nrm) ? (float)(clip / nrm) : NAN;
  const int64_t lo = (int64_t)(blockIdx.x - L.first[t]) * L.piece;
  const int64_t n = L.n[t] - lo < L.piece ? L.n[t] - lo : L.piece;
  const typename T::elem* g = reinterpret_cast<const typename T::elem*>(L.src[t]) + lo;
  typename T::elem* o = reinterpret_cast<typename T::elem*>(L.dst[t]) + lo;
  int64_t c = (int64_t)threadIdx.x * C;
  for (; c + C <= n; c += CLIP_THREADS * C) {
    float v[C];
    T::widen(vt_load16(g + c), v);
#pragma unroll
    for (int j = 0; j < C; ++j) v[j] *= f;
    vt_store16(o + c, T::pack(v));
  }
  for (int64_t k = c; k < n && k < c + C; ++k) o[k] = T::put(T::one(g[k]) * f);
}

static int64_t clip_piece(const int64_t* n_h, int32_t n_tensors) {
  int64_t total = 0;
  for (int32_t i = 0; i < n_tensors; ++i) total += n_h[i];
  int64_t piece = (total + CLIP_PIECES - 1) / CLIP_PIECES;
  if (piece < CLIP_MIN_PIECE) piece = CLIP_MIN_PIECE;
  const int64_t step = CLIP_THREADS * 8;       // whole rounds of a workgroup in either element size
  return (piece + step - 1) / step * step;
}

// pieces of a tensor (an empty one keeps a workgroup: its norm is written too)
static int64_t clip_pieces_of(int64_t n, int64_t piece) {
  return n > 0 ? (n + piece - 1) / piece : 1;
}

static int clip_check(const int64_t* n_h, int32_t n_tensors, int32_t dtype) {
  if (n_h == nullptr || n_tensors <= 0 || dtype < AA_DT_F32 || dtype > AA_DT_F16)
    return AA_ERR_INVALID;
  for (int32_t i = 0; i < n_tensors; ++i)
    if (n_h[i] < 0) return AA_ERR_INVALID;
  return AA_OK;
}

template <typename T>
static void clip_launch(const ClipList& L, unsigned blocks, bool scale, const double* partial,
                        int64_t count, double clip, int each, float* norm, hipStream_t st) {
  if (scale)
    aa_clip_scale_kernel<T><<<dim3(blocks), dim3(CLIP_THREADS), 0, st>>>(L, partial, count, clip,
                                                                         each, norm);
  else
    aa_clip_sumsq_kernel<T><<<dim3(blocks), dim3(CLIP_THREADS), 0, st>>>(
        L, const_cast<double*>(partial));
}

extern "C" {

int64_t aa_clip_tensors_workspace_bytes(const int64_t* n_h, int32_t n_tensors) {
  if (clip_check(n_h, n_tensors, AA_DT_F32) != AA_OK) return -1;
  const int64_t piece = clip_piece(n_h, n_tensors);
  int64_t total = 1;                           // the joined sum
  for (int32_t i = 0; i < n_tensors; ++i) total += clip_pieces_of(n_h[i], piece);
  return total * (int64_t)sizeof(double);
}

int aa_clip_tensors(const void* const* src_h, void* const* dst_h, const int64_t* n_h,
                    int32_t n_tensors, int32_t dtype, double clip, int32_t each, float* norm,
                    void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = clip_check(n_h, n_tensors, dtype);
  if (rc != AA_OK) return rc;
  const bool scale = dst_h != nullptr;           // without destinations: the global norm only
  if (src_h == nullptr || norm == nullptr || (scale ? !(clip > 0.0) : each != 0))
    return AA_ERR_INVALID;
  for (int32_t i = 0; i < n_tensors; ++i)
    if (n_h[i] > 0 && (src_h[i] == nullptr || (scale && dst_h[i] == nullptr)))
      return AA_ERR_INVALID;
  if (workspace == nullptr || workspace_bytes < aa_clip_tensors_workspace_bytes(n_h, n_tensors))
    return AA_ERR_RANGE;
  const int64_t piece = clip_piece(n_h, n_tensors);
  double* joined = (double*)workspace;
  double* partial = joined + 1;
  hipStream_t st = (hipStream_t)stream;
  int64_t total = 0;
  for (int32_t i = 0; i < n_tensors; ++i) total += clip_pieces_of(n_h[i], piece);
  if (total > 0x7fffffff) return AA_ERR_RANGE;
  for (int pass = 0; pass < (scale ? 2 : 1); ++pass) {
    int64_t done = 0;
    for (int32_t base = 0; base < n_tensors; base += AA_CLIP_TENSORS) {
      ClipList L;
      L.count = n_tensors - base < AA_CLIP_TENSORS ? n_tensors - base : AA_CLIP_TENSORS;
      L.piece = piece;
      uint32_t blocks = 0;
      for (int i = 0; i < AA_CLIP_TENSORS; ++i) {
        const bool in = i < L.count;
        L.src[i] = in ? src_h[base + i] : nullptr;
        L.dst[i] = in && scale ? dst_h[base + i] : nullptr;
        L.n[i] = in ? n_h[base + i] : 0;
        L.first[i] = blocks;
        if (in) blocks += (uint32_t)clip_pieces_of(L.n[i], piece);
      }
      L.first[AA_CLIP_TENSORS] = blocks;
      const double* sums = partial;
      int64_t count = total;
      if (pass == 0 || each) sums = partial + done;
      else if (total > CLIP_JOIN) { sums = joined; count = 1; }
      float* nrm = each ? norm + base : (base == 0 ? norm : nullptr);
      if (dtype == AA_DT_F32)
        clip_launch<VtF32>(L, blocks, pass == 1, sums, count, clip, each, nrm, st);
      else if (dtype == AA_DT_BF16)
        clip_launch<VtBf16>(L, blocks, pass == 1, sums, count, clip, each, nrm, st);
      else
        clip_launch<VtF16>(L, blocks, pass == 1, sums, count, clip, each, nrm, st);
      done += blocks;
    }
    if (pass == 0 && !each && (!scale || total > CLIP_JOIN))
      aa_clip_join_kernel<<<dim3(1), dim3(1024), 0, st>>>(partial, total, joined,
                                                          scale ? nullptr : norm);
  }
  return aa_launch_status();
}

}  // extern "C"
