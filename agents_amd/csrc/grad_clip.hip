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
// the join costs no launch.  14 bf16 tensors of 333 MB: 56 .. 58 us (5.8 TB/s) and 108 .. 110 (6.1); 10
// f32 tensors of 7 MB: 4.1 and 5.7.  Past AA_CLIP_JOIN pieces a launch of one workgroup adds them first.
#include <math.h>
#include "common.h"
#include "agents_amd.h"
#include "vec_types.h"

#define CLIP_THREADS 256
#define CLIP_MIN_PIECE 8192        // elements
#define CLIP_PIECES 2048           // workgroups a large list is cut into: 8 per CU
#define CLIP_JOIN 4096
#define CLIP_UNROLL 4
// Clipped tensors of this many bytes are stored past the caches (the memory-side one holds 256 MB), so
// that they do not push out the gradients that the second pass reads again.  bf16, us a call: 268 MB
// 148 -> 122, 333 MB 200 -> 167; with an update of the clipped tensors behind it 344 -> 348.  Below it
// costs whoever reads them next: 134 MB 64 -> 64 alone, 137 -> 171 with the update.
#define CLIP_PAST_CACHE (256ll << 20)
#define CLIP_FEW 32

template <int N>
struct ClipList {
  const void* src[N];
  void* dst[N];
  int64_t n[N];
  int64_t piece;                         // elements per workgroup
  uint32_t first[N + 1];                 // first workgroup of every tensor
  int32_t count;
};

template <int N>
__device__ static inline int clip_find(const ClipList<N>& L, unsigned b) {
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

// U loads of a lane are in flight at once
template <typename T, int U>
__device__ static inline void clip_load(const typename T::elem* g, int64_t c, uint4 (&q)[U]) {
#pragma unroll
  for (int u = 0; u < U; ++u) q[u] = vt_load16(g + c + (int64_t)u * CLIP_THREADS * T::C);
}

template <typename T, int N>
__global__ void __launch_bounds__(CLIP_THREADS)
aa_clip_sumsq_kernel(ClipList<N> L, double* __restrict__ partial) {
  constexpr int C = T::C, U = CLIP_UNROLL, ROUND = CLIP_THREADS * C;
  __shared__ double red[16];
  const int t = clip_find(L, blockIdx.x);
  const int64_t lo = (int64_t)(blockIdx.x - L.first[t]) * L.piece;
  const int64_t n = L.n[t] - lo < L.piece ? L.n[t] - lo : L.piece;
  const typename T::elem* g = reinterpret_cast<const typename T::elem*>(L.src[t]) + lo;
  double s0 = 0.0, s1 = 0.0;
  auto add = [&](const uint4& q) {
    float v[C];
    T::widen(q, v);
#pragma unroll
    for (int j = 0; j < C; j += 2) {
      s0 = fma((double)v[j], (double)v[j], s0);
      s1 = fma((double)v[j + 1], (double)v[j + 1], s1);
    }
  };
  int64_t c = (int64_t)threadIdx.x * C;
  for (; c + (U - 1) * ROUND + C <= n; c += U * ROUND) {
    uint4 q[U];
    clip_load<T, U>(g, c, q);
#pragma unroll
    for (int u = 0; u < U; ++u) add(q[u]);
  }
  for (; c + C <= n; c += ROUND) add(vt_load16(g + c));
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

template <typename T, int N>
__global__ void __launch_bounds__(CLIP_THREADS)
aa_clip_scale_kernel(ClipList<N> L, const double* __restrict__ partial, int64_t count, double clip,
                     int each, int past_cache, float* __restrict__ norm) {
  constexpr int C = T::C, U = CLIP_UNROLL, ROUND = CLIP_THREADS * C;
  __shared__ double red[16];
  // the pieces in the opposite order of the first pass: what it read last is still cached
  const unsigned block = gridDim.x - 1 - blockIdx.x;
  const int t = clip_find(L, block);
  const int64_t lo = (int64_t)(block - L.first[t]) * L.piece;
  const int64_t n = L.n[t] - lo < L.piece ? L.n[t] - lo : L.piece;
  const typename T::elem* g = reinterpret_cast<const typename T::elem*>(L.src[t]) + lo;
  typename T::elem* o = reinterpret_cast<typename T::elem*>(L.dst[t]) + lo;
  int64_t c = (int64_t)threadIdx.x * C;
  bool full = c + (U - 1) * ROUND + C <= n;
  uint4 q[U];
  if (full) clip_load<T, U>(g, c, q);          // in flight while the pieces' sums are added
  // `partial` is the list's own in `each` mode, the whole call's otherwise
  const int64_t p0 = each ? L.first[t] : 0, p1 = each ? L.first[t + 1] : count;
  double s = 0.0;
  for (int64_t i = p0 + threadIdx.x; i < p1; i += CLIP_THREADS) s += partial[i];
  const double nrm = sqrt(clip_block_sum(s, red));
  if (threadIdx.x == 0 && norm != nullptr) {
    if (each) {
      if (block == L.first[t]) norm[t] = (float)nrm;
    } else if (block == 0) {
      norm[0] = (float)nrm;
    }
  }
  // the factor is rounded to fp32 once; no clipping gives exactly 1
  const float f = !isfinite(nrm) ? NAN : nrm <= clip ? 1.f : (float)(clip / nrm);
  auto put = [&](const uint4& q, int64_t at) {
    float v[C];
    T::widen(q, v);
#pragma unroll
    for (int j = 0; j < C; ++j) v[j] *= f;
    if (past_cache) vt_store16_nt(o + at, T::pack(v));
    else vt_store16(o + at, T::pack(v));
  };
  while (full) {
#pragma unroll
    for (int u = 0; u < U; ++u) put(q[u], c + u * ROUND);
    c += U * ROUND;
    full = c + (U - 1) * ROUND + C <= n;
    if (full) clip_load<T, U>(g, c, q);
  }
  for (; c + C <= n; c += ROUND) put(vt_load16(g + c), c);
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

template <typename T, int N>
static void clip_launch(const ClipList<N>& L, unsigned blocks, bool scale, const double* partial,
                        int64_t count, double clip, int each, int past_cache, float* norm,
                        hipStream_t st) {
  if (scale)
    aa_clip_scale_kernel<T, N><<<dim3(blocks), dim3(CLIP_THREADS), 0, st>>>(
        L, partial, count, clip, each, past_cache, norm);
  else
    aa_clip_sumsq_kernel<T, N><<<dim3(blocks), dim3(CLIP_THREADS), 0, st>>>(
        L, const_cast<double*>(partial));
}

struct ClipCall {
  const void* const* src;
  void* const* dst;                // null: the global norm only
  const int64_t* n;
  int32_t n_tensors, dtype, each, past_cache;
  int64_t piece, total;            // elements of a piece, pieces of the call
  double clip;
  float* norm;
  double* joined;
  double* partial;
};

template <int N>
static void clip_run(const ClipCall& c, hipStream_t st) {
  for (int pass = 0; pass < (c.dst != nullptr ? 2 : 1); ++pass) {
    int64_t done = 0;
    for (int32_t base = 0; base < c.n_tensors; base += N) {
      ClipList<N> L;
      L.count = c.n_tensors - base < N ? c.n_tensors - base : N;
      L.piece = c.piece;
      uint32_t blocks = 0;
      for (int i = 0; i < N; ++i) {
        const bool in = i < L.count;
        L.src[i] = in ? c.src[base + i] : nullptr;
        L.dst[i] = in && c.dst != nullptr ? c.dst[base + i] : nullptr;
        L.n[i] = in ? c.n[base + i] : 0;
        L.first[i] = blocks;
        if (in) blocks += (uint32_t)clip_pieces_of(L.n[i], c.piece);
      }
      L.first[N] = blocks;
      const double* sums = c.partial;
      int64_t count = c.total;
      if (pass == 0 || c.each) sums = c.partial + done;
      else if (c.total > CLIP_JOIN) { sums = c.joined; count = 1; }
      float* nrm = c.each ? c.norm + base : (base == 0 ? c.norm : nullptr);
      if (c.dtype == AA_DT_F32)
        clip_launch<VtF32, N>(L, blocks, pass == 1, sums, count, c.clip, c.each, c.past_cache, nrm,
                               st);
      else if (c.dtype == AA_DT_BF16)
        clip_launch<VtBf16, N>(L, blocks, pass == 1, sums, count, c.clip, c.each, c.past_cache, nrm,
                               st);
      else
        clip_launch<VtF16, N>(L, blocks, pass == 1, sums, count, c.clip, c.each, c.past_cache, nrm,
                               st);
      done += blocks;
    }
    if (pass == 0 && !c.each && (c.dst == nullptr || c.total > CLIP_JOIN))
      aa_clip_join_kernel<<<dim3(1), dim3(1024), 0, st>>>(c.partial, c.total, c.joined,
                                                          c.dst == nullptr ? c.norm : nullptr);
  }
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
  ClipCall c = {src_h, dst_h, n_h, n_tensors, dtype, each != 0, 0, clip_piece(n_h, n_tensors), 0,
                clip, norm, (double*)workspace, (double*)workspace + 1};
  int64_t elements = 0;
  for (int32_t i = 0; i < n_tensors; ++i) {
    c.total += clip_pieces_of(n_h[i], c.piece);
    elements += n_h[i];
  }
  c.past_cache = elements * (dtype == AA_DT_F32 ? 4 : 2) >= CLIP_PAST_CACHE;
  if (c.total > 0x7fffff) return AA_ERR_RANGE;
  // the arguments of a launch are written by the host for every call: a short list for few tensors
  if (n_tensors <= CLIP_FEW) clip_run<CLIP_FEW>(c, (hipStream_t)stream);
  else clip_run<AA_CLIP_TENSORS>(c, (hipStream_t)stream);
  return aa_launch_status();
}

}  // extern "C"
