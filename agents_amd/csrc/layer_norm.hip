// Layer normalisation over the last axis, forward and backward (keras LayerNormalization).
//   mean = sum x / D;  var = sum (x - mean)^2 / D;  rstd = 1 / sqrt(var + eps);  h = (x - mean) rstd
//   y = h gamma + beta
//   g = dy gamma;  dx = rstd (g - mean(g) - h mean(g h)) * act'(x);  dgamma = sum_rows dy h;
//   dbeta = sum_rows dy
// Everything is held in fp32; x, dy, y and dx are rounded once on their way to memory.  Bound by HBM:
// a row is read once into registers by one team (a wave up to 1,024 columns, a workgroup of
// 256 / 512 / 1,024 lanes beyond), the mean and the squares about it come from the registers, so the
// variance has no cancellation and the row is not read a second time.  The weight gradients need every
// row: a team walks many rows with its columns' sums in registers and leaves one partial per
// workgroup, a second launch adds the partials in a fixed order (no atomics: same bits every call).
// Rows wider than 16,384 columns do not fit the registers beside these sums and take loops.
#include <math.h>
#include "common.h"
#include "agents_amd.h"
#include "vec_types.h"
#include "wave_ops.h"

#define LN_MAX_WIDTH_REG 16384
#define LN_PER_LANE 16

struct LnArgs {
  int64_t rows, inner;
  int width;
  const void* x; int64_t x_outer, x_inner;
  const void* dy; int64_t dy_outer, dy_inner;
  void* out; int64_t out_outer, out_inner;     // y or dx
  const float* gamma;
  const float* beta;
  float epsilon;
  float* stats;                                // [rows][2] mean, rstd
  float* partial;                              // [groups][2][width]
  int mask_act;
};

template <int TEAM>
__device__ static inline float ln_team_sum(float v, float* red) {
  v = wv_sum(v);
  if constexpr (TEAM == 64) return v;
  constexpr int NW = TEAM / 64;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) s += red[w];
  return s;
}

// two sums behind one pair of barriers
template <int TEAM>
__device__ static inline void ln_team_sum2(float& a, float& b, float* red) {
  a = wv_sum(a);
  b = wv_sum(b);
  if constexpr (TEAM == 64) return;
  constexpr int NW = TEAM / 64;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    red[threadIdx.x >> 6] = a;
    red[NW + (threadIdx.x >> 6)] = b;
  }
  __syncthreads();
  a = b = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) { a += red[w]; b += red[NW + w]; }
}

template <typename T, int NCH>
__device__ static inline void ln_load(const typename T::elem* p, int lane, int team, int width,
                                      uint4 (&q)[NCH]) {
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = (lane + i * team) * T::C;
    q[i] = make_uint4(0u, 0u, 0u, 0u);
    if (c + T::C <= width) {
      q[i] = vt_load16(p + c);
    } else if (c < width) {
      float v[T::C];
      vt_load_part<T>(p + c, width - c, 0.f, v);
      q[i] = T::pack(v);       // back to the type it came from: exact
    }
  }
}

// fp32 weights of this lane's columns; `fill` beyond the row and where there is no such weight
template <int C, int NCH>
__device__ static inline void ln_load_weight(const float* w, int lane, int team, int width,
                                             float fill, float (&v)[NCH][C]) {
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = (lane + i * team) * C;
#pragma unroll
    for (int j = 0; j < C; j += 4) {
      if (w != nullptr && c + j + 4 <= width) {
        const uint4 q = vt_load16(w + c + j);
        v[i][j] = __uint_as_float(q.x); v[i][j + 1] = __uint_as_float(q.y);
        v[i][j + 2] = __uint_as_float(q.z); v[i][j + 3] = __uint_as_float(q.w);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          v[i][j + k] = (w != nullptr && c + j + k < width) ? w[c + j + k] : fill;
      }
    }
  }
}

// A team walks rows `stride` apart: the weights are read once, the next row's loads are in flight while
// this one is worked on.
template <typename T, int TEAM, int NCH>
__global__ void __launch_bounds__(TEAM == 64 ? 256 : TEAM)
aa_layer_norm_fwd_kernel(LnArgs a) {
  constexpr int C = T::C;
  constexpr int PER = TEAM == 64 ? 4 : 1;        // teams of a workgroup
  __shared__ float red[32];
  const int64_t row0 = (int64_t)blockIdx.x * PER + (TEAM == 64 ? threadIdx.x >> 6 : 0);
  const int64_t stride = (int64_t)gridDim.x * PER;
  const int lane = TEAM == 64 ? (threadIdx.x & 63) : threadIdx.x;
  if (row0 >= a.rows) return;      // (the whole workgroup, or a wave that meets no barrier)
  const typename T::elem* x = reinterpret_cast<const typename T::elem*>(a.x);
  typename T::elem* out = reinterpret_cast<typename T::elem*>(a.out);
  uint4 next[NCH];
  ln_load<T, NCH>(x + vt_row(row0, a.inner, a.x_outer, a.x_inner), lane, TEAM, a.width, next);
  float gm[NCH][C], bt[NCH][C];
  ln_load_weight<C, NCH>(a.gamma, lane, TEAM, a.width, 1.f, gm);
  ln_load_weight<C, NCH>(a.beta, lane, TEAM, a.width, 0.f, bt);
  // (a quotient, not a product with 1 / D: a constant row's mean is its value, its y is beta)
  const float width = (float)a.width;
  for (int64_t row = row0; row < a.rows; row += stride) {
    float v[NCH][C];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      T::widen(next[i], v[i]);
#pragma unroll
      for (int j = 0; j < C; ++j) s += v[i][j];
    }
    if (row + stride < a.rows)
      ln_load<T, NCH>(x + vt_row(row + stride, a.inner, a.x_outer, a.x_inner), lane, TEAM, a.width,
                      next);
    const float mean = ln_team_sum<TEAM>(s, red) / width;
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int n = a.width - (lane + i * TEAM) * C;
#pragma unroll
      for (int j = 0; j < C; ++j) {
        v[i][j] -= mean;
        ss += j < n ? v[i][j] * v[i][j] : 0.f;
      }
    }
    const float var = ln_team_sum<TEAM>(ss, red) / width;
    const float rstd = 1.f / sqrtf(var + a.epsilon);
    if (lane == 0 && a.stats != nullptr) {
      a.stats[2 * row] = mean;
      a.stats[2 * row + 1] = rstd;
    }
    typename T::elem* y = out + vt_row(row, a.inner, a.out_outer, a.out_inner);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = (lane + i * TEAM) * C;
#pragma unroll
      for (int j = 0; j < C; ++j) v[i][j] = v[i][j] * rstd * gm[i][j] + bt[i][j];
      if (c + C <= a.width) vt_store16(y + c, T::pack(v[i]));
      else if (c < a.width) vt_store_part<T>(y + c, a.width - c, v[i]);
    }
  }
}

// rows wider than the registers hold: a workgroup per row, three passes
template <typename T>
__global__ void __launch_bounds__(1024) aa_layer_norm_fwd_wide_kernel(LnArgs a) {
  __shared__ float red[32];
  const int64_t row = vt_block();
  if (row >= a.rows) return;
  const typename T::elem* x = reinterpret_cast<const typename T::elem*>(a.x) +
                              vt_row(row, a.inner, a.x_outer, a.x_inner);
  typename T::elem* y = reinterpret_cast<typename T::elem*>(a.out) +
                        vt_row(row, a.inner, a.out_outer, a.out_inner);
  const float width = (float)a.width;
  float s = 0.f;
  for (int c = threadIdx.x; c < a.width; c += 1024) s += T::one(x[c]);
  const float mean = ln_team_sum<1024>(s, red) / width;
  float ss = 0.f;
  for (int c = threadIdx.x; c < a.width; c += 1024) {
    const float d = T::one(x[c]) - mean;
    ss += d * d;
  }
  const float rstd = 1.f / sqrtf(ln_team_sum<1024>(ss, red) / width + a.epsilon);
  if (threadIdx.x == 0 && a.stats != nullptr) {
    a.stats[2 * row] = mean;
    a.stats[2 * row + 1] = rstd;
  }
  for (int c = threadIdx.x; c < a.width; c += 1024) {
    const float g = a.gamma != nullptr ? a.gamma[c] : 1.f;
    const float b = a.beta != nullptr ? a.beta[c] : 0.f;
    y[c] = T::put((T::one(x[c]) - mean) * rstd * g + b);
  }
}

__device__ static inline float ln_act_grad(float y, int kind) {
  if (kind == AA_ACT_RELU) return y > 0.f ? 1.f : 0.f;
  if (kind == AA_ACT_TANH) return 1.f - y * y;
  return 1.f;
}

template <typename T, int TEAM, int NCH, bool WEIGHTS>
__global__ void __launch_bounds__(TEAM == 64 ? 256 : TEAM)
aa_layer_norm_bwd_kernel(LnArgs a) {
  constexpr int C = T::C;
  constexpr int PER = TEAM == 64 ? 4 : 1;        // teams of a workgroup
  // the next row in flight and gamma in registers; 1,024 lanes have 128 registers each and need them
  // for the sums (spills cost more than reading gamma again)
  constexpr bool AHEAD = TEAM < 1024;
  __shared__ float red[32];
  __shared__ float sums[(WEIGHTS && TEAM == 64) ? 2 * 64 * NCH * C : 1];
  const int sub = TEAM == 64 ? (threadIdx.x >> 6) : 0;
  const int lane = TEAM == 64 ? (threadIdx.x & 63) : threadIdx.x;
  const float inv = 1.f / (float)a.width;
  const int64_t row0 = (int64_t)blockIdx.x * PER + sub, stride = (int64_t)gridDim.x * PER;
  const typename T::elem* x = reinterpret_cast<const typename T::elem*>(a.x);
  const typename T::elem* dy = reinterpret_cast<const typename T::elem*>(a.dy);
  uint4 nx[NCH], nd[NCH];          // the next row
  float nmean = 0.f, nrstd = 0.f;
  auto fetch = [&](int64_t r) {
    ln_load<T, NCH>(x + vt_row(r, a.inner, a.x_outer, a.x_inner), lane, TEAM, a.width, nx);
    ln_load<T, NCH>(dy + vt_row(r, a.inner, a.dy_outer, a.dy_inner), lane, TEAM, a.width, nd);
    nmean = a.stats[2 * r];
    nrstd = a.stats[2 * r + 1];
  };
  if (AHEAD && row0 < a.rows) fetch(row0);
  float gm[NCH][C], dg[NCH][C], db[NCH][C];
  if (AHEAD) ln_load_weight<C, NCH>(a.gamma, lane, TEAM, a.width, 1.f, gm);
#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int j = 0; j < C; ++j) dg[i][j] = db[i][j] = 0.f;
  for (int64_t row = row0; row < a.rows; row += stride) {
    if (!AHEAD) {
      fetch(row);
      ln_load_weight<C, NCH>(a.gamma, lane, TEAM, a.width, 1.f, gm);
    }
    uint4 qx[NCH], qd[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) { qx[i] = nx[i]; qd[i] = nd[i]; }
    const float mean = nmean, rstd = nrstd;
    if (AHEAD && row + stride < a.rows) fetch(row + stride);
    float c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      float xv[C], dv[C];
      T::widen(qx[i], xv);
      T::widen(qd[i], dv);
#pragma unroll
      for (int j = 0; j < C; ++j) {
        // (beyond the row dy reads as 0: nothing is added to any sum)
        const float h = (xv[j] - mean) * rstd, g = dv[j] * gm[i][j];
        c1 += g;
        c2 += g * h;
        if (WEIGHTS) {
          dg[i][j] += dv[j] * h;
          db[i][j] += dv[j];
        }
      }
    }
    ln_team_sum2<TEAM>(c1, c2, red);
    c1 *= inv;
    c2 *= inv;
    if (a.out != nullptr) {
      typename T::elem* dx = reinterpret_cast<typename T::elem*>(a.out) +
                             vt_row(row, a.inner, a.out_outer, a.out_inner);
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const int c = (lane + i * TEAM) * C;
        float xv[C], dv[C], r[C];
        T::widen(qx[i], xv);
        T::widen(qd[i], dv);
#pragma unroll
        for (int j = 0; j < C; ++j) {
          const float h = (xv[j] - mean) * rstd;
          r[j] = rstd * (dv[j] * gm[i][j] - c1 - h * c2);
          if (a.mask_act != AA_ACT_NONE) r[j] *= ln_act_grad(xv[j], a.mask_act);
        }
        if (c + C <= a.width) vt_store16(dx + c, T::pack(r));
        else if (c < a.width) vt_store_part<T>(dx + c, a.width - c, r);
      }
    }
  }
  if constexpr (WEIGHTS) {
    float* out = a.partial + (int64_t)blockIdx.x * 2 * a.width;
    if constexpr (TEAM == 64) {
      // the four waves' sums, added in the order of the waves
      for (int w = 0; w < 4; ++w) {
        if (sub == w) {
#pragma unroll
          for (int i = 0; i < NCH; ++i)
#pragma unroll
            for (int j = 0; j < C; ++j) {
              const int at = (lane + i * 64) * C + j;
              const int at2 = at + 64 * NCH * C;
              sums[at] = w == 0 ? dg[i][j] : sums[at] + dg[i][j];
              sums[at2] = w == 0 ? db[i][j] : sums[at2] + db[i][j];
            }
        }
        __syncthreads();
      }
      for (int c = threadIdx.x; c < a.width; c += 256) {
        out[c] = sums[c];
        out[a.width + c] = sums[64 * NCH * C + c];
      }
    } else {
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int j = 0; j < C; ++j) {
          const int c = (lane + i * TEAM) * C + j;
          if (c < a.width) {
            out[c] = dg[i][j];
            out[a.width + c] = db[i][j];
          }
        }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(1024) aa_layer_norm_dx_wide_kernel(LnArgs a) {
  __shared__ float red[32];
  const int64_t row = vt_block();
  if (row >= a.rows) return;
  const typename T::elem* x = reinterpret_cast<const typename T::elem*>(a.x) +
                              vt_row(row, a.inner, a.x_outer, a.x_inner);
  const typename T::elem* dy = reinterpret_cast<const typename T::elem*>(a.dy) +
                               vt_row(row, a.inner, a.dy_outer, a.dy_inner);
  typename T::elem* dx = reinterpret_cast<typename T::elem*>(a.out) +
                         vt_row(row, a.inner, a.out_outer, a.out_inner);
  const float mean = a.stats[2 * row], rstd = a.stats[2 * row + 1];
  const float inv = 1.f / (float)a.width;
  float c1 = 0.f, c2 = 0.f;
  for (int c = threadIdx.x; c < a.width; c += 1024) {
    const float g = T::one(dy[c]) * (a.gamma != nullptr ? a.gamma[c] : 1.f);
    c1 += g;
    c2 += g * ((T::one(x[c]) - mean) * rstd);
  }
  ln_team_sum2<1024>(c1, c2, red);
  c1 *= inv;
  c2 *= inv;
  for (int c = threadIdx.x; c < a.width; c += 1024) {
    const float xv = T::one(x[c]), h = (xv - mean) * rstd;
    const float g = T::one(dy[c]) * (a.gamma != nullptr ? a.gamma[c] : 1.f);
    float r = rstd * (g - c1 - h * c2);
    if (a.mask_act != AA_ACT_NONE) r *= ln_act_grad(xv, a.mask_act);
    dx[c] = T::put(r);
  }
}

// weight gradients of wide rows: a lane owns a column, grid = (column blocks, row groups)
template <typename T>
__global__ void __launch_bounds__(256) aa_layer_norm_dw_wide_kernel(LnArgs a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.width) return;
  float dg = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float xv = T::one(reinterpret_cast<const typename T::elem*>(
        a.x)[vt_row(row, a.inner, a.x_outer, a.x_inner) + c]);
    const float dv = T::one(reinterpret_cast<const typename T::elem*>(
        a.dy)[vt_row(row, a.inner, a.dy_outer, a.dy_inner) + c]);
    dg += dv * ((xv - a.stats[2 * row]) * a.stats[2 * row + 1]);
    db += dv;
  }
  float* out = a.partial + (int64_t)blockIdx.y * 2 * a.width;
  out[c] = dg;
  out[a.width + c] = db;
}

// sums of the partials' columns: 32 columns x 32 lanes along the partials per workgroup
__global__ void __launch_bounds__(1024)
aa_layer_norm_join_kernel(const float* __restrict__ partial, int groups, int width,
                          float* __restrict__ dgamma, float* __restrict__ dbeta) {
  __shared__ float red[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + tx;
  float s = 0.f;
  if (c < 2 * width)
    for (int p = ty; p < groups; p += 32) s += partial[(int64_t)p * 2 * width + c];
  red[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && c < 2 * width) {
    float t = 0.f;
#pragma unroll
    for (int j = 0; j < 32; ++j) t += red[j][tx];
    if (c < width) {
      if (dgamma != nullptr) dgamma[c] = t;
    } else if (dbeta != nullptr) {
      dbeta[c - width] = t;
    }
  }
}

// lanes of a row's team (0: the loops)
static int ln_team(int64_t width) {
  if (width <= 64 * LN_PER_LANE) return 64;
  if (width <= 256 * LN_PER_LANE) return 256;
  if (width <= 512 * LN_PER_LANE) return 512;
  if (width <= LN_MAX_WIDTH_REG) return 1024;
  return 0;
}

// workgroups of the forward pass: enough to fill the machine, several rows each beyond that
static unsigned ln_fwd_blocks(int64_t rows, int team) {
  const int64_t teams = team == 64 ? (rows + 3) / 4 : rows;
  const int64_t most = team <= 256 ? 2048 : team == 512 ? 1024 : 512;
  return (unsigned)(teams < most ? teams : most);
}

// workgroups of the backward pass = partials of the weight gradients
static int64_t ln_groups(int64_t rows, int64_t width) {
  const int team = ln_team(width);
  if (team == 0) return rows < 64 ? rows : 64;
  const int64_t teams = team == 64 ? (rows + 3) / 4 : rows;
  const int64_t most = team == 64 ? 1024 : team == 256 ? 512 : 256;
  return teams < most ? teams : most;
}

static int ln_check(const aa_layer_norm_desc* d) {
  if (d == nullptr || d->rows <= 0 || d->width <= 0 || d->inner <= 0 || d->x == nullptr)
    return AA_ERR_INVALID;
  if (d->dtype < AA_DT_F32 || d->dtype > AA_DT_F16) return AA_ERR_INVALID;
  if (d->mask_act < AA_ACT_NONE || d->mask_act > AA_ACT_TANH) return AA_ERR_INVALID;
  if (d->width > (1 << 30) || d->rows > VT_MAX_BLOCKS) return AA_ERR_RANGE;
  return AA_OK;
}

static LnArgs ln_args(const aa_layer_norm_desc* d) {
  LnArgs a;
  a.rows = d->rows; a.inner = d->inner; a.width = (int)d->width;
  a.x = d->x; a.x_outer = d->x_outer; a.x_inner = d->x_inner;
  a.dy = d->dy; a.dy_outer = d->dy_outer; a.dy_inner = d->dy_inner;
  a.out = nullptr; a.out_outer = a.out_inner = 0;
  a.gamma = d->gamma; a.beta = d->beta; a.epsilon = d->epsilon; a.stats = d->stats;
  a.partial = nullptr; a.mask_act = d->mask_act;
  return a;
}

template <typename T>
static void ln_launch_fwd(const LnArgs& a, hipStream_t st) {
  constexpr int NCH = LN_PER_LANE / T::C;
  const int team = ln_team(a.width);
  const dim3 grid(ln_fwd_blocks(a.rows, team));
  switch (team) {
    case 64:
      if (a.width <= 64 * LN_PER_LANE / 2)
        aa_layer_norm_fwd_kernel<T, 64, NCH / 2><<<grid, dim3(256), 0, st>>>(a);
      else
        aa_layer_norm_fwd_kernel<T, 64, NCH><<<grid, dim3(256), 0, st>>>(a);
      break;
    case 256: aa_layer_norm_fwd_kernel<T, 256, NCH><<<grid, dim3(256), 0, st>>>(a); break;
    case 512: aa_layer_norm_fwd_kernel<T, 512, NCH><<<grid, dim3(512), 0, st>>>(a); break;
    case 1024: aa_layer_norm_fwd_kernel<T, 1024, NCH><<<grid, dim3(1024), 0, st>>>(a); break;
    default: aa_layer_norm_fwd_wide_kernel<T><<<vt_grid(a.rows), dim3(1024), 0, st>>>(a);
  }
}

template <typename T, bool WEIGHTS>
static void ln_launch_bwd(const LnArgs& a, unsigned groups, hipStream_t st) {
  constexpr int NCH = LN_PER_LANE / T::C;
  switch (ln_team(a.width)) {
    case 64:
      if (a.width <= 64 * LN_PER_LANE / 2)
        aa_layer_norm_bwd_kernel<T, 64, NCH / 2, WEIGHTS><<<dim3(groups), dim3(256), 0, st>>>(a);
      else
        aa_layer_norm_bwd_kernel<T, 64, NCH, WEIGHTS><<<dim3(groups), dim3(256), 0, st>>>(a);
      break;
    case 256:
      aa_layer_norm_bwd_kernel<T, 256, NCH, WEIGHTS><<<dim3(groups), dim3(256), 0, st>>>(a);
      break;
    case 512:
      aa_layer_norm_bwd_kernel<T, 512, NCH, WEIGHTS><<<dim3(groups), dim3(512), 0, st>>>(a);
      break;
    case 1024:
      aa_layer_norm_bwd_kernel<T, 1024, NCH, WEIGHTS><<<dim3(groups), dim3(1024), 0, st>>>(a);
      break;
    default:
      // (the weights first: dx may be stored over x or dy)
      if (WEIGHTS)
        aa_layer_norm_dw_wide_kernel<T><<<dim3((unsigned)((a.width + 255) / 256), groups),
                                          dim3(256), 0, st>>>(a);
      if (a.out != nullptr)
        aa_layer_norm_dx_wide_kernel<T><<<vt_grid(a.rows), dim3(1024), 0, st>>>(a);
  }
}

extern "C" {

int aa_layer_norm_forward(const aa_layer_norm_desc* d, void* stream) {
  const int rc = ln_check(d);
  if (rc != AA_OK) return rc;
  if (d->y == nullptr) return AA_ERR_INVALID;
  LnArgs a = ln_args(d);
  a.out = d->y; a.out_outer = d->y_outer; a.out_inner = d->y_inner;
  hipStream_t st = (hipStream_t)stream;
  if (d->dtype == AA_DT_F32) ln_launch_fwd<VtF32>(a, st);
  else if (d->dtype == AA_DT_BF16) ln_launch_fwd<VtBf16>(a, st);
  else ln_launch_fwd<VtF16>(a, st);
  return aa_launch_status();
}

int64_t aa_layer_norm_backward_workspace_bytes(const aa_layer_norm_desc* d) {
  if (ln_check(d) != AA_OK) return -1;
  if (d->dgamma == nullptr && d->dbeta == nullptr) return 0;
  return ln_groups(d->rows, d->width) * 2 * d->width * (int64_t)sizeof(float);
}

int aa_layer_norm_backward(const aa_layer_norm_desc* d, void* workspace, int64_t workspace_bytes,
                           void* stream) {
  const int rc = ln_check(d);
  if (rc != AA_OK) return rc;
  const bool weights = d->dgamma != nullptr || d->dbeta != nullptr;
  if (d->dy == nullptr || d->stats == nullptr || (d->dx == nullptr && !weights))
    return AA_ERR_INVALID;
  if (weights && (workspace == nullptr ||
                  workspace_bytes < aa_layer_norm_backward_workspace_bytes(d)))
    return AA_ERR_RANGE;
  LnArgs a = ln_args(d);
  a.out = d->dx; a.out_outer = d->dx_outer; a.out_inner = d->dx_inner;
  a.partial = (float*)workspace;
  const unsigned groups = (unsigned)ln_groups(d->rows, d->width);
  hipStream_t st = (hipStream_t)stream;
  if (weights) {
    if (d->dtype == AA_DT_F32) ln_launch_bwd<VtF32, true>(a, groups, st);
    else if (d->dtype == AA_DT_BF16) ln_launch_bwd<VtBf16, true>(a, groups, st);
    else ln_launch_bwd<VtF16, true>(a, groups, st);
    aa_layer_norm_join_kernel<<<dim3((unsigned)((2 * d->width + 31) / 32)), dim3(1024), 0, st>>>(
        a.partial, (int)groups, a.width, d->dgamma, d->dbeta);
  } else {
    if (d->dtype == AA_DT_F32) ln_launch_bwd<VtF32, false>(a, groups, st);
    else if (d->dtype == AA_DT_BF16) ln_launch_bwd<VtBf16, false>(a, groups, st);
    else ln_launch_bwd<VtF16, false>(a, groups, st);
  }
  return aa_launch_status();
}

}  // extern "C"
