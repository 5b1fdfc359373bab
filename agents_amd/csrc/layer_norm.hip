// Layer normalisation over the last axis, forward and backward (keras LayerNormalization).
//   mean = sum x / D;  var = sum (x - mean)^2 / D;  rstd = 1 / sqrt(var + eps);  h = (x - mean) rstd
//   y = h gamma + beta
//   g = dy gamma;  dx = rstd (g - mean(g) - h mean(g h)) * act'(x);  dgamma = sum_rows dy h;
//   dbeta = sum_rows dy
// Everything is held in fp32; x, dy, y and dx are rounded once on their way to memory.  Bound by HBM: a
// row is read once into registers by one team of lanes -- 8 for up to 64 columns, a workgroup for
// thousands --, the mean and the squares about it come from the registers, so the variance has no
// cancellation and the row is not read a second time; a team's next row is in flight meanwhile.
// The weight gradients need every row: a team walks many rows with its columns' sums in registers, the
// teams of a workgroup add theirs in LDS, and a second launch adds the workgroups' partials, all in a
// fixed order (no atomics: same bits every call).  One workgroup of 1,024 lanes per CU: the partials
// cost a write and a read of 8 bytes a column and workgroup, which at 512 workgroups of 256 lanes was
// as much as the rows themselves for 2000 rows of 2048.
// bf16 8192x4096 (67 MB an array): forward 28 .. 30 us, 4.5 TB/s, backward 39 .. 42, 5.0 TB/s, and 5 for
// the join; f32 256x512, by latency: 3.5, 5.7 and 2 us.
// Rows past 8,192 columns have no registers left for the weights' sums: their columns are summed by a
// pass of its own; past 16,384 the rows are walked in loops.
#include <math.h>
#include "common.h"
#include "agents_amd.h"
#include "vec_types.h"
#include "wave_ops.h"

#define LN_FWD_COLUMNS 16384       // columns that a workgroup's registers hold
#define LN_BWD_COLUMNS 8192        // the same beside the weights' sums

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
  float* dgamma;
  float* dbeta;
  int mask_act;
};

// Sums over a team of TEAM lanes in every one of them.  Teams past a wave meet in `red`, each call in
// a half of its own (`turn` alternates): one barrier.  TEAMS teams of a workgroup call in step.
template <int TEAM, int TEAMS>
__device__ static inline void ln_team_sum2(float& a, float& b, float (*red)[2][16], int& turn) {
  a = wv_group_sum<(TEAM < 64 ? TEAM : 64)>(a);
  b = wv_group_sum<(TEAM < 64 ? TEAM : 64)>(b);
  if constexpr (TEAM > 64) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
      red[turn][0][wave] = a;
      red[turn][1][wave] = b;
    }
    __syncthreads();
    const int w0 = TEAMS == 1 ? 0 : wave & ~(TEAM / 64 - 1);
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < TEAM / 64; ++w) {
      a += red[turn][0][w0 + w];
      b += red[turn][1][w0 + w];
    }
    turn ^= 1;
  }
}
template <int TEAM>
__device__ static inline float ln_team_sum(float v, float (*red)[2][16], int& turn) {
  v = wv_group_sum<(TEAM < 64 ? TEAM : 64)>(v);
  if constexpr (TEAM > 64) {       // (one team: the workgroup)
    if ((threadIdx.x & 63) == 0) red[turn][0][threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < TEAM / 64; ++w) v += red[turn][0][w];
    turn ^= 1;
  }
  return v;
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
__global__ void __launch_bounds__(TEAM <= 256 ? 256 : TEAM)
aa_layer_norm_fwd_kernel(LnArgs a) {
  constexpr int C = T::C;
  constexpr int PER = TEAM <= 256 ? 256 / TEAM : 1;        // teams of a workgroup
  static_assert(TEAM <= 64 || PER == 1, "teams that meet a barrier fill the workgroup");
  __shared__ float red[2][2][16];
  int turn = 0;
  const int64_t stride = (int64_t)gridDim.x * PER;
  const int lane = threadIdx.x % TEAM;
  // Teams of one wave stay in step: those past the last row work on it once more, their loop ends
  // with the wave's and they store nothing.
  const int64_t wave0 = (int64_t)blockIdx.x * PER + (TEAM < 64 ? (threadIdx.x & ~63u) / TEAM
                                                               : threadIdx.x / TEAM);
  const int ahead = TEAM < 64 ? (int)(threadIdx.x & 63u) / TEAM : 0;
  if (wave0 >= a.rows) return;     // (the whole workgroup, or a wave that meets no barrier)
  const int64_t last = a.rows - 1;
  const typename T::elem* x = reinterpret_cast<const typename T::elem*>(a.x);
  typename T::elem* out = reinterpret_cast<typename T::elem*>(a.out);
  uint4 next[NCH];
  const int64_t row0 = wave0 + ahead < last ? wave0 + ahead : last;
  ln_load<T, NCH>(x + vt_row(row0, a.inner, a.x_outer, a.x_inner), lane, TEAM, a.width, next);
  float gm[NCH][C], bt[NCH][C];
  ln_load_weight<C, NCH>(a.gamma, lane, TEAM, a.width, 1.f, gm);
  ln_load_weight<C, NCH>(a.beta, lane, TEAM, a.width, 0.f, bt);
  // (A quotient, not a product with 1 / D: one rounding less.  A constant row's y is beta where the sum is
  // exact, as for 2; else its mean is as far off as the sum of its values, a few 2^-24 of their size, and y by
  // that over sqrt(epsilon): 1000 columns of 100.1, epsilon 1e-3: mean 1.5e-5, y 4.9e-4 gamma.)
  const float width = (float)a.width;
  for (int64_t base = wave0; base < a.rows; base += stride) {
    const int64_t row = base + ahead;
    float v[NCH][C];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      T::widen(next[i], v[i]);
#pragma unroll
      for (int j = 0; j < C; ++j) s += v[i][j];
    }
    if (base + stride < a.rows) {
      const int64_t r = row + stride < last ? row + stride : last;
      ln_load<T, NCH>(x + vt_row(r, a.inner, a.x_outer, a.x_inner), lane, TEAM, a.width, next);
    }
    const float mean = ln_team_sum<TEAM>(s, red, turn) / width;
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
    const float var = ln_team_sum<TEAM>(ss, red, turn) / width;
    const float rstd = 1.f / sqrtf(var + a.epsilon);
    if (row > last) continue;
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

// one chunk of a row as fp32 (0 past its end)
template <typename T>
__device__ static inline void ln_chunk(const typename T::elem* x, int c, int width, float (&v)[T::C]) {
  if (c + T::C <= width) T::widen(vt_load16(x + c), v);
  else vt_load_part<T>(x + c, width - c, 0.f, v);
}
template <typename T>
__device__ static inline void ln_put(typename T::elem* y, int c, int width, const float (&v)[T::C]) {
  if (c + T::C <= width) vt_store16(y + c, T::pack(v));
  else vt_store_part<T>(y + c, width - c, v);
}

// rows wider than the registers hold: a workgroup per row, three passes
template <typename T>
__global__ void __launch_bounds__(1024) aa_layer_norm_fwd_wide_kernel(LnArgs a) {
  constexpr int C = T::C;
  __shared__ float red[2][2][16];
  int turn = 0;
  const int64_t row = vt_block();
  if (row >= a.rows) return;
  const typename T::elem* x = reinterpret_cast<const typename T::elem*>(a.x) +
                              vt_row(row, a.inner, a.x_outer, a.x_inner);
  typename T::elem* y = reinterpret_cast<typename T::elem*>(a.out) +
                        vt_row(row, a.inner, a.out_outer, a.out_inner);
  const float width = (float)a.width;
  float s = 0.f;
  for (int c = threadIdx.x * C; c < a.width; c += 1024 * C) {
    float v[C];
    ln_chunk<T>(x, c, a.width, v);
#pragma unroll
    for (int j = 0; j < C; ++j) s += v[j];
  }
  const float mean = ln_team_sum<1024>(s, red, turn) / width;
  float ss = 0.f;
  for (int c = threadIdx.x * C; c < a.width; c += 1024 * C) {
    float v[C];
    ln_chunk<T>(x, c, a.width, v);
#pragma unroll
    for (int j = 0; j < C; ++j) ss += c + j < a.width ? (v[j] - mean) * (v[j] - mean) : 0.f;
  }
  const float rstd = 1.f / sqrtf(ln_team_sum<1024>(ss, red, turn) / width + a.epsilon);
  if (threadIdx.x == 0 && a.stats != nullptr) {
    a.stats[2 * row] = mean;
    a.stats[2 * row + 1] = rstd;
  }
  for (int c = threadIdx.x * C; c < a.width; c += 1024 * C) {
    float v[C], gm[1][C], bt[1][C];
    ln_chunk<T>(x, c, a.width, v);
    ln_load_weight<C, 1>(a.gamma, c / C, 0, a.width, 1.f, gm);
    ln_load_weight<C, 1>(a.beta, c / C, 0, a.width, 0.f, bt);
#pragma unroll
    for (int j = 0; j < C; ++j) v[j] = (v[j] - mean) * rstd * gm[0][j] + bt[0][j];
    ln_put<T>(y, c, a.width, v);
  }
}

__device__ static inline float ln_act_grad(float y, int kind) {
  if (kind == AA_ACT_RELU) return y > 0.f ? 1.f : 0.f;
  if (kind == AA_ACT_TANH) return 1.f - y * y;
  return 1.f;
}

// Workgroups of 1,024 lanes = PER teams, each a row at a time.
template <typename T, int TEAM, int NCH, bool WEIGHTS>
__global__ void __launch_bounds__(1024) aa_layer_norm_bwd_kernel(LnArgs a) {
  constexpr int C = T::C;
  constexpr int PER = 1024 / TEAM;
  // gamma and the next row in registers: 128 registers a lane hold them beside the sums of 8 columns (110 ..
  // 127 are used; teams of 512 need a few more and leave 9 values in fp16, 3 in fp32, in scratch memory)
  constexpr bool AHEAD = NCH * C <= 8;
  constexpr int COLS = TEAM * NCH * C;           // columns of a team
  constexpr int UNIT = TEAM < 64 ? 64 : TEAM;    // lanes that hold one set of sums at the end
  constexpr int UNITS = 1024 / UNIT;
  __shared__ float red[2][2][16];
  __shared__ float sums[WEIGHTS && UNITS > 1 ? UNITS / 2 : 1][2][WEIGHTS && UNITS > 1 ? COLS : 1];
  int turn = 0;
  const int sub = threadIdx.x / TEAM, lane = threadIdx.x % TEAM;
  const float inv = 1.f / (float)a.width;
  const int64_t row0 = (int64_t)blockIdx.x * PER, stride = (int64_t)gridDim.x * PER;
  const typename T::elem* x = reinterpret_cast<const typename T::elem*>(a.x);
  const typename T::elem* dy = reinterpret_cast<const typename T::elem*>(a.dy);
  uint4 nx[NCH], nd[NCH];          // the next row; zeros past the last one, which add nothing
  float nmean, nrstd;
  auto fetch = [&](int64_t r) {
    nmean = nrstd = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) nx[i] = nd[i] = make_uint4(0u, 0u, 0u, 0u);
    if (r < a.rows) {
      ln_load<T, NCH>(x + vt_row(r, a.inner, a.x_outer, a.x_inner), lane, TEAM, a.width, nx);
      ln_load<T, NCH>(dy + vt_row(r, a.inner, a.dy_outer, a.dy_inner), lane, TEAM, a.width, nd);
      nmean = a.stats[2 * r];
      nrstd = a.stats[2 * r + 1];
    }
  };
  if (AHEAD) fetch(row0 + sub);
  float gm[NCH][C], dg[NCH][C], db[NCH][C];
  if (AHEAD) ln_load_weight<C, NCH>(a.gamma, lane, TEAM, a.width, 1.f, gm);
#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int j = 0; j < C; ++j) dg[i][j] = db[i][j] = 0.f;
  for (int64_t base = row0; base < a.rows; base += stride) {       // (workgroup-uniform)
    const int64_t row = base + sub;
    if (!AHEAD) {
      fetch(row);
      ln_load_weight<C, NCH>(a.gamma, lane, TEAM, a.width, 1.f, gm);
    }
    uint4 qx[NCH], qd[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) { qx[i] = nx[i]; qd[i] = nd[i]; }
    const float mean = nmean, rstd = nrstd;
    if (AHEAD && base + stride < a.rows) fetch(row + stride);
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
    ln_team_sum2<TEAM, PER>(c1, c2, red, turn);
    c1 *= inv;
    c2 *= inv;
    if (a.out != nullptr && row < a.rows) {
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
        if (c < a.width) ln_put<T>(dx, c, a.width, r);
      }
    }
  }
  if constexpr (WEIGHTS) {
    // teams of a wave, then the units of the workgroup in halves
    if constexpr (TEAM < 64) {
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int j = 0; j < C; ++j) {
          const auto add = [](float p, float q) { return p + q; };
          if constexpr (TEAM <= 8) {      // (lane ^ 8: a row rotated by half of it)
            dg[i][j] += __uint_as_float(wv_xor<8>(__float_as_uint(dg[i][j]), 0));
            db[i][j] += __uint_as_float(wv_xor<8>(__float_as_uint(db[i][j]), 0));
          }
          if constexpr (TEAM <= 16) {
            dg[i][j] = wv_step<16>(dg[i][j], add);
            db[i][j] = wv_step<16>(db[i][j], add);
          }
          dg[i][j] = wv_step<32>(dg[i][j], add);
          db[i][j] = wv_step<32>(db[i][j], add);
        }
    }
    const int unit = threadIdx.x / UNIT;
    const bool speaks = TEAM >= 64 || (threadIdx.x & 63) < TEAM;
#pragma unroll
    for (int half = UNITS / 2; half >= 1; half >>= 1) {
      if (unit >= half && unit < 2 * half && speaks) {
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
          for (int j = 0; j < C; j += 4) {
            *(float4*)&sums[unit - half][0][(lane + i * TEAM) * C + j] =
                make_float4(dg[i][j], dg[i][j + 1], dg[i][j + 2], dg[i][j + 3]);
            *(float4*)&sums[unit - half][1][(lane + i * TEAM) * C + j] =
                make_float4(db[i][j], db[i][j + 1], db[i][j + 2], db[i][j + 3]);
          }
      }
      __syncthreads();
      if (unit < half && speaks) {
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
          for (int j = 0; j < C; j += 4) {
            const float4 g = *(const float4*)&sums[unit][0][(lane + i * TEAM) * C + j];
            const float4 b = *(const float4*)&sums[unit][1][(lane + i * TEAM) * C + j];
            dg[i][j] += g.x; dg[i][j + 1] += g.y; dg[i][j + 2] += g.z; dg[i][j + 3] += g.w;
            db[i][j] += b.x; db[i][j + 1] += b.y; db[i][j + 2] += b.z; db[i][j + 3] += b.w;
          }
      }
      __syncthreads();
    }
    if (unit == 0 && speaks) {
      // (as 16-byte stores: single floats, 32 bytes apart, took 13 us of 33 for 1000x8192)
      float* og = a.partial + (int64_t)blockIdx.x * 2 * a.width;
      float* ob = og + a.width;
      if (gridDim.x == 1) {        // nothing to join
        og = a.dgamma;
        ob = a.dbeta;
      }
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int j = 0; j < C; j += 4) {
          const int c = (lane + i * TEAM) * C + j;
          const float g[4] = {dg[i][j], dg[i][j + 1], dg[i][j + 2], dg[i][j + 3]};
          const float b[4] = {db[i][j], db[i][j + 1], db[i][j + 2], db[i][j + 3]};
          if (c < a.width) {
            if (og != nullptr) ln_put<VtF32>(og, c, a.width, g);
            if (ob != nullptr) ln_put<VtF32>(ob, c, a.width, b);
          }
        }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(1024) aa_layer_norm_dx_wide_kernel(LnArgs a) {
  constexpr int C = T::C;
  __shared__ float red[2][2][16];
  int turn = 0;
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
  for (int c = threadIdx.x * C; c < a.width; c += 1024 * C) {
    float xv[C], dv[C], gm[1][C];
    ln_chunk<T>(x, c, a.width, xv);
    ln_chunk<T>(dy, c, a.width, dv);
    ln_load_weight<C, 1>(a.gamma, c / C, 0, a.width, 1.f, gm);
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const float g = dv[j] * gm[0][j];
      c1 += g;
      c2 += g * ((xv[j] - mean) * rstd);
    }
  }
  ln_team_sum2<1024, 1>(c1, c2, red, turn);
  c1 *= inv;
  c2 *= inv;
  for (int c = threadIdx.x * C; c < a.width; c += 1024 * C) {
    float xv[C], dv[C], gm[1][C];
    ln_chunk<T>(x, c, a.width, xv);
    ln_chunk<T>(dy, c, a.width, dv);
    ln_load_weight<C, 1>(a.gamma, c / C, 0, a.width, 1.f, gm);
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const float h = (xv[j] - mean) * rstd;
      dv[j] = rstd * (dv[j] * gm[0][j] - c1 - h * c2);
      if (a.mask_act != AA_ACT_NONE) dv[j] *= ln_act_grad(xv[j], a.mask_act);
    }
    ln_put<T>(dx, c, a.width, dv);
  }
}

// weight gradients of wide rows: a lane owns a chunk of columns, grid = (column blocks, row groups)
template <typename T>
__global__ void __launch_bounds__(256) aa_layer_norm_dw_wide_kernel(LnArgs a) {
  constexpr int C = T::C, U = 4;
  const int c = (blockIdx.x * 256 + threadIdx.x) * C;
  if (c >= a.width) return;
  const typename T::elem* x = reinterpret_cast<const typename T::elem*>(a.x) + c;
  const typename T::elem* dy = reinterpret_cast<const typename T::elem*>(a.dy) + c;
  float dg[C], db[C];
#pragma unroll
  for (int j = 0; j < C; ++j) dg[j] = db[j] = 0.f;
  for (int64_t row = blockIdx.y; row < a.rows; row += (int64_t)U * gridDim.y) {
    float xv[U][C], dv[U][C];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = row + (int64_t)u * gridDim.y;
#pragma unroll
      for (int j = 0; j < C; ++j) xv[u][j] = dv[u][j] = 0.f;
      if (r < a.rows) {
        ln_chunk<T>(x + vt_row(r, a.inner, a.x_outer, a.x_inner), 0, a.width - c, xv[u]);
        ln_chunk<T>(dy + vt_row(r, a.inner, a.dy_outer, a.dy_inner), 0, a.width - c, dv[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = row + (int64_t)u * gridDim.y;
      if (r >= a.rows) break;
      const float mean = a.stats[2 * r], rstd = a.stats[2 * r + 1];
#pragma unroll
      for (int j = 0; j < C; ++j) {
        dg[j] += dv[u][j] * ((xv[u][j] - mean) * rstd);
        db[j] += dv[u][j];
      }
    }
  }
  float* og = a.partial + (int64_t)blockIdx.y * 2 * a.width;
  float* ob = og + a.width;
  if (gridDim.y == 1) {            // nothing to join
    og = a.dgamma;
    ob = a.dbeta;
  }
#pragma unroll
  for (int j = 0; j < C; j += 4) {
    const float g[4] = {dg[j], dg[j + 1], dg[j + 2], dg[j + 3]};
    const float b[4] = {db[j], db[j + 1], db[j + 2], db[j + 3]};
    if (c + j < a.width) {
      if (og != nullptr) ln_put<VtF32>(og, c + j, a.width, g);
      if (ob != nullptr) ln_put<VtF32>(ob, c + j, a.width, b);
    }
  }
}

// sums of the partials' columns: 32 columns x 32 lanes along the partials per workgroup
__global__ void __launch_bounds__(1024)
aa_layer_norm_join_kernel(const float* __restrict__ partial, int groups, int width,
                          float* __restrict__ dgamma, float* __restrict__ dbeta) {
  __shared__ float red[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + tx;
  float s = 0.f;
  if (c < 2 * width) {
    const float* q = partial + c;
    int p = ty;
    for (; p + 7 * 32 < groups; p += 8 * 32) {       // (eight loads in flight)
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = q[(int64_t)(p + 32 * i) * 2 * width];
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[i];
    }
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = p + 32 * i < groups ? q[(int64_t)(p + 32 * i) * 2 * width] : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += v[i];
  }
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

// lanes of a row's team, forward (0: the loops)
static int ln_fwd_team(int64_t width) {
  if (width <= 64) return 8;
  if (width <= 256) return 32;
  if (width <= 1024) return 64;
  if (width <= 4096) return 256;
  if (width <= 8192) return 512;
  return width <= LN_FWD_COLUMNS ? 1024 : 0;
}

// workgroups of the forward pass: enough to fill the machine, several rows each beyond that
static unsigned ln_fwd_blocks(int64_t rows, int team) {
  const int per = team <= 256 ? 256 / team : 1;
  const int64_t teams = (rows + per - 1) / per;
  const int64_t most = team <= 256 ? 2048 : team == 512 ? 1024 : 256;
  return (unsigned)(teams < most ? teams : most);
}

// lanes of a row's team, backward: 8 columns each (0: two passes)
static int ln_bwd_team(int64_t width) {
  if (width > LN_BWD_COLUMNS) return 0;
  int team = 8;
  while (team * 8 < width) team *= team == 8 ? 4 : 2;
  return team;
}

// workgroups of the backward pass = partials of the weight gradients: one per CU at most, and no more
// than share the rounds evenly
static int64_t ln_groups(int64_t rows, int64_t width) {
  const int team = ln_bwd_team(width);
  if (team == 0) {
    // row groups of the columns' pass, 32 .. 128: f16 2000x12000 backward 86 us at 64, 71 at 128;
    // f32 200x9000 18 at 64, 21 at 128.  Few rows: one group, which needs no launch to join it (one
    // group | a group a row: f32 4x9001 9.2 | 11.0 us, 4x65536 20 | 29, 16x65536 23 | 34; the other
    // way round for bf16 8x9001 13.5 | 11.8, 16x16384 15 | 12, 64x65536 68 | 42).  Between 16,384 and
    // 65,536 columns, where the rule goes from 4 rows to 16, nothing was measured, nor a size in both types.
    if (rows <= (width < 65536 ? 4 : 16)) return 1;
    const int64_t want = rows / 8 < 32 ? 32 : rows / 8 > 128 ? 128 : rows / 8;
    return rows < want ? rows : want;
  }
  const int64_t sets = (rows + 1024 / team - 1) / (1024 / team);
  // two rounds of one workgroup cost less than the launch that would join two (one | joined, bf16: two
  // rounds 32x512 5.8 | 6.5 us, 4x4096 6.1 | 6.9; three 48x512 7.0 | 6.8, 6x4096 7.5 | 6.8)
  if (sets <= 2) return 1;
  const int64_t rounds = (sets + 255) / 256;
  return (sets + rounds - 1) / rounds;
}

static int ln_check(const aa_layer_norm_desc* d) {
  if (d == nullptr || d->rows <= 0 || d->width <= 0 || d->inner <= 0 || d->x == nullptr)
    return AA_ERR_INVALID;
  if (d->dtype < AA_DT_F32 || d->dtype > AA_DT_F16) return AA_ERR_INVALID;
  if (d->mask_act < AA_ACT_NONE || d->mask_act > AA_ACT_TANH) return AA_ERR_INVALID;
  if (d->width > (1 << 29) || d->rows > VT_MAX_BLOCKS) return AA_ERR_RANGE;
  return AA_OK;
}

// whether the weights' gradients pass through partials
static bool ln_joins(const aa_layer_norm_desc* d) {
  return ln_groups(d->rows, d->width) > 1;
}

static LnArgs ln_args(const aa_layer_norm_desc* d) {
  LnArgs a;
  a.rows = d->rows; a.inner = d->inner; a.width = (int)d->width;
  a.x = d->x; a.x_outer = d->x_outer; a.x_inner = d->x_inner;
  a.dy = d->dy; a.dy_outer = d->dy_outer; a.dy_inner = d->dy_inner;
  a.out = nullptr; a.out_outer = a.out_inner = 0;
  a.gamma = d->gamma; a.beta = d->beta; a.epsilon = d->epsilon; a.stats = d->stats;
  a.partial = nullptr; a.dgamma = d->dgamma; a.dbeta = d->dbeta; a.mask_act = d->mask_act;
  return a;
}

template <typename T>
static void ln_launch_fwd(const LnArgs& a, hipStream_t st) {
  constexpr int N8 = 8 / T::C, N16 = 16 / T::C;       // chunks of a lane
  const int team = ln_fwd_team(a.width);
  const dim3 grid(team != 0 ? ln_fwd_blocks(a.rows, team) : 1);
  switch (team) {
    case 8: aa_layer_norm_fwd_kernel<T, 8, N8><<<grid, dim3(256), 0, st>>>(a); break;
    case 32: aa_layer_norm_fwd_kernel<T, 32, N8><<<grid, dim3(256), 0, st>>>(a); break;
    case 64:
      if (a.width <= 512) aa_layer_norm_fwd_kernel<T, 64, N8><<<grid, dim3(256), 0, st>>>(a);
      else aa_layer_norm_fwd_kernel<T, 64, N16><<<grid, dim3(256), 0, st>>>(a);
      break;
    case 256: aa_layer_norm_fwd_kernel<T, 256, N16><<<grid, dim3(256), 0, st>>>(a); break;
    case 512: aa_layer_norm_fwd_kernel<T, 512, N16><<<grid, dim3(512), 0, st>>>(a); break;
    case 1024: aa_layer_norm_fwd_kernel<T, 1024, N16><<<grid, dim3(1024), 0, st>>>(a); break;
    default: aa_layer_norm_fwd_wide_kernel<T><<<vt_grid(a.rows), dim3(1024), 0, st>>>(a);
  }
}

template <typename T, bool WEIGHTS>
static void ln_launch_bwd(const LnArgs& a, unsigned groups, hipStream_t st) {
  constexpr int N8 = 8 / T::C, N16 = 16 / T::C;
  const dim3 grid(groups), block(1024);
  switch (ln_bwd_team(a.width)) {
    case 8: aa_layer_norm_bwd_kernel<T, 8, N8, WEIGHTS><<<grid, block, 0, st>>>(a); break;
    case 32: aa_layer_norm_bwd_kernel<T, 32, N8, WEIGHTS><<<grid, block, 0, st>>>(a); break;
    case 64: aa_layer_norm_bwd_kernel<T, 64, N8, WEIGHTS><<<grid, block, 0, st>>>(a); break;
    case 128: aa_layer_norm_bwd_kernel<T, 128, N8, WEIGHTS><<<grid, block, 0, st>>>(a); break;
    case 256: aa_layer_norm_bwd_kernel<T, 256, N8, WEIGHTS><<<grid, block, 0, st>>>(a); break;
    case 512: aa_layer_norm_bwd_kernel<T, 512, N8, WEIGHTS><<<grid, block, 0, st>>>(a); break;
    case 1024: aa_layer_norm_bwd_kernel<T, 1024, N8, WEIGHTS><<<grid, block, 0, st>>>(a); break;
    default:
      // (the weights first: dx may be stored over x or dy)
      if (WEIGHTS) {
        const unsigned blocks = (unsigned)((a.width + 256 * T::C - 1) / (256 * T::C));
        aa_layer_norm_dw_wide_kernel<T><<<dim3(blocks, groups), dim3(256), 0, st>>>(a);
      }
      if (a.out == nullptr) break;
      if (a.width <= LN_FWD_COLUMNS)
        aa_layer_norm_bwd_kernel<T, 1024, N16, false>
            <<<dim3((unsigned)(a.rows < 512 ? a.rows : 512)), block, 0, st>>>(a);
      else
        aa_layer_norm_dx_wide_kernel<T><<<vt_grid(a.rows), block, 0, st>>>(a);
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
  if (!ln_joins(d)) return 0;
  return ln_groups(d->rows, d->width) * 2 * d->width * (int64_t)sizeof(float);
}

int aa_layer_norm_backward(const aa_layer_norm_desc* d, void* workspace, int64_t workspace_bytes,
                           void* stream) {
  const int rc = ln_check(d);
  if (rc != AA_OK) return rc;
  const bool weights = d->dgamma != nullptr || d->dbeta != nullptr;
  if (d->dy == nullptr || d->stats == nullptr || (d->dx == nullptr && !weights))
    return AA_ERR_INVALID;
  const bool joins = weights && ln_joins(d);
  if (joins && (workspace == nullptr ||
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
    if (joins)
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
