// Log-probabilities of given actions (tokens) of Categorical(logits / temperature), with the entropy
// and the most likely alternatives, and the gradient with respect to the logits.
//   x = logits, -inf where the mask excludes an action;  c = 1 / temperature;  m: a reference of the row
//   S = sum exp(c (x - m));   ln p_v = c (x_v - m) - ln S;   H = ln S - c sum exp(c (x - m)) (x - m) / S
//   d x_v = c [ g (1{v = a} - p_v) - h p_v (ln p_v + H) ]        (g = d log_prob, h = d entropy)
// One pass over a row: every lane keeps a reference r, S and sum e (x - r) relative to it, and moves r
// only when a chunk exceeds it by CAT_MARGIN powers of two (exp never overflows, the sums lose nothing:
// they are floating point); the lanes' triples are joined at the end.  Entropy is formed from
// differences to the reference, never from two large numbers.  All sums are fp32.
// The alternatives ride in the same pass: a wave keeps its 64 best keys (value, then lower index)
// sorted across its lanes, a chunk whose maximum stays below the k-th costs one comparison, the others
// collect in LDS and are merged 64 at a time by a bitonic network.
// Bound by HBM for vocabularies (268 MB of bf16, 4096x32768: forward 56 .. 60 us, 4.5 TB/s; gradient,
// which reads and writes them, 82 .. 85 us, 6.4 TB/s; f16 2044x50001, 204 MB, 43 .. 46 and 64 .. 66),
// by launch and latency for a few actions (f32 4096x18 with an int32 mask: 3.6 and 4.0 us).  Few rows:
// a row is split over workgroups and the parts joined by a second launch (bf16 1x131072 with 20
// alternatives: 8.8 + 4.2 us).
#include <math.h>
#include "common.h"
#include "agents_amd.h"
#include "vec_types.h"
#include "wave_ops.h"

#define CAT_MARGIN 4.f             // powers of two a value may exceed its lane's reference by
#define CAT_LOWEST (-3.402823466e+38f)
#define CAT_LOG2E 1.4426950408889634f
#define CAT_LN2 0.6931471805599453f
#define CAT_FEW 512                // up to here a row is held in registers
#define CAT_WAVE_VOCAB 4096        // up to here a wave takes a row, beyond a workgroup
#define CAT_SPLIT_ROWS 256         // (one workgroup a CU)
#define CAT_SPLIT_BLOCKS 1024      // workgroups that fill the machine
// A gradient of this many bytes is stored past the caches: with the logits it exceeds the 256 MB of the
// memory-side cache, and its dirty lines would be written back under the next reads.  Forward and
// gradient of bf16 rows of 32768, us a pass, and with a copy of the gradient behind it:
// 134 MB 84.7 -> 71.0 (137 -> 126), 268 MB 160 -> 132 (259 -> 245); below it costs the reader:
// 101 MB 58.6 -> 55.4 (88 -> 99), 67 MB 38.0 -> 37.8 (59 -> 64).
#define CAT_PAST_CACHE (128ll << 20)
#define CAT_EMPTY_KEY 0x007fffffffffffffull   // key of -inf: no alternative

typedef unsigned long long u64;

struct CatArgs {
  int64_t rows, inner;
  int vocab;
  const void* logits; int64_t x_outer, x_inner;
  const void* actions; int64_t a_outer, a_inner, first_action;
  int action_bytes, no_padding;
  const void* mask; int64_t k_outer, k_inner;
  float inv_t;                     // 1 / temperature
  int top_k;
  float* log_prob;
  float* entropy;
  float* stats;                    // [rows][2]: reference, ln S ((0, +inf) for a row without a distribution)
  int64_t* top_ids;
  float* top_log_prob;
  int splits;                      // parts of a row
  float* part;                     // [rows][splits][4]
  u64* part_keys;                  // [rows][top_k][splits]
};

struct CatSum {
  float r, s, t;
};

__device__ static inline float cat_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// moves `a` to the reference `to` (at or above a.r); a part whose weight vanishes leaves no trace
// (its t may be infinite there), a NaN stays in s
__device__ static inline CatSum cat_move(CatSum a, float to, float c2) {
  const float d = fmaxf(a.r - to, CAT_LOWEST);
  const float w = cat_exp2((a.r - to) * c2);
  CatSum o;
  o.r = to;
  o.s = a.r == to ? a.s : a.s * w;
  o.t = a.r == to ? a.t : w > 0.f ? w * (a.t + d * a.s) : 0.f;
  return o;
}

__device__ static inline CatSum cat_join(CatSum a, CatSum b, float c2) {
  const float to = fmaxf(a.r, b.r);
  a = cat_move(a, to, c2);
  b = cat_move(b, to, c2);
  a.s += b.s;
  a.t += b.t;
  return a;
}

// the triples of a wave's lanes, in every lane
__device__ static inline CatSum cat_wave_join(CatSum a, float c2) {
  a = cat_move(a, wv_max(a.r), c2);
  a.s = wv_sum(a.s);
  a.t = wv_sum(a.t);
  return a;
}

// ---- alternatives: keys that order as (value, then lower index) ---------------------------------
__device__ static inline u64 cat_key(float v, int index) {
  const unsigned b = __float_as_uint(v + 0.f);             // -0 counts as 0
  const unsigned hi = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return ((u64)hi << 32) | (unsigned)~index;
}
__device__ static inline float cat_key_value(u64 k) {
  const unsigned hi = (unsigned)(k >> 32);
  return __uint_as_float((hi & 0x80000000u) ? (hi & 0x7fffffffu) : ~hi);
}
__device__ static inline int cat_key_index(u64 k) { return (int)~(unsigned)k; }

__device__ static inline u64 cat_lane(u64 v, int from) {       // `from` is wave-uniform
  const unsigned lo = __builtin_amdgcn_readlane((int)(unsigned)v, from);
  const unsigned hi = __builtin_amdgcn_readlane((int)(unsigned)(v >> 32), from);
  return ((u64)hi << 32) | lo;
}

struct CatTop {
  u64 list;          // this lane's place of the wave's best 64, descending (0: none yet)
  u64 bar;           // a key must exceed it (wave-uniform)
  float low;         // its value
  int held;          // keys waiting in `buf` (wave-uniform)
  bool sorted;       // `list` holds keys (wave-uniform)
  u64* buf;          // LDS of this wave's own: 64 keys and what is offered between two flushes
};

__device__ static inline CatTop cat_top(u64* buf) {
  return CatTop{0ull, CAT_EMPTY_KEY, -INFINITY, 0, false, buf};
}

__device__ static inline void cat_top_raise(CatTop& t, u64 bar) {
  if (bar > t.bar) {
    t.bar = bar;
    t.low = cat_key_value(bar);
  }
}

__device__ static inline void cat_wave_fence() {
  // LDS of one wave: executed in order, the compiler must keep it so
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// the newest up to 64 waiting keys join the list
__device__ static inline void cat_top_flush(CatTop& t, int lane, int k) {
  const int n = t.held < 64 ? t.held : 64;
  cat_wave_fence();
  const u64 cand = lane < n ? t.buf[t.held - n + lane] : 0ull;
  t.held -= n;
  cat_wave_fence();
  const u64 order = wv_sort_desc(cand, lane, t.sorted);      // ascending for the merge
  t.list = t.sorted ? wv_merge_desc(t.list, order, lane) : order;
  t.sorted = true;
  cat_top_raise(t, cat_lane(t.list, k - 1));
}

__device__ static inline void cat_top_offer_key(CatTop& t, u64 key, int lane) {
  const bool in = key > t.bar;
  const u64 b = __ballot(in);
  if (b == 0ull) return;
  if (in) t.buf[t.held + __popcll(b & ((1ull << lane) - 1ull))] = key;
  t.held += __popcll(b);
}

// (a comparison of values first: most places hold no candidate; a NaN is none)
__device__ static inline void cat_top_offer(CatTop& t, float v, int index, int lane) {
  if (__any(v >= t.low)) cat_top_offer_key(t, v >= t.low ? cat_key(v, index) : 0ull, lane);
}

// ---- the row's end: log_prob, entropy, stats, alternatives -----------------------------------------
template <int MB>
__device__ static inline bool cat_allowed(const void* mask, int64_t at) {
  if (MB == 1) return reinterpret_cast<const uint8_t*>(mask)[at] != 0;
  if (MB == 4) return reinterpret_cast<const int32_t*>(mask)[at] != 0;
  return true;
}

// a row's index of an action; negative: a padding row
__device__ static inline int64_t cat_action(const CatArgs& a, int64_t row) {
  if (a.actions == nullptr) return 0;
  const int64_t at = vt_row(row, a.inner, a.a_outer, a.a_inner);
  const int64_t v = a.action_bytes == 8 ? reinterpret_cast<const int64_t*>(a.actions)[at]
                                        : (int64_t)reinterpret_cast<const int32_t*>(a.actions)[at];
  // (compared first: the difference may need a 65th bit)
  if (v < a.first_action) return a.no_padding ? (int64_t)a.vocab : -1;
  const uint64_t index = (uint64_t)v - (uint64_t)a.first_action;
  return index < (uint64_t)a.vocab ? (int64_t)index : (int64_t)a.vocab;
}

// the action's logit, -inf where it is masked (read before the row, so that nothing waits for it)
template <typename T, int MB>
__device__ static inline float cat_action_logit(const CatArgs& a, int64_t row, int64_t action) {
  if (action < 0 || action >= a.vocab) return 0.f;
  const float x = T::one(reinterpret_cast<const typename T::elem*>(
      a.logits)[vt_row(row, a.inner, a.x_outer, a.x_inner) + action]);
  return cat_allowed<MB>(a.mask, vt_row(row, a.inner, a.k_outer, a.k_inner) + action) ? x
                                                                                     : -INFINITY;
}

__device__ static inline float cat_nan() { return __uint_as_float(0x7fc00000u); }

// one lane: everything of a row but its alternatives; returns ln S (+inf: no distribution)
// (the reference may lie CAT_MARGIN powers of two below the row's maximum, so the value of an action that
// is all but certain is a difference of two numbers of up to 2.8: off by some 2e-7, on either side of 0)
__device__ static inline float cat_finish(const CatArgs& a, int64_t row, int64_t action, float x,
                                          CatSum u) {
  const bool empty = u.s == 0.f;
  const float ls = empty ? INFINITY : logf(u.s);
  if (a.stats != nullptr) {
    a.stats[2 * row] = empty ? 0.f : u.r;
    a.stats[2 * row + 1] = ls;
  }
  if (a.entropy != nullptr) a.entropy[row] = empty ? 0.f : ls - a.inv_t * (u.t / u.s);
  if (a.log_prob != nullptr)
    a.log_prob[row] = action >= a.vocab ? cat_nan()
                      : empty           ? -INFINITY
                                        : (x - u.r) * a.inv_t - ls;
  return ls;
}

// one wave: the row's alternatives from the sorted list
__device__ static inline void cat_write_top(const CatArgs& a, int64_t row, int lane, u64 key, float r,
                                            float ls) {
  if (lane >= a.top_k) return;
  const bool real = key > CAT_EMPTY_KEY && !isnan(ls);
  a.top_ids[row * a.top_k + lane] = real ? cat_key_index(key) : -1;
  a.top_log_prob[row * a.top_k + lane] =
      real ? (cat_key_value(key) - r) * a.inv_t - ls : isnan(ls) ? ls : -INFINITY;
}

// a padding row (negative action): its logits are not used (the first tile of them, for few actions the
// row, is on its way before the action is known)
__device__ static inline void cat_pad_row(const CatArgs& a, int64_t row, int lane) {
  if (lane == 0) {
    a.log_prob[row] = 0.f;
    if (a.entropy != nullptr) a.entropy[row] = 0.f;
    if (a.stats != nullptr) {
      a.stats[2 * row] = 0.f;
      a.stats[2 * row + 1] = INFINITY;
    }
  }
  if (lane < a.top_k) {
    a.top_ids[row * a.top_k + lane] = -1;
    a.top_log_prob[row * a.top_k + lane] = -INFINITY;
  }
}

// U chunks of a lane, TEAM apart, and their masks: all loads in flight together
template <typename T, int MB, int U>
struct CatTile {
  static constexpr int C = T::C;
  static constexpr int W = MB == 0 ? 1 : MB * C / 4;       // mask words of a chunk
  uint4 q[U];
  unsigned m[U][W];
};

// `kb`: its wave's first chunk; chunks from k1 on read as -inf
template <typename T, int MB, int U, int TEAM>
__device__ static inline void cat_load(const typename T::elem* x, const uint8_t* mk, int kb, int lane,
                                       int k1, int skew, CatTile<T, MB, U>& t) {
  constexpr int C = T::C;
  const int e0 = (kb + lane) * C - skew;
  if (kb + (U - 1) * TEAM + 64 <= k1) {                    // (wave-uniform: all there)
#pragma unroll
    for (int u = 0; u < U; ++u) {
      t.q[u] = vt_load16(x + e0 + u * TEAM * C);
      if (MB != 0) __builtin_memcpy(t.m[u], mk + (int64_t)MB * (e0 + u * TEAM * C), MB * C);
    }
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned w = T::LOWEST_WORD;
      t.q[u] = make_uint4(w, w, w, w);
      if (kb + lane + u * TEAM < k1) {
        t.q[u] = vt_load16(x + e0 + u * TEAM * C);
        if (MB != 0) __builtin_memcpy(t.m[u], mk + (int64_t)MB * (e0 + u * TEAM * C), MB * C);
      }
    }
  }
}

// chunk u as fp32, -inf where it is masked
template <typename T, int MB, int U>
__device__ static inline void cat_values(const CatTile<T, MB, U>& t, int u, float (&v)[T::C]) {
  T::widen(t.q[u], v);
#pragma unroll
  for (int j = 0; j < T::C; ++j) {
    if (MB == 1 && ((t.m[u][j / 4] >> (8 * (j % 4))) & 0xffu) == 0u) v[j] = -INFINITY;
    if (MB == 4 && t.m[u][j] == 0u) v[j] = -INFINITY;
  }
}

// a value into the sums of its lane
__device__ static inline void cat_add(CatSum& u, float v, float c2) {
  const float d = v - u.r;
  const float e = cat_exp2(d * c2);
  u.s += e;
  u.t = fmaf(e, fmaxf(d, CAT_LOWEST), u.t);
}

// TEAM = 64: a wave per row, four rows per workgroup.  TEAM = 256: a workgroup per part of a row.
template <typename T, int MB, int TEAM, bool TOP>
__global__ void __launch_bounds__(256) aa_categorical_kernel(CatArgs a) {
  // Two chunks a tile without alternatives (registers for seven waves a SIMD: bf16 30000x2000 30 -> 27
  // us, f16 2044x50001 48.6 -> 46.7 against four); four with them, where a tile's first look at its
  // candidates is what costs (bf16 2044x50001 with 20: 66 against 71).  Reading a row from a tile that
  // depends on the row, so that rows of a power of two bytes spread over the channels, gained nothing.
  constexpr int C = T::C, U = MB == 4 || !TOP ? 2 : 4;
  __shared__ float red[3][4];
  __shared__ u64 keys[TOP ? 4 : 1][TOP ? 64 * (C + 1) : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int me = TEAM == 64 ? lane : threadIdx.x;
  const int64_t item = TEAM == 64 ? vt_block() * 4 + wave : vt_block();
  const int64_t row = TEAM == 64 ? item : item / a.splits;
  const int part = TEAM == 64 ? 0 : (int)(item - row * a.splits);
  if (row >= a.rows) return;       // (the whole workgroup, or a wave that meets no barrier)
  const int64_t action = cat_action(a, row);
  const typename T::elem* x = reinterpret_cast<const typename T::elem*>(a.logits) +
                              vt_row(row, a.inner, a.x_outer, a.x_inner);
  const uint8_t* mk = MB == 0 ? nullptr : reinterpret_cast<const uint8_t*>(a.mask) +
                                              MB * vt_row(row, a.inner, a.k_outer, a.k_inner);
  // Whole chunks lie on 16-byte addresses: chunk k holds elements k C - skew ..; the elements in front
  // of the first and behind the last one are taken one by one, by the first wave of their part.
  const int skew = (int)(((uintptr_t)x & 15u) / sizeof(typename T::elem));
  const int whole0 = skew > 0 ? 1 : 0;
  int whole1 = (int)(((int64_t)a.vocab + skew) / C);
  if (whole1 < whole0) whole1 = whole0;
  const int chunks = whole1 - whole0;
  const int each = TEAM == 64 ? chunks : (chunks + a.splits - 1) / a.splits;
  const int k0 = whole0 + part * each;
  const int k1 = k0 + each < whole1 ? k0 + each : whole1;
  const int first = k0 + (TEAM == 64 ? 0 : wave * 64);
  CatTile<T, MB, U> next;
  if (first < k1) cat_load<T, MB, U, TEAM>(x, mk, first, lane, k1, skew, next);
  const float chosen = cat_action_logit<T, MB>(a, row, action);
  if (action < 0) {
    if (a.splits == 1) cat_pad_row(a, row, me);
    return;                        // the whole team returns; the joining launch writes
  }
  const float c2 = a.inv_t * CAT_LOG2E;
  const float margin = CAT_MARGIN / c2;
  CatSum u = {CAT_LOWEST, 0.f, 0.f};
  CatTop top = cat_top(TOP ? keys[wave] : nullptr);
  if ((TEAM == 64 || wave == 0) && (part == 0 || part == a.splits - 1)) {
    const int head = part == 0 ? whole0 * C - skew : 0;                  // (skew 0: none)
    const int tail = part == a.splits - 1 ? whole1 * C - skew : a.vocab;
    // lanes 0 .. 31 the front, 32 .. 63 the end: fewer than 8 elements each
    const int e = lane < 32 ? lane : tail + lane - 32;
    const bool here = lane < 32 ? e < head && e < a.vocab : e >= head && e < a.vocab;
    float v = -INFINITY;
    if (here && cat_allowed<MB>(mk, e)) v = T::one(x[e]);
    if (v > u.r + margin) u.r = v;
    cat_add(u, v, c2);
    if (TOP) cat_top_offer(top, v, e, lane);
  }
  for (int kb = first; kb < k1; kb += TEAM * U) {          // (wave-uniform)
    const CatTile<T, MB, U> tile = next;
    if (kb + TEAM * U < k1) cat_load<T, MB, U, TEAM>(x, mk, kb + TEAM * U, lane, k1, skew, next);
    float v[U][C], high[U];
    float highest = -INFINITY;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      cat_values<T, MB, U>(tile, i, v[i]);
      high[i] = v[i][0];
#pragma unroll
      for (int j = 1; j < C; ++j) high[i] = fmaxf(high[i], v[i][j]);
      highest = fmaxf(highest, high[i]);
    }
    if (highest > u.r + margin) u = cat_move(u, highest, c2);
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int j = 0; j < C; ++j) cat_add(u, v[i][j], c2);
    if (TOP) {
      if (kb == first) {
        // k lanes hold a value at or above the k-th of the lanes' maxima, so the row's k best are too
        const unsigned sorted = wv_sort_desc((unsigned)(cat_key(highest, 0) >> 32), lane);
        cat_top_raise(top, (u64)(unsigned)__builtin_amdgcn_readlane((int)sorted, a.top_k - 1) << 32);
      }
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (__any(high[i] >= top.low)) {
          const int ku = kb + i * TEAM + lane;
#pragma unroll
          for (int j = 0; j < C; ++j)
            cat_top_offer(top, v[i][j], ku * C - skew + j, lane);
          // (once a chunk: a copy of the sort at every place would not fit the instruction cache)
          while (top.held >= 64) cat_top_flush(top, lane, a.top_k);
        }
    }
  }
  if (TOP)
    while (top.held > 0) cat_top_flush(top, lane, a.top_k);
  u = cat_wave_join(u, c2);
  if constexpr (TEAM == 64) {
    float ls = 0.f;
    if (lane == 0) ls = cat_finish(a, row, action, chosen, u);
    if (TOP) cat_write_top(a, row, lane, top.list, u.r, __shfl(ls, 0, 64));
  } else {
    if (lane == 0) { red[0][wave] = u.r; red[1][wave] = u.s; red[2][wave] = u.t; }
    if (TOP) keys[wave][lane] = top.list;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      CatSum o = {red[0][w], red[1][w], red[2][w]};
      u = cat_join(u, o, c2);
      if (TOP) top.list = wv_merge_desc(top.list, keys[w][63 - lane], lane);
    }
    if (a.splits == 1) {
      float ls = 0.f;
      if (lane == 0) ls = cat_finish(a, row, action, chosen, u);
      if (TOP) cat_write_top(a, row, lane, top.list, u.r, __shfl(ls, 0, 64));
    } else {
      if (lane == 0) {
        float* p = a.part + item * 4;
        p[0] = u.r; p[1] = u.s; p[2] = u.t; p[3] = 0.f;
      }
      // the parts' lists interleaved by rank: the first keys that the join reads are the best ones
      if (TOP && lane < a.top_k)
        a.part_keys[(row * a.top_k + lane) * a.splits + part] = top.list;
    }
  }
}

template <int U>
__device__ static inline void cat_join_load(const u64* src, int at, int n, int lane, u64 (&v)[U]) {
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = at + u * 64 + lane;
    v[u] = i < n ? src[i] : 0ull;
  }
}

// joins the parts of a row: a wave per row, by latency: its keys are loaded eight at a time (one at a
// time, both launches of f32 1x262144 with 40 took 23.7 us, of bf16 18.7; now 15.1 and 14.5)
template <typename T, int MB, bool TOP>
__global__ void __launch_bounds__(64) aa_categorical_join_kernel(CatArgs a) {
  constexpr int U = 8;             // keys of a lane in flight together
  __shared__ u64 keys[TOP ? 64 * (U + 1) : 1];
  const int lane = threadIdx.x;
  const int64_t row = vt_block();
  if (row >= a.rows) return;
  const int n = a.splits * a.top_k;
  u64 v[U];
  if (TOP) cat_join_load<U>(a.part_keys + row * n, 0, n, lane, v);
  const int64_t action = cat_action(a, row);
  if (action < 0) {
    cat_pad_row(a, row, lane);
    return;
  }
  const float chosen = cat_action_logit<T, MB>(a, row, action);
  const float c2 = a.inv_t * CAT_LOG2E;
  CatSum u = {CAT_LOWEST, 0.f, 0.f};
  for (int p = lane; p < a.splits; p += 64) {
    const float* q = a.part + (row * a.splits + p) * 4;
    CatSum o = {q[0], q[1], q[2]};
    u = cat_join(u, o, c2);
  }
  u = cat_wave_join(u, c2);
  float ls = 0.f;
  if (lane == 0) ls = cat_finish(a, row, action, chosen, u);
  if (TOP) {
    CatTop top = cat_top(keys);
    for (int i = 0; i < n; i += 64 * U) {
      if (i > 0) cat_join_load<U>(a.part_keys + row * n, i, n, lane, v);
      if (i == 0 && n > 64) {      // (as for a row's first tile; 64 keys are one flush in any case)
        u64 high = 0ull;
#pragma unroll
        for (int u = 0; u < U; ++u) high = high > v[u] ? high : v[u];
        const unsigned sorted = wv_sort_desc((unsigned)(high >> 32), lane);
        cat_top_raise(top, (u64)(unsigned)__builtin_amdgcn_readlane((int)sorted, a.top_k - 1) << 32);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) cat_top_offer_key(top, v[u], lane);
      while (top.held >= 64) cat_top_flush(top, lane, a.top_k);
    }
    while (top.held > 0) cat_top_flush(top, lane, a.top_k);
    cat_write_top(a, row, lane, top.list, u.r, __shfl(ls, 0, 64));
  }
}

// Few actions: a team of G lanes holds a row in registers, F elements a lane in chunks G apart, so the
// maximum is the row's own and the sums are taken once.  Bound by the instructions around a row (its
// reductions, its logarithm), so several rows share a wave: bf16 38000x300 takes 23 us with a wave a row.

// the lane's elements and which of them exist and are allowed, one bit each
template <typename T, int MB, int G, int F>
__device__ static inline unsigned cat_few_load(const CatArgs& a, int64_t row, int lane, float (&v)[F]) {
  constexpr int C = T::C;
  const typename T::elem* x = reinterpret_cast<const typename T::elem*>(a.logits) +
                              vt_row(row, a.inner, a.x_outer, a.x_inner);
  const uint8_t* mk = MB == 0 ? nullptr : reinterpret_cast<const uint8_t*>(a.mask) +
                                              MB * vt_row(row, a.inner, a.k_outer, a.k_inner);
  unsigned in = 0u;
#pragma unroll
  for (int i = 0; i < F / C; ++i) {
    const int e0 = (i * G + lane) * C, n = a.vocab - e0;
    float w[C];
    unsigned bits = (1u << C) - 1u;
    if (n >= C) {
      T::widen(vt_load16(x + e0), w);
      if constexpr (MB != 0) {
        unsigned m[MB * C / 4];
        __builtin_memcpy(m, mk + MB * e0, MB * C);
#pragma unroll
        for (int j = 0; j < C; ++j)
          if (MB == 1 ? ((m[j / 4] >> (8 * (j % 4))) & 0xffu) == 0u : m[MB * j / 4] == 0u)
            bits &= ~(1u << j);
      }
    } else {
      vt_load_part<T>(x + e0, n, 0.f, w);
#pragma unroll
      for (int j = 0; j < C; ++j)
        if (j >= n || !cat_allowed<MB>(mk, e0 + j)) bits &= ~(1u << j);
    }
    in |= bits << (i * C);
#pragma unroll
    for (int j = 0; j < C; ++j) v[i * C + j] = w[j];
  }
  return in;
}

template <typename T, int MB, int G, int F>
__global__ void __launch_bounds__(256) aa_categorical_few_kernel(CatArgs a) {
  constexpr int PER = 256 / G;
  const int lane = threadIdx.x % G;
  const int64_t wanted = vt_block() * PER + threadIdx.x / G;
  // (teams past the last row stay in step with their wave on the last one and store nothing)
  const int64_t row = wanted < a.rows ? wanted : a.rows - 1;
  float v[F];
  const unsigned in = cat_few_load<T, MB, G, F>(a, row, lane, v);
  const int64_t action = cat_action(a, row);
  const float chosen = cat_action_logit<T, MB>(a, row, action);
  const float c2 = a.inv_t * CAT_LOG2E;
  CatSum u = {CAT_LOWEST, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < F; ++i) {
    if (((in >> i) & 1u) == 0u) v[i] = -INFINITY;
    u.r = fmaxf(u.r, v[i]);
  }
  u.r = wv_group_max<G>(u.r);
#pragma unroll
  for (int i = 0; i < F; ++i) cat_add(u, v[i], c2);
  u.s = wv_group_sum<G>(u.s);
  u.t = wv_group_sum<G>(u.t);
  if (wanted >= a.rows || lane != 0) return;
  if (action < 0) cat_pad_row(a, row, 0);
  else cat_finish(a, row, action, chosen, u);
}

// ---- gradient --------------------------------------------------------------------------------------
struct CatGradArgs {
  CatArgs f;                       // the forward's operands; stats and entropy as it left them
  const float* dlog_prob;          // [rows], nullable
  const float* dentropy;           // [rows], nullable
  void* dx; int64_t dx_outer, dx_inner;
  int blocks;                      // workgroups per row
  int past_cache;                  // see CAT_PAST_CACHE
};

struct CatRow {
  float ref, c2, l2s, a0, a1, hit;
  int action;
  bool zero;
};

// d x_v = p_v (a0 + a1 (c2 (x - ref) - l2s)) + hit [v = action], p_v = 2^(c2 (x - ref) - l2s)
__device__ static inline CatRow cat_row_grad(const CatGradArgs& a, int64_t row) {
  CatRow o;
  const int64_t action = cat_action(a.f, row);
  const float ls = a.f.stats[2 * row + 1];
  const float g = a.dlog_prob != nullptr ? a.dlog_prob[row] : 0.f;
  const float h = a.dentropy != nullptr ? a.dentropy[row] : 0.f;
  o.ref = a.f.stats[2 * row];
  o.c2 = a.f.inv_t * CAT_LOG2E;
  o.l2s = ls * CAT_LOG2E;
  o.zero = action < 0 || (isinf(ls) && ls > 0.f);
  const float ent = (a.dentropy != nullptr && !o.zero) ? a.f.entropy[row] : 0.f;
  o.a0 = -a.f.inv_t * (g + h * ent);
  o.a1 = -a.f.inv_t * h * CAT_LN2;
  o.hit = a.f.inv_t * g;
  // an action past the end: its log-probability is NaN, and so is the gradient
  if (action >= a.f.vocab && a.dlog_prob != nullptr) o.a0 = cat_nan();
  o.action = (a.dlog_prob != nullptr && action < a.f.vocab) ? (int)action : -1;
  return o;
}

__device__ static inline float cat_grad_one(const CatRow& r, float x) {
  const float l = fmaf(x - r.ref, r.c2, -r.l2s);
  const float p = cat_exp2(l);
  return p * fmaf(r.a1, fmaxf(l, -200.f), r.a0);       // (p is 0 from -150 on)
}

// TEAM = 64: a wave per row, four rows per workgroup.  TEAM = 256: a workgroup per part of a row.
template <typename T, int MB, int TEAM>
__global__ void __launch_bounds__(256) aa_categorical_grad_kernel(CatGradArgs a) {
  constexpr int C = T::C;
  const int64_t item = TEAM == 64 ? vt_block() * 4 + (threadIdx.x >> 6) : vt_block();
  const int64_t row = TEAM == 64 ? item : item / a.blocks;
  const int block = TEAM == 64 ? 0 : (int)(item - row * a.blocks);
  if (row >= a.f.rows) return;
  const typename T::elem* x = reinterpret_cast<const typename T::elem*>(a.f.logits) +
                              vt_row(row, a.f.inner, a.f.x_outer, a.f.x_inner);
  typename T::elem* dx = reinterpret_cast<typename T::elem*>(a.dx) +
                         vt_row(row, a.f.inner, a.dx_outer, a.dx_inner);
  const uint8_t* mk = MB == 0 ? nullptr : reinterpret_cast<const uint8_t*>(a.f.mask) +
                                              MB * vt_row(row, a.f.inner, a.f.k_outer, a.f.k_inner);
  const CatRow r = cat_row_grad(a, row);
  // chunks lie on the destination's 16-byte addresses
  const int skew = (int)(((uintptr_t)dx & 15u) / sizeof(typename T::elem));
  const int chunks = (int)(((int64_t)a.f.vocab + skew + C - 1) / C);
  const int step = TEAM == 64 ? 64 : a.blocks * 256;
  if (r.zero) {                    // padding, or nothing allowed: its logits are not read
    float v[C];
#pragma unroll
    for (int j = 0; j < C; ++j) v[j] = 0.f;
    for (int k = block * 256 + threadIdx.x % TEAM; k < chunks; k += step) {
      const int e0 = k * C - skew;
      if (e0 >= 0 && e0 + C <= a.f.vocab) {
        vt_store16(dx + e0, T::pack(v));
      } else {
#pragma unroll
        for (int j = 0; j < C; ++j)
          if (e0 + j >= 0 && e0 + j < a.f.vocab) dx[e0 + j] = T::put(0.f);
      }
    }
    return;
  }
  for (int k = block * 256 + threadIdx.x % TEAM; k < chunks; k += step) {
    const int e0 = k * C - skew;
    if (e0 >= 0 && e0 + C <= a.f.vocab) {
      float v[C];
      T::widen(vt_load16(x + e0), v);
#pragma unroll
      for (int j = 0; j < C; ++j) v[j] = cat_grad_one(r, v[j]);
      if ((unsigned)(r.action - e0) < (unsigned)C) {
#pragma unroll
        for (int j = 0; j < C; ++j)
          if (e0 + j == r.action) v[j] += r.hit;
      }
      if (MB == 1) {
#pragma unroll
        for (int j = 0; j < C; ++j)
          if (mk[e0 + j] == 0) v[j] = 0.f;
      }
      if (MB == 4) {
#pragma unroll
        for (int j = 0; j < C; j += 4) {
          const uint4 m = vt_load16(mk + 4 * (int64_t)(e0 + j));
          if (m.x == 0u) v[j] = 0.f;
          if (m.y == 0u) v[j + 1] = 0.f;
          if (m.z == 0u) v[j + 2] = 0.f;
          if (m.w == 0u) v[j + 3] = 0.f;
        }
      }
      if (a.past_cache) vt_store16_nt(dx + e0, T::pack(v));
      else vt_store16(dx + e0, T::pack(v));
    } else {
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const int e = e0 + j;
        if (e < 0 || e >= a.f.vocab) continue;
        float v = cat_grad_one(r, T::one(x[e]));
        if (e == r.action) v += r.hit;
        if (MB == 1 && mk[e] == 0) v = 0.f;
        if (MB == 4 && reinterpret_cast<const int32_t*>(mk)[e] == 0) v = 0.f;
        dx[e] = T::put(v);
      }
    }
  }
}

// few actions: as the forward call, G lanes a row
template <typename T, int MB, int G, int F>
__global__ void __launch_bounds__(256) aa_categorical_few_grad_kernel(CatGradArgs a) {
  constexpr int C = T::C;
  const int lane = threadIdx.x % G;
  const int64_t row = vt_block() * (256 / G) + threadIdx.x / G;
  if (row >= a.f.rows) return;
  float v[F];
  const unsigned in = cat_few_load<T, MB, G, F>(a.f, row, lane, v);
  const CatRow r = cat_row_grad(a, row);
  typename T::elem* dx = reinterpret_cast<typename T::elem*>(a.dx) +
                         vt_row(row, a.f.inner, a.dx_outer, a.dx_inner);
#pragma unroll
  for (int i = 0; i < F / C; ++i) {
    const int e0 = (i * G + lane) * C, n = a.f.vocab - e0;
    float w[C];
#pragma unroll
    for (int j = 0; j < C; ++j) {
      w[j] = cat_grad_one(r, v[i * C + j]) + (e0 + j == r.action ? r.hit : 0.f);
      if (r.zero || ((in >> (i * C + j)) & 1u) == 0u) w[j] = 0.f;
    }
    if (n >= C) vt_store16(dx + e0, T::pack(w));
    else if (n > 0) vt_store_part<T>(dx + e0, n, w);
  }
}

// ---- host ------------------------------------------------------------------------------------------
static int cat_check(const aa_categorical_desc* d) {
  if (d == nullptr || d->rows <= 0 || d->inner <= 0 || d->vocab <= 0 || d->logits == nullptr)
    return AA_ERR_INVALID;
  if (d->dtype < AA_DT_F32 || d->dtype > AA_DT_F16) return AA_ERR_INVALID;
  if (d->actions != nullptr && d->action_bytes != 4 && d->action_bytes != 8) return AA_ERR_INVALID;
  if (d->mask != nullptr && d->mask_bytes != 1 && d->mask_bytes != 4) return AA_ERR_INVALID;
  if (!(d->temperature >= 1e-30f && d->temperature <= 1e30f)) return AA_ERR_INVALID;
  if (d->top_k < 0 || d->top_k > AA_CATEGORICAL_MAX_TOP || d->top_k > d->vocab)
    return AA_ERR_INVALID;
  if (d->vocab > (1 << 30)) return AA_ERR_RANGE;
  return AA_OK;
}

// Rows are split where a workgroup for each leaves CUs idle (up to CAT_SPLIT_ROWS rows) and a row is
// longer than what a workgroup reads while the joining launch runs (32 KB).  us without / with:
// bf16 16000 x 64 rows 5.6 / 6.9, 50001 x 64 11.4 / 7.5, x 256 13.1 / 14.3, x 384 16.3 / 18.8,
// 131072 x 1 19 / 6.3, x 256 20.8 / 19.3, x 384 29 / 32; f32 131072 x 192 42 / 29, x 384 54 / 50.
static int cat_splits(const aa_categorical_desc* d) {
  const int per = d->dtype == AA_DT_F32 ? 4 : 8;
  if (d->rows > CAT_SPLIT_ROWS || d->vocab <= 2048 * per) return 1;
  int64_t want = (CAT_SPLIT_BLOCKS + d->rows - 1) / d->rows;
  const int64_t most = (d->vocab / per + 1023) / 1024;     // four rounds of a workgroup at least
  if (want > most) want = most;
  return want < 1 ? 1 : (int)want;
}

static CatArgs cat_args(const aa_categorical_desc* d) {
  CatArgs a;
  a.rows = d->rows; a.inner = d->inner; a.vocab = (int)d->vocab;
  a.logits = d->logits; a.x_outer = d->x_outer; a.x_inner = d->x_inner;
  a.actions = d->actions; a.a_outer = d->a_outer; a.a_inner = d->a_inner;
  a.first_action = d->first_action; a.action_bytes = d->action_bytes; a.no_padding = d->no_padding;
  a.mask = d->mask; a.k_outer = d->k_outer; a.k_inner = d->k_inner;
  a.inv_t = 1.f / d->temperature; a.top_k = d->top_k;
  a.log_prob = d->log_prob; a.entropy = d->entropy; a.stats = d->stats;
  a.top_ids = d->top_ids; a.top_log_prob = d->top_log_prob;
  a.splits = 1; a.part = nullptr; a.part_keys = nullptr;
  return a;
}

template <typename T, int MB>
static void cat_launch(const CatArgs& a, hipStream_t st) {
  if (a.top_k == 0 && a.vocab <= CAT_FEW) {
    const dim3 by8 = vt_grid((a.rows + 31) / 32), by16 = vt_grid((a.rows + 15) / 16), block(256);
    if (a.vocab <= 64) aa_categorical_few_kernel<T, MB, 8, 8><<<by8, block, 0, st>>>(a);
    else if (a.vocab <= 128) aa_categorical_few_kernel<T, MB, 16, 8><<<by16, block, 0, st>>>(a);
    else if (a.vocab <= 256) aa_categorical_few_kernel<T, MB, 16, 16><<<by16, block, 0, st>>>(a);
    else aa_categorical_few_kernel<T, MB, 16, 32><<<by16, block, 0, st>>>(a);
    return;
  }
  if (a.vocab <= CAT_WAVE_VOCAB) {
    const dim3 grid = vt_grid((a.rows + 3) / 4);
    if (a.top_k > 0) aa_categorical_kernel<T, MB, 64, true><<<grid, dim3(256), 0, st>>>(a);
    else aa_categorical_kernel<T, MB, 64, false><<<grid, dim3(256), 0, st>>>(a);
    return;
  }
  const dim3 grid = vt_grid(a.rows * a.splits);
  if (a.top_k > 0) aa_categorical_kernel<T, MB, 256, true><<<grid, dim3(256), 0, st>>>(a);
  else aa_categorical_kernel<T, MB, 256, false><<<grid, dim3(256), 0, st>>>(a);
  if (a.splits > 1) {
    const dim3 rows = vt_grid(a.rows);
    if (a.top_k > 0) aa_categorical_join_kernel<T, MB, true><<<rows, dim3(64), 0, st>>>(a);
    else aa_categorical_join_kernel<T, MB, false><<<rows, dim3(64), 0, st>>>(a);
  }
}

template <typename T, int MB>
static void cat_launch_grad(const CatGradArgs& g, hipStream_t st) {
  const int64_t rows = g.f.rows;
  const dim3 block(256);
  const dim3 by8 = vt_grid((rows + 31) / 32), by16 = vt_grid((rows + 15) / 16);
  if (g.f.vocab <= 64)
    aa_categorical_few_grad_kernel<T, MB, 8, 8><<<by8, block, 0, st>>>(g);
  else if (g.f.vocab <= 128)
    aa_categorical_few_grad_kernel<T, MB, 16, 8><<<by16, block, 0, st>>>(g);
  else if (g.f.vocab <= 256)
    aa_categorical_few_grad_kernel<T, MB, 16, 16><<<by16, block, 0, st>>>(g);
  else if (g.f.vocab <= CAT_FEW)
    aa_categorical_few_grad_kernel<T, MB, 16, 32><<<by16, block, 0, st>>>(g);
  else if (g.f.vocab <= CAT_WAVE_VOCAB)
    aa_categorical_grad_kernel<T, MB, 64><<<vt_grid((rows + 3) / 4), block, 0, st>>>(g);
  else
    aa_categorical_grad_kernel<T, MB, 256><<<vt_grid(rows * g.blocks), block, 0, st>>>(g);
}

template <typename T>
static void cat_launch_grad_mask(const CatGradArgs& g, int mask_bytes, hipStream_t st) {
  if (mask_bytes == 0) cat_launch_grad<T, 0>(g, st);
  else if (mask_bytes == 1) cat_launch_grad<T, 1>(g, st);
  else cat_launch_grad<T, 4>(g, st);
}

template <typename T>
static void cat_launch_mask(const CatArgs& a, int mask_bytes, hipStream_t st) {
  if (mask_bytes == 0) cat_launch<T, 0>(a, st);
  else if (mask_bytes == 1) cat_launch<T, 1>(a, st);
  else cat_launch<T, 4>(a, st);
}

extern "C" {

int64_t aa_categorical_workspace_bytes(const aa_categorical_desc* d) {
  if (cat_check(d) != AA_OK) return -1;
  const int splits = cat_splits(d);
  return splits == 1 ? 0 : d->rows * splits * (16 + 8 * (int64_t)d->top_k);
}

int aa_categorical_log_prob(const aa_categorical_desc* d, void* workspace, int64_t workspace_bytes,
                            void* stream) {
  const int rc = cat_check(d);
  if (rc != AA_OK) return rc;
  if ((d->actions == nullptr) != (d->log_prob == nullptr)) return AA_ERR_INVALID;
  if (d->top_k > 0 && (d->top_ids == nullptr || d->top_log_prob == nullptr)) return AA_ERR_INVALID;
  const int64_t need = aa_categorical_workspace_bytes(d);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return AA_ERR_RANGE;
  CatArgs a = cat_args(d);
  a.splits = cat_splits(d);
  if (a.rows * a.splits > VT_MAX_BLOCKS) return AA_ERR_RANGE;
  if (a.splits > 1) {
    a.part = (float*)workspace;
    a.part_keys = (u64*)(a.part + 4 * a.rows * a.splits);
  }
  const int mb = d->mask == nullptr ? 0 : d->mask_bytes;
  hipStream_t st = (hipStream_t)stream;
  if (d->dtype == AA_DT_F32) cat_launch_mask<VtF32>(a, mb, st);
  else if (d->dtype == AA_DT_BF16) cat_launch_mask<VtBf16>(a, mb, st);
  else cat_launch_mask<VtF16>(a, mb, st);
  return aa_launch_status();
}

int aa_categorical_log_prob_backward(const aa_categorical_desc* d, const float* dlog_prob,
                                     const float* dentropy, void* dlogits, int64_t dx_outer,
                                     int64_t dx_inner, void* stream) {
  const int rc = cat_check(d);
  if (rc != AA_OK) return rc;
  if (d->stats == nullptr || dlogits == nullptr || (dlog_prob == nullptr && dentropy == nullptr) ||
      (dlog_prob != nullptr && d->actions == nullptr) ||
      (dentropy != nullptr && d->entropy == nullptr))
    return AA_ERR_INVALID;
  CatGradArgs g;
  g.f = cat_args(d);
  g.dlog_prob = dlog_prob; g.dentropy = dentropy;
  g.dx = dlogits; g.dx_outer = dx_outer; g.dx_inner = dx_inner;
  const int per = d->dtype == AA_DT_F32 ? 4 : 8;
  const int64_t rounds = (d->vocab / per + 256) / 256;
  g.blocks = (int)((rounds + 3) / 4);
  g.past_cache = d->rows * d->vocab * (d->dtype == AA_DT_F32 ? 4 : 2) >= CAT_PAST_CACHE;
  if (g.f.rows * g.blocks > VT_MAX_BLOCKS) return AA_ERR_RANGE;
  const int mb = d->mask == nullptr ? 0 : d->mask_bytes;
  hipStream_t st = (hipStream_t)stream;
  if (d->dtype == AA_DT_F32) cat_launch_grad_mask<VtF32>(g, mb, st);
  else if (d->dtype == AA_DT_BF16) cat_launch_grad_mask<VtBf16>(g, mb, st);
  else cat_launch_grad_mask<VtF16>(g, mb, st);
  return aa_launch_status();
}

}  // extern "C"
