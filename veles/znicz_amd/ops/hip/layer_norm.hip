// Layer normalisation of the rows of a matrix, forward and backward.
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) r
//   y  = xh w + b
//   g  = dy w;  dx = r (g - mean(g) - xh mean(g xh))
//   dw = sum over rows of dy xh,  db = sum over rows of dy
// The variance is taken around the mean (no difference of large numbers);
// statistics and sums are held in 32 bits, and dx, y are rounded once.
#include <stdexcept>

#include "rows.h"

#define LN_THREADS 256
#define LN_LONG 1024
// Partial column sums of long rows that a backward pass leaves to be joined:
// one for each 32 rows within these bounds (1024 x 40000 bf16 with 32 of them
// 110 us, 64 117, 128 127, 256 154, since each is as long as two rows of fp32;
// 4096 x 17000 with 64 of them 183, 128 192; 16 x 40000 with 8 17, 16 21)
#define LN_PARTS_FEW 8
#define LN_PARTS 64

// A row that is too long for registers: f(first element, number) for each of
// this thread's packs and for one of the elements behind the last pack.
template <int N>
struct Count {
  static constexpr int n = N;
};
template <int N, typename F>
__device__ __forceinline__ void over_row(int cols, F f) {
  const int packs = cols / N, single = packs * N + threadIdx.x;
#pragma unroll 2
  for (int p = threadIdx.x; p < packs; p += LN_LONG) f(p * N, Count<N>());
  if (single < cols) f(single, Count<1>());
}
template <typename T, int N>
__device__ __forceinline__ void get_some(float* e, const T* x, Count<N>) {
  if constexpr (N == 1) {
    e[0] = (float)x[0];
  } else {
    Pack<T> v;
    v.load(x);
    v.get(e);
  }
}
template <typename T, int N>
__device__ __forceinline__ void put_some(T* y, const float* e, Count<N>) {
  if constexpr (N == 1) {
    y[0] = from_f<T>(e[0]);
  } else {
    Pack<T> v;
    v.set(e);
    v.store(y);
  }
}

// (16 bytes at a time, which a loop over p[k] does not become)
template <int N>
__device__ __forceinline__ void get_param(float* v, const float* p, int j,
                                          float none, Count<N>) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = none;
  if (p) __builtin_memcpy(v, p + j, sizeof(float) * N);
}

// One workgroup to such a row; it is read three times (backward: twice), from
// the caches after the first, 16 bytes at a time.  1024 x 40000 bf16: 54 us,
// 3.0 TB/s of one read and one write (with single elements, or the parameters
// one by one, 175 to 260); bound by the waits between its three readings.
template <typename T>
__global__ __launch_bounds__(LN_LONG) void ln_fwd_k(
    RowsIn x_, RowsOut y_, const float* __restrict__ w,
    const float* __restrict__ b, float* __restrict__ mean,
    float* __restrict__ rstd, long rows, int cols, float eps) {
  __shared__ float tmp[LN_LONG / WAVE];
  constexpr int N = Pack<T>::N;
  for (long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* x = (const T*)x_.p + row * x_.stride;
    T* y = (T*)y_.p + row * y_.stride;
    float s = 0.f, v = 0.f;
    over_row<N>(cols, [&](int j, auto count) {
      float e[count.n];
      get_some(e, x + j, count);
#pragma unroll
      for (int k = 0; k < count.n; ++k) s += e[k];
    });
    const float mu = block_sum(s, tmp) / cols;
    over_row<N>(cols, [&](int j, auto count) {
      float e[count.n];
      get_some(e, x + j, count);
#pragma unroll
      for (int k = 0; k < count.n; ++k) v = fmaf(e[k] - mu, e[k] - mu, v);
    });
    const float r = 1.f / sqrtf(block_sum(v, tmp) / cols + eps);
    over_row<N>(cols, [&](int j, auto count) {
      float e[count.n], gain[count.n], shift[count.n];
      get_some(e, x + j, count);
      get_param(gain, w, j, 1.f, count);
      get_param(shift, b, j, 0.f, count);
#pragma unroll
      for (int k = 0; k < count.n; ++k)
        e[k] = fmaf((e[k] - mu) * r, gain[k], shift[k]);
      put_some(y + j, e, count);
    });
    if (threadIdx.x == 0) {
      if (mean) mean[row] = mu;
      if (rstd) rstd[row] = r;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(LN_LONG) void ln_bwd_k(
    RowsIn dy_, RowsIn x_, const float* __restrict__ w,
    const float* __restrict__ mean, const float* __restrict__ rstd,
    RowsOut dx_, long rows, int cols) {
  __shared__ float tmp[LN_LONG / WAVE];
  constexpr int N = Pack<T>::N;
  for (long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* dy = (const T*)dy_.p + row * dy_.stride;
    const T* x = (const T*)x_.p + row * x_.stride;
    T* dx = (T*)dx_.p + row * dx_.stride;
    const float mu = mean[row], r = rstd[row];
    float s1 = 0.f, s2 = 0.f;
    over_row<N>(cols, [&](int j, auto count) {
      float e[count.n], g[count.n], gain[count.n];
      get_some(e, x + j, count);
      get_some(g, dy + j, count);
      get_param(gain, w, j, 1.f, count);
#pragma unroll
      for (int k = 0; k < count.n; ++k) {
        const float d = g[k] * gain[k];
        s1 += d;
        s2 = fmaf(d, (e[k] - mu) * r, s2);
      }
    });
    s1 = block_sum(s1, tmp) / cols;
    s2 = block_sum(s2, tmp) / cols;
    over_row<N>(cols, [&](int j, auto count) {
      float e[count.n], g[count.n], gain[count.n];
      get_some(e, x + j, count);
      get_some(g, dy + j, count);
      get_param(gain, w, j, 1.f, count);
#pragma unroll
      for (int k = 0; k < count.n; ++k) {
        const float d = g[k] * gain[k];
        g[k] = r * (d - s1 - (e[k] - mu) * r * s2);
      }
      put_some(dx + j, g, count);
    });
  }
}

// Column sums of dy xh and dy over this workgroup's rows: one thread to a
// pack of columns (the last one ends with the row), part[blockIdx.y] =
// [2][cols].  With ln_bwd_k and ln_join_k, 1024 x 40000 bf16: 110 us, 2.2 TB/s
// of dy, x and dx once; they are read twice.
template <typename T>
__global__ __launch_bounds__(LN_THREADS) void ln_cols_k(
    RowsIn dy_, RowsIn x_, const float* __restrict__ mean,
    const float* __restrict__ rstd, float* __restrict__ part, long rows,
    int cols) {
  constexpr int N = Pack<T>::N;
  const int own = (blockIdx.x * LN_THREADS + threadIdx.x) * N;
  if (own >= cols) return;
  const int j = min(own, cols - N);
  const long per = (rows + gridDim.y - 1) / gridDim.y;
  const long lo = blockIdx.y * per, hi = min(lo + per, rows);
  float sw[N], sb[N];
#pragma unroll
  for (int k = 0; k < N; ++k) sw[k] = sb[k] = 0.f;
#pragma unroll 4
  for (long row = lo; row < hi; ++row) {
    Pack<T> vg, vx;
    float g[N], e[N];
    vg.load((const T*)dy_.p + row * dy_.stride + j);
    vx.load((const T*)x_.p + row * x_.stride + j);
    vg.get(g);
    vx.get(e);
    const float mu = mean[row], rs = rstd[row];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      sw[k] = fmaf(g[k], (e[k] - mu) * rs, sw[k]);
      sb[k] += g[k];
    }
  }
  float* out = part + (long)blockIdx.y * 2 * cols;
#pragma unroll
  for (int k = 0; k < N; ++k)
    if (j + k >= own) {
      out[j + k] = sw[k];
      out[cols + j + k] = sb[k];
    }
}

// The partial sums [parts][2][cols] joined, always in the same order: 32 of
// the 2 cols columns to a workgroup, 8 slices of the parts (256 parts of 4096
// columns, 8 MB: 4.8 us, of which 4 are the launch and one load's delay)
#define LN_SLICES 8
__global__ __launch_bounds__(LN_THREADS) void ln_join_k(
    const float* __restrict__ part, int parts, float* __restrict__ dw,
    float* __restrict__ db, int cols, int accumulate) {
  __shared__ float tmp[LN_SLICES][32];
  const int lane = threadIdx.x % 32, slice = threadIdx.x / 32;
  const long c = (long)blockIdx.x * 32 + lane;
  const long all = 2l * cols;
  float s = 0.f;
  if (c < all) {
#pragma unroll 8
    for (int i = slice; i < parts; i += LN_SLICES) s += part[i * all + c];
  }
  tmp[slice][lane] = s;
  __syncthreads();
  if (slice || c >= all) return;
#pragma unroll
  for (int i = 1; i < LN_SLICES; ++i) s += tmp[i][lane];
  float* out = c < cols ? dw : db;
  if (!out) return;
  const long j = c < cols ? c : c - cols;
  out[j] = accumulate ? out[j] + s : s;
}

// ---------------------------------------------------------------------------
// rows in registers
// ---------------------------------------------------------------------------
// A team of lanes has a row, 8, 16 or (forward) 32 elements a lane: a part of a
// wave, a wave, or a whole workgroup, as the row is long.  It goes through the rows
// in steps, several at a time, with the gain and the shift (backward: the
// gain and the two column sums) in registers all along.

// the team's sums of R values each, in all its lanes; `tmp`: [2][R][waves],
// used in turn so that one barrier does for a call
template <int THREADS, int TEAM, int R>
struct TeamSum {
  float* tmp;
  int turn;

  __device__ __forceinline__ void operator()(float* v) {
    if constexpr (TEAM <= WAVE) {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if constexpr (TEAM == WAVE) {
          v[i] = wave_sum(v[i]);
        } else {
          v[i] += other_lane<0xb1>(v[i]);
          v[i] += other_lane<0x4e>(v[i]);
          if (TEAM > 4) v[i] += other_lane<0x141>(v[i]);
          if (TEAM > 8) v[i] += other_lane<0x140>(v[i]);
          if (TEAM > 16) v[i] += __shfl_xor(v[i], 16);
        }
      }
    } else {
      // a wave's sum comes to its last lane; the waves' are joined by a lane
      // to each
      constexpr int WAVES = TEAM / WAVE, ALL = THREADS / WAVE;
      float* t = tmp + turn * R * ALL;
      turn ^= 1;
      const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float w = wave_sum_last(v[i]);
        if (lane == WAVE - 1) t[i * ALL + wave] = w;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < R; ++i) {
        v[i] = t[i * ALL + wave / WAVES * WAVES + lane % WAVES];
        v[i] += other_lane<0xb1>(v[i]);
        if (WAVES > 2) v[i] += other_lane<0x4e>(v[i]);
        if (WAVES > 4) v[i] += other_lane<0x141>(v[i]);
        if (WAVES > 8) v[i] += other_lane<0x140>(v[i]);
      }
    }
  }
};

// 1 / sqrt(v): one unit in the last place (v_rsq_f32, which takes numbers
// below 2^-126 for 0)
__device__ __forceinline__ float inv_sqrt(float v) {
  const bool small = v < 0x1p-100f;
  const float r = __builtin_amdgcn_rsqf(small ? v * 0x1p100f : v);
  return small ? r * 0x1p50f : r;
}

// sum / cols to the nearest: the product with the rounded reciprocal `per` and
// the rest that it leaves, which is exact.  The product alone is off by a step
// for 3.0 at 1000 columns, say, and what a row of equal values then keeps of
// itself is multiplied by a deviation of up to 1 / sqrt(eps).  (A sum that is
// no number or infinite has no rest.)
__device__ __forceinline__ float mean_of(float sum, int cols, float per) {
  const float q = sum * per, rest = fmaf(-q, (float)cols, sum);
  return rest == rest ? fmaf(rest, per, q) : q;
}

// Where a lane's packs of a row lie.  The last pack of a row that is no
// whole number of packs ends with the row, so that its first elements are
// the pack's before, too; a lane beyond the last pack has that one again.
// Both are loaded and stored like any other (the same values to the same
// place), which spares the branches, and are left out of the sums.  A row
// shorter than a pack (TINY) is read and written one by one.  Rows may begin at
// any element; off multiples of 16 bytes loads and stores are slower: 16384 x
// 4096 bf16, rows 4097 apart, 63 us instead of 50, backward 86 instead of 80.
template <typename T, int TEAM, int NV, bool TINY>
struct Slots {
  static constexpr int N = Pack<T>::N;
  int lane, cols, packs;

  __device__ __forceinline__ Slots(int cols_) {
    lane = threadIdx.x % TEAM;
    cols = cols_;
    packs = (cols + N - 1) / N;
  }
  __device__ __forceinline__ bool has(int i) const {
    return i * TEAM + lane < packs;
  }
  __device__ __forceinline__ int at(int i) const {
    const int j = (i * TEAM + lane) * N;
    return TINY ? 0 : min(j, cols - N);
  }
  // whether element k of pack i is this pack's own
  __device__ __forceinline__ bool own(int i, int k) const {
    return column(lane, i, k) >= 0;
  }
  // the column of element k of a lane's pack i, -1 if it is another's
  __device__ __forceinline__ int column(int of, int i, int k) const {
    const int j = (i * TEAM + of) * N;
    const int c = (TINY ? 0 : min(j, cols - N)) + k;
    return i * TEAM + of < packs && c >= j && c < cols ? c : -1;
  }
  __device__ __forceinline__ void load(Pack<T>& v, const T* row, int i) const {
    if (TINY) {
      float e[N];
#pragma unroll
      for (int k = 0; k < N; ++k) e[k] = k < cols ? (float)row[k] : 0.f;
      v.set(e);
    } else {
      v.load(row + at(i));
    }
  }
  __device__ __forceinline__ void store(const Pack<T>& v, T* row,
                                        int i) const {
    if (TINY) {
      T e[N];
      __builtin_memcpy(e, &v.raw, 16);
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (k < cols) row[k] = e[k];
    } else {
      v.store(row + at(i));
    }
  }
  // parameters of the lane's columns, 16 bytes at a time
  __device__ __forceinline__ void load_param(float* v, const float* p,
                                             float none) const {
#pragma unroll
    for (int k = 0; k < NV * N; ++k) v[k] = none;
    if (!p) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (TINY) {
#pragma unroll
        for (int k = 0; k < N; ++k)
          if (k < cols) v[i * N + k] = p[k];
      } else {
        __builtin_memcpy(v + i * N, p + at(i), sizeof(float) * N);
      }
    }
  }
};

// The rows of a team: those of a workgroup's teams from `start`, and `teams`
// apart.  All lanes of a workgroup make the same number of steps.
template <int THREADS, int TEAM>
struct Steps {
  long start, teams;
  int mine;        // this lane's team among those of its workgroup

  __device__ __forceinline__ Steps() {
    constexpr int TEAMS = THREADS / TEAM;
    teams = (long)gridDim.x * TEAMS;
    start = (long)blockIdx.x * TEAMS;
    // (the same number for a wave, where it is one)
    mine = TEAM < WAVE ? (int)threadIdx.x / TEAM
                       : __builtin_amdgcn_readfirstlane(threadIdx.x / TEAM);
  }
  // whether all rows of the step from `first` exist
  __device__ __forceinline__ bool full(long first, long rows) const {
    return first + THREADS / TEAM - 1 < rows;
  }
};

// All loads so far have arrived.  (Before a loop whose first loads were
// issued outside, so that within it the compiler counts those of the loop
// alone.)
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt(0x0f70);      // vmcnt 0
}

// In each step the next one's loads come before this one's stores: memory
// operations are waited for in their order, and what waits for a load would
// otherwise wait for stores to reach memory (16384 x 4096 bf16: 61 us before,
// 51 so, 5.2 TB/s, where a bare copy reaches 6.5).  For the same reason nothing
// after those loads is on a condition; the last step is apart.
template <typename T, int THREADS, int TEAM, int NV, bool EXACT, bool TINY>
__global__ __launch_bounds__(THREADS) void ln_fwd_team_k(
    RowsIn x_, RowsOut y_, const float* __restrict__ w,
    const float* __restrict__ b, float* __restrict__ mean,
    float* __restrict__ rstd, long rows, int cols, float eps) {
  constexpr int N = Pack<T>::N;
  constexpr bool AHEAD = NV < 8;       // (fp32 of 32 elements: no registers)
  __shared__ float tmp[2 * (THREADS / WAVE)];
  TeamSum<THREADS, TEAM, 1> sum{tmp, 0};
  const Slots<T, TEAM, NV, TINY> at(cols);
  const Steps<THREADS, TEAM> steps;
  float gain[NV * N], shift[NV * N];
  const float per = 1.f / cols;
  Pack<T> v[NV];
  auto load = [&](long row) {
    row = min(row, rows - 1);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      at.load(v[i], (const T*)x_.p + row * x_.stride, i);
  };
  auto step = [&](long row, bool last) {
    float mu = 0.f, rs = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float e[N], q = 0.f;
      v[i].get(e);
#pragma unroll
      for (int k = 0; k < N; ++k) q += EXACT || at.own(i, k) ? e[k] : 0.f;
      mu += at.has(i) ? q : 0.f;
    }
    sum(&mu);
    mu = mean_of(mu, cols, per);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float e[N], q = 0.f;
      v[i].forget();
      v[i].get(e);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        float d = e[k] - mu;
        if (!EXACT) d = at.own(i, k) ? d : 0.f;
        q = fmaf(d, d, q);
      }
      rs += at.has(i) ? q : 0.f;
    }
    sum(&rs);
    rs = inv_sqrt(fmaf(rs, per, eps));
    if (at.lane == 0 && mean && row < rows) mean[row] = mu;
    if (at.lane == 0 && rstd && row < rows) rstd[row] = rs;
    Pack<T> y[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float e[N];
      v[i].forget();
      v[i].get(e);
#pragma unroll
      for (int k = 0; k < N; ++k)
        e[k] = fmaf((e[k] - mu) * rs, gain[i * N + k], shift[i * N + k]);
      y[i].set(e);
    }
    if (AHEAD && !last) load(row + steps.teams);
    if (last && row >= rows) return;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      at.store(y[i], (T*)y_.p + row * y_.stride, i);
    if (!AHEAD && !last) load(row + steps.teams);
  };
  load(steps.start + steps.mine);
  at.load_param(gain, w, 1.f);
  at.load_param(shift, b, 0.f);
  wait_loads();
  long first = steps.start;
  for (; steps.full(first, rows); first += steps.teams)
    step(first + steps.mine, false);
  if (first < rows) step(first + steps.mine, true);
}

// The backward pass of the same teams; part[block] = [2][cols], the
// workgroup's column sums.  SUMS: dw or db is asked for, DX: dx is.  16384 x
// 4096 bf16 with the joining: 79 us, 5.1 TB/s; bound by memory and by the one
// workgroup that a compute unit has.
template <typename T, int THREADS, int TEAM, int NV, bool EXACT, bool SUMS,
          bool DX, bool TINY>
__global__ __launch_bounds__(THREADS) void ln_bwd_team_k(
    RowsIn dy_, RowsIn x_, const float* __restrict__ w,
    const float* __restrict__ mean, const float* __restrict__ rstd,
    RowsOut dx_, float* __restrict__ part, long rows, int cols) {
  constexpr int N = Pack<T>::N, E = NV * N;
  __shared__ float tmp[4 * (THREADS / WAVE)];
  TeamSum<THREADS, TEAM, 2> sum{tmp, 0};
  const Slots<T, TEAM, NV, TINY> at(cols);
  const Steps<THREADS, TEAM> steps;
  float gain[E], dw[E], db[E];
  const float per = 1.f / cols;
  Pack<T> vx[NV], vg[NV];
  float mu, rs;
  auto load = [&](long row) {
    row = min(row, rows - 1);
    mu = mean[row];
    rs = rstd[row];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      at.load(vx[i], (const T*)x_.p + row * x_.stride, i);
      at.load(vg[i], (const T*)dy_.p + row * dy_.stride, i);
    }
  };
  auto step = [&](long row, bool last) {
    if (last && row >= rows) {
      mu = rs = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        vx[i].fill(0.f);
        vg[i].fill(0.f);
      }
    }
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float e[N], g[N], s1 = 0.f, s2 = 0.f;
      vx[i].get(e);
      vg[i].get(g);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float h = (e[k] - mu) * rs;
        if (SUMS) {
          dw[i * N + k] = fmaf(g[k], h, dw[i * N + k]);
          db[i * N + k] += g[k];
        }
        float d = g[k] * gain[i * N + k];
        if (!EXACT) d = at.own(i, k) ? d : 0.f;
        s1 += d;
        s2 = fmaf(d, h, s2);
      }
      s[0] += at.has(i) ? s1 : 0.f;
      s[1] += at.has(i) ? s2 : 0.f;
    }
    if (!DX) {
      if (!last) load(row + steps.teams);
      return;
    }
    sum(s);
    const float s1 = mean_of(s[0], cols, per), s2 = mean_of(s[1], cols, per);
    Pack<T> out[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float e[N], g[N];
      vx[i].forget();
      vg[i].forget();
      vx[i].get(e);
      vg[i].get(g);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float h = (e[k] - mu) * rs;
        g[k] = rs * (fmaf(g[k], gain[i * N + k], -s1) - h * s2);
      }
      out[i].set(g);
    }
    if (!last) load(row + steps.teams);
    if (last && row >= rows) return;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      at.store(out[i], (T*)dx_.p + row * dx_.stride, i);
  };
  load(steps.start + steps.mine);
  at.load_param(gain, w, 1.f);
#pragma unroll
  for (int k = 0; k < E; ++k) dw[k] = db[k] = 0.f;
  wait_loads();
  long first = steps.start;
  for (; steps.full(first, rows); first += steps.teams)
    step(first + steps.mine, false);
  if (first < rows) step(first + steps.mine, true);
  if (!SUMS) return;
  // the workgroup's sums: over the teams of a wave, then over the waves that
  // have the same columns
  constexpr int LANES = TEAM < WAVE ? TEAM : WAVE;     // of a wave
  constexpr int SETS = TEAM < WAVE ? THREADS / WAVE : THREADS / TEAM;
  __shared__ alignas(16) float all[SETS][E * TEAM];
  const int set = TEAM < WAVE ? threadIdx.x / WAVE : threadIdx.x / TEAM;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float d[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        d[k] = half ? db[i * N + k] : dw[i * N + k];
#pragma unroll
        for (int off = LANES; off < WAVE; off *= 2)
          d[k] += __shfl_xor(d[k], off);
      }
      if (TEAM >= WAVE || (threadIdx.x & (WAVE - 1)) < TEAM)
        __builtin_memcpy(&all[set][(i * TEAM + at.lane) * N], d, sizeof(d));
    }
    __syncthreads();
    float* out = part + (2l * blockIdx.x + half) * cols;
    // (in the columns' order, so that a wave's stores lie together)
    for (int a = threadIdx.x; a < E * TEAM; a += THREADS) {
      const int c = at.column(a / N % TEAM, a / N / TEAM, a % N);
      if (c < 0) continue;
      float d = all[0][a];
#pragma unroll
      for (int v = 1; v < SETS; ++v) d += all[v][a];
      out[c] = d;
    }
    __syncthreads();
  }
}

static unsigned row_grid(long rows) {
  return (unsigned)(rows < 65536 ? rows : 65536);
}

// Rows of up to LN_MOST elements are held by teams, forward, and up to
// LN_MOST_SUMS backward: of 8 a lane as far as 1024 lanes go, then 16 and 32.
// 2048 x 32000 bf16 forward: held 62 us, read three times 83.  Backward 4096 x
// 16000: held 99, read twice 154; 32 elements a lane have no registers for the
// sums, and without them were slower than reading twice (2048 x 32000: 219,
// 179).  With 16 elements a lane from the start: 16384 x 4096 forward 56
// instead of 51 us, 8000 x 1000 9.3 instead of 8.2 (65536 x 1000, where the
// barriers of two waves weigh more, 54.6 instead of 59.9), backward 65536 x
// 1000 87 instead of 78, 193600 x 96 31 instead of 27.
#define LN_MOST 32768
#define LN_MOST_SUMS 16384
// Workgroups at most: 2048 of 256 threads forward (16384 x 4096 bf16 in 51
// us, with 4096 of them 71, 8192 87).  Backward 256 of 1024 threads, one to a
// compute unit, so that few column sums are left to be joined (79 us; 512 of
// them, in turns, 90; 128 118).
#define LN_FORWARD 2048
#define LN_BACKWARD 256

// F(threads, team, elements of a lane) of the first team that holds a row
#define LN_TEAMS(cols, F)                                                    \
  do {                                                                       \
    if (cols <= 32) {                                                        \
      F(256, 4, 8);                                                          \
    } else if (cols <= 64) {                                                 \
      F(256, 8, 8);                                                          \
    } else if (cols <= 128) {                                                \
      F(256, 16, 8);                                                         \
    } else if (cols <= 256) {                                                \
      F(256, 32, 8);                                                         \
    } else if (cols <= 512) {                                                \
      F(256, 64, 8);                                                         \
    } else if (cols <= 1024) {                                               \
      F(128, 128, 8);                                                        \
    } else if (cols <= 2048) {                                               \
      F(256, 256, 8);                                                        \
    } else if (cols <= 4096) {                                               \
      F(512, 512, 8);                                                        \
    } else if (cols <= 8192) {                                               \
      F(1024, 1024, 8);                                                      \
    } else if (cols <= 16384) {                                              \
      F(1024, 1024, 16);                                                     \
    } else {                                                                 \
      F(1024, 1024, 32);                                                     \
    }                                                                        \
  } while (0)

static unsigned team_grid(long rows, int teams, long most) {
  const long n = (rows + teams - 1) / teams;
  return (unsigned)(n < most ? n : most);
}

template <typename T>
static void ln_fwd_run(RowsIn x, RowsOut y, const float* w, const float* b,
                       float* mean, float* rstd, long rows, int cols,
                       float eps, hipStream_t s) {
  constexpr int N = Pack<T>::N;
  if (cols > LN_MOST) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(ln_fwd_k<T>), dim3(row_grid(rows)),
                       dim3(LN_LONG), 0, s, x, y, w, b, mean, rstd, rows,
                       cols, eps);
    return;
  }
#define RUN2(THREADS, TEAM, E, EXACT, TINY)                                  \
  hipLaunchKernelGGL(                                                        \
      HIP_KERNEL_NAME(ln_fwd_team_k<T, THREADS, TEAM, E / N, EXACT, TINY>),  \
      dim3(team_grid(rows, THREADS / TEAM, LN_FORWARD * 256 / THREADS)),     \
      dim3(THREADS), 0, s, x, y, w, b, mean, rstd, rows, cols, eps)
#define RUN(THREADS, TEAM, E)                                                \
  if (cols % N == 0)                                                         \
    RUN2(THREADS, TEAM, E, true, false);                                     \
  else                                                                       \
    RUN2(THREADS, TEAM, E, false, false)
  if (cols < N)
    RUN2(256, 4, 8, false, true);
  else
    LN_TEAMS(cols, RUN);
#undef RUN
#undef RUN2
}

void layer_norm_fwd_launch(int type, RowsIn x, RowsOut y, const float* w,
                           const float* b, float* mean, float* rstd,
                           long rows, int cols, float eps, hipStream_t s) {
  if (rows == 0) return;
#define RUN(T) ln_fwd_run<T>(x, y, w, b, mean, rstd, rows, cols, eps, s)
  ROW_TYPE_SWITCH(type, RUN)
#undef RUN
  HIP_CHECK_LAST();
}

// workgroups of a backward pass, or partial sums that it leaves
static long ln_parts(long rows, int cols) {
  if (cols > LN_MOST_SUMS) {
    long n = rows < LN_PARTS_FEW ? rows : LN_PARTS_FEW;
    if (n < rows / 32) n = rows / 32;
    return n < LN_PARTS ? n : LN_PARTS;
  }
  long n = 0;
#define GRID(THREADS, TEAM, E) n = team_grid(rows, 1024 / TEAM, LN_BACKWARD)
  LN_TEAMS(cols, GRID);
#undef GRID
  return n;
}

// floats that layer_norm_bwd_launch needs at `part` where it is asked for
// dw or db
long layer_norm_bwd_scratch(long rows, int cols) {
  return ln_parts(rows, cols) * 2 * cols;
}

template <typename T>
static void ln_bwd_run(RowsIn dy, RowsIn x, const float* w,
                       const float* mean, const float* rstd, RowsOut dx,
                       bool sums, float* part, long rows, int cols,
                       hipStream_t s) {
  constexpr int N = Pack<T>::N;
  if (cols > LN_MOST_SUMS) {
    // the sums first: dx may be written over dy or x
    if (sums) {
      const int packs = (cols + N - 1) / N;
      hipLaunchKernelGGL(HIP_KERNEL_NAME(ln_cols_k<T>),
                         dim3((packs + LN_THREADS - 1) / LN_THREADS,
                              (unsigned)ln_parts(rows, cols)),
                         dim3(LN_THREADS), 0, s, dy, x, mean, rstd, part,
                         rows, cols);
      HIP_CHECK_LAST();
    }
    if (dx.p)
      hipLaunchKernelGGL(HIP_KERNEL_NAME(ln_bwd_k<T>), dim3(row_grid(rows)),
                         dim3(LN_LONG), 0, s, dy, x, w, mean, rstd, dx,
                         rows, cols);
    return;
  }
  const dim3 grid((unsigned)ln_parts(rows, cols));
#define RUN2(TEAM, E, EXACT, SUMS, DX, TINY)                                 \
  hipLaunchKernelGGL(                                                        \
      HIP_KERNEL_NAME(                                                       \
          ln_bwd_team_k<T, 1024, TEAM, E / N, EXACT, SUMS, DX, TINY>),       \
      grid, dim3(1024), 0, s, dy, x, w, mean, rstd, dx, part, rows, cols)
#define RUN(THREADS, TEAM, E)                                                \
  if constexpr (E == 32)                                                     \
    return;                                                                  \
  else if (cols % N == 0 && sums && dx.p)                                    \
    RUN2(TEAM, E, true, true, true, false);                                  \
  else if (sums && dx.p)                                                     \
    RUN2(TEAM, E, false, true, true, false);                                 \
  else if (sums)                                                             \
    RUN2(TEAM, E, false, true, false, false);                                \
  else                                                                       \
    RUN2(TEAM, E, false, false, true, false)
  if (cols >= N)
    LN_TEAMS(cols, RUN);
  else if (sums && dx.p)
    RUN2(4, 8, false, true, true, true);
  else if (sums)
    RUN2(4, 8, false, true, false, true);
  else
    RUN2(4, 8, false, false, true, true);
#undef RUN
#undef RUN2
}

void layer_norm_bwd_launch(int type, RowsIn dy, RowsIn x, const float* w,
                           const float* mean, const float* rstd, RowsOut dx,
                           float* dw, float* db, bool accumulate,
                           float* part, long rows, int cols,
                           hipStream_t s) {
  const bool sums = dw || db;
  if (rows && (sums || dx.p)) {
#define RUN(T)                                                               \
  ln_bwd_run<T>(dy, x, w, mean, rstd, dx, sums, part, rows, cols, s)
    ROW_TYPE_SWITCH(type, RUN)
#undef RUN
    HIP_CHECK_LAST();
  }
  if (!sums) return;
  hipLaunchKernelGGL(ln_join_k, dim3((2l * cols + 31) / 32),
                     dim3(LN_THREADS), 0, s, part,
                     (int)ln_parts(rows, cols), dw, db, cols,
                     (int)accumulate);
  HIP_CHECK_LAST();
}
