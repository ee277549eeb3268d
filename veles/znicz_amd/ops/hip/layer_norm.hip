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
// rows of partial column sums that a backward pass leaves to be joined
#define LN_PARTS 256
// workgroups of 256 threads that a backward pass of teams has at most
#define LN_BLOCKS 768
#ifndef LN_RA
#define LN_RA 2
#define LN_RB 2
#define LN_RC 1
#define LN_FB 2048
#define LN_ONCE 0
#endif

// one workgroup to a row; the row is read three times, from the caches
// after the first
template <typename T>
__global__ __launch_bounds__(LN_THREADS) void ln_fwd_k(
    RowsIn x_, RowsOut y_, const float* __restrict__ w,
    const float* __restrict__ b, float* __restrict__ mean,
    float* __restrict__ rstd, long rows, int cols, float eps) {
  __shared__ float tmp[LN_THREADS / WAVE];
  for (long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* x = (const T*)x_.p + row * x_.stride;
    T* y = (T*)y_.p + row * y_.stride;
    float s = 0.f;
    for (int j = threadIdx.x; j < cols; j += LN_THREADS) s += (float)x[j];
    const float mu = block_sum(s, tmp) / cols;
    float v = 0.f;
    for (int j = threadIdx.x; j < cols; j += LN_THREADS) {
      const float d = (float)x[j] - mu;
      v += d * d;
    }
    const float r = 1.f / sqrtf(block_sum(v, tmp) / cols + eps);
    for (int j = threadIdx.x; j < cols; j += LN_THREADS) {
      float h = ((float)x[j] - mu) * r;
      if (w) h *= w[j];
      if (b) h += b[j];
      y[j] = from_f<T>(h);
    }
    if (threadIdx.x == 0) {
      if (mean) mean[row] = mu;
      if (rstd) rstd[row] = r;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(LN_THREADS) void ln_bwd_k(
    RowsIn dy_, RowsIn x_, const float* __restrict__ w,
    const float* __restrict__ mean, const float* __restrict__ rstd,
    RowsOut dx_, long rows, int cols) {
  __shared__ float tmp[LN_THREADS / WAVE];
  for (long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* dy = (const T*)dy_.p + row * dy_.stride;
    const T* x = (const T*)x_.p + row * x_.stride;
    T* dx = (T*)dx_.p + row * dx_.stride;
    const float mu = mean[row], r = rstd[row];
    float s1 = 0.f, s2 = 0.f;
    for (int j = threadIdx.x; j < cols; j += LN_THREADS) {
      const float g = (float)dy[j] * (w ? w[j] : 1.f);
      s1 += g;
      s2 += g * (((float)x[j] - mu) * r);
    }
    s1 = block_sum(s1, tmp) / cols;
    s2 = block_sum(s2, tmp) / cols;
    for (int j = threadIdx.x; j < cols; j += LN_THREADS) {
      const float g = (float)dy[j] * (w ? w[j] : 1.f);
      const float h = ((float)x[j] - mu) * r;
      dx[j] = from_f<T>(r * (g - s1 - h * s2));
    }
  }
}

// column sums of dy xh and dy over this workgroup's rows: one thread to a
// column, part[blockIdx.y] = [2][cols]
template <typename T>
__global__ __launch_bounds__(LN_THREADS) void ln_cols_k(
    RowsIn dy_, RowsIn x_, const float* __restrict__ mean,
    const float* __restrict__ rstd, float* __restrict__ part, long rows,
    int cols) {
  const int j = blockIdx.x * LN_THREADS + threadIdx.x;
  if (j >= cols) return;
  const long per = (rows + gridDim.y - 1) / gridDim.y;
  const long lo = blockIdx.y * per;
  const long hi = lo + per < rows ? lo + per : rows;
  float sw = 0.f, sb = 0.f;
  for (long row = lo; row < hi; ++row) {
    const float g = (float)((const T*)dy_.p)[row * dy_.stride + j];
    const float h =
        ((float)((const T*)x_.p)[row * x_.stride + j] - mean[row]) *
        rstd[row];
    sw += g * h;
    sb += g;
  }
  float* out = part + (long)blockIdx.y * 2 * cols;
  out[j] = sw;
  out[cols + j] = sb;
}

// The partial sums [parts][2][cols] joined, always in the same order: 32 of
// the 2 cols columns to a workgroup, 8 slices of the parts
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
// A team of lanes has a row, 8 or 16 elements a lane: a part of a wave, a
// wave, or a whole workgroup, as the row is long.  It goes through the rows
// in steps, several at a time, with the gain and the shift (backward: the
// gain and the two column sums) in registers all along.

// the team's sums of R values each, in all its lanes; `tmp`: [2][R][waves],
// used in turn so that one barrier does for a call
template <int TEAM, int R>
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
      constexpr int WAVES = TEAM / WAVE;
      float* t = tmp + turn * R * WAVES;
      turn ^= 1;
      const int lane = threadIdx.x & (WAVE - 1);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float w = wave_sum_last(v[i]);
        if (lane == WAVE - 1) t[i * WAVES + threadIdx.x / WAVE] = w;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < R; ++i) {
        v[i] = t[i * WAVES + lane % WAVES];
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

// Where a lane's packs of a row lie.  The last pack of a row that is no
// whole number of packs ends with the row, so that its first elements are
// the pack's before, too; a lane beyond the last pack has that one again.
// Both are loaded and stored like any other (the same values to the same
// place), which spares the branches, and are left out of the sums.  A row
// shorter than a pack (TINY) is read and written one by one.
template <typename T, int TEAM, int NV, bool TINY>
struct Slots {
  static constexpr int N = Pack<T>::N;
  int lane, cols, packs;

  __device__ __forceinline__ Slots(int cols_) {
    lane = TEAM <= WAVE ? threadIdx.x % TEAM : threadIdx.x;
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
    const int j = (i * TEAM + lane) * N;
    return has(i) && at(i) + k >= j && at(i) + k < cols;
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
  // parameters of the lane's columns
  __device__ __forceinline__ void load_param(float* v, const float* p,
                                             float none) const {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k)
        v[i * N + k] = p && (!TINY || k < cols) ? p[at(i) + k] : none;
  }
};

// The rows of a team: from `start`, `step` apart R at a time.  All lanes of
// a wave (a workgroup, where it is the team) make the same number of steps.
template <int THREADS, int TEAM, int R>
struct Steps {
  long start, teams;
  int mine;        // this lane's team among those of its wave

  __device__ __forceinline__ Steps() {
    constexpr int TEAMS = THREADS / TEAM;
    teams = (long)gridDim.x * TEAMS;
    start = (long)blockIdx.x * TEAMS;
    if (TEAM < THREADS)
      start += __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE) *
               (TEAM < WAVE ? WAVE / TEAM : 1);
    mine = TEAM < WAVE ? (threadIdx.x & (WAVE - 1)) / TEAM : 0;
  }
  // whether all rows of the step from `first` exist
  __device__ __forceinline__ bool full(long first, long rows) const {
    return first + (R - 1) * teams + (TEAM < WAVE ? WAVE / TEAM - 1 : 0) <
           rows;
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
// otherwise wait for stores to reach memory.  For the same reason nothing
// after those loads is on a condition; the last step is apart.
template <typename T, int THREADS, int TEAM, int NV, int R, bool EXACT,
          bool TINY>
__global__ __launch_bounds__(THREADS) void ln_fwd_team_k(
    RowsIn x_, RowsOut y_, const float* __restrict__ w,
    const float* __restrict__ b, float* __restrict__ mean,
    float* __restrict__ rstd, long rows, int cols, float eps) {
  constexpr int N = Pack<T>::N;
  __shared__ float tmp[2 * R * (THREADS / WAVE)];
  TeamSum<TEAM, R> sum{tmp, 0};
  const Slots<T, TEAM, NV, TINY> at(cols);
  const Steps<THREADS, TEAM, R> steps;
  float gain[NV * N], shift[NV * N];
  const float per = 1.f / cols;
  Pack<T> v[R][NV];
  auto load = [&](long row0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long row = min(row0 + r * steps.teams, rows - 1);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        at.load(v[r][i], (const T*)x_.p + row * x_.stride, i);
    }
  };
  auto step = [&](long row0, bool last) {
    float mu[R], rs[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mu[r] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float e[N], q = 0.f;
        v[r][i].get(e);
#pragma unroll
        for (int k = 0; k < N; ++k)
          q += EXACT || at.own(i, k) ? e[k] : 0.f;
        mu[r] += at.has(i) ? q : 0.f;
      }
    }
    sum(mu);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mu[r] *= per;
      rs[r] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float e[N], q = 0.f;
        v[r][i].forget();
        v[r][i].get(e);
#pragma unroll
        for (int k = 0; k < N; ++k) {
          float d = e[k] - mu[r];
          if (!EXACT) d = at.own(i, k) ? d : 0.f;
          q = fmaf(d, d, q);
        }
        rs[r] += at.has(i) ? q : 0.f;
      }
    }
    sum(rs);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long row = row0 + r * steps.teams;
      rs[r] = inv_sqrt(fmaf(rs[r], per, eps));
      if (at.lane == 0 && mean && row < rows) mean[row] = mu[r];
      if (at.lane == 0 && rstd && row < rows) rstd[row] = rs[r];
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float e[N];
        v[r][i].forget();
        v[r][i].get(e);
#pragma unroll
        for (int k = 0; k < N; ++k)
          e[k] = fmaf((e[k] - mu[r]) * rs[r], gain[i * N + k],
                      shift[i * N + k]);
        v[r][i].set(e);
      }
    Pack<T> y[R][NV];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < NV; ++i) y[r][i] = v[r][i];
    if (!last) load(row0 + R * steps.teams);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long row = row0 + r * steps.teams;
      if (last && row >= rows) continue;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        at.store(y[r][i], (T*)y_.p + row * y_.stride, i);
    }
  };
  load(steps.start + steps.mine);
  at.load_param(gain, w, 1.f);
  at.load_param(shift, b, 0.f);
  long first = steps.start;
  wait_loads();
  for (; steps.full(first, rows); first += R * steps.teams)
    step(first + steps.mine, false);
  if (first < rows) step(first + steps.mine, true);
}

// The backward pass of the same teams; part[block] = [2][cols], the
// workgroup's column sums.  SUMS: dw and db are asked for.
template <typename T, int THREADS, int TEAM, int NV, int R, bool EXACT,
          bool SUMS, bool TINY>
__global__ __launch_bounds__(THREADS) void ln_bwd_team_k(
    RowsIn dy_, RowsIn x_, const float* __restrict__ w,
    const float* __restrict__ mean, const float* __restrict__ rstd,
    RowsOut dx_, float* __restrict__ part, long rows, int cols) {
  constexpr int N = Pack<T>::N, E = NV * N;
  __shared__ float tmp[4 * R * (THREADS / WAVE)];
  TeamSum<TEAM, 2 * R> sum{tmp, 0};
  const Slots<T, TEAM, NV, TINY> at(cols);
  const Steps<THREADS, TEAM, R> steps;
  float gain[E], dw[E], db[E];
  const float per = 1.f / cols;
  Pack<T> vx[R][NV], vg[R][NV];
  float mu[R], rs[R];
  auto load = [&](long row0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long row = min(row0 + r * steps.teams, rows - 1);
      mu[r] = mean[row];
      rs[r] = rstd[row];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        at.load(vx[r][i], (const T*)x_.p + row * x_.stride, i);
        at.load(vg[r][i], (const T*)dy_.p + row * dy_.stride, i);
      }
    }
  };
  auto step = [&](long row0, bool last) {
    float s[2 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (last && row0 + r * steps.teams >= rows) {
        mu[r] = rs[r] = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          vx[r][i].fill(0.f);
          vg[r][i].fill(0.f);
        }
      }
      s[2 * r] = s[2 * r + 1] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float e[N], g[N], s1 = 0.f, s2 = 0.f;
        vx[r][i].get(e);
        vg[r][i].get(g);
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const float h = (e[k] - mu[r]) * rs[r];
          if (SUMS) {
            dw[i * N + k] = fmaf(g[k], h, dw[i * N + k]);
            db[i * N + k] += g[k];
          }
          float d = g[k] * gain[i * N + k];
          if (!EXACT) d = at.own(i, k) ? d : 0.f;
          s1 += d;
          s2 = fmaf(d, h, s2);
        }
        s[2 * r] += at.has(i) ? s1 : 0.f;
        s[2 * r + 1] += at.has(i) ? s2 : 0.f;
      }
    }
    if (!dx_.p) {
      if (!last) load(row0 + R * steps.teams);
      return;
    }
    sum(s);
    Pack<T> out[R][NV];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float s1 = s[2 * r] * per, s2 = s[2 * r + 1] * per;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float e[N], g[N];
        vx[r][i].forget();
        vg[r][i].forget();
        vx[r][i].get(e);
        vg[r][i].get(g);
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const float h = (e[k] - mu[r]) * rs[r];
          g[k] = rs[r] * (fmaf(g[k], gain[i * N + k], -s1) - h * s2);
        }
        out[r][i].set(g);
      }
    }
    if (!last) load(row0 + R * steps.teams);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long row = row0 + r * steps.teams;
      if (last && row >= rows) continue;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        at.store(out[r][i], (T*)dx_.p + row * dx_.stride, i);
    }
  };
  load(steps.start + steps.mine);
  at.load_param(gain, w, 1.f);
#pragma unroll
  for (int k = 0; k < E; ++k) dw[k] = db[k] = 0.f;
  long first = steps.start;
  wait_loads();
  for (; steps.full(first, rows); first += R * steps.teams)
    step(first + steps.mine, false);
  if (first < rows) step(first + steps.mine, true);
  if (!SUMS) return;
  // the workgroup's sums: over the teams of a wave, then over the waves
  float* out = part + (long)blockIdx.x * 2 * cols;
  if constexpr (TEAM < THREADS) {
    __shared__ float all[2 * E * TEAM];
#pragma unroll
    for (int k = 0; k < E; ++k) {
#pragma unroll
      for (int off = TEAM; off < WAVE; off *= 2) {
        dw[k] += __shfl_xor(dw[k], off);
        db[k] += __shfl_xor(db[k], off);
      }
    }
    const int lane = threadIdx.x & (WAVE - 1);
    for (int v = 0; v < THREADS / WAVE; ++v) {
      if ((int)threadIdx.x / WAVE == v && lane < TEAM) {
#pragma unroll
        for (int k = 0; k < E; ++k) {
          const int a = k * TEAM + lane;
          all[a] = v ? all[a] + dw[k] : dw[k];
          all[E * TEAM + a] = v ? all[E * TEAM + a] + db[k] : db[k];
        }
      }
      __syncthreads();
    }
    if ((int)threadIdx.x >= TEAM) return;
#pragma unroll
    for (int k = 0; k < E; ++k) {
      dw[k] = all[k * TEAM + lane];
      db[k] = all[E * TEAM + k * TEAM + lane];
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (at.own(i, k)) {
        out[at.at(i) + k] = dw[i * N + k];
        out[cols + at.at(i) + k] = db[i * N + k];
      }
}

static unsigned row_grid(long rows) {
  return (unsigned)(rows < 65536 ? rows : 65536);
}

// the elements of a row that a team of lanes holds at most: 8 or 16 each
#define LN_MOST 16384

// F(threads, team, elements of a lane, rows at a time) of the first team
// that holds a row
#define LN_TEAMS(cols, F)                                                    \
  do {                                                                       \
    if (cols <= 32) {                                                        \
      F(256, 4, 8, LN_RA);                                                   \
    } else if (cols <= 64) {                                                 \
      F(256, 8, 8, LN_RA);                                                   \
    } else if (cols <= 128) {                                                \
      F(256, 16, 8, LN_RA);                                                  \
    } else if (cols <= 256) {                                                \
      F(256, 32, 8, LN_RA);                                                  \
    } else if (cols <= 512) {                                                \
      F(256, 64, 8, LN_RA);                                                  \
    } else if (cols <= 1024) {                                               \
      F(128, 128, 8, LN_RB);                                                 \
    } else if (cols <= 2048) {                                               \
      F(256, 256, 8, LN_RB);                                                 \
    } else if (cols <= 4096) {                                               \
      F(512, 512, 8, LN_RB);                                                 \
    } else if (cols <= 8192) {                                               \
      F(1024, 1024, 8, LN_RB);                                               \
    } else {                                                                 \
      F(1024, 1024, 16, LN_RC);                                              \
    }                                                                        \
  } while (0)

static unsigned team_grid(long rows, int teams, int at_once, long most) {
  const long n = (rows + (long)teams * at_once - 1) / ((long)teams * at_once);
  return (unsigned)(n < most ? n : most);
}

template <typename T>
static void ln_fwd_run(RowsIn x, RowsOut y, const float* w, const float* b,
                       float* mean, float* rstd, long rows, int cols,
                       float eps, hipStream_t s) {
  constexpr int N = Pack<T>::N;
  if (cols > LN_MOST) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(ln_fwd_k<T>), dim3(row_grid(rows)),
                       dim3(LN_THREADS), 0, s, x, y, w, b, mean, rstd, rows,
                       cols, eps);
    return;
  }
  const bool exact = cols % N == 0;
#define RUN2(THREADS, TEAM, E, R, EXACT, TINY)                               \
  hipLaunchKernelGGL(                                                        \
      HIP_KERNEL_NAME(                                                       \
          ln_fwd_team_k<T, THREADS, TEAM, E / N, R, EXACT, TINY>),           \
      dim3(team_grid(rows, THREADS / TEAM, R, LN_FB * 256 / THREADS)),        \
      dim3(THREADS), 0, s, x, y, w, b, mean, rstd, rows, cols, eps)
#define RUN(THREADS, TEAM, E, R)                                             \
  if (exact)                                                                 \
    RUN2(THREADS, TEAM, E, R, true, false);                                  \
  else                                                                       \
    RUN2(THREADS, TEAM, E, R, false, false)
  if (cols < N)
    RUN2(256, 4, 8, LN_RA, false, true);
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

// workgroups of a backward pass that leaves partial sums
static long ln_parts(long rows, int cols) {
  if (cols > LN_MOST) return rows < LN_PARTS ? rows : LN_PARTS;
  long n = 0;
#define GRID(THREADS, TEAM, E, R)                                            \
  n = team_grid(rows, THREADS / TEAM, R, LN_BLOCKS * 256 / THREADS)
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
  if (cols > LN_MOST) {
    // the sums first: dx may be written over dy or x
    if (sums)
      hipLaunchKernelGGL(
          HIP_KERNEL_NAME(ln_cols_k<T>),
          dim3((cols + LN_THREADS - 1) / LN_THREADS,
               (unsigned)ln_parts(rows, cols)),
          dim3(LN_THREADS), 0, s, dy, x, mean, rstd, part, rows, cols);
    HIP_CHECK_LAST();
    if (dx.p)
      hipLaunchKernelGGL(HIP_KERNEL_NAME(ln_bwd_k<T>), dim3(row_grid(rows)),
                         dim3(LN_THREADS), 0, s, dy, x, w, mean, rstd, dx,
                         rows, cols);
    return;
  }
  const unsigned grid = (unsigned)ln_parts(rows, cols);
  const bool exact = cols % N == 0;
#define RUN2(THREADS, TEAM, E, R, EXACT, SUMS, TINY)                         \
  hipLaunchKernelGGL(                                                        \
      HIP_KERNEL_NAME(                                                       \
          ln_bwd_team_k<T, THREADS, TEAM, E / N, R, EXACT, SUMS, TINY>),     \
      dim3(grid), dim3(THREADS), 0, s, dy, x, w, mean, rstd, dx, part, rows, \
      cols)
#define RUN(THREADS, TEAM, E, R)                                             \
  if (exact && sums)                                                         \
    RUN2(THREADS, TEAM, E, R, true, true, false);                            \
  else if (sums)                                                             \
    RUN2(THREADS, TEAM, E, R, false, true, false);                           \
  else                                                                       \
    RUN2(THREADS, TEAM, E, R, false, false, false)
  if (cols < N && sums)
    RUN2(256, 4, 8, LN_RA, false, true, true);
  else if (cols < N)
    RUN2(256, 4, 8, LN_RA, false, false, true);
  else
    LN_TEAMS(cols, RUN);
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
