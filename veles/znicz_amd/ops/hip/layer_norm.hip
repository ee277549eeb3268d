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
          if (TEAM > 4) {
            v[i] += other_lane<0x141>(v[i]);
            v[i] += other_lane<0x140>(v[i]);
          }
        }
      }
    } else {
      constexpr int WAVES = TEAM / WAVE;
      float* t = tmp + turn * R * WAVES;
      turn ^= 1;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float w = wave_sum(v[i]);
        if ((threadIdx.x & (WAVE - 1)) == 0) t[i * WAVES + threadIdx.x / WAVE] = w;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < R; ++i) {
        v[i] = 0.f;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) v[i] += t[i * WAVES + k];
      }
    }
  }
};

// Where a lane's packs of a row lie.  The last pack of a row that is no
// whole number of packs ends with the row, so that its first elements are
// the pack's before, too: `lo` of them count there.  A row shorter than a
// pack is read one by one.
template <typename T, int TEAM, int NV>
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
    return max(min(j, cols - N), 0);
  }
  // whether element k of pack i is this pack's own
  template <bool EXACT>
  __device__ __forceinline__ bool own(int i, int k) const {
    if (EXACT) return has(i);
    const int j = (i * TEAM + lane) * N;
    return has(i) && at(i) + k >= j && at(i) + k < cols;
  }
  __device__ __forceinline__ void load(Pack<T>& v, const T* row, int i) const {
    if (cols >= N) {
      v.load(row + at(i));
    } else {
      float e[N];
#pragma unroll
      for (int k = 0; k < N; ++k) e[k] = k < cols ? (float)row[k] : 0.f;
      v.set(e);
    }
  }
  __device__ __forceinline__ void store(const Pack<T>& v, T* row,
                                        int i) const {
    if (cols >= N) {
      v.store(row + at(i));
    } else {
      T e[N];
      __builtin_memcpy(e, &v.raw, 16);
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (k < cols) row[k] = e[k];
    }
  }
  // parameters of the lane's columns
  __device__ __forceinline__ void load_param(float* v, const float* p,
                                             float none) const {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int j = at(i) + k;
        v[i * N + k] = p && has(i) && j < cols ? p[j] : none;
      }
  }
};

template <typename T, int THREADS, int TEAM, int NV, int R, bool EXACT>
__global__ __launch_bounds__(THREADS) void ln_fwd_team_k(
    RowsIn x_, RowsOut y_, const float* __restrict__ w,
    const float* __restrict__ b, float* __restrict__ mean,
    float* __restrict__ rstd, long rows, int cols, float eps) {
  constexpr int N = Pack<T>::N, TEAMS = THREADS / TEAM;
  __shared__ float tmp[2 * R * (THREADS / WAVE)];
  TeamSum<TEAM, R> sum{tmp, 0};
  const Slots<T, TEAM, NV> at(cols);
  float gain[NV * N], shift[NV * N];
  at.load_param(gain, w, 1.f);
  at.load_param(shift, b, 0.f);
  const long teams = (long)gridDim.x * TEAMS;
  const float per = 1.f / cols;
  // (all lanes of a wave make the same number of steps)
  for (long first = (long)blockIdx.x * TEAMS + (TEAM < THREADS
                        ? (int)threadIdx.x / WAVE * (WAVE / TEAM) : 0);
       first < rows; first += teams * R) {
    const long row0 =
        first + (TEAM < WAVE ? (threadIdx.x & (WAVE - 1)) / TEAM : 0);
    Pack<T> v[R][NV];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long row = row0 + r * teams;
      const T* x = (const T*)x_.p + row * x_.stride;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        v[r][i].fill(0.f);
        if (row < rows && at.has(i)) at.load(v[r][i], x, i);
      }
    }
    float mu[R], rs[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mu[r] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float e[N];
        v[r][i].get(e);
#pragma unroll
        for (int k = 0; k < N; ++k)
          mu[r] += EXACT || at.template own<EXACT>(i, k) ? e[k] : 0.f;
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
          if (!EXACT) d = at.template own<EXACT>(i, k) ? d : 0.f;
          q = fmaf(d, d, q);
        }
        rs[r] += at.has(i) ? q : 0.f;
      }
    }
    sum(rs);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long row = row0 + r * teams;
      rs[r] = 1.f / sqrtf(fmaf(rs[r], per, eps));
      if (row >= rows) continue;
      T* y = (T*)y_.p + row * y_.stride;
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
        if (at.has(i)) at.store(v[r][i], y, i);
      }
      if (at.lane == 0) {
        if (mean) mean[row] = mu[r];
        if (rstd) rstd[row] = rs[r];
      }
    }
  }
}

// The backward pass of the same teams; part[block] = [2][cols], the
// workgroup's column sums.  SUMS: dw and db are asked for.
template <typename T, int THREADS, int TEAM, int NV, int R, bool EXACT,
          bool SUMS>
__global__ __launch_bounds__(THREADS) void ln_bwd_team_k(
    RowsIn dy_, RowsIn x_, const float* __restrict__ w,
    const float* __restrict__ mean, const float* __restrict__ rstd,
    RowsOut dx_, float* __restrict__ part, long rows, int cols) {
  constexpr int N = Pack<T>::N, TEAMS = THREADS / TEAM, E = NV * N;
  __shared__ float tmp[4 * R * (THREADS / WAVE)];
  TeamSum<TEAM, 2 * R> sum{tmp, 0};
  const Slots<T, TEAM, NV> at(cols);
  float gain[E], dw[E], db[E];
  at.load_param(gain, w, 1.f);
#pragma unroll
  for (int k = 0; k < E; ++k) dw[k] = db[k] = 0.f;
  const long teams = (long)gridDim.x * TEAMS;
  const float per = 1.f / cols;
  for (long first = (long)blockIdx.x * TEAMS + (TEAM < THREADS
                        ? (int)threadIdx.x / WAVE * (WAVE / TEAM) : 0);
       first < rows; first += teams * R) {
    const long row0 =
        first + (TEAM < WAVE ? (threadIdx.x & (WAVE - 1)) / TEAM : 0);
    Pack<T> vx[R][NV], vg[R][NV];
    float mu[R], rs[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long row = row0 + r * teams;
      const T* x = (const T*)x_.p + row * x_.stride;
      const T* g = (const T*)dy_.p + row * dy_.stride;
      mu[r] = rs[r] = 0.f;
      if (row < rows) {
        mu[r] = mean[row];
        rs[r] = rstd[row];
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        vx[r][i].fill(0.f);
        vg[r][i].fill(0.f);
        if (row < rows && at.has(i)) {
          at.load(vx[r][i], x, i);
          at.load(vg[r][i], g, i);
        }
      }
    }
    float s[2 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s[2 * r] = s[2 * r + 1] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float e[N], g[N];
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
          if (!EXACT) d = at.template own<EXACT>(i, k) ? d : 0.f;
          s[2 * r] += d;
          s[2 * r + 1] = fmaf(d, h, s[2 * r + 1]);
        }
      }
    }
    if (!dx_.p) continue;
    sum(s);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long row = row0 + r * teams;
      if (row >= rows) continue;
      T* dx = (T*)dx_.p + row * dx_.stride;
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
        vg[r][i].set(g);
        if (at.has(i)) at.store(vg[r][i], dx, i);
      }
    }
  }
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
      if (at.template own<false>(i, k)) {
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
      F(256, 4, 8, 4);                                                       \
    } else if (cols <= 64) {                                                 \
      F(256, 4, 16, 2);                                                      \
    } else if (cols <= 128) {                                                \
      F(256, 16, 8, 4);                                                      \
    } else if (cols <= 256) {                                                \
      F(256, 16, 16, 2);                                                     \
    } else if (cols <= 512) {                                                \
      F(256, 64, 8, 4);                                                      \
    } else if (cols <= 1024) {                                               \
      F(256, 64, 16, 2);                                                     \
    } else if (cols <= 2048) {                                               \
      F(256, 256, 8, 4);                                                     \
    } else if (cols <= 4096) {                                               \
      F(256, 256, 16, 2);                                                    \
    } else if (cols <= 8192) {                                               \
      F(1024, 1024, 8, 2);                                                   \
    } else {                                                                 \
      F(1024, 1024, 16, 1);                                                  \
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
#define RUN2(THREADS, TEAM, E, R, EXACT)                                     \
  hipLaunchKernelGGL(                                                        \
      HIP_KERNEL_NAME(ln_fwd_team_k<T, THREADS, TEAM, E / N, R, EXACT>),     \
      dim3(team_grid(rows, THREADS / TEAM, R, 2048 * 256 / THREADS)),        \
      dim3(THREADS), 0, s, x, y, w, b, mean, rstd, rows, cols, eps)
#define RUN(THREADS, TEAM, E, R)                                             \
  if (exact)                                                                 \
    RUN2(THREADS, TEAM, E, R, true);                                         \
  else                                                                       \
    RUN2(THREADS, TEAM, E, R, false)
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
#define RUN2(THREADS, TEAM, E, R, EXACT, SUMS)                               \
  hipLaunchKernelGGL(                                                        \
      HIP_KERNEL_NAME(                                                       \
          ln_bwd_team_k<T, THREADS, TEAM, E / N, R, EXACT, SUMS>),           \
      dim3(grid), dim3(THREADS), 0, s, dy, x, w, mean, rstd, dx, part, rows, \
      cols)
#define RUN(THREADS, TEAM, E, R)                                             \
  if (exact && sums)                                                         \
    RUN2(THREADS, TEAM, E, R, true, true);                                   \
  else if (sums)                                                             \
    RUN2(THREADS, TEAM, E, R, false, true);                                  \
  else                                                                       \
    RUN2(THREADS, TEAM, E, R, false, false)
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
