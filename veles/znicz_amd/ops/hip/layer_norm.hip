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

// the columns' partial sums joined, always in the same order
__global__ __launch_bounds__(LN_THREADS) void ln_join_k(
    const float* __restrict__ part, int parts, float* __restrict__ dw,
    float* __restrict__ db, int cols, int accumulate) {
  const int j = blockIdx.x * LN_THREADS + threadIdx.x;
  if (j >= cols) return;
  float sw = 0.f, sb = 0.f;
  for (int i = 0; i < parts; ++i) {
    sw += part[(long)i * 2 * cols + j];
    sb += part[(long)i * 2 * cols + cols + j];
  }
  if (dw) dw[j] = accumulate ? dw[j] + sw : sw;
  if (db) db[j] = accumulate ? db[j] + sb : sb;
}

static unsigned row_grid(long rows) {
  return (unsigned)(rows < 65536 ? rows : 65536);
}

void layer_norm_fwd_launch(int type, RowsIn x, RowsOut y, const float* w,
                           const float* b, float* mean, float* rstd,
                           long rows, int cols, float eps, hipStream_t s) {
  if (rows == 0) return;
#define RUN(T)                                                               \
  hipLaunchKernelGGL(HIP_KERNEL_NAME(ln_fwd_k<T>), dim3(row_grid(rows)),     \
                     dim3(LN_THREADS), 0, s, x, y, w, b, mean, rstd, rows,   \
                     cols, eps)
  ROW_TYPE_SWITCH(type, RUN)
#undef RUN
  HIP_CHECK_LAST();
}

// floats that layer_norm_bwd_launch needs at `part` where it is asked for
// dw or db
long layer_norm_bwd_scratch(int type, long rows, int cols) {
  (void)type;
  const long parts = rows < LN_PARTS ? rows : LN_PARTS;
  return parts * 2 * cols;
}

void layer_norm_bwd_launch(int type, RowsIn dy, RowsIn x, const float* w,
                           const float* mean, const float* rstd, RowsOut dx,
                           float* dw, float* db, bool accumulate,
                           float* part, long rows, int cols,
                           hipStream_t s) {
  const unsigned cblocks = (cols + LN_THREADS - 1) / LN_THREADS;
  // the sums first: dx may be written over dy or x
  if (dw || db) {
    const unsigned parts = (unsigned)(rows < LN_PARTS ? rows : LN_PARTS);
    if (parts) {
#define RUN(T)                                                               \
  hipLaunchKernelGGL(HIP_KERNEL_NAME(ln_cols_k<T>), dim3(cblocks, parts),    \
                     dim3(LN_THREADS), 0, s, dy, x, mean, rstd, part, rows,  \
                     cols)
      ROW_TYPE_SWITCH(type, RUN)
#undef RUN
      HIP_CHECK_LAST();
    }
    hipLaunchKernelGGL(ln_join_k, dim3(cblocks), dim3(LN_THREADS), 0, s,
                       part, (int)parts, dw, db, cols, (int)accumulate);
    HIP_CHECK_LAST();
  }
  if (dx.p && rows) {
#define RUN(T)                                                               \
  hipLaunchKernelGGL(HIP_KERNEL_NAME(ln_bwd_k<T>), dim3(row_grid(rows)),     \
                     dim3(LN_THREADS), 0, s, dy, x, w, mean, rstd, dx, rows, \
                     cols)
    ROW_TYPE_SWITCH(type, RUN)
#undef RUN
    HIP_CHECK_LAST();
  }
}
