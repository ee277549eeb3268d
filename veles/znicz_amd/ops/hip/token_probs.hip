// Rows of logits x[0..V): log probabilities of given classes with the
// entropy and the top alternatives, and distillation from a teacher's top
// logits.
//   m = max x, s = sum exp(x - m), ln p_j = x_j - m - ln s
//   H = ln s - sum exp(x - m) (x - m) / s
// Exponents are taken to base 2 by one fused product for each class:
//   u_j = C x_j - M, M = C m rounded, d = C m - M the rounding's remainder,
//   exp(x_j - m) = 2^(u_j - d), so that ln s = (log2 sum 2^u - d) ln 2 holds
// to the last bit of its 32 whatever the size of the logits, and
//   H = (log2 sum 2^u - sum 2^u u / sum 2^u) ln 2.
// Where C m is so large that d is no longer small against 1, or no number at
// all (a row whose classes all hold the type's lowest value), u = (x - m) C
// takes its place, with d = 0.
// Minus infinity is a class that is not allowed.  A row with NaN or plus
// infinity has no distribution: its sum is NaN, and so is what it gives.
#include <stdexcept>

#include "rows.h"

#define TP_THREADS 256
#define LOG2E 1.44269504088896340736f
#define LN2 0.69314718055994530942f
// u is cut here where it is multiplied by its power, which is 0 by then
#define U_MIN -200.f

// largest allowed logit, and the sums over the row relative to it
struct RowSums {
  float m;      // -inf: no class is allowed
  float um;     // C m, rounded, 0 for a row without classes
  float d;      // C m - um
  float s;      // sum 2^u; NaN: the row has a NaN or plus infinity
  float w;      // sum 2^u u
  bool far;     // u = (x - m) C
};

__device__ __forceinline__ void row_reference(RowSums& r, float c) {
  const float m = r.m == -INFINITY ? 0.f : r.m;
  r.um = m * c;
  r.far = !(fabsf(r.um) < 0x1p20f);      // (d is below 1/16 then)
  r.d = r.far ? 0.f : fmaf(m, c, -r.um);
}

// (v_exp_f32, v_log_f32: one unit in the last place; powers below 2^-126
// are 0, and the sums are 1 at least)
template <bool FAR>
__device__ __forceinline__ float exponent(float x, float c,
                                          const RowSums& r) {
  return FAR ? (x - r.m) * c : fmaf(x, c, -r.um);
}
__device__ __forceinline__ float pow2(float u) {
  return __builtin_amdgcn_exp2f(u);
}
__device__ __forceinline__ float log2_of(float s) {
  return __builtin_amdgcn_logf(s);
}

// ln of the sum of exp((x - m) / tau)
__device__ __forceinline__ float ln_sum(const RowSums& r) {
  return (log2_of(r.s) - r.d) * LN2;
}

// an order of the values in whole numbers; the two zeros are one
__device__ __forceinline__ int order_of(float x) {
  const int i = __float_as_int(x + 0.f);
  return i < 0 ? i ^ 0x7fffffff : i;
}
__device__ __forceinline__ float value_of(int i) {
  return __int_as_float(i < 0 ? i ^ 0x7fffffff : i);
}

// Value and class in one number: a larger value is first, of equal values
// the lower class.  0 is below every class.
typedef unsigned long long rank_t;
__device__ __forceinline__ rank_t key_of(float x, int j) {
  return ((rank_t)((unsigned)order_of(x) ^ 0x80000000u) << 32) |
         (unsigned)(0x7fffffff - j);
}
__device__ __forceinline__ float key_value(rank_t k) {
  return value_of((int)((unsigned)(k >> 32) ^ 0x80000000u));
}
__device__ __forceinline__ int key_class(rank_t k) {
  return 0x7fffffff - (int)(unsigned)k;
}

__device__ __forceinline__ rank_t block_max_key(rank_t v, rank_t* tmp) {
#pragma unroll
  for (int off = 32; off; off >>= 1) {
    const rank_t o = __shfl_xor(v, off);
    v = o > v ? o : v;
  }
  if ((threadIdx.x & (WAVE - 1)) == 0) tmp[threadIdx.x / WAVE] = v;
  __syncthreads();
  v = tmp[0];
  for (int i = 1; i < (int)blockDim.x / WAVE; ++i) v = tmp[i] > v ? tmp[i] : v;
  __syncthreads();
  return v;
}

template <bool FAR, typename T>
__device__ __forceinline__ void add_row(const T* x, int cols, float c,
                                        const RowSums& r, float& s,
                                        float& w) {
  for (int j = threadIdx.x; j < cols; j += blockDim.x) {
    const float u = exponent<FAR>((float)x[j], c, r);
    const float e = pow2(u);
    s += e;
    w = fmaf(e, fmaxf(u, U_MIN), w);
  }
}

template <typename T>
__device__ RowSums row_sums(const T* x, int cols, float c, float* tmp) {
  RowSums r;
  float m = -INFINITY;
  for (int j = threadIdx.x; j < cols; j += blockDim.x)
    m = fmaxf(m, (float)x[j]);
  r.m = block_max(m, tmp);
  row_reference(r, c);
  float s = 0.f, w = 0.f;
  if (r.far)
    add_row<true>(x, cols, c, r, s, w);
  else
    add_row<false>(x, cols, c, r, s, w);
  r.s = block_sum(s, tmp);
  r.w = block_sum(w, tmp);
  return r;
}

// one workgroup to a row; the row is read again for each alternative
template <typename T>
__global__ __launch_bounds__(TP_THREADS) void logprobs_k(
    RowsIn x_, const int* __restrict__ labels, float* __restrict__ logprob,
    float* __restrict__ entropy, int* __restrict__ top_idx,
    float* __restrict__ top_lp, int top, long rows, long live, int cols) {
  __shared__ float tmp[TP_THREADS / WAVE];
  __shared__ rank_t ktmp[TP_THREADS / WAVE];
  for (long row = blockIdx.x; row < rows; row += gridDim.x) {
    const int tid = threadIdx.x;
    if (row >= live) {
      if (tid == 0) {
        if (logprob) logprob[row] = 0.f;
        if (entropy) entropy[row] = 0.f;
      }
      for (int k = tid; k < top; k += TP_THREADS) {
        top_idx[row * top + k] = -1;
        top_lp[row * top + k] = 0.f;
      }
      continue;
    }
    const T* x = (const T*)x_.p + row * x_.stride;
    const RowSums r = row_sums(x, cols, LOG2E, tmp);
    const bool none = r.m == -INFINITY && r.s == 0.f;
    const bool bad = r.s != r.s;
    const float ln = ln_sum(r);
    if (tid == 0) {
      if (entropy)
        entropy[row] = none ? 0.f : (log2_of(r.s) - r.w / r.s) * LN2;
      if (logprob) {
        const int l = labels[row];
        float v = 0.f;
        if (l >= cols)
          v = NAN;
        else if (l >= 0)
          v = bad ? NAN : none ? -INFINITY : ((float)x[l] - r.m) - ln;
        logprob[row] = v;
      }
    }
    rank_t last = ~0ull;
    for (int k = 0; k < top; ++k) {
      rank_t best = 0;
      if (!bad && !none && last)
        for (int j = tid; j < cols; j += TP_THREADS) {
          const float v = (float)x[j];
          const rank_t key = v == -INFINITY ? 0 : key_of(v, j);
          if (key < last && key > best) best = key;
        }
      best = block_max_key(best, ktmp);
      if (tid == 0) {
        top_idx[row * top + k] = best ? key_class(best) : -1;
        top_lp[row * top + k] =
            bad ? NAN : best ? (key_value(best) - r.m) - ln : -INFINITY;
      }
      last = best;
    }
  }
}

// Distillation: q = softmax(z / tau) over the teacher's classes, p =
// softmax(x / tau) over all;
//   loss = tau^2 sum q (ln q - ln p),  dloss/dx_j = tau (p_j - q_j).
// One workgroup to a row.  A class that is named twice has the sum of both.
template <typename T, typename O>
__global__ __launch_bounds__(TP_THREADS) void distill_k(
    RowsIn x_, const int* __restrict__ idx, const float* __restrict__ z,
    RowsOut err_, float* __restrict__ loss, const int* __restrict__ labels,
    int* __restrict__ n_err, int top, long rows, long live, int cols,
    float tau) {
  __shared__ float tmp[TP_THREADS / WAVE];
  __shared__ int sid[MAX_TOP];
  __shared__ float sq[MAX_TOP];
  const int tid = threadIdx.x;
  for (long row = blockIdx.x; row < rows; row += gridDim.x) {
    O* err = (O*)err_.p + row * err_.stride;
    if (row >= live) {
      for (int j = tid; j < cols; j += TP_THREADS) err[j] = from_f<O>(0.f);
      if (tid == 0 && loss) loss[row] = 0.f;
      continue;
    }
    const T* x = (const T*)x_.p + row * x_.stride;
    const float c = LOG2E / tau;
    const RowSums r = row_sums(x, cols, c, tmp);
    const bool none = r.m == -INFINITY && r.s == 0.f;
    // the teacher's distribution: thread k has its k-th class
    int id = -1;
    float t = -INFINITY, xk = 0.f;
    bool wrong = false;
    if (tid < top) {
      id = idx[row * top + tid];
      if (id >= cols) {
        wrong = true;
      } else if (id >= 0) {
        t = z[row * top + tid];
        wrong = !(t < INFINITY);
        xk = (float)x[id];
      }
      if (wrong || t == -INFINITY) id = -1;
    }
    const bool bad = __syncthreads_or(wrong) || r.s != r.s;
    const float zm = block_max(id >= 0 ? t : -INFINITY, tmp);
    const float g = id >= 0 ? expf((t - zm) / tau) : 0.f;
    const float gs = block_sum(g, tmp);
    const bool lost = none || zm == -INFINITY;
    float q = 0.f, part = 0.f;
    if (!lost && id >= 0) {
      q = g / gs;
      // tau (ln q - ln p)
      const float far = (t - zm) - (xk - r.m) + tau * (ln_sum(r) - logf(gs));
      part = q > 0.f ? q * far : 0.f;
    }
    if (tid < top) {
      sid[tid] = id;
      sq[tid] = q;
    }
    part = block_sum(part, tmp);          // (and sid, sq are there)
    if (tid == 0 && loss)
      loss[row] = bad ? NAN : lost ? 0.f : tau * part;
    if (labels) {
      const int l = labels[row];
      int first = 0x7fffffff;
      for (int j = tid; j < cols; j += TP_THREADS)
        if ((float)x[j] == r.m) {
          first = j;
          break;
        }
#pragma unroll
      for (int off = 32; off; off >>= 1)
        first = min(first, __shfl_xor(first, off));
      if ((tid & (WAVE - 1)) == 0) ((int*)tmp)[tid / WAVE] = first;
      __syncthreads();
      if (tid == 0 && l >= 0) {
        for (int i = 1; i < TP_THREADS / WAVE; ++i)
          first = min(first, ((int*)tmp)[i]);
        if (bad || none || first != l) atomicAdd(n_err, 1);
      }
    }
    // err may lie over x: what is read of x is read before
    float mine = 0.f, sum = 0.f;
    if (id >= 0) {
      mine = r.far ? pow2(exponent<true>(xk, c, r))
                   : pow2(exponent<false>(xk, c, r));
      for (int k = 0; k < top; ++k)
        if (sid[k] == id) sum += sq[k];
    }
    __syncthreads();
    const float a = bad ? NAN : lost ? 0.f : tau / r.s;
    for (int j = tid; j < cols; j += TP_THREADS) {
      const float v = (float)x[j];
      const float e = r.far ? pow2(exponent<true>(v, c, r))
                            : pow2(exponent<false>(v, c, r));
      err[j] = from_f<O>(lost && !bad ? 0.f : a * e);
    }
    __syncthreads();
    if (id >= 0 && !bad && !lost)
      err[id] = from_f<O>(fmaf(a, mine, -tau * sum));
    __syncthreads();
  }
}

static unsigned row_grid(long rows) {
  return (unsigned)(rows < 65536 ? rows : 65536);
}

void token_logprobs_launch(int type, RowsIn x, const int* labels,
                           float* logprob, float* entropy, int* top_idx,
                           float* top_lp, int top, long rows, long live,
                           int cols, hipStream_t s) {
  if (rows == 0) return;
#define RUN(T)                                                               \
  hipLaunchKernelGGL(HIP_KERNEL_NAME(logprobs_k<T>), dim3(row_grid(rows)),   \
                     dim3(TP_THREADS), 0, s, x, labels, logprob, entropy,    \
                     top_idx, top_lp, top, rows, live, cols)
  ROW_TYPE_SWITCH(type, RUN)
#undef RUN
  HIP_CHECK_LAST();
}

void eval_distill_launch(int type, int err_type, RowsIn x, const int* idx, const float* z,
                         RowsOut err, float* loss, const int* labels,
                         int* n_err, int top, long rows, long live, int cols,
                         float tau, hipStream_t s) {
  if (rows == 0) return;
#define RUN2(T, O)                                                           \
  hipLaunchKernelGGL(HIP_KERNEL_NAME(distill_k<T, O>), dim3(row_grid(rows)), \
                     dim3(TP_THREADS), 0, s, x, idx, z, err, loss, labels,   \
                     n_err, top, rows, live, cols, tau)
#define RUN(T) RUN2(T, T)
  if (type == ROW_F32 && err_type == ROW_BF16) {
    RUN2(float, bf16_t);
  } else {
    ROW_TYPE_SWITCH(type, RUN)
  }
#undef RUN
#undef RUN2
  HIP_CHECK_LAST();
}
