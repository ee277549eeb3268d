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

#define LOG2E 1.44269504088896340736f
#define LN2 0.69314718055994530942f
// u is cut here where it is multiplied by its power, which is 0 by then
#define U_MIN -200.f
// a thread's M is no lower, so that it stands for a thread without classes
// too: 2^(M - M') of it and of any that counts is 0, and d is below 16
#define M_MIN -0x1p28f
// from here on u = (x - m) C (d is below 1/16 up to it)
#define M_FAR 0x1p20f

// (v_exp_f32, v_log_f32: one unit in the last place; powers below 2^-126
// are 0, and the sums of a row are 1/2 at least)
__device__ __forceinline__ float pow2(float u) {
  return __builtin_amdgcn_exp2f(u);
}
__device__ __forceinline__ float log2_of(float s) {
  return __builtin_amdgcn_logf(s);
}

// ---------------------------------------------------------------------------
// order of classes
// ---------------------------------------------------------------------------

// an order of the values in whole numbers; the two zeros are one
__device__ __forceinline__ int order_of(float x) {
  const int i = __float_as_int(x + 0.f);
  return i < 0 ? i ^ 0x7fffffff : i;
}
__device__ __forceinline__ float value_of(int i) {
  return __int_as_float(i < 0 ? i ^ 0x7fffffff : i);
}
#define ORDER_NONE ((int)0x807fffff)    // of minus infinity

// Value and class in one number: a larger value is first, of equal values
// the lower class.  0 is below every class.
typedef unsigned long long rank_t;
__device__ __forceinline__ rank_t rank_of(float x, int j) {
  return ((rank_t)((unsigned)order_of(x) ^ 0x80000000u) << 32) |
         (unsigned)(0x7fffffff - j);
}
__device__ __forceinline__ float rank_value(rank_t k) {
  return value_of((int)((unsigned)(k >> 32) ^ 0x80000000u));
}
// (of key 0: below that of every value)
__device__ __forceinline__ int rank_order(rank_t k) {
  return (int)((unsigned)(k >> 32) ^ 0x80000000u);
}
__device__ __forceinline__ int rank_class(rank_t k) {
  return 0x7fffffff - (int)(unsigned)k;
}

// how many of the list are before one
__device__ __forceinline__ int ranks_before(const rank_t* list, int n,
                                            rank_t key) {
  int before = 0;
#pragma unroll 8
  for (int j = 0; j < n; ++j) before += list[j] > key;
  return before;
}

// ---------------------------------------------------------------------------
// sums over a row
// ---------------------------------------------------------------------------

// largest logit and the sums relative to it
struct Sums {
  float m;      // -inf: no class is allowed
  float um;     // M
  float s;      // sum 2^u; NaN: the row has a NaN or plus infinity
  float w;      // sum 2^u u (entropy alone)

  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    um = M_MIN;
    s = w = 0.f;
  }
  // the same sums to a larger m
  __device__ __forceinline__ void raise(float to, float c) {
    const float um2 = fmaxf(to * c, M_MIN);
    const float by = um - um2, f = pow2(by);
    w = f * fmaf(by, s, w);
    s *= f;
    m = to;
    um = um2;
  }
  __device__ __forceinline__ void add(float x, float c) {
    const float u = fmaf(x, c, -um);
    const float e = pow2(u);
    s += e;
    w = fmaf(e, fmaxf(u, U_MIN), w);
  }
};

// what a row's outputs are made of
struct Row {
  float m, c;
  float um;      // of u = C x - um, unless `far`
  bool far;
  bool none;     // no class is allowed
  bool bad;      // NaN or plus infinity
  float s;       // sum 2^u
  float ln;      // ln of the sum of exp((x - m) / tau)
  float entropy;

  __device__ __forceinline__ float u(float x) const {
    return far ? (x - m) * c : fmaf(x, c, -um);
  }
  __device__ __forceinline__ void finish(const Sums& a, float c_) {
    m = a.m;
    c = c_;
    um = a.um;
    s = a.s;
    far = !(fabsf(m * c) < M_FAR) && m != -INFINITY;
    bad = s != s;
    none = !bad && m == -INFINITY;
    const float d = far ? 0.f : fmaf(m, c, -um);
    ln = (log2_of(s) - d) * LN2;
    entropy = none ? 0.f : (log2_of(s) - a.w / s) * LN2;
  }
};

__device__ __forceinline__ bool is_far(float m, float c) {
  return !(fabsf(m * c) < M_FAR) && m != -INFINITY;
}

// the waves' sums joined, in every thread; `tmp`: one for each wave
template <int THREADS>
__device__ __forceinline__ Sums join_block(Sums a, float c, Sums* tmp) {
  constexpr int WAVES = THREADS / WAVE;
  a.raise(wave_max(a.m), c);
  a.s = wave_sum(a.s);
  a.w = wave_sum(a.w);
  if (WAVES == 1) return a;
  if ((threadIdx.x & (WAVE - 1)) == 0) tmp[threadIdx.x / WAVE] = a;
  __syncthreads();
  float m = tmp[0].m;
#pragma unroll
  for (int i = 1; i < WAVES; ++i) m = fmaxf(m, tmp[i].m);
  Sums t;
  t.clear();
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    Sums b = tmp[i];
    b.raise(m, c);
    t.m = b.m;
    t.um = b.um;
    t.s += b.s;
    t.w += b.w;
  }
  return t;
}

// Sums of a part of a row, to the exact C m: parts are joined by
// 2^((m - m') C)
struct Part {
  float m, s, w;
  int first;     // lowest class with the value m
};

__device__ __forceinline__ Part part_of(const Sums& a, float c, int first) {
  const float d = is_far(a.m, c) || a.m == -INFINITY
                      ? 0.f : fmaf(a.m, c, -a.um);
  const float f = pow2(-d);
  return Part{a.m, f * a.s, f * fmaf(-d, a.s, a.w), first};
}

// Up to 64 parts of a row joined, by every wave for itself: lane i has the
// i-th.
__device__ __forceinline__ Row join_parts(const Part* p, int n, float c,
                                          int* first) {
  const int lane = threadIdx.x & (WAVE - 1);
  Part a{-INFINITY, 0.f, 0.f, 0x7fffffff};
  if (lane < n) a = p[lane];
  const float m = wave_max(a.m);
  // (an empty part beside an empty row: no difference of infinities)
  const float by = a.m == m ? 0.f : fmaxf((a.m - m) * c, M_MIN);
  const float f = pow2(by);
  Sums t;
  t.m = m;
  t.um = fmaxf(m * c, M_MIN);
  t.s = wave_sum(f * a.s);
  t.w = wave_sum(f * fmaf(by, a.s, a.w));
  *first = wave_min(a.m == m ? a.first : 0x7fffffff);
  Row r;
  r.finish(t, c);
  r.ln = log2_of(t.s) * LN2;             // (the parts are to the exact C m)
  return r;
}

// ---------------------------------------------------------------------------
// a row, or a part of it, in the registers of a workgroup
// ---------------------------------------------------------------------------

// A row's elements: up to N - 1 before the first multiple of 16 bytes (loads
// off such a multiple are slower: 4096 x 50001 bf16 in 95 us, x 50000 in 79),
// whole packs, and up to N - 1 behind them.  The single ones are one each for
// the first 2 N threads.
template <typename T>
struct Cut {
  static constexpr int N = Pack<T>::N;
  int head, packs, single;     // single: this thread's, or -1

  __device__ __forceinline__ Cut(const T* x, int n) {
    head = (int)((16 - ((unsigned long long)x & 15)) & 15) / (int)sizeof(T);
    head = min(head, n);
    packs = (n - head) / N;
    const int tail = head + packs * N, t = threadIdx.x;
    single = t < head ? t : t >= N && tail + t - N < n ? tail + t - N : -1;
  }
  __device__ __forceinline__ float load_single(const T* x) const {
    return single >= 0 ? (float)x[single] : -INFINITY;
  }
};

// Thread t holds packs t, t + THREADS, ... and one of the single elements.
// Places without an element hold minus infinity.
template <typename T, int THREADS, int NV>
struct Held {
  static constexpr int N = Pack<T>::N;
  Pack<T> v[NV];
  float rest;

  __device__ __forceinline__ void load(const T* x, const Cut<T>& cut) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      v[i].fill(-INFINITY);
      // (one offset for all, from bases that are the same for a wave)
      if (i * THREADS + (int)threadIdx.x < cut.packs)
        v[i].load_once(x + cut.head + i * THREADS * N + threadIdx.x * N);
    }
    rest = cut.load_single(x);
  }
};

// Packs are summed CHUNK at a time, relative to the thread's largest so far:
// what follows a load of 16 bytes is done while the next ones are under way,
// and no element is read twice.
#define CHUNK 2

template <typename T, int COUNT>
__device__ __forceinline__ void add_packs(const Pack<T>* v, Sums& a, float c,
                                          float* high) {
  constexpr int N = Pack<T>::N;
  float m;
#pragma unroll
  for (int i = 0; i < COUNT; ++i) {
    float e[N];
    v[i].get(e);
    float h = max3(e[0], e[1], e[2]);
#pragma unroll
    for (int j = 3; j + 1 < N; j += 2) h = max3(h, e[j], e[j + 1]);
    h = max3(h, e[N - 1], h);
    if (high) high[i] = h;
    m = i ? max3(m, h, m) : h;
  }
  a.raise(fmaxf(a.m, m), c);
#pragma unroll
  for (int i = 0; i < COUNT; ++i) {
    float e[N];
    v[i].get(e);
#pragma unroll
    for (int j = 0; j < N; ++j) a.add(e[j], c);
  }
}

template <typename T, int THREADS, int NV>
__device__ __forceinline__ Sums held_sums(const Held<T, THREADS, NV>& h,
                                          int packs, float c, float* high) {
  constexpr int STEP = NV < CHUNK ? NV : CHUNK;
  Sums a;
  a.clear();
#pragma unroll
  for (int i = 0; i < NV; i += STEP) {
    if (i * THREADS >= packs) break;
    add_packs<T, STEP>(h.v + i, a, c, high ? high + i : nullptr);
  }
  a.raise(fmaxf(a.m, h.rest), c);
  a.add(h.rest, c);
  return a;
}

// ---------------------------------------------------------------------------
// token_logprobs
// ---------------------------------------------------------------------------

#define LP_THREADS 256
// classes that may be looked at more closely; more of them (many equal
// values) are thinned out first
#define LP_CAND 512

struct LogprobsOut {
  const int* labels;
  float* logprob;
  float* entropy;
  int* idx;
  float* lp;
  int top;
};

__device__ __forceinline__ void logprobs_padding(const LogprobsOut& o,
                                                 long row) {
  if (threadIdx.x == 0) {
    if (o.logprob) o.logprob[row] = 0.f;
    if (o.entropy) o.entropy[row] = 0.f;
  }
  for (int k = threadIdx.x; k < o.top; k += blockDim.x) {
    o.idx[row * o.top + k] = -1;
    o.lp[row * o.top + k] = 0.f;
  }
}

// Logit of the class that is asked for: -inf if there is none, NaN for one
// that does not exist; in thread 0.  (Read before the row is, as two loads
// that wait for each other.)
template <typename T>
__device__ __forceinline__ float given_logit(const LogprobsOut& o, long row,
                                             const T* x, int cols) {
  if (threadIdx.x || !o.logprob) return 0.f;
  const int l = o.labels[row];
  return l >= cols ? NAN : l >= 0 ? (float)x[l] : -INFINITY;
}

__device__ __forceinline__ void logprobs_row(const LogprobsOut& o, long row,
                                             float given, const Row& r) {
  if (threadIdx.x) return;
  if (o.entropy) o.entropy[row] = r.entropy;
  if (o.logprob) {
    const bool named = o.labels[row] >= 0;
    const float v = given == -INFINITY ? given : (given - r.m) - r.ln;
    o.logprob[row] = !named ? 0.f : r.bad ? NAN : v;
  }
}

// the alternative of rank k; key 0: there is none
__device__ __forceinline__ void logprobs_top(const LogprobsOut& o, long row,
                                             int k, rank_t key,
                                             const Row& r) {
  o.idx[row * o.top + k] = key ? rank_class(key) : -1;
  o.lp[row * o.top + k] =
      r.bad ? NAN : key ? (rank_value(key) - r.m) - r.ln : -INFINITY;
}

template <int THREADS>
__device__ __forceinline__ int block_count(int n, int* tmp) {
  constexpr int WAVES = THREADS / WAVE;
  n = wave_sum(n);
  __syncthreads();
  if ((threadIdx.x & (WAVE - 1)) == 0) tmp[threadIdx.x / WAVE] = n;
  __syncthreads();
  n = 0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) n += tmp[i];
  return n;
}

// Among the threads' largest values, in `high`, one that at least `top` of
// them reach, and not many more; by one wave.  All classes that reach it are
// few, and the first `top` are among them.  Fewer than `top` threads with a
// class: the lowest of all.
template <int THREADS>
__device__ __forceinline__ int find_bound(const int* high, int top) {
  constexpr int PER = THREADS / WAVE;
  int v[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) v[i] = high[threadIdx.x + i * WAVE];
  int hi = v[0];
#pragma unroll
  for (int i = 1; i < PER; ++i) hi = max(hi, v[i]);
  hi = wave_max(hi);
  int lo = ORDER_NONE + 1;
  auto reach = [&](int b) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) n += __popcll(__ballot(v[i] >= b));
    return n;
  };
  if (reach(lo) < top) return lo;
  // reach(lo) >= top > reach(hi + 1)
  while (lo < hi) {
    const int mid = lo + (int)(((unsigned)hi - (unsigned)lo + 1u) / 2u);
    const int n = reach(mid);
    if (n >= top) {
      lo = mid;
      if (n <= top + top / 4) break;
    } else {
      hi = mid - 1;
    }
  }
  return lo;
}

template <int THREADS>
struct TopSpace {
  int high[THREADS];
  rank_t cand[LP_CAND];
  int n, bound, groups;
  int list[LP_CAND];
  int tmp[THREADS / WAVE];

  __device__ __forceinline__ void put(float x, float from, int j) {
    if (x >= from) {
      const int at = atomicAdd(&n, 1);
      if (at < LP_CAND) cand[at] = rank_of(x, j);
    }
  }
};

// The bound for all threads, from their largest values in sp.high
template <int THREADS>
__device__ __forceinline__ float share_bound(TopSpace<THREADS>& sp, int top) {
  if (threadIdx.x < WAVE) {
    const int b = find_bound<THREADS>(sp.high, top);
    if (threadIdx.x == 0) {
      sp.bound = b;
      sp.n = sp.groups = 0;
    }
  }
  __syncthreads();
  return value_of(sp.bound);
}

// Too many classes reach the bound (one value many times): the top-th value
// itself, then among the classes that hold it the last that is needed, by
// halving; the part x[0..n) is read from the caches each time.
template <typename T, int THREADS>
__device__ __noinline__ void thin_out(const T* x, int n, int base, int top,
                                      TopSpace<THREADS>& sp) {
  const int tid = threadIdx.x;
  int lo = sp.bound, hi = 0x7f800000;
  while (lo < hi) {
    const int mid = lo + (int)(((unsigned)hi - (unsigned)lo + 1u) / 2u);
    int c = 0;
    for (int j = tid; j < n; j += THREADS) c += order_of(x[j]) >= mid;
    if (block_count<THREADS>(c, sp.tmp) >= top)
      lo = mid;
    else
      hi = mid - 1;
  }
  int c = 0;
  for (int j = tid; j < n; j += THREADS) c += order_of(x[j]) > lo;
  const int need = top - block_count<THREADS>(c, sp.tmp);
  int a = 0, b = n - 1;
  while (a < b) {
    const int mid = a + (b - a) / 2;
    c = 0;
    for (int j = tid; j <= mid; j += THREADS) c += order_of(x[j]) == lo;
    if (block_count<THREADS>(c, sp.tmp) >= need)
      b = mid;
    else
      a = mid + 1;
  }
  if (tid == 0) sp.n = 0;
  __syncthreads();
  for (int j = tid; j < n; j += THREADS) {
    const int o = order_of(x[j]);
    if (o > lo || (o == lo && j <= a))
      sp.cand[atomicAdd(&sp.n, 1)] = rank_of(x[j], base + j);
  }
  __syncthreads();
}

// what a workgroup's part of a row gives
struct PartOut {
  LogprobsOut o;
  Part* parts;       // null: the part is the whole row
  rank_t* keys;

  __device__ __forceinline__ void put(long row, long item, int k, rank_t key,
                                      const Row& r) const {
    if (parts)
      keys[item * o.top + k] = key;
    else
      logprobs_top(o, row, k, key, r);
  }
};

// The `found` classes in sp.cand in their order: the place of each is the
// number of those before it.
template <int THREADS>
__device__ __forceinline__ void put_top(const PartOut& p, long row, long item,
                                        int found, const Row& r,
                                        const TopSpace<THREADS>& sp) {
  for (int i = threadIdx.x; i < found; i += THREADS) {
    const rank_t mine = sp.cand[i];
    const int before = ranks_before(sp.cand, found, mine);
    if (before < p.o.top) p.put(row, item, before, mine, r);
  }
  for (int k = found + threadIdx.x; k < p.o.top; k += THREADS)
    p.put(row, item, k, 0, r);
}

// Where u = C x - M does not do: the sums of the part x[0..n) once more
template <typename T>
__device__ __noinline__ Sums far_sums(const T* x, int n, float m, float c,
                                      float* tmp) {
  Sums a;
  a.m = m;
  a.um = 0.f;
  a.s = a.w = 0.f;
  for (int j = threadIdx.x; j < n; j += blockDim.x) {
    const float u = ((float)x[j] - m) * c, e = pow2(u);
    a.s += e;
    a.w = fmaf(e, fmaxf(u, U_MIN), a.w);
  }
  __syncthreads();
  a.s = block_sum(a.s, tmp);
  a.w = block_sum(a.w, tmp);
  return a;
}

// row, part and element range of this workgroup in a grid of parts x rows,
// the rows in two dimensions
struct Place {
  long row, item;
  int base, n;

  __device__ __forceinline__ Place(int cols, int size) {
    row = (long)blockIdx.z * gridDim.y + blockIdx.y;
    item = row * gridDim.x + blockIdx.x;
    base = blockIdx.x * size;
    n = min(size, cols - base);
  }
};

// One workgroup to a part of a row, which it holds in registers
template <typename T, int NV>
__global__ __launch_bounds__(LP_THREADS) void logprobs_held_k(
    RowsIn x_, PartOut p, long rows, long live, int cols, int size) {
  __shared__ TopSpace<LP_THREADS> sp;
  __shared__ Sums tmp[LP_THREADS / WAVE];
  constexpr int N = Pack<T>::N;
  const int tid = threadIdx.x;
  const Place at(cols, size);
  if (at.row >= rows) return;
  if (at.row >= live) {
    logprobs_padding(p.o, at.row);
    return;
  }
  const T* row = (const T*)x_.p + at.row * x_.stride;
  const T* x = row + at.base;
  const float given = p.parts ? 0.f : given_logit(p.o, at.row, row, cols);
  const Cut<T> cut(x, at.n);
  Held<T, LP_THREADS, NV> h;
  h.load(x, cut);
  float high[NV];
  Sums a = held_sums(h, cut.packs, LOG2E, high);
  sp.high[tid] = order_of(a.m);
  a = join_block<LP_THREADS>(a, LOG2E, tmp);
  if (is_far(a.m, LOG2E)) a = far_sums(x, at.n, a.m, LOG2E, (float*)tmp);
  Row r;
  r.finish(a, LOG2E);
  if (!p.parts)
    logprobs_row(p.o, at.row, given, r);
  else if (tid == 0)
    p.parts[at.item] = part_of(a, LOG2E, 0);
  if (!p.o.top) return;
  int found = 0;
  if (!r.bad && !r.none) {
    const float bound = share_bound(sp, p.o.top);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (i * LP_THREADS >= cut.packs) break;
      if (high[i] >= bound) {
        float e[N];
        h.v[i].forget();
        h.v[i].get(e);
        const int j0 = at.base + cut.head + (i * LP_THREADS + tid) * N;
#pragma unroll
        for (int j = 0; j < N; ++j) sp.put(e[j], bound, j0 + j);
      }
    }
    sp.put(h.rest, bound, at.base + cut.single);
    __syncthreads();
    if (sp.n > LP_CAND)
      thin_out<T, LP_THREADS>(x, at.n, at.base, p.o.top, sp);
    found = sp.n;
  }
  put_top(p, at.row, at.item, found, r, sp);
}

// largest value of the eight lanes' own, for four values; in all lanes
__device__ __forceinline__ void max_of_eight_lanes(float* h) {
  // (two wait states between a write and its use by another lane)
  asm volatile("s_nop 1\n\t"
      "v_max_f32_dpp %0, %0, %0 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n\t"
      "v_max_f32_dpp %1, %1, %1 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n\t"
      "v_max_f32_dpp %2, %2, %2 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n\t"
      "v_max_f32_dpp %3, %3, %3 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n\t"
      "v_max_f32_dpp %0, %0, %0 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n\t"
      "v_max_f32_dpp %1, %1, %1 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n\t"
      "v_max_f32_dpp %2, %2, %2 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n\t"
      "v_max_f32_dpp %3, %3, %3 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n\t"
      "v_max_f32_dpp %0, %0, %0 row_half_mirror row_mask:0xf bank_mask:0xf\n\t"
      "v_max_f32_dpp %1, %1, %1 row_half_mirror row_mask:0xf bank_mask:0xf\n\t"
      "v_max_f32_dpp %2, %2, %2 row_half_mirror row_mask:0xf bank_mask:0xf\n\t"
      "v_max_f32_dpp %3, %3, %3 row_half_mirror row_mask:0xf bank_mask:0xf"
      : "+v"(h[0]), "+v"(h[1]), "+v"(h[2]), "+v"(h[3]));
}

// One workgroup to a part of a row that streams past it, four packs of a
// thread at a time.  The largest value of each eight packs (128 bytes) stays
// in LDS; for the alternatives those are read again that reach the bound.
#define GROUP 8
template <typename T, bool TOP>
__global__ __launch_bounds__(LP_THREADS) void logprobs_stream_k(
    RowsIn x_, PartOut p, long rows, long live, int cols, int size) {
  __shared__ TopSpace<LP_THREADS> sp;
  __shared__ Sums tmp[LP_THREADS / WAVE];
  extern __shared__ float groups[];
  constexpr int N = Pack<T>::N;
  constexpr int U = 4, STEP = U * LP_THREADS;
  const int tid = threadIdx.x;
  const Place at(cols, size);
  if (at.row >= rows) return;
  if (at.row >= live) {
    logprobs_padding(p.o, at.row);
    return;
  }
  const T* row = (const T*)x_.p + at.row * x_.stride;
  const T* x = row + at.base;
  const float given = p.parts ? 0.f : given_logit(p.o, at.row, row, cols);
  const Cut<T> cut(x, at.n);
  const int packs = cut.packs;
  const float rest = cut.load_single(x);
  const T* body = x + cut.head;
  Sums a;
  a.clear();
  a.raise(rest, LOG2E);
  a.add(rest, LOG2E);
  for (int b = 0; b < packs; b += STEP) {
    Pack<T> v[U];
    if (b + STEP <= packs) {
#pragma unroll
      for (int i = 0; i < U; ++i)
        v[i].load_once(body + (long)(b + i * LP_THREADS) * N + tid * N);
    } else {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        v[i].fill(-INFINITY);
        if (b + i * LP_THREADS + tid < packs)
          v[i].load_once(body + (long)(b + i * LP_THREADS) * N + tid * N);
      }
    }
    float high[U];
    add_packs<T, U>(v, a, LOG2E, high);
    if (TOP) {
      max_of_eight_lanes(high);
      // lane i of each eight has that of pack row i
      const int i = tid % GROUP;
      const float h = i == 0 ? high[0] : i == 1 ? high[1]
                    : i == 2 ? high[2] : high[3];
      const int g = (b + i * LP_THREADS + tid) / GROUP;
      if (i < U && g * GROUP < packs) groups[g] = h;
    }
  }
  a = join_block<LP_THREADS>(a, LOG2E, tmp);
  if (is_far(a.m, LOG2E)) a = far_sums(x, at.n, a.m, LOG2E, (float*)tmp);
  Row r;
  r.finish(a, LOG2E);
  if (!p.parts)
    logprobs_row(p.o, at.row, given, r);
  else if (tid == 0)
    p.parts[at.item] = part_of(a, LOG2E, 0);
  if (!TOP) return;
  int found = 0;
  if (!r.bad && !r.none) {
    const int n = (packs + GROUP - 1) / GROUP;
    float h = rest;
    for (int g = tid; g < n; g += LP_THREADS) h = fmaxf(h, groups[g]);
    sp.high[tid] = order_of(h);
    __syncthreads();
    const float bound = share_bound(sp, p.o.top);
    if (h >= bound)
      for (int g = tid; g < n; g += LP_THREADS)
        if (groups[g] >= bound) {
          const int k = atomicAdd(&sp.groups, 1);
          if (k < LP_CAND) sp.list[k] = g;
        }
    sp.put(rest, bound, at.base + cut.single);
    __syncthreads();
    const int m = min(sp.groups, LP_CAND);
    for (int k = tid / GROUP; k < m; k += LP_THREADS / GROUP) {
      const int q = sp.list[k] * GROUP + tid % GROUP;
      if (q < packs) {
        Pack<T> v;
        float e[N];
        v.load(body + (long)q * N);
        v.get(e);
#pragma unroll
        for (int j = 0; j < N; ++j)
          sp.put(e[j], bound, at.base + cut.head + q * N + j);
      }
    }
    __syncthreads();
    if (sp.n > LP_CAND || sp.groups > LP_CAND)
      thin_out<T, LP_THREADS>(x, at.n, at.base, p.o.top, sp);
    found = sp.n;
  }
  put_top(p, at.row, at.item, found, r, sp);
}

// A row's parts joined.  Each part's list is in order, so that the first few
// of all lists, one to a thread, have a bound as the threads' largest values
// have within a part.
template <typename T>
__global__ __launch_bounds__(LP_THREADS) void logprobs_join_k(
    RowsIn x_, LogprobsOut o, const Part* __restrict__ parts,
    const rank_t* __restrict__ keys, long rows, long live, int cols,
    int split) {
  extern __shared__ rank_t list[];
  __shared__ int high[LP_THREADS];
  __shared__ int count, bound;
  const int tid = threadIdx.x;
  for (long row = blockIdx.x; row < rows; row += gridDim.x) {
    if (row >= live) {
      logprobs_padding(o, row);
      continue;
    }
    const T* x = (const T*)x_.p + row * x_.stride;
    const int all = split * o.top;
    const rank_t* mine = keys + row * all;
    const int place = tid / split;
    rank_t k = 0;
    if (place < o.top && place < LP_THREADS / split)
      k = mine[tid % split * o.top + place];
    const float given = given_logit(o, row, x, cols);
    int first;
    const Row r = join_parts(parts + row * split, split, LOG2E, &first);
    logprobs_row(o, row, given, r);
    if (!o.top) continue;
    high[tid] = rank_order(k);
    __syncthreads();
    if (tid < WAVE) {
      const int b = find_bound<LP_THREADS>(high, o.top);
      if (tid == 0) {
        bound = b;
        count = 0;
      }
    }
    __syncthreads();
    if (!r.bad && !r.none)
      for (int i = tid; i < all; i += LP_THREADS) {
        const rank_t k = mine[i];
        if (rank_order(k) >= bound) list[atomicAdd(&count, 1)] = k;
      }
    __syncthreads();
    const int found = count;
    for (int i = tid; i < found; i += LP_THREADS) {
      const int before = ranks_before(list, found, list[i]);
      if (before < o.top) logprobs_top(o, row, before, list[i], r);
    }
    for (int k = found + tid; k < o.top; k += LP_THREADS)
      logprobs_top(o, row, k, 0, r);
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// eval_distill
// ---------------------------------------------------------------------------

#define TP_THREADS 256

__device__ __forceinline__ Row plain_row(const Sums& a, float c) {
  Row r;
  r.finish(a, c);
  return r;
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
    float m = -INFINITY;
    for (int j = tid; j < cols; j += TP_THREADS) m = fmaxf(m, (float)x[j]);
    m = block_max(m, tmp);
    Sums sums;
    sums.clear();
    sums.m = m;
    sums.um = fmaxf(m * c, M_MIN);
    const bool far = is_far(m, c);
    for (int j = tid; j < cols; j += TP_THREADS) {
      const float v = (float)x[j];
      sums.s += pow2(far ? (v - m) * c : fmaf(v, c, -sums.um));
    }
    sums.s = block_sum(sums.s, tmp);
    const Row r = plain_row(sums, c);
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
    const bool bad = __syncthreads_or(wrong) || r.bad;
    const float zm = block_max(id >= 0 ? t : -INFINITY, tmp);
    const float g = id >= 0 ? expf((t - zm) / tau) : 0.f;
    const float gs = block_sum(g, tmp);
    const bool lost = r.none || zm == -INFINITY;
    float q = 0.f, part = 0.f;
    if (!lost && id >= 0) {
      q = g / gs;
      // tau (ln q - ln p)
      const float apart = (t - zm) - (xk - r.m) + tau * (r.ln - logf(gs));
      part = q > 0.f ? q * apart : 0.f;
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
        if (bad || r.none || first != l) atomicAdd(n_err, 1);
      }
    }
    // err may lie over x: what is read of x is read before
    float mine = 0.f, sum = 0.f;
    if (id >= 0) {
      mine = pow2(r.u(xk));
      for (int k = 0; k < top; ++k)
        if (sid[k] == id) sum += sq[k];
    }
    __syncthreads();
    const float a = bad ? NAN : lost ? 0.f : tau / r.s;
    for (int j = tid; j < cols; j += TP_THREADS) {
      const float e = pow2(r.u((float)x[j]));
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

static dim3 parts_grid(int split, long rows) {
  const long y = rows < 32768 ? rows : 32768;
  return dim3((unsigned)split, (unsigned)y, (unsigned)((rows + y - 1) / y));
}

// parts of a row that are joined at most, and groups that a part may have
#define LP_PARTS 64
#define LP_GROUPS 16384
// Few rows are cut until there are two workgroups for each compute unit, but
// into parts of 4 packs a thread at least.  One row of 131072 bf16: 11.0 us
// with 4 packs, 11.0 with 2; 600 rows: 38 us with two workgroups, 41 with
// four, 39 with eight (the parts' own ends and their joining weigh more).
#define LP_LEAST 4
#define LP_BLOCKS 512

// How a call is laid out: parts of a row, elements of a part, and packs of
// a thread where they are held (0: they stream past)
struct LogprobsPlan {
  int split, size, nv;
};

static LogprobsPlan logprobs_plan(int type, long rows, int cols) {
  const int n = type == ROW_F32 ? 4 : 8;
  const long held = LP_THREADS * 16 * n;
  const long most = (long)LP_GROUPS * GROUP * n;
  long split = (cols + most - 1) / most;
  const long least = LP_THREADS * LP_LEAST * n;
  while (split < LP_PARTS && rows * split < LP_BLOCKS &&
         cols / (split + 1) >= least)
    ++split;
  // whole packs to a part
  long size = (cols + split - 1) / split;
  size = (size + n - 1) / n * n;
  LogprobsPlan p;
  p.size = (int)size;
  p.split = (int)((cols + size - 1) / size);
  p.nv = 0;
  if (size <= held) {
    p.nv = 1;
    while ((long)LP_THREADS * p.nv * n < size) p.nv *= 2;
  }
  return p;
}

// bytes that token_logprobs_launch needs at `scratch`
long token_logprobs_scratch(int type, long live, int cols, int top) {
  const LogprobsPlan p = logprobs_plan(type, live, cols);
  if (p.split == 1) return 0;
  return live * p.split * ((long)sizeof(Part) + top * (long)sizeof(rank_t));
}

template <typename T>
static void logprobs_run(RowsIn x, LogprobsOut o, LogprobsPlan l, long rows,
                         long live, int cols, void* scratch, hipStream_t s) {
  const bool joined = l.split > 1;
  PartOut p{o, nullptr, nullptr};
  if (joined) {
    p.keys = (rank_t*)scratch;
    p.parts = (Part*)(p.keys + live * l.split * (long)o.top);
  }
  const long some = joined ? live : rows;
#define HELD(NV)                                                             \
  case NV:                                                                   \
    hipLaunchKernelGGL(HIP_KERNEL_NAME(logprobs_held_k<T, NV>),              \
                       parts_grid(l.split, some), dim3(LP_THREADS), 0, s, x, \
                       p, some, live, cols, l.size);                         \
    break;
#define STREAM(TOP)                                                          \
  hipLaunchKernelGGL(                                                        \
      HIP_KERNEL_NAME(logprobs_stream_k<T, TOP>), parts_grid(l.split, some), \
      dim3(LP_THREADS),                                                      \
      TOP ? (l.size / Pack<T>::N + GROUP - 1) / GROUP * sizeof(float) : 0,   \
      s, x, p, some, live, cols, l.size)
  if (some) {
    switch (l.nv) {
      HELD(1) HELD(2) HELD(4) HELD(8) HELD(16)
      default:
        if (o.top)
          STREAM(true);
        else
          STREAM(false);
    }
    HIP_CHECK_LAST();
  }
#undef HELD
#undef STREAM
  if (!joined) return;
  hipLaunchKernelGGL(HIP_KERNEL_NAME(logprobs_join_k<T>),
                     dim3(row_grid(rows)), dim3(LP_THREADS),
                     sizeof(rank_t) * l.split * o.top, s, x, o, p.parts,
                     p.keys, rows, live, cols, l.split);
  HIP_CHECK_LAST();
}

void token_logprobs_launch(int type, RowsIn x, const int* labels,
                           float* logprob, float* entropy, int* top_idx,
                           float* top_lp, int top, long rows, long live,
                           int cols, void* scratch, hipStream_t s) {
  if (rows == 0) return;
  const LogprobsOut o{labels, logprob, entropy, top_idx, top_lp, top};
  const LogprobsPlan p = logprobs_plan(type, live, cols);
#define RUN(T) logprobs_run<T>(x, o, p, rows, live, cols, scratch, s)
  ROW_TYPE_SWITCH(type, RUN)
#undef RUN
}

void eval_distill_launch(int type, int err_type, RowsIn x, const int* idx,
                         const float* z, RowsOut err, float* loss,
                         const int* labels, int* n_err, int top, long rows,
                         long live, int cols, float tau, hipStream_t s) {
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
