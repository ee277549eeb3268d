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
  // the same sums to a larger m (W: that of the entropy too)
  template <bool W>
  __device__ __forceinline__ void raise(float to, float c) {
    const float um2 = fmaxf(to * c, M_MIN);
    const float by = um - um2, f = pow2(by);
    if (W) w = f * fmaf(by, s, w);
    s *= f;
    m = to;
    um = um2;
  }
  template <bool W>
  __device__ __forceinline__ void add(float x, float c) {
    const float u = fmaf(x, c, -um);
    const float e = pow2(u);
    s += e;
    if (W) w = fmaf(e, fmaxf(u, U_MIN), w);
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
template <bool W, int THREADS>
__device__ __forceinline__ Sums join_block(Sums a, float c, Sums* tmp) {
  constexpr int WAVES = THREADS / WAVE;
  a.raise<W>(wave_max(a.m), c);
  a.s = wave_sum(a.s);
  if (W) a.w = wave_sum(a.w);
  if (WAVES == 1) return a;
  if ((threadIdx.x & (WAVE - 1)) == 0) tmp[threadIdx.x / WAVE] = a;
  __syncthreads();
  // (every wave joins them for itself, a lane to each)
  const int lane = threadIdx.x & (WAVE - 1);
  a.clear();
  if (lane < WAVES) a = tmp[lane];
  a.raise<W>(wave_max(a.m), c);
  a.s = wave_sum(a.s);
  if (W) a.w = wave_sum(a.w);
  return a;
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
  // from the exact C m to M
  if (m != -INFINITY && !is_far(m, c)) {
    const float d = fmaf(m, c, -t.um), f = pow2(d);
    t.w = f * fmaf(d, t.s, t.w);
    t.s *= f;
  }
  Row r;
  r.finish(t, c);
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
    for (int i = 0; i < NV; ++i) load_pack(i, x, cut);
    rest = cut.load_single(x);
  }
  __device__ __forceinline__ void load_pack(int i, const T* x,
                                            const Cut<T>& cut) {
    v[i].fill(-INFINITY);
    // (one offset for all, from bases that are the same for a wave)
    if (i * THREADS + (int)threadIdx.x < cut.packs)
      v[i].load_once(x + cut.head + i * THREADS * N + threadIdx.x * N);
  }
};

// Packs are summed CHUNK at a time, relative to the thread's largest so far:
// what follows a load of 16 bytes is done while the next ones are under way,
// and no element is read twice.
#define CHUNK 2

template <bool W, typename T, int COUNT>
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
  a.raise<W>(fmaxf(a.m, m), c);
#pragma unroll
  for (int i = 0; i < COUNT; ++i) {
    float e[N];
    v[i].get(e);
#pragma unroll
    for (int j = 0; j < N; ++j) a.add<W>(e[j], c);
  }
}

template <bool W, typename T, int THREADS, int NV>
__device__ __forceinline__ Sums held_sums(const Held<T, THREADS, NV>& h,
                                          int packs, float c, float* high) {
  constexpr int STEP = NV < CHUNK ? NV : CHUNK;
  Sums a;
  a.clear();
#pragma unroll
  for (int i = 0; i < NV; i += STEP) {
    if (i * THREADS >= packs) break;
    add_packs<W, T, STEP>(h.v + i, a, c, high ? high + i : nullptr);
  }
  a.raise<W>(fmaxf(a.m, h.rest), c);
  a.add<W>(h.rest, c);
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

// Among a wave's values, PER of a lane, one that at least `top` of them reach,
// and not many more; fewer than `top` that belong to a class: the lowest.
// Three values in between are tried at a time, from the least that is reached
// on (one row of 131072 bf16, two such searches, in a graph: 8.7 us; one at a
// time from the lowest value on 10.4).
template <int PER>
__device__ __forceinline__ int narrow_down(const int* v, int lo, int hi,
                                           int top) {
  auto reach = [&](int b) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) n += __popcll(__ballot(v[i] >= b));
    return n;
  };
  if (lo <= ORDER_NONE) {
    lo = ORDER_NONE + 1;
    if (reach(lo) < top) return lo;
  }
  // reach(lo) >= top > reach(hi + 1)
  while (lo < hi) {
    const unsigned d = (unsigned)hi - (unsigned)lo, q = d / 4 + 1;
    int at[3], n[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      at[i] = (int)((unsigned)lo + min(q * (i + 1), d));
      n[i] = reach(at[i]);
    }
    int now = 0;
    if (n[2] >= top) {
      lo = at[2];
      now = n[2];
    } else if (n[1] >= top) {
      lo = at[1];
      hi = at[2] - 1;
      now = n[1];
    } else if (n[0] >= top) {
      lo = at[0];
      hi = at[1] - 1;
      now = n[0];
    } else {
      hi = at[0] - 1;
    }
    if (now && now <= top + top / 4) break;
  }
  return lo;
}

// Such a value for the threads' largest ones, in `high`; by one wave.  All
// classes that reach it are few, and the first `top` are among them.
template <int THREADS>
__device__ __forceinline__ int find_bound(const int* high, int top) {
  constexpr int PER = THREADS / WAVE;
  int v[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) v[i] = high[threadIdx.x + i * WAVE];
  int most = v[0], least = v[0];
#pragma unroll
  for (int i = 1; i < PER; ++i) {
    most = max(most, v[i]);
    least = min(least, v[i]);
  }
  // (as many as there are lanes reach the least of the lanes' largest)
  return narrow_down<PER>(v, wave_min(top <= WAVE ? most : least),
                          wave_max(most), top);
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
// halving; the part x[0..n) is read from the caches each time, up to 32 + log2
// n times with two barriers each.  Rows of one value, or with fewer classes than
// alternatives above a finite lowest value, all come here: 256 x 1000 fp32 24
// to 29 us in place of 4.5, 8192 x 8000 bf16 1.4 to 1.5 ms in place of 38 us,
// 2048 x 131072 8.7 to 9.2 ms in place of 97 us.
template <typename T, int THREADS>
__device__ __forceinline__ void thin_out(const T* x, int n, int base, int top,
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
__device__ __forceinline__ Sums far_sums(const T* x, int n, float m, float c,
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

// Rows so short that half the threads or more have no pack: in place of each
// thread's largest value that of each half, quarter, ... of a pack, as many as
// there are threads, of which the bound is less often too low.  4096 x 1000
// bf16 with 128 alternatives, for which 125 threads have too few values: 92 us
// without, 29 so; 4096 x 500 70 and 26.  Not where there are many threads to an
// alternative, or few classes in all (4096 x 1000, 20 of them: 13.9 us without,
// 14.3 so; 6 x 72: 5.4, 5.8).
template <typename T, int S = 2>
__device__ __forceinline__ bool put_pieces(
    const Held<T, LP_THREADS, 1>& h, int packs, int* high) {
  constexpr int N = Pack<T>::N, LANES = LP_THREADS / S;
  if (packs > LANES) return false;
  if constexpr (S < N)
    if (packs <= LANES / 2) return put_pieces<T, 2 * S>(h, packs, high);
  if (threadIdx.x < LANES) {
    float e[N];
    h.v[0].get(e);
#pragma unroll
    for (int g = 0; g < S; ++g) {
      float m = g ? -INFINITY : h.rest;
#pragma unroll
      for (int j = 0; j < N / S; ++j) m = fmaxf(m, e[g * (N / S) + j]);
      high[g * LANES + threadIdx.x] = order_of(m);
    }
  }
  return true;
}

// One workgroup to a part of a row, which it holds in registers, so that the
// alternatives are found without reading it again.  8192 x 8000 bf16, 20 of
// them: 38 us, 3.5 TB/s; 4096 x 8000 fp32 27 us, 4.8 TB/s.  Bound by the
// delays of its steps one after another (load, sums, bound, order), which the
// other workgroups of the compute unit cover as far as they fit; 256 x 1000
// fp32 takes 4.5 us, of which 2.3 are a launch.
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
  Sums a = held_sums<true>(h, cut.packs, LOG2E, high);
  bool pieces = false;
  if constexpr (NV == 1)
    if (at.n > 128 && cut.packs < 4 * p.o.top)
      pieces = put_pieces<T>(h, cut.packs, sp.high);
  if (!pieces) sp.high[tid] = order_of(a.m);
  a = join_block<true, LP_THREADS>(a, LOG2E, tmp);
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
// 4096 x 50001 bf16, 20 alternatives: 77 us, 5.2 TB/s; 2048 x 131072, 64 of
// them: 96 us, 5.6 TB/s, of 6.9 that bare loads reach.  Bound by memory, and
// for some 10 us by the alternatives, which the workgroups of a compute unit
// come to at about the same time.  Loads of the next four packs before the
// sums of these took 4% off a call without alternatives and nothing off one
// with them, for 20 registers more.
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
  a.raise<true>(rest, LOG2E);
  a.add<true>(rest, LOG2E);
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
    add_packs<true, T, U>(v, a, LOG2E, high);
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
  a = join_block<true, LP_THREADS>(a, LOG2E, tmp);
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
// have within a part.  One row of 131072 bf16 in 16 parts, with the parts: 8.7
// us in a graph, 5 alternatives; bound by two launches and the steps' delays.
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
// q = softmax(z / tau) over the teacher's classes (one that is named more than
// once has the sum of its shares), p = softmax(x / tau) over all;
//   loss = tau^2 sum q (ln q - ln p),  dloss/dx_j = tau (p_j - q_j).
// The row is read once: it stays in registers until its sum is known.  The
// teacher's classes are taken off the gradients in registers too, by the
// threads that hold them, so that each gradient is written once.

struct DistillArgs {
  RowsIn x;
  const int* idx;
  const float* z;
  RowsOut err;
  float* loss;
  const int* labels;
  int* n_err;
  int top;
  long rows, live;
  int cols, size;
  float tau, c;      // c = log2 e / tau
  Part* parts;       // of split rows
  float* xk;         // their logits of the teacher's classes
  bool past;         // gradients are stored past the caches
};

// Gradients of so many bytes are not in the caches any more when the next
// operator reads them.  Stored past them: 2048 x 30000 bf16 (123 MB) 54
// instead of 62 us, 2048 x 131072 220 instead of 224; but a kernel that reads
// 67 MB just written takes 10 us longer (134 MB: 11 us less).  For gradients of
// the logits' type; a bf16 gradient of fp32 logits is 8 bytes a lane and pack,
// and goes through the caches.
#define PAST_CACHES (96l << 20)

template <int THREADS>
struct DistillSpace {
  int id[MAX_TOP];           // -1: no class, or one that came before
  float take[MAX_TOP];       // what it takes off its gradient
  int next[MAX_TOP];         // the next one of the same thread
  int head[THREADS];         // a thread's first one, or -1
  unsigned where[THREADS];   // its packs with one; bit 31: its single element
  int wrong, empty, first;
};
#define WHERE_MORE 30        // packs beyond those that are held
#define WHERE_SINGLE 31

// The teacher's side of a row; lane i of the first wave has its classes i
// and i + 64.
struct Teacher {
  int id[2];
  float z[2], x[2], q[2];      // (z: from softmax on less the largest, zm)
  float zm, gs;
  bool wrong;

  __device__ __forceinline__ void load(const DistillArgs& a, long row) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = threadIdx.x + h * WAVE;
      id[h] = -1;
      z[h] = -INFINITY;
      if (k < a.top) {
        id[h] = a.idx[row * a.top + k];
        z[h] = a.z[row * a.top + k];
      }
    }
  }
  // its logits in the student's row
  template <typename T>
  __device__ __forceinline__ void gather(const DistillArgs& a, const T* row) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      x[h] = id[h] >= 0 && id[h] < a.cols ? (float)row[id[h]] : 0.f;
  }
  __device__ __forceinline__ void gathered(const DistillArgs& a, long row) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = threadIdx.x + h * WAVE;
      x[h] = k < a.top ? a.xk[row * a.top + k] : 0.f;
    }
  }
  __device__ __forceinline__ void softmax(const DistillArgs& a) {
    bool w = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      w |= id[h] >= a.cols || (id[h] >= 0 && !(z[h] < INFINITY));
      if (id[h] >= a.cols || z[h] == -INFINITY) id[h] = -1;
      if (id[h] < 0) z[h] = -INFINITY;
    }
    wrong = __any(w);
    zm = wave_max(fmaxf(z[0], z[1]));
    float g[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      z[h] -= zm;
      g[h] = id[h] >= 0 ? pow2(z[h] * a.c) : 0.f;
    }
    gs = wave_sum(g[0] + g[1]);
#pragma unroll
    for (int h = 0; h < 2; ++h) q[h] = g[h] / gs;
  }
  // Leaves what each class takes off its gradient, all places of a class
  // together, with the thread that holds the element of x[0..n).  Places that
  // share a class get the logit z that belongs to the sum Q of their shares
  // (tau ln Q/q more), so that the loss, which goes over the places, is
  // sum Q (ln Q - ln p) over the classes.
  template <typename T, int THREADS, int NV>
  __device__ __forceinline__ void place(const DistillArgs& a, int base, int n,
                                        const Cut<T>& cut,
                                        DistillSpace<THREADS>& sp) {
    constexpr int N = Pack<T>::N;
    const int tid = threadIdx.x;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sp.id[tid + h * WAVE] = id[h];
      sp.take[tid + h * WAVE] = q[h];
    }
    wave_fence();
    float sum[2] = {0.f, 0.f};
    bool again[2] = {id[0] < 0, id[1] < 0};
#pragma unroll 4
    for (int j = 0; j < (a.top + 3) / 4 * 4; ++j) {
      const int other = sp.id[j];
      const float share = sp.take[j];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool same = other == id[h];
        sum[h] += same ? share : 0.f;
        again[h] |= same && j < tid + h * WAVE;
      }
    }
    // (all reads of the wave are before its writes)
    wave_fence();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = tid + h * WAVE;
      const int j = id[h] - base;
      if (q[h] > 0.f && sum[h] != q[h])
        z[h] = fmaf(a.tau * LN2, log2_of(sum[h] / q[h]), z[h]);
      sp.id[k] = -1;
      if (again[h] || j < 0 || j >= n) continue;
      sp.id[k] = j;
      sp.take[k] = a.tau * sum[h];
      const int p = j - cut.head, tail = cut.packs * N;
      int owner, bit = WHERE_SINGLE;
      if (p < 0) {
        owner = j;
      } else if (p >= tail) {
        owner = N + p - tail;
      } else {
        owner = p / N % THREADS;
        bit = p / N / THREADS;
        if (bit >= NV) bit = WHERE_MORE;
      }
      sp.next[k] = atomicExch(&sp.head[owner], k);
      atomicOr(&sp.where[owner], 1u << bit);
    }
  }
  // tau sum q (ln q - ln p), after place()
  __device__ __forceinline__ float loss(const DistillArgs& a, const Row& r) {
    const float apart = a.tau * (r.ln - log2_of(gs) * LN2);
    float s = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (id[h] >= 0 && q[h] > 0.f)
        s += q[h] * (z[h] - (x[h] - r.m) + apart);
    return wave_sum(s);
  }
};

// the first class with the value m among those that this thread holds
template <typename T, int THREADS, int NV>
__device__ __forceinline__ int first_held(Held<T, THREADS, NV>& h, const T* x,
                                          const Cut<T>& cut, float m) {
  constexpr int N = Pack<T>::N;
  const int tid = threadIdx.x;
  int at = 0x7fffffff;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (i * THREADS >= cut.packs) break;
    float e[N];
    h.v[i].forget();
    h.v[i].get(e);
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (e[j] == m) at = min(at, cut.head + (i * THREADS + tid) * N + j);
  }
  for (int p = NV * THREADS + tid; p < cut.packs; p += THREADS)
    for (int j = 0; j < N; ++j) {
      const int k = cut.head + p * N + j;
      if ((float)x[k] == m) at = min(at, k);
    }
  if (h.rest == m && cut.single >= 0) at = min(at, cut.single);
  return at;
}

// sums of the packs beyond those that are held
template <typename T, int THREADS, int NV>
__device__ __forceinline__ void add_more(const T* x, const Cut<T>& cut,
                                         Sums& a, float c) {
  constexpr int N = Pack<T>::N;
  for (int b = NV * THREADS; b < cut.packs; b += CHUNK * THREADS) {
    Pack<T> v[CHUNK];
#pragma unroll
    for (int i = 0; i < CHUNK; ++i) {
      const int p = b + i * THREADS + threadIdx.x;
      v[i].fill(-INFINITY);
      if (p < cut.packs) v[i].load(x + cut.head + (long)p * N);
    }
    add_packs<false, T, CHUNK>(v, a, c, nullptr);
  }
}

template <typename T, typename O, int N>
__device__ __forceinline__ void put_gradients(O* to, const float* g,
                                              bool past) {
  if constexpr (__is_same(T, O)) {
    Pack<O> v;
    v.set(g);
    if (past) {
      // (else both become one store, without the mark)
      asm volatile("");
      v.store_once(to);
      asm volatile("");
    } else {
      v.store(to);
    }
  } else {
    O t[N];
#pragma unroll
    for (int j = 0; j < N; ++j) t[j] = from_f<O>(g[j]);
    __builtin_memcpy(to, t, sizeof(t));
  }
}

// One workgroup to a row, or (JOINED) to a part of a row whose sums
// distill_part_k has left.  The teacher's side is done by the first wave
// while the row is under way.  2048 x 131072 bf16: 219 us, 4.9 TB/s of one
// read and one write; 4096 x 32000: 103 us, 5.1 TB/s; 1023 x 50001 fp32: 79
// us, 5.1 TB/s.  Bound by memory and by the turns that a row takes: a compute
// unit has registers for one row of 256 KB, so that nothing is loaded while it
// is stored (a copy laid out the same takes 192 us of the 219).  Loading the
// next row into the registers that the gradients leave was no faster.  The form
// that the evaluator calls, fp32 logits with a bf16 gradient, labels and n_err:
// 1023 x 50001 71 us, 4.3 TB/s; 256 x 1000 4.8 us; the first largest class and
// its barrier are 0.3 to 2 us of that.  Wrong rows add to one number, each for
// itself: 4096 x 1000 takes 15 us with all of them right, 21 with a third of
// them wrong and 53 with all wrong (eval_softmax: 9 and 53).
template <typename T, typename O, int THREADS, int NV, bool JOINED>
__global__ __launch_bounds__(THREADS) void distill_k(DistillArgs a) {
  __shared__ DistillSpace<THREADS> sp;
  __shared__ Sums tmp[THREADS / WAVE];
  constexpr int N = Pack<T>::N;
  const int tid = threadIdx.x;
  const Place at(a.cols, a.size);
  if (at.row >= a.rows) return;
  O* err = (O*)a.err.p + at.row * a.err.stride + at.base;
  if (at.row >= a.live) {
    for (int j = tid; j < at.n; j += THREADS) err[j] = from_f<O>(0.f);
    if (tid == 0 && at.base == 0 && a.loss) a.loss[at.row] = 0.f;
    return;
  }
  const bool leads = tid < WAVE;
  const T* row = (const T*)a.x.p + at.row * a.x.stride;
  const T* x = row + at.base;
  const Cut<T> cut(x, at.n);
  Teacher t;
  if (leads) t.load(a, at.row);
  Held<T, THREADS, NV> h;
  h.load(x, cut);
  sp.head[tid] = -1;
  sp.where[tid] = 0;
  __syncthreads();
  if (leads) {
    if (JOINED)
      t.gathered(a, at.row);
    else
      t.gather(a, row);
    t.softmax(a);
    t.place<T, THREADS, NV>(a, at.base, at.n, cut, sp);
    if (tid == 0) {
      sp.wrong = t.wrong;
      sp.empty = t.zm == -INFINITY;
      sp.first = 0x7fffffff;
    }
  }
  Row r;
  int first = 0x7fffffff;
  if (JOINED) {
    r = join_parts(a.parts + at.row * gridDim.x, gridDim.x, a.c, &first);
    __syncthreads();
  } else {
    Sums s = held_sums<false>(h, cut.packs, a.c, nullptr);
    add_more<T, THREADS, NV>(x, cut, s, a.c);
    const float own = s.m;
    s = join_block<false, THREADS>(s, a.c, tmp);
    if (is_far(s.m, a.c)) s = far_sums(x, at.n, s.m, a.c, (float*)tmp);
    r.finish(s, a.c);
    if (a.labels) {
      if (own == r.m && !r.none)
        atomicMin(&sp.first, first_held(h, x, cut, r.m));
      __syncthreads();
      first = sp.first;
    }
  }
  const bool bad = r.bad || sp.wrong;
  const bool lost = r.none || sp.empty;
  if (leads && at.base == 0) {
    const float loss = bad ? NAN : lost ? 0.f : a.tau * t.loss(a, r);
    if (tid == 0) {
      if (a.loss) a.loss[at.row] = loss;
      if (a.labels) {
        // (the student's errors: what the teacher gives is no part of them)
        const int l = a.labels[at.row];
        if (l >= 0 && (r.bad || r.none || first != l)) atomicAdd(a.n_err, 1);
      }
    }
  }

  const float scale = bad ? NAN : lost ? 0.f : a.tau / r.s;
  if (r.far) {
    // (all classes one by one; the places of the teacher's are searched)
    for (int j = tid; j < at.n; j += THREADS) {
      float g = bad ? NAN : lost ? 0.f : scale * pow2(r.u((float)x[j]));
      if (!bad && !lost)
        for (int k = 0; k < a.top; ++k)
          if (sp.id[k] == j) g -= sp.take[k];
      err[j] = from_f<O>(g);
    }
    return;
  }
  const unsigned where = lost ? 0 : sp.where[tid];
  // gradients of a pack; `some`: with classes of the teacher's
  auto pack = [&](const Pack<T>& v, int p, bool some) {
    float g[N];
    v.get(g);
#pragma unroll
    for (int j = 0; j < N; ++j) g[j] = scale * pow2(fmaf(g[j], a.c, -r.um));
    const int j = cut.head + p * N;
    if (some) {
      for (int k = sp.head[tid]; k >= 0; k = sp.next[k]) {
        const int d = sp.id[k] - j;
        const float by = sp.take[k];
#pragma unroll
        for (int i = 0; i < N; ++i) g[i] -= d == i ? by : 0.f;
      }
    }
    put_gradients<T, O, N>(err + j, g, a.past);
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (i * THREADS >= cut.packs) break;
    const int p = i * THREADS + tid;
    h.v[i].forget();
    if (p < cut.packs) pack(h.v[i], p, where >> i & 1);
  }
  for (int p = NV * THREADS + tid; p < cut.packs; p += THREADS) {
    Pack<T> v;
    v.load(x + cut.head + (long)p * N);
    pack(v, p, where >> WHERE_MORE & 1);
  }
  if (cut.single >= 0) {
    float g = scale * pow2(fmaf(h.rest, a.c, -r.um));
    if (where >> WHERE_SINGLE & 1)
      for (int k = sp.head[tid]; k >= 0; k = sp.next[k])
        g -= sp.id[k] == cut.single ? sp.take[k] : 0.f;
    err[cut.single] = from_f<O>(g);
  }
}

// Sums of a part of a row, and the row's logits of the teacher's classes.  One
// row of 131072 bf16 in 16 parts, with their gradients: 9.8 us, two launches
// and the delays of their steps.
template <typename T, int THREADS, int NV>
__global__ __launch_bounds__(THREADS) void distill_part_k(DistillArgs a) {
  __shared__ Sums tmp[THREADS / WAVE];
  __shared__ int first;
  const Place at(a.cols, a.size);
  if (at.row >= a.live) return;
  const T* row = (const T*)a.x.p + at.row * a.x.stride;
  const T* x = row + at.base;
  if (at.base == 0)
    for (int k = threadIdx.x; k < a.top; k += THREADS) {
      const int id = a.idx[at.row * a.top + k];
      a.xk[at.row * a.top + k] =
          id >= 0 && id < a.cols ? (float)row[id] : 0.f;
    }
  if (threadIdx.x == 0) first = 0x7fffffff;
  const Cut<T> cut(x, at.n);
  Held<T, THREADS, NV> h;
  h.load(x, cut);
  Sums s = held_sums<false>(h, cut.packs, a.c, nullptr);
  add_more<T, THREADS, NV>(x, cut, s, a.c);
  const float own = s.m;
  s = join_block<false, THREADS>(s, a.c, tmp);
  if (is_far(s.m, a.c)) s = far_sums(x, at.n, s.m, a.c, (float*)tmp);
  if (a.labels) {
    if (own == s.m) atomicMin(&first, first_held(h, x, cut, s.m));
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const int at_first = a.labels && first < at.n ? at.base + first
                                                  : 0x7fffffff;
    a.parts[at.item] = part_of(s, a.c, at_first);
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
// Fewer rows than LP_ROWS are cut until there are four workgroups for each
// compute unit, but into parts of 4 packs a thread at least.  In a graph, rows
// of 131072 bf16, 64 alternatives, whole and cut: 60 rows 26.1 and 18.5 us, 100
// rows 27.2 and 22.3, 200 28.5 and 29.4, 300 31.1 and 32.2, 511 33.1 and 44.2;
// of 50001, 20 alternatives: 100 rows 14.0 and 14.0, 200 14.4 and 16.6.  One
// row with 5 alternatives: parts of 4 packs 8.8 us, 8 10.2, 2 8.8 (30 rows, 64
// alternatives: 15.9, 16.9, 17.1).
#define LP_LEAST 4
#define LP_ROWS 192
#define LP_BLOCKS 1024

// Packs of a thread at most that are held (4096 rows of 8000 fp32: 26.9 us,
// streamed 30.8; 8192 of 8000 bf16 37.9, 42.0).  With 16 of them too few waves
// fit a compute unit: 4096 x 20000 bf16 42.5 us, streamed 38.4.
#define LP_HELD 8

// How a call is laid out: parts of a row, elements of a part, and packs of
// a thread where they are held (0: they stream past)
struct LogprobsPlan {
  int split, size, nv;
};

static LogprobsPlan logprobs_plan(int type, long rows, int cols) {
  const int n = type == ROW_F32 ? 4 : 8;
  const long held = LP_THREADS * LP_HELD * n;
  const long most = (long)LP_GROUPS * GROUP * n;
  long split = (cols + most - 1) / most;
  const long least = LP_THREADS * LP_LEAST * n;
  while (rows < LP_ROWS && split < LP_PARTS && rows * split < LP_BLOCKS &&
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
      HELD(1) HELD(2) HELD(4) HELD(8)
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

// Rows are cut into parts up to as many rows: a part's sums are a pass of
// their own, and what that costs is gained back where few compute units would
// have work.  Whole rows of 131072 bf16 against parts: 1 row 17.0 and 9.8 us,
// 30 rows 19.0 and 13.0, 60 22.1 and 19.6, 100 22.9 and 23.7, 200 26.3 and
// 39.8.
#define DISTILL_CUT 64

// How a call is laid out: parts of a row, elements of a part, threads and
// packs of a thread.  Rows that 256 threads hold in 16 packs each are left to
// them (4096 x 32000 bf16: 103 us; to 512 threads 107), since a workgroup's
// loads, sums and stores then overlap another's; of longer ones as many
// threads as hold them (2048 x 60000: 512 threads 101 us, 1024 124); what 1024
// do not hold is read twice.
struct DistillPlan {
  int split, size, threads, nv;
};

static DistillPlan distill_plan(int type, long rows, int cols) {
  const int n = type == ROW_F32 ? 4 : 8;
  DistillPlan p{1, cols, 256, 1};
  const long least = 256 * 4 * n;
  long split = 1;
  if (rows <= DISTILL_CUT)
    while (split < 64 && rows * split < 512 && cols / (split + 1) >= least)
      ++split;
  if (split > 1) {
    long size = (cols + split - 1) / split;
    p.size = (int)((size + n - 1) / n * n);
    p.split = (cols + p.size - 1) / p.size;
  }
  p.threads = (long)p.size <= 256 * 16 * n ? 256
              : (long)p.size <= 512 * 16 * n ? 512 : 1024;
  p.nv = p.threads > 256 ? 16 : 1;
  while (p.nv < 16 && (long)p.threads * p.nv * n < p.size) p.nv *= 2;
  return p;
}

// bytes that eval_distill_launch needs at `scratch`
long eval_distill_scratch(int type, long live, int cols, int top) {
  const DistillPlan p = distill_plan(type, live, cols);
  if (p.split == 1) return 0;
  return live * (p.split * (long)sizeof(Part) + top * (long)sizeof(float));
}

template <typename T, typename O>
static void distill_run(DistillArgs a, DistillPlan p, hipStream_t s) {
#define CASE(THREADS, NV)                                                    \
  if (p.threads == THREADS && p.nv == NV) {                                  \
    if (p.split == 1) {                                                      \
      hipLaunchKernelGGL(                                                    \
          HIP_KERNEL_NAME(distill_k<T, O, THREADS, NV, false>),              \
          parts_grid(1, a.rows), dim3(THREADS), 0, s, a);                    \
    } else {                                                                 \
      if (a.live)                                                            \
        hipLaunchKernelGGL(HIP_KERNEL_NAME(distill_part_k<T, THREADS, NV>),  \
                           parts_grid(p.split, a.live), dim3(THREADS), 0, s, \
                           a);                                               \
      hipLaunchKernelGGL(                                                    \
          HIP_KERNEL_NAME(distill_k<T, O, THREADS, NV, true>),               \
          parts_grid(p.split, a.rows), dim3(THREADS), 0, s, a);              \
    }                                                                        \
  }
  CASE(256, 1) CASE(256, 2) CASE(256, 4) CASE(256, 8) CASE(256, 16)
  CASE(512, 16) CASE(1024, 16)
#undef CASE
  HIP_CHECK_LAST();
}

void eval_distill_launch(int type, int err_type, RowsIn x, const int* idx,
                         const float* z, RowsOut err, float* loss,
                         const int* labels, int* n_err, int top, long rows,
                         long live, int cols, float tau, void* scratch,
                         hipStream_t s) {
  if (rows == 0) return;
  const DistillPlan p = distill_plan(type, live, cols);
  Part* parts = (Part*)scratch;
  DistillArgs a{x, idx, z, err, loss, labels, n_err, top, rows, live, cols,
                p.size, tau, LOG2E / tau, parts,
                p.split > 1 ? (float*)(parts + live * p.split) : nullptr,
                rows * cols * (err_type == ROW_F32 ? 4 : 2) >= PAST_CACHES};
#define RUN(T) distill_run<T, T>(a, p, s)
  if (type == ROW_F32 && err_type == ROW_BF16) {
    distill_run<float, bf16_t>(a, p, s);
  } else {
    ROW_TYPE_SWITCH(type, RUN)
  }
#undef RUN
}
