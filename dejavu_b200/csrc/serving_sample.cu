// Sampling of one token per row of logits: temperature, top-k, top-p, min-p, from a given random number.
//
// Entries are ordered without being sorted. (logit, index) is a 64-bit number, larger for what comes first, so that every cut is a
// threshold on it and ties need no rule of their own. A cluster of up to 8 blocks takes a row, each a slice of it in shared memory:
//   1. the slices arrive, and the row's largest entry;
//   2. a histogram of 2048 equal steps of the logit: how many entries, and how far into the step they are on average;
//   3. top-k: what lies in the step of the k-th entry, or, where few enough do, in all steps up to it, is collected in the first block and
//      sorted there; top-p: count and average bound a step's weight from both sides (the exponential is convex; the bounds are a 10^-4th
//      apart, where the steps' borders alone would leave thousands of entries between them), the entries between the bounds are
//      collected, those outside summed;
//   4. if all that can be kept is in the list, the first block makes the rest of it alone; else the sum of what is kept, warp by warp in
//      index order, and the place where the running sum passes u times it.
// Rows of more ties than the list takes, and comparisons that come out closer than the weights' errors allow (of 151936 entries with top-p 0.9 one
// row in 700, which then takes 0.3 to 0.8 ms; of 50272 one in 15000), go to one block, which reads the row from L2 as often as it needs, narrows the range by 2048 steps of the 64-bit number at
// a time, and has weights from exp in 64 bits: the token is that of the 64-bit definition.
//
// The steps lie between the largest entry and the smallest, at most 45 temperatures below it, so that ids masked by -1e4 rather than -inf make
// them coarser, and more entries lie between the bounds. Of flat rows that can be more than the list takes: 32 rows of 151936 of a spread
// of 0.5, top-p 0.9, take 53 us with -inf and 940 with -1e4 (top-p 0.5: 960 and 1230); with a spread of 2.5 both take 50.
//
// Weights: 2^(n/256) from a table, 2^f for the rest |f| <= 1/512 by its series in 32 bits, off by 1.2e-9 at most; sums have 64 bits. (32-bit
// weights would leave every tenth row of a flat distribution undecided.) Rows whose differences two floats do not hold (a largest entry of
// +inf, temperatures below 1e-30 or above 1e25) are left to one block too.
//
// A row is read once, then swept two or three times in shared memory between block and cluster barriers. One row of 50272 entries (top-k 50,
// top-p): 14 us, a chain of barriers and fetched code; 256 rows of settings of their own: 80 us, four waves of such chains and sweeps;
// 32 rows of 151936 (top-p 0.9): 49 us, a third of it the weights and their sums. (With pairs of floats as sums, and a warp alone
// with the share that the token is in: 88 and 65.)
#include <math.h>
#include <string.h>

#include <cooperative_groups.h>
#include <utility>

#include "pairs.cuh"
#include "serving.cuh"

namespace djv {

constexpr int SA_THREADS = 512, SA_WARPS = SA_THREADS / WARP, SA_BINS = 2048, SA_LIST = 2048, SA_CLUSTER = 8;
constexpr int SA_EACH = SA_BINS / SA_THREADS;  // steps, or entries of the list, of a thread
constexpr double SA_CLOSE = 3e-9;   // what counts as close, of a sum: more than twice the weights' relative error (and what they lose in sums)
constexpr int SA_TABLE = 256;
constexpr float SA_MAGIC = 12582912.f;  // added to a number below 2^22 rounds it: the lowest bits are then the number's
constexpr uint32_t SA_ROUND = 0x4b400000u;  // (its bits)
constexpr float SA_FAR = 45.f;      // temperatures below the largest entry from where on nothing counts (e^-45 = 3e-20)
constexpr double SA_TINY = 1e-10;   // unless u is less than what 2^30 of them make up together (3e-11): 0, or no usual random number

struct SampleArgs {
  long long *token;
  const void *logits;
  long long ld;
  const float *u, *temperature;
  double temperature0;
  const int *top_k;
  int top_k0;
  const float *top_p;
  double top_p0;
  const float *min_p;
  double min_p0;
  int V;
};

using u64 = unsigned long long;

// Larger for larger logits; NaN counts as -inf, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) x = -INFINITY;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
__device__ __forceinline__ u64 place_of(uint32_t key, int i) { return (u64)key << 32 | (uint32_t)~i; }

struct SampleShared {
  u64 list[SA_LIST];
  union {
    struct {
      union {
        unsigned count[SA_BINS];  // of this block's slice
        int owned[SA_LIST];       // later: its entries between the bounds of top-p
      };
      unsigned upto[SA_BINS];   // of the row, in this step and those in front of it
    };
    double mass[SA_BINS];       // (of a block that works alone)
  };
  unsigned into[SA_BINS], all_into[SA_BINS];  // sum of how far into the step entries are, in parts; of the slice, of the row
  uint2 table[SA_TABLE];      // 2^(30 + j / 256), rounded, less SA_ROUND; and as a float
  double part[SA_WARPS], part2[SA_WARPS], part3[SA_WARPS];
  u64 wide[SA_WARPS];
  float narrow[SA_WARPS], narrow2[SA_WARPS];
  unsigned counts[SA_WARPS];
  // written by the blocks of the cluster
  u64 best[SA_CLUSTER];
  float least[SA_CLUSTER];
  double sums[SA_CLUSTER][2], kept[SA_CLUSTER];
  int listed, own;
  u64 cut;                    // by the first block: entries whose place is lower are dropped
  int done;                   // by the first block: 1: it has the token, or finds it alone
  int found[4];
  u64 lo, hi, place;
};

// ---- what a block does together -------------------------------------------------------------------------------------
template <typename V, typename F>
__device__ __forceinline__ V block_all(V v, V *slots, F f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if (threadIdx.x % WARP == 0) slots[threadIdx.x / WARP] = v;
  __syncthreads();
  v = slots[threadIdx.x % SA_WARPS];
#pragma unroll
  for (int o = SA_WARPS / 2; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ double block_total(double v, SampleShared &s) {
  return block_all(v, s.part, [](double a, double b) { return a + b; });
}
// (Out of line, like other things that are used in several places: a row goes through most of the code once, and fetching that is a
// large part of its time.)
__device__ __noinline__ u64 block_most(u64 v, u64 *slots) {
  return block_all(v, slots, [](u64 a, u64 b) { return a > b ? a : b; });
}
__device__ __forceinline__ u64 block_least(u64 v, u64 *slots) { return ~block_most(~v, slots); }
__device__ __noinline__ double power_of_2(double x) { return exp2(x); }

// f(x, index) for the row's entries from lo to hi (multiples of the chunk, or the row's end), a thread every `step`-th chunk
template <typename T, bool VEC, typename F>
__device__ __forceinline__ void sweep(const T *row, int lo, int hi, int at, int step, F f) {
  constexpr int N = VEC ? Chunk<T>::N : 1, DEEP = 4;
  int i = lo + at * N;
  if (VEC) {
    for (; i + (DEEP - 1) * step * N + N <= hi; i += DEEP * step * N) {
      uint4 v[DEEP];
#pragma unroll
      for (int d = 0; d < DEEP; ++d) v[d] = *reinterpret_cast<const uint4 *>(row + i + d * step * N);
#pragma unroll
      for (int d = 0; d < DEEP; ++d) {
        float x[N];
        unpack_chunk<T>(v[d], x);
#pragma unroll
        for (int e = 0; e < N; ++e) f(x[e], i + d * step * N + e);
      }
    }
  }
  for (; i < hi; i += step * N)
    for (int e = 0; e < N; ++e)
      if (i + e < hi) f(to_f(row[i + e]), i + e);
}

// The places of a warp's 64 entries, two to a lane (lane and lane + 32), through the steps j <= 32 of a bitonic merge of blocks of k.
__device__ __forceinline__ void merge_in_warp(u64 &x, u64 &y, int first, int k, int from) {
  const int lane = threadIdx.x % WARP;
  if (from >= 32) {
    const bool falls = ((first + lane) & k) == 0;
    if ((x < y) == falls) {
      const u64 t = x;
      x = y;
      y = t;
    }
    from = 16;
  }
  for (int j = from; j > 0; j >>= 1) {
    const u64 a = __shfl_xor_sync(0xffffffffu, x, j), b = __shfl_xor_sync(0xffffffffu, y, j);
    const bool low = (lane & j) == 0;  // of a pair, the one that gets the larger where the block falls
    if ((low == (((first + lane) & k) == 0)) == (a > x)) x = a;
    if ((low == (((first + 32 + lane) & k) == 0)) == (b > y)) y = b;
  }
}

// Sorts list[0 .. n), largest first; n <= SA_LIST; entries are different, the filling is 0. Steps inside 64 entries stay in a warp.
__device__ __noinline__ void sort_list(u64 *list, int n) {
  int size = 64;
  while (size < n) size *= 2;
  const int lane = threadIdx.x % WARP, warp = threadIdx.x / WARP;
  for (int i = n + threadIdx.x; i < size; i += SA_THREADS) list[i] = 0;
  __syncthreads();
  for (int at = warp * 64; at < size; at += SA_WARPS * 64) {
    u64 x = list[at + lane], y = list[at + 32 + lane];
    for (int k = 2; k <= 64; k *= 2) merge_in_warp(x, y, at, k, k / 2);
    list[at + lane] = x;
    list[at + 32 + lane] = y;
  }
  __syncthreads();
  for (int k = 128; k <= size; k *= 2) {
    for (int j = k / 2; j >= 64; j /= 2) {
      for (int i = threadIdx.x; i < size / 2; i += SA_THREADS) {
        const int a = 2 * i - (i & (j - 1)), b = a + j;
        const u64 x = list[a], y = list[b];
        if ((x < y) == ((a & k) == 0)) {
          list[a] = y;
          list[b] = x;
        }
      }
      __syncthreads();
    }
    for (int at = warp * 64; at < size; at += SA_WARPS * 64) {
      u64 x = list[at + lane], y = list[at + 32 + lane];
      merge_in_warp(x, y, at, k, 32);
      list[at + lane] = x;
      list[at + 32 + lane] = y;
    }
    __syncthreads();
  }
}

// Sum of v over the threads in front of this one; total receives the block's.
template <typename V>
__device__ __noinline__ V block_before(V v, V *slots, V &total) {
  const int lane = threadIdx.x % WARP, warp = threadIdx.x / WARP;
  V sum = v;
#pragma unroll
  for (int o = 1; o < WARP; o <<= 1) {
    const V up = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += up;
  }
  __syncthreads();
  if (lane == WARP - 1) slots[warp] = sum;
  __syncthreads();
  V run = slots[lane % SA_WARPS];
#pragma unroll
  for (int o = 1; o < SA_WARPS; o <<= 1) {
    const V up = __shfl_up_sync(0xffffffffu, run, o, SA_WARPS);
    if (lane % SA_WARPS >= o) run += up;
  }
  total = __shfl_sync(0xffffffffu, run, SA_WARPS - 1);
  const V front = __shfl_sync(0xffffffffu, run, warp ? warp - 1 : 0);
  return (warp ? front : V(0)) + (sum - v);
}

// The largest entry of a row and what follows from it.
struct SampleScale {
  float top, inv;       // largest logit, steps per unit of the logit
  float fine, inv_fine; // parts of a step, and per unit of the logit
  int fine_bits;
  double temperature;
  float c_hi, c_lo;     // log2(e) / temperature
  float reach;          // entries further below the largest are dropped
  double close;         // see SA_CLOSE

  __device__ __forceinline__ bool counts(float x) const { return top - x <= reach || x == top; }
  // For x that counts: how many parts of a step, `fine` of them to one, are in front of it, rounded, plus 2^23: a number whose lowest bits
  // are the part and those above the step, and which compares with parts(step).
  __device__ __forceinline__ float part_of(float x) const { return x == top ? 8388608.f : fmaf(top - x, inv_fine, 8388608.f); }
  __device__ __forceinline__ float parts(float step) const { return fmaf(step, fine, 8388608.f); }
  __device__ __forceinline__ double exact(float x) const { return x == top ? 1.0 : exp(((double)x - (double)top) / temperature); }
  // For x that counts (for others a number that means nothing): 2^((x - top) c) = 2^(n / 256) (1 + q), in two at a time; bits receives n as
  // the lowest bits of SA_MAGIC + n. |q| <= 0.00136, so that two terms of its series are left to 3e-13.
  __device__ __forceinline__ uint64_t reduced(uint64_t t, uint64_t x, uint64_t &bits) const {  // t: x - top, rounded
    const uint64_t ch = pack2(c_hi, c_hi), zero = pack2(0.f, 0.f);
    const uint64_t v = sub2(t, x), e = sub2(sub2(x, sub2(t, v)), add2(pack2(top, top), v));  // x - top = t + e
    const uint64_t ny = fma2(t, pack2(-c_hi, -c_hi), zero);                                   // -y, and what it lacks:
    const uint64_t rest = add2(fma2(t, ch, ny), fma2(t, pack2(c_lo, c_lo), fma2(e, ch, zero)));
    bits = fma2(ny, pack2(-256.f, -256.f), pack2(SA_MAGIC, SA_MAGIC));
    const uint64_t n = sub2(bits, pack2(SA_MAGIC, SA_MAGIC)), nf = fma2(n, pack2(0.00390625f, 0.00390625f), ny);  // (exact)
    const uint64_t f = fma2(sub2(rest, nf), pack2(0.69314718f, 0.69314718f), zero);
    return fma2(fma2(f, f, zero), fma2(f, pack2(0.16666667f, 0.16666667f), pack2(0.5f, 0.5f)), f);
  }
  // 2^(n / 256) (1 + q) as an integer times 2^(-30 - down): off by 1.2e-9 of it at most (the table by 2^-31, the rounding by as much)
  __device__ __forceinline__ static uint32_t mantissa(float bits, float q, const uint2 *table, unsigned &down) {
    const uint32_t n = __float_as_uint(bits);
    const uint2 w = table[n % SA_TABLE];
    down = SA_ROUND / SA_TABLE - n / SA_TABLE;
    return w.x + __float_as_uint(fmaf(__uint_as_float(w.y), q, SA_MAGIC));
  }
  __device__ __forceinline__ double weight(float x, const uint2 *table) const {  // the same in 64 bits
    uint64_t bits;
    float b0, b1, q0, q1;
    const uint64_t x2 = pack2(x, x);
    unpack2(reduced(sub2(x2, pack2(top, top)), x2, bits), q0, q1);
    unpack2(bits, b0, b1);
    unsigned down;
    const uint32_t m = mantissa(b0, q0, table, down);
    return (double)m * __longlong_as_double((long long)(1023 - 30 - down) << 52);
  }
};
// (where a few are made in cold code)
__device__ __noinline__ double weight_of(const SampleScale &z, float x, const uint2 *table) { return z.weight(x, table); }
constexpr int SA_UNITS = 52;  // sums are integers, 2^52 to the largest weight: 4096 of those fit. Entries 36 temperatures below it are 0 in them.
__device__ __forceinline__ u64 shifted(u64 v, unsigned down) {  // (0 from 64 on)
  u64 r;
  asm("shr.u64 %0, %1, %2;" : "=l"(r) : "l"(v), "r"(down));
  return r;
}

// One row by one block, in 64 bits, from global memory: nothing is too close and nothing too much.
template <typename T, bool VEC>
struct SampleAlone {
  const T *row;
  int V;
  SampleShared &s;
  SampleScale z;

  template <typename F>
  __device__ __forceinline__ void all(F f) const {
    sweep<T, VEC>(row, 0, V, threadIdx.x, SA_THREADS, f);
  }

  // Of the entries between places lo and hi (inclusive), those in front first: the place of entry number `rank` (from 0), or, by
  // mass, of the last entry in front of which less than `mass` lies. Cuts the range until what is left fits the list.
  template <bool MASS>
  __device__ u64 narrow(u64 lo, u64 hi, int rank, double mass) {
    for (;;) {
      __syncthreads();
      if (threadIdx.x == 0) s.listed = 0;
      __syncthreads();
      u64 first = 0, last = ~0ull;
      all([&](float x, int i) {
        const u64 p = place_of(order_of(x), i);
        if (p < lo || p > hi || !z.counts(x)) return;
        first = p > first ? p : first;
        last = p < last ? p : last;
        const int at = atomicAdd(&s.listed, 1);
        if (at < SA_LIST) s.list[at] = p;
      });
      __syncthreads();
      const int n = s.listed;
      if (n <= SA_LIST) break;
      hi = block_most(first, s.wide);
      lo = block_least(last, s.wide);
      int shift = 0;
      while (((hi - lo) >> shift) >= SA_BINS) ++shift;
      for (int i = threadIdx.x; i < SA_BINS; i += SA_THREADS) {
        if (MASS) s.mass[i] = 0;
        else s.count[i] = 0;
      }
      __syncthreads();
      all([&](float x, int i) {
        const u64 p = place_of(order_of(x), i);
        if (p < lo || p > hi || !z.counts(x)) return;
        const int bin = (int)((hi - p) >> shift);
        if (MASS) atomicAdd(&s.mass[bin], z.exact(x));
        else atomicAdd(&s.count[bin], 1u);
      });
      __syncthreads();
      if (threadIdx.x == 0) {
        int bin = 0;
        if (MASS) {  // the last step in front of which less than `mass` lies and that holds anything
          double run = 0, before = 0;
          int best = 0;
          for (; bin < SA_BINS; ++bin) {
            if (s.mass[bin] == 0) continue;
            if (bin > 0 && run >= mass) break;
            best = bin;
            before = run;
            run += s.mass[bin];
          }
          s.found[0] = best;
          s.sums[0][0] = before;
        } else {
          int run = 0;
          while (bin < SA_BINS - 1 && run + (int)s.count[bin] <= rank) run += s.count[bin++];
          s.found[0] = bin;
          s.found[1] = run;
        }
      }
      __syncthreads();
      const int bin = s.found[0];
      if (MASS) mass -= s.sums[0][0];
      else rank -= s.found[1];
      const u64 step = 1ull << shift, up = hi - (u64)bin * step;
      lo = up - lo >= step ? up - (step - 1) : lo;
      hi = up;
    }
    const int n = s.listed;
    sort_list(s.list, n);
    if (threadIdx.x == 0) {
      int at = min(rank, n - 1);
      if (MASS) {
        double run = 0;
        at = 0;
        for (int i = 0; i < n && (i == 0 || run < mass); ++i) {
          at = i;
          run += z.exact(logit_of((uint32_t)(s.list[i] >> 32)));
        }
      }
      s.place = s.list[at];
    }
    __syncthreads();
    const u64 place = s.place;
    __syncthreads();
    return place;
  }

  __device__ __noinline__ int token(int k, double p, double min_p, double u) {
    u64 cut = 0;
    const u64 most = place_of(order_of(z.top), 0);
    if (k > 0 && k < V) {
      int n = 0;
      all([&](float x, int) { n += z.counts(x); });
      if ((int)block_total(n, s) > k) cut = narrow<false>(0, most, k - 1, 0);
    }
    if (p < 1) {
      double sum = 0;
      all([&](float x, int i) {
        if (z.counts(x) && place_of(order_of(x), i) >= cut) sum += z.exact(x);
      });
      cut = narrow<true>(cut, most, 0, p * block_total(sum, s));
    }
    return draw(row, 0, V, cut, u, min_p, [&](float x) { return z.exact(x); }, [&](float x) { return z.exact(x); });
  }

  // The first index of from .. to - 1 at which the running sum of what is kept passes u times its total.
  template <typename W, typename E>
  __device__ int draw(const T *entries, int from, int to, u64 cut, double u, double min_p, W weight, E exact) {
    const int warp = threadIdx.x / WARP, lane = threadIdx.x % WARP;
    constexpr int N = VEC ? Chunk<T>::N : 1;
    const int share = ((to - from + SA_WARPS - 1) / SA_WARPS + WARP * N - 1) / (WARP * N) * (WARP * N);
    const int lo = min(to, from + warp * share), hi = min(to, lo + share);
    auto kept = [&](float x, int i) -> double {
      if (!z.counts(x) || place_of(order_of(x), i) < cut) return 0.0;
      const double w = weight(x);
      if (min_p > 0 && w < min_p * (1 + 1e-8) && (w < min_p * (1 - 1e-8) || exact(x) < min_p)) return 0.0;
      return w;
    };
    double sum = 0;
    sweep<T, VEC>(entries, lo, hi, lane, WARP, [&](float x, int i) { sum += kept(x, i); });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    __syncthreads();
    if (lane == 0) s.part[warp] = sum;
    __syncthreads();
    double total = 0;
    for (int w = 0; w < SA_WARPS; ++w) total += s.part[w];
    return locate(entries, from, to, share, 0.0, u * total, total, kept);
  }

  // The first of SA_WARPS sums at which the running sum exceeds target (before: in front of the first, then of that one); SA_WARPS: none, and
  // last has the last that is not 0.
  __device__ __forceinline__ static int passed(const double *sums, double &before, double target, int &last) {
    last = 0;
    double run = before;
    for (int w = 0; w < SA_WARPS; ++w) {
      if (sums[w] > 0) last = w;
      if (run + sums[w] > target) {
        before = run;
        return w;
      }
      run += sums[w];
    }
    return SA_WARPS;
  }
  // s.part has the sums of shares of the entries from .. to - 1, `before` is in front of the first: where the running sum passes target.
  // found[1]: too close to tell.
  template <typename K>
  __device__ int locate(const T *entries, int from, int to, int share, double before, double target, double total, K kept) {
    const int warp = threadIdx.x / WARP, lane = threadIdx.x % WARP;
    int last;
    int at = passed(s.part, before, target, last);
    if (at == SA_WARPS) {  // (rounding: the last entry that is kept)
      at = last;
      target = INFINITY;
      before = 0;
    }
    // that share by all warps
    from = min(to, from + at * share);
    to = min(to, from + share);
    share = (share + SA_THREADS - 1) / SA_THREADS * WARP;
    const int lo = min(to, from + warp * share), hi = min(to, lo + share);
    double sum = 0;
    for (int i = lo + lane; i < hi; i += WARP) sum += kept(to_f(entries[i]), i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s.part2[warp] = sum;
    __syncthreads();
    at = passed(s.part2, before, target, last);
    bool near = false;
    if (at == SA_WARPS) {
      near = target < INFINITY;  // (the two sums differ in their rounding)
      at = last;
    }
    if (warp == at) {
      double run = before;
      int token = -1, latest = -1;
      near |= fabs(before - target) <= z.close * total;
      for (int i0 = lo; i0 < hi && token < 0; i0 += WARP) {
        const int i = i0 + lane;
        const double w = i < hi ? kept(to_f(entries[i]), i) : 0.0;
        const unsigned any = __ballot_sync(0xffffffffu, w > 0);
        if (any == 0) continue;
        sum = w;
#pragma unroll
        for (int o = 1; o < WARP; o <<= 1) {
          const double up = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += up;
        }
        const unsigned over = __ballot_sync(0xffffffffu, w > 0 && run + sum > target);
        near |= __any_sync(0xffffffffu, w > 0 && fabs(run + sum - target) <= z.close * total) != 0;
        latest = i0 + 31 - __clz(any);
        if (over) token = i0 + __ffs(over) - 1;
        run += __shfl_sync(0xffffffffu, sum, WARP - 1);
      }
      if (lane == 0) {
        s.found[0] = token >= 0 ? token : latest;
        s.found[1] = near;
      }
    }
    __syncthreads();
    return s.found[0];
  }
};

// The sorted list holds all entries that can be kept, n of them, `behind` is the weight of the others that top-p counts: the token.
// found[1]: too close to tell. By all of a block.
__device__ __noinline__ int sample_list(SampleShared &s, const SampleScale &z, int n, double behind, double p, double min_p, double u) {
  const int at = threadIdx.x * SA_EACH;
  double w[SA_EACH], mine = 0, total;
  if (threadIdx.x == 0) s.found[1] = 0;
#pragma unroll
  for (int e = 0; e < SA_EACH; ++e) {
    w[e] = at + e < n ? weight_of(z, logit_of((uint32_t)(s.list[at + e] >> 32)), s.table) : 0.0;
    mine += w[e];
  }
  double run = block_before(mine, s.part, total);
  const double mass = p * (total + behind);
  int left = 0;
  bool near = false;
#pragma unroll
  for (int e = 0; e < SA_EACH; ++e) {
    bool in = at + e < n;
    if (in && p < 1 && at + e > 0) {
      in = run < mass;
      near |= fabs(run - mass) <= z.close * (total + behind);
    }
    if (in && min_p > 0 && w[e] < min_p * (1 + 1e-8)) in = w[e] >= min_p * (1 - 1e-8) && z.exact(logit_of((uint32_t)(s.list[at + e] >> 32))) >= min_p;
    left += in;
    run += w[e];
  }
  n = (int)block_total(left, s);  // (what is kept are the first ones)
  // by index: the halves of a place change sides
  for (int i = threadIdx.x; i < n; i += SA_THREADS) s.list[i] = s.list[i] << 32 | s.list[i] >> 32;
  __syncthreads();
  sort_list(s.list, n);
  mine = 0;
#pragma unroll
  for (int e = 0; e < SA_EACH; ++e) {
    w[e] = at + e < n ? weight_of(z, logit_of((uint32_t)s.list[at + e]), s.table) : 0.0;
    mine += w[e];
  }
  run = block_before(mine, s.part, total);
  const double target = u * total;
  int over = n - 1;  // (rounding: the last one)
#pragma unroll
  for (int e = SA_EACH - 1; e >= 0; --e) {
    double upto = run;
    for (int x = 0; x <= e; ++x) upto += w[x];
    if (at + e >= n) continue;
    near |= fabs(upto - target) <= z.close * total;
    if (upto > target) over = min(over, at + e);
  }
  over = (int)block_least((u64)over, s.wide);
  if (near) s.found[1] = 1;
  __syncthreads();
  return (int)~(uint32_t)(s.list[over] >> 32);
}

// The same for a list of up to 64 entries that is not sorted, of which the first `most` can be kept: by one warp, two entries to a lane, without
// a barrier. -1: too close to tell.
__device__ __noinline__ int sample_short(const SampleShared &s, const SampleScale &z, int n, int most, double behind, double p, double min_p, double u) {
  const int lane = threadIdx.x % WARP;
  u64 v[2];
  for (int h = 0; h < 2; ++h) v[h] = lane + 32 * h < n ? s.list[lane + 32 * h] : 0;
  bool near = false;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {  // the first ones first: what is kept; by index: the token
#pragma unroll 1
    for (int k = 2; k <= 64; k *= 2) merge_in_warp(v[0], v[1], 0, k, k / 2);
    double w[2], upto[2], total = 0;
    bool in[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      in[h] = v[h] != 0 && (pass || lane + 32 * h < most);
      w[h] = in[h] ? weight_of(z, logit_of((uint32_t)(pass ? v[h] : v[h] >> 32)), s.table) : 0.0;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      double sum = w[h];
#pragma unroll
      for (int o = 1; o < WARP; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
      }
      upto[h] = total + sum;
      total += __shfl_sync(0xffffffffu, sum, WARP - 1);
    }
    if (pass == 0) {
      const double all = total + behind, mass = p * all;
      double last = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const double up = __shfl_up_sync(0xffffffffu, upto[h], 1), before = lane ? up : last;
        last = __shfl_sync(0xffffffffu, upto[h], WARP - 1);
        if (in[h] && p < 1 && lane + h > 0) {
          in[h] = before < mass;
          near |= fabs(before - mass) <= z.close * all;
        }
        if (in[h] && min_p > 0 && w[h] < min_p * (1 + 1e-8))
          in[h] = w[h] >= min_p * (1 - 1e-8) && z.exact(logit_of((uint32_t)(v[h] >> 32))) >= min_p;
        v[h] = in[h] ? v[h] << 32 | v[h] >> 32 : 0;
      }
    } else {
      const double target = u * total;
      unsigned over[2], some[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        near |= in[h] && fabs(upto[h] - target) <= z.close * total;
        over[h] = __ballot_sync(0xffffffffu, in[h] && upto[h] > target);
        some[h] = __ballot_sync(0xffffffffu, in[h]);
      }
      const int at = over[0] ? __ffs(over[0]) - 1 : over[1] ? 31 + __ffs(over[1]) : __popc(some[0]) + __popc(some[1]) - 1;  // (rounding: the last one)
      const u64 found = __shfl_sync(0xffffffffu, at < 32 ? v[0] : v[1], at % WARP);
      n = (int)~(uint32_t)(found >> 32);
    }
  }
  return __any_sync(0xffffffffu, near) ? -1 : n;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(SA_THREADS, 2) sample_kernel(SampleArgs a, int slice, int stored) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  SampleShared &s = *reinterpret_cast<SampleShared *>(smem_raw);
  T *const copy = reinterpret_cast<T *>(smem_raw + (sizeof(SampleShared) + 15) / 16 * 16);
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), b = blockIdx.x / C;
  const int tid = threadIdx.x, warp = tid / WARP, lane = tid % WARP;
  auto started = cluster.barrier_arrive();
  pdl_prologue();
  const double temperature = a.temperature ? (double)a.temperature[b] : a.temperature0;
  const double p = a.top_p ? (double)a.top_p[b] : a.top_p0, min_p = fmin(a.min_p ? (double)a.min_p[b] : a.min_p0, 1.0), u = a.u[b];
  const int k = a.top_k ? a.top_k[b] : a.top_k0;
  const T *const row = static_cast<const T *>(a.logits) + b * a.ld;
  constexpr int N = VEC ? Chunk<T>::N : 1;
  const int from = min(a.V, rank * slice), to = min(a.V, from + slice);
  const T *const entries = stored ? copy - from : row;  // entries[i], from <= i < to
  // a warp's share of the slice, in index order
  const int share = ((to - from + SA_WARPS - 1) / SA_WARPS + WARP * N - 1) / (WARP * N) * (WARP * N);
  const int lo = min(to, from + warp * share), hi = min(to, lo + share);
  SampleShared &first = *cluster.map_shared_rank(&s, 0);
  SampleAlone<T, VEC> r{row, a.V, s, {}};
  SampleScale &z = r.z;
  // four entries at a time, whatever their type: short code
  constexpr int FOUR = VEC ? 4 : 2;
  auto four = [&](int i, float (&x)[FOUR]) {
    if (VEC && i + FOUR <= hi) {
      if (sizeof(T) == 4) {
        *reinterpret_cast<uint4 *>(x) = *reinterpret_cast<const uint4 *>(entries + i);
      } else {
        T y[4];
        *reinterpret_cast<uint2 *>(y) = *reinterpret_cast<const uint2 *>(entries + i);
#pragma unroll
        for (int e = 0; e < FOUR; ++e) x[e] = to_f(y[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < FOUR; ++e) x[e] = i + e < hi ? to_f(entries[i + e]) : -INFINITY;
    }
  };
  // f(x, index) for the warp's entries, and for some of -inf behind its last
  auto mine = [&](auto f) {
    for (int i = lo + lane * FOUR; i < hi; i += WARP * FOUR) {
      float x[FOUR];
      four(i, x);
#pragma unroll
      for (int e = 0; e < FOUR; ++e) f(x[e], i + e);
    }
  };

  // 1. the slice, and the row's largest and smallest entries
  float top = -INFINITY, bottom = INFINITY;
  int top_at = 0;
  {
    auto see = [&](float x, int i) {
      if (x > top) {  // (not -inf, not NaN; of equal ones the first)
        top = x;
        top_at = i;
      }
      if (x > -INFINITY) bottom = fminf(bottom, x);
    };
    if (VEC) {
      constexpr int DEEP = 4;
      for (int i0 = lo + lane * N; i0 < hi; i0 += DEEP * WARP * N) {
        uint4 v[DEEP];
#pragma unroll
        for (int d = 0; d < DEEP; ++d)
          if (i0 + d * WARP * N + N <= hi) v[d] = ld_stream16(row + i0 + d * WARP * N);
#pragma unroll 1
        for (int d = 0; d < DEEP; ++d) {
          const int i = i0 + d * WARP * N;
          if (i + N <= hi) {
            float x[N];
            unpack_chunk<T>(v[0], x);
            if (stored) *reinterpret_cast<uint4 *>(copy + (i - from)) = v[0];
#pragma unroll
            for (int e = 0; e < N; ++e) see(x[e], i + e);
#pragma unroll
            for (int e = 0; e + 1 < DEEP; ++e) v[e] = v[e + 1];
          } else {
            for (int e = i; e < hi; ++e) {
              if (stored) copy[e - from] = row[e];
              see(to_f(row[e]), e);
            }
          }
        }
      }
    } else {
      for (int i = lo + lane; i < hi; i += WARP) {
        if (stored) copy[i - from] = row[i];
        see(to_f(row[i]), i);
      }
    }
  }
  if (tid < SA_TABLE) {
    const double w = power_of_2(30.0 + tid * (1.0 / SA_TABLE));
    s.table[tid] = make_uint2(__double2uint_rn(w) - SA_ROUND, __float_as_uint((float)w));
  }
  for (int i = tid; i < SA_BINS; i += SA_THREADS) s.count[i] = s.into[i] = 0;
  if (tid == 0) s.listed = s.own = 0;
  u64 best = top > -INFINITY ? place_of(order_of(top), top_at) : 0;
  best = block_most(best, s.wide);
  bottom = block_all(bottom, s.narrow, [](float x, float y) { return fminf(x, y); });
  cluster.barrier_wait(std::move(started));  // (all blocks of the cluster have started)
  if (tid < C) {
    SampleShared &other = *cluster.map_shared_rank(&s, tid);
    other.best[rank] = best;
    other.least[rank] = bottom;
  }
  cluster.sync();
#pragma unroll
  for (int c = 0; c < SA_CLUSTER; ++c) {
    if (c < C) {
      best = s.best[c] > best ? s.best[c] : best;
      bottom = fminf(bottom, s.least[c]);
    }
  }
  const int arg = best ? (int)~(uint32_t)best : -1;
  if (arg < 0 || !(temperature > 0) || k == 1) {
    if (rank == 0 && tid == 0) a.token[b] = arg;
    return;
  }
  z.top = logit_of((uint32_t)(best >> 32));
  z.temperature = temperature;
  z.close = SA_CLOSE + a.V * (1.0 / (1ll << SA_UNITS));  // (a sum is 1 or more, and each entry loses less than a unit of it)
  const double log2_unit = 1.4426950408889634 / temperature;
  z.c_hi = (float)log2_unit;
  z.c_lo = (float)(log2_unit - (double)z.c_hi);
  z.reach = (float)fmin(SA_FAR * temperature, 3e38);
  const float range = fminf(z.top - bottom, z.reach);
  // (one step for all where they would be too fine or too coarse for floats, their parts, 2^23 in all, among them)
  z.inv = range > 1e-30f && range < 3e38f ? SA_BINS / range * 0.99999f : 0.f;
  z.fine_bits = min(12, __clz(a.V) - 1);  // (the sum of parts over the row stays below 2^31)
  z.fine = (float)(1 << z.fine_bits);
  z.inv_fine = z.inv * z.fine;
  bool by_rank = k > 0 && k < a.V;
  const bool by_mass = p < 1;
  u64 cut = 0;
  int rank_bin = SA_BINS;  // the step with the last entry that top-k keeps

  // One block goes on alone; the others have nothing left to do.
  auto alone = [&]() {
    const int token = r.token(k, p, min_p, u);
    if (tid == 0) a.token[b] = token;
  };
  if (!(u >= SA_TINY)) {  // falls among the first entries that are kept, even if they weigh next to nothing: down to where 64 bits end (2^-1074)
    z.reach = (float)fmin(746.0 * temperature, 3e38);
    if (rank == 0) alone();
    return;
  }
  if (z.top == INFINITY || !(log2_unit > 1e-25 && log2_unit < 1e30)) {  // (not for sums of two floats)
    if (rank == 0) alone();
    return;
  }
  // The block's own list (indices; fewer than SA_LIST, as the counts say): begun, an entry, and sent to the first block's list.
  auto begin_list = [&]() {
    if (tid == 0) s.own = 0;
    __syncthreads();
  };
  auto own = [&](int i) { s.owned[atomicAdd(&s.own, 1) & (SA_LIST - 1)] = i; };
  auto send_list = [&]() {
    __syncthreads();
    const int n = s.own;
    if (tid == 0) s.found[0] = n ? atomicAdd(&first.listed, n) : 0;
    __syncthreads();
    const int at = s.found[0];
    for (int i = tid; i < n && at + i < SA_LIST; i += SA_THREADS) {
      const int j = s.owned[i];
      first.list[at + i] = place_of(order_of(to_f(entries[j])), j);
    }
  };
  // Entries of steps from .. to - 1 go to the first block's list.
  auto collect = [&](float from, float to) {
    begin_list();
    from = z.parts(from);
    to = z.parts(to);
    mine([&](float x, int i) {
      const float at = z.part_of(x);
      if (at >= from && at < to && z.counts(x)) own(i);
    });
    send_list();
    cluster.sync();
  };
  const bool by_min = min_p > 0;
  const float min_high = (float)min_p * 1.000001f, min_low = (float)min_p * 0.999999f;  // (of weights in 32 bits)
  auto enough = [&](float x, double w) { return w >= min_p * (1 + 1e-8) || (w >= min_p * (1 - 1e-8) && z.exact(x) >= min_p); };
  // Weights of the entries that top-k keeps: in front of step `from` and from step `to` on (to the first block's sums), and, in s.part, of the
  // first ones that min-p keeps too, warp by warp. Those between go to the lists. (No branches around the weights, so that those
  // of a chunk overlap. Sums are integers: exact whatever their order, and a third of what pairs of floats take.)
  auto weigh = [&](float from, float to) {
    begin_list();
    from = z.parts(from);  // (infinite ones stay so)
    to = z.parts(to);
    const float rank_from = z.parts((float)rank_bin), rank_to = z.parts((float)rank_bin + 1);
    double x0 = 0, x1 = 0, x2 = 0;
    const uint64_t top2 = pack2(z.top, z.top), down2 = pack2(-z.inv_fine, -z.inv_fine), zero_part = pack2(8388608.f, 8388608.f);
    constexpr int RUN = ((1 << (64 - SA_UNITS)) - FOUR) / FOUR * WARP * FOUR;  // so many of a warp's entries leave room in its lanes' sums
    for (int begin = lo; begin < hi; begin += RUN) {
      u64 front = 0, behind = 0, enough_too = 0;
      const int end = min(hi, begin + RUN);
      for (int i = begin + lane * FOUR; i < end; i += WARP * FOUR) {
        float x[FOUR];
        four(i, x);
        unsigned between = 0;
#pragma unroll
        for (int e = 0; e < FOUR; e += 2) {
          const uint64_t xx = pack2(x[e], x[e + 1]), t2 = sub2(xx, top2);
          uint64_t bits2;
          float t[2], at[2], bits[2], q[2];
          unpack2(z.reduced(t2, xx, bits2), q[0], q[1]);
          unpack2(t2, t[0], t[1]);
          unpack2(fma2(t2, down2, zero_part), at[0], at[1]);
          unpack2(bits2, bits[0], bits[1]);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            bool keep = -t[h] <= z.reach;
            if (rank_bin < SA_BINS) keep = keep && (at[h] < rank_from || (at[h] < rank_to && place_of(order_of(x[e + h]), i + e + h) >= cut));
            unsigned down;
            const uint32_t m = z.mantissa(bits[h], q[h], s.table, down);
            const u64 w = shifted((u64)m << (SA_UNITS - 30), down);
            const bool first_ones = keep && at[h] < from, last_ones = keep && at[h] >= to;
            if (first_ones) front += w;
            if (last_ones) behind += w;
            if (by_min && first_ones) {
              const float about = (float)m * __uint_as_float((127 - 30 - down) << 23);
              if (about >= min_high || (about >= min_low && z.exact(x[e + h]) >= min_p)) enough_too += w;
            }
            between |= (unsigned)(keep && !first_ones && !last_ones) << (e + h);
          }
        }
        while (between) {
          own(i + __ffs(between) - 1);
          between &= between - 1;
        }
      }
      x0 += (double)front;
      x1 += (double)behind;
      x2 += (double)(by_min ? enough_too : front);
    }
    constexpr double UNIT = 1.0 / (1ll << SA_UNITS);
    x0 *= UNIT;
    x1 *= UNIT;
    x2 *= UNIT;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      x0 += __shfl_xor_sync(0xffffffffu, x0, o);
      x1 += __shfl_xor_sync(0xffffffffu, x1, o);
      x2 += __shfl_xor_sync(0xffffffffu, x2, o);
    }
    if (lane == 0) {
      s.part[warp] = x2;
      s.part2[warp] = x0;
      s.part3[warp] = x1;
    }
    send_list();
    if (tid < 2) {
      double sum = 0;
      for (int w = 0; w < SA_WARPS; ++w) sum += tid ? s.part3[w] : s.part2[w];
      first.sums[rank][tid] = sum;
    }
  };
  // The first block tells all the cut, or that they are not needed any more.
  auto tell = [&](u64 value, bool done) {
    if (rank == 0) {
      __syncthreads();  // (the list has been read)
      if (tid == 0) s.listed = 0;
      if (tid < C) {
        SampleShared &other = *cluster.map_shared_rank(&s, tid);
        other.cut = value;
        other.done = done;
      }
    }
    cluster.sync();
    cut = s.cut;
    return s.done != 0;
  };
  // The first block makes the rest of what it has in the list, `behind` is the weight of the others that top-p counts.
  auto finish = [&](int most, double behind) {
    const int n = s.listed;
    if (n <= 64) {
      if (warp == 0) {
        const int token = sample_short(s, z, n, most, behind, p, min_p, u);
        if (lane == 0) s.found[0] = token;
      }
      __syncthreads();
      const int token = s.found[0];
      __syncthreads();
      if (token < 0) alone();
      else if (tid == 0) a.token[b] = token;
      return;
    }
    sort_list(s.list, n);
    const int token = sample_list(s, z, min(n, most), behind, p, min_p, u);
    const bool close = s.found[1] != 0;
    __syncthreads();
    if (close) alone();
    else if (tid == 0) a.token[b] = token;
  };

  float weigh_from = INFINITY, weigh_to = INFINITY;  // (without top-p all that top-k keeps)
  bool all_listed = false;
  if (by_rank || by_mass) {
    // 2. counts of the steps: of the slice, then of the row and running
    mine([&](float x, int) {
      if (!z.counts(x)) return;
      const unsigned at = __float_as_uint(z.part_of(x)) & 0x7fffffu;
      atomicAdd(&s.count[at >> z.fine_bits], 1u);
      if (by_mass) atomicAdd(&s.into[at >> z.fine_bits], at & ((1u << z.fine_bits) - 1));
    });
    cluster.sync();
    // a block adds up its share of the steps, for all
    const int steps = SA_BINS / C, at = tid * SA_EACH;
    for (int i = tid; i < steps * (by_mass ? 2 : 1); i += SA_THREADS) {
      const bool second = i >= steps;
      const int bin = rank * steps + (second ? i - steps : i);
      unsigned v[SA_CLUSTER], sum = 0;
#pragma unroll
      for (int c = 0; c < SA_CLUSTER; ++c) {
        v[c] = 0;
        if (c < C) {
          const SampleShared &other = *cluster.map_shared_rank(&s, c);
          v[c] = second ? other.into[bin] : other.count[bin];
        }
      }
#pragma unroll
      for (int c = 0; c < SA_CLUSTER; ++c) sum += v[c];
#pragma unroll
      for (int c = 0; c < SA_CLUSTER; ++c)
        if (c < C) {
          SampleShared &other = *cluster.map_shared_rank(&s, c);
          (second ? other.all_into : other.upto)[bin] = sum;
        }
    }
    cluster.sync();
    static_assert(SA_EACH == 4, "16-byte loads of counts");
    const uint4 n4 = *reinterpret_cast<const uint4 *>(&s.upto[at]);
    const unsigned n[SA_EACH] = {n4.x, n4.y, n4.z, n4.w};
    unsigned total;
    const unsigned run = block_before(n[0] + n[1] + n[2] + n[3], s.counts, total);
    by_rank = by_rank && total > (unsigned)k;
    {
      unsigned upto = run;
#pragma unroll
      for (int e = 0; e < SA_EACH; ++e) {
        if (by_rank && (int)upto < k && (int)(upto + n[e]) >= k) s.found[2] = at + e;
        upto += n[e];
        s.upto[at + e] = upto;
      }
    }
    __syncthreads();
    if (by_rank) rank_bin = s.found[2];
    const int rank_upto = by_rank ? (int)s.upto[rank_bin] : 0, rank_before = by_rank && rank_bin ? (int)s.upto[rank_bin - 1] : 0;
    if (by_rank) {
      // 3. top-k
      const bool whole = rank_upto <= SA_LIST;
      if (!whole && rank_upto - rank_before > SA_LIST) {
        if (rank == 0) alone();
        return;
      }
      collect(whole ? 0 : rank_bin, rank_bin + 1);
      if (whole) {
        if (rank == 0) finish(k, 0);
        return;
      }
      u64 place = 0;
      if (rank == 0) {
        sort_list(s.list, s.listed);
        place = s.list[k - 1 - rank_before];
      }
      tell(place, false);
    }
    if (by_mass) {
      // top-p: bounds of the running sums at the steps' borders. A step's n entries at f_i of it (0 .. 1) weigh E 2^(-c f_i) each, E at its
      // beginning: together at least E n 2^(-c F), with F the average, and at most E n (1 - F (1 - 2^-c)). For the half a
      // part that places are rounded by, and 32-bit arithmetic here (sums of 2048 numbers, 2^-18 at most), the bounds are widened.
      const double per_step = z.inv > 0.f ? log2_unit / z.inv : 0.0;
      const float per = (float)per_step, full = exp2f(-per), wider = 1.f + 1e-5f + per / z.fine, less = fmaxf(0.f, 2.f - wider);
      float low[SA_EACH], high[SA_EACH], low_total, high_total;
#pragma unroll
      for (int e = 0; e < SA_EACH; ++e) {
        const int bin = at + e;
        const float begin = exp2f((float)(-per_step * bin));
        low[e] = high[e] = 0;
        if (n[e] && bin <= rank_bin) {
          if (bin < rank_bin) {
            const float f = __fdividef((float)s.all_into[bin], (float)n[e] * z.fine);
            high[e] = begin * n[e] * (1.f - f * (1.f - full)) * wider;
            low[e] = begin * n[e] * exp2f(-per * (f + 1.f / z.fine)) * less;
          } else {  // only the first ones of the step
            high[e] = begin * (k - rank_before) * wider;
            low[e] = begin * (k - rank_before) * full * less;
          }
          if (z.inv == 0.f) low[e] = 0;  // (no steps: equal entries, or a range that floats do not hold)
        }
      }
      float high_run = block_before(high[0] + high[1] + high[2] + high[3], s.narrow, high_total);
      float low_run = block_before(low[0] + low[1] + low[2] + low[3], s.narrow2, low_total);
      const float reach_high = (float)p * high_total * 1.00001f, reach_low = (float)p * low_total * 0.99999f;
      // can: the first step at whose end the sum can have reached p of the total; must: the first at whose end it has to have
      unsigned can = SA_BINS - 1, must = SA_BINS - 1;
#pragma unroll
      for (int e = 0; e < SA_EACH; ++e) {
        high_run += high[e];
        low_run += low[e];
        if (can == SA_BINS - 1 && high_run >= reach_low) can = at + e;
        if (must == SA_BINS - 1 && low_run >= reach_high) must = at + e;
      }
      const u64 both = block_all((u64)can << 32 | must, s.wide, [](u64 x, u64 y) { return min(x >> 32, y >> 32) << 32 | min((unsigned)x, (unsigned)y); });
      can = (unsigned)(both >> 32);
      must = (unsigned)both;
      int most = (int)s.upto[must], least = can ? (int)s.upto[can - 1] : 0;
      if (by_rank) {
        most = min(most, k);
        least = min(least, k);
      }
      const bool whole = most <= SA_LIST / 4;  // (a longer list is sorted in more time than it saves)
      if (!whole && most - least > SA_LIST) {
        if (rank == 0) alone();
        return;
      }
      all_listed = whole;
      weigh_from = whole ? 0.f : (float)can;
      weigh_to = (float)must + 1.f;
    }
  }
  weigh(weigh_from, weigh_to);
  if (by_mass) {
    cluster.sync();
    if (all_listed) {
      if (rank == 0) {
        double behind = 0;
        for (int c = 0; c < C; ++c) behind += s.sums[c][1];
        finish(SA_LIST, behind);
      }
      return;
    }
    const int at = tid * SA_EACH;
    u64 place = cut;
    bool close = false;
    if (rank == 0 && s.listed > 0) {
      const int length = s.listed;
      double in_front = 0, behind = 0, w[SA_EACH], sum = 0, between;
      for (int c = 0; c < C; ++c) {
        in_front += s.sums[c][0];
        behind += s.sums[c][1];
      }
      sort_list(s.list, length);
#pragma unroll
      for (int e = 0; e < SA_EACH; ++e) {
        w[e] = at + e < length ? z.weight(logit_of((uint32_t)(s.list[at + e] >> 32)), s.table) : 0.0;
        sum += w[e];
      }
      double before = in_front + block_before(sum, s.part2, between);
      const double all = in_front + between + behind, mass = p * all;
      bool near = false;
      unsigned last = 0;
#pragma unroll
      for (int e = 0; e < SA_EACH; ++e) {
        if (at + e < length && at + e > 0) {
          near |= fabs(before - mass) <= z.close * all;
          if (before < mass) last = at + e;
        }
        before += w[e];
      }
      const u64 found = block_all((u64)near << 32 | last, s.wide, [](u64 x, u64 y) { return max(x >> 32, y >> 32) << 32 | max((unsigned)x, (unsigned)y); });
      close = (found >> 32) != 0;
      place = s.list[(unsigned)found];
    }
    if (tell(place, close)) {
      if (rank == 0) alone();
      return;
    }
    // the block's own entries between the bounds, as far as they are kept, join their warps' sums
    for (int i = tid; i < s.own; i += SA_THREADS) {
      const int j = s.owned[i];
      const float x = to_f(entries[j]);
      if (place_of(order_of(x), j) < cut) continue;
      const double w = z.weight(x, s.table);
      if (!by_min || enough(x, w)) atomicAdd(&s.part[(j - from) / share], w);
    }
    __syncthreads();
  }

  // 4. the sums of what is kept, in index order
  __syncthreads();
  double sum = 0;
  for (int w = 0; w < SA_WARPS; ++w) sum += s.part[w];
  if (tid < C) cluster.map_shared_rank(&s, tid)->kept[rank] = sum;
  cluster.sync();
  double total = 0, before = 0, in_front = 0;
  for (int c = 0; c < C; ++c) total += s.kept[c];
  const double target = u * total;
  int owner = C, last = 0;
  for (int c = 0; c < C; ++c) {
    if (s.kept[c] > 0) last = c;
    if (owner == C && before + s.kept[c] > target) {
      owner = c;
      in_front = before;
    }
    before += s.kept[c];
  }
  if (owner == C) {  // (rounding: the last entry that is kept)
    owner = last;
    in_front = before;
  }
  if (rank != owner) return;
  const int token = r.locate(entries, from, to, share, in_front, target, total, [&](float x, int i) -> double {
    if (!z.counts(x) || place_of(order_of(x), i) < cut) return 0.0;
    const double w = z.weight(x, s.table);
    return !by_min || enough(x, w) ? w : 0.0;
  });
  const bool close = s.found[1] != 0;
  __syncthreads();
  if (close) alone();
  else if (tid == 0) a.token[b] = token;
}

// Blocks of a row: as many as are resident at once with B rows, two to a multiprocessor (clusters stay inside a group of multiprocessors, so
// fewer of the larger ones fit), but not so few that a slice finds no room beside another one. Slices that find none are read from L2
// in every sweep. (256 rows of 50272 entries: 88 us with four blocks per row in four waves, 134 with one block per row and L2; 80 by now.)
template <typename T>
static cudaError_t launch_sample(const SampleArgs &a, int B, bool vec, cudaStream_t st) {
  constexpr int N = Chunk<T>::N, fixed = ((int)sizeof(SampleShared) + 15) / 16 * 16, most = 200 * 1024, beside = 112 * 1024;
  static DevicePrep prep;
  const int(*resident)[4];
  cudaError_t e = prep.get(
      [&](int(&clusters)[4]) {
        cudaError_t f = cluster_residency(sample_kernel<T, true>, SA_THREADS, beside, 2, clusters);
        if (f == cudaSuccess) f = cudaFuncSetAttribute(sample_kernel<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        return f != cudaSuccess ? f : cudaFuncSetAttribute(sample_kernel<T, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
      },
      resident);
  if (e != cudaSuccess) return e;
  int log = 3;
  static_assert(SA_CLUSTER == 8, "clusters of up to 2^3 blocks");
  while (log > 0 && (a.V >> log < 512 || (B > (*resident)[log] && (long long)(a.V >> log) * 2 * (int)sizeof(T) <= beside - fixed))) --log;
  const int C = 1 << log, slice = ceil_div(ceil_div(a.V, C), N) * N;
  const int room = ((long long)B * C <= sm_count() ? most : beside) - fixed;
  const bool stored = (long long)slice * (int)sizeof(T) <= room;
  const int smem = fixed + (stored ? slice * (int)sizeof(T) : 0);
  return djv::launch_kernel_cluster(vec ? sample_kernel<T, true> : sample_kernel<T, false>, dim3(B * C), dim3(SA_THREADS), smem, st, dim3(C, 1, 1),
                                    a, slice, (int)stored);
}

static double double_of(long long bits) {
  double v;
  memcpy(&v, &bits, sizeof(v));
  return v;
}

}  // namespace djv

using namespace djv;

extern "C" int djv_sample(int dtype, long long *token, const void *logits, long long ld, const float *u, const float *temperature,
                          long long temperature_bits, const int32_t *top_k, int top_k_all, const float *top_p, long long top_p_bits,
                          const float *min_p, long long min_p_bits, int B, int V, void *stream) {
  DJV_REQUIRE(is_dtype(dtype), "sample: dtype %d", dtype);
  DJV_REQUIRE(token && logits && u, "sample: null pointer");
  DJV_REQUIRE(B >= 0 && B <= (1 << 27) && V >= 1 && V <= (1 << 30) && ld >= V, "sample: B=%d V=%d ld=%lld", B, V, ld);
  const SampleArgs a{token, logits, ld, u, temperature, double_of(temperature_bits), top_k, top_k_all, top_p, double_of(top_p_bits),
                     min_p, double_of(min_p_bits), V};
  DJV_REQUIRE((temperature || (a.temperature0 >= 0 && a.temperature0 < 1e30)) && (top_k || top_k_all >= 0) && (top_p || a.top_p0 >= 0) &&
                  (min_p || (a.min_p0 >= 0 && a.min_p0 <= 1)),
              "sample: temperature %g, top_k %d, top_p %g, min_p %g", a.temperature0, top_k_all, a.top_p0, a.min_p0);
  if (B == 0) return DJV_OK;
  const bool vec = aligned16(logits) && ld % (16 / (int)dtype_bytes(dtype)) == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == DJV_DTYPE_F16    ? launch_sample<__half>(a, B, vec, st)
                        : dtype == DJV_DTYPE_BF16 ? launch_sample<bf16>(a, B, vec, st)
                                                  : launch_sample<float>(a, B, vec, st);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_error("sample: CUDA error %d (%s)", (int)e, cudaGetErrorString(e));
    return DJV_ERR_CUDA;
  }
  count_launch();
  return check_launch("sample");
}
