// The next token of every row of logits from a given random number (ah_sample, include/alpha_hip.h).
//
// A workgroup to a row.  Every question asked of a row (which is the k-th largest, where does a mass end, which token does the number fall on) is
// "the first, from the largest down, at which a running sum passes a number", and is answered by descending into bins of the logit: the masses (or
// counts) of 2048 bins between the row's bounds are added up in LDS, the bin that holds the answer is found by a scan, and its members are
// gathered, sorted and scanned; if they are too many, the bin is cut again between its own bounds, and if they are all equal the answer is one of them by
// index.  Where no nucleus is asked for the walk is by index: sums of runs of 64 vectors, a scan over those, and the one run again.
// With a small top_k all of that happens in the list of the few candidates that the threads' maxima leave.
//
// Weights are whole numbers of 2^-43 of the largest, so sums are exact and the same in every order.  2^(y/256) for whole y is read from a table, the
// rest is e^g with |g| <= 2^-9.5: 1 + g + g^2 (1/2 + g/6 + g^2/24), the parentheses in 32 bits (2^-43 of the result), all else in 64.
#include "common.h"

using namespace ah;

namespace {

struct SampleArgs {
  const void *logits;
  const float *temperature, *top_p, *min_p, *uniform;
  const int32_t *top_k;
  int32_t *tokens;
  float *logprobs;
  int64_t ld;
  int32_t vocab;
};

constexpr int THREADS = 512, WAVES = THREADS / 64, BINS = 2048, LIST = 2048, EACH = LIST / THREADS, STEPS = 256;
static_assert(BINS == LIST, "EACH bins, or entries, to a thread");
constexpr int MAX_VOCAB = 1 << 20;              // sums of as many weights of 2^43 stay below 2^63
constexpr double UNIT = 0x1p43;
constexpr int FEW = THREADS / 2;                 // a top_k up to this goes through the threads' maxima, which leave about k candidates

// f32 -> whole numbers of the same order, -0 as 0; back
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float of_order(uint32_t o) { return __uint_as_float((o >> 31) ? o ^ 0x80000000u : ~o); }
// a list's entries: the larger logit first, then the lower index
__device__ __forceinline__ uint64_t entry_of(float l, int index) { return (uint64_t)order_of(l) << 32 | (0xffffffffu - (uint32_t)index); }
__device__ __forceinline__ float entry_logit(uint64_t e) { return of_order((uint32_t)(e >> 32)); }
__device__ __forceinline__ int entry_index(uint64_t e) { return (int)(0xffffffffu - (uint32_t)e); }

constexpr int RUNS = MAX_VOCAB / 256 + 1;         // (one more where a row begins inside a vector)

struct Shared {
  uint64_t bins[2][BINS];                        // running sums, of the row's own bins and of a bin's bins
  uint64_t list[LIST], sorted[LIST];
  uint64_t runs[RUNS];                           // sums of 64 vectors of four (or eight) logits
  double   steps[STEPS];                         // 2^(i / 256)
  uint64_t part[WAVES];
  float    low[WAVES], high[WAVES];
  uint64_t found_before;
  int      found, listed;
};
static_assert(sizeof(Shared) <= 160 * 1024, "a workgroup's LDS");

// ------------------------------------------------------------------------------------------ a workgroup's sums
// What every lane has read from the same place, told the compiler: branches on it, with barriers behind them, are branches of the whole wave.
__device__ __forceinline__ int same(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ float same(float v) { return __uint_as_float((uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(v))); }
__device__ __forceinline__ uint64_t same(uint64_t v) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
}
__device__ __forceinline__ uint64_t wave_running(uint64_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) { const uint64_t x = __shfl_up(v, o); v += lane >= o ? x : 0; }
  return v;
}
// the sum over the threads before this one, and over all
__device__ __forceinline__ uint64_t block_before(uint64_t v, Shared &s, uint64_t &all) {
  const int wave = threadIdx.x >> 6;
  const uint64_t upto = wave_running(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) s.part[wave] = upto;
  __syncthreads();
  uint64_t before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; w++) { const uint64_t x = s.part[w]; all += x; before += w < wave ? x : 0; }
  all = same(all);
  return before + upto - v;
}
__device__ __forceinline__ uint64_t block_sum(uint64_t v, Shared &s) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.part[threadIdx.x >> 6] = v;
  __syncthreads();
  uint64_t all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; w++) all += s.part[w];
  return same(all);
}
__device__ __forceinline__ void block_bounds(float &low, float &high, Shared &s) {
  low = -wave_max(-low);
  high = wave_max(high);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) { s.low[threadIdx.x >> 6] = low; s.high[threadIdx.x >> 6] = high; }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; w++) { low = fminf(low, s.low[w]); high = fmaxf(high, s.high[w]); }
  low = same(low);
  high = same(high);
}

// The first n entries of `list` in order, into `sorted`.  Up to 256 by counting the larger ones of each, 2 to 8 threads to an entry; more by exchanges,
// whose steps between neighbours of 128 need no barrier.
__device__ __forceinline__ void sort_list(Shared &s, int n) {
  const int t = threadIdx.x;
  __syncthreads();
  if (n <= THREADS / 2) {
    const int shift = n <= THREADS / 8 ? 3 : n <= THREADS / 4 ? 2 : 1, i = t >> shift;
    const uint64_t mine = i < n ? s.list[i] : 0;
    uint32_t larger = 0;
    for (int j = t & ((1 << shift) - 1); j < n; j += 1 << shift) larger += s.list[j] > mine;
    larger += lane_xor<1>(larger);
    if (shift > 1) larger += lane_xor<2>(larger);
    if (shift > 2) larger += lane_xor<4>(larger);
    if (i < n && (t & ((1 << shift) - 1)) == 0) s.sorted[larger] = mine;
  } else {
    int size = THREADS;
    while (size < n) size <<= 1;
    for (int i = t; i < size; i += THREADS) s.sorted[i] = i < n ? s.list[i] : 0;
    __syncthreads();
    for (int run = 2; run <= size; run <<= 1)
      for (int apart = run >> 1; apart; apart >>= 1) {
        for (int q = t; q < size / 2; q += THREADS) {
          const int i = 2 * q - (q & (apart - 1)), j = i + apart;
          const uint64_t x = s.sorted[i], y = s.sorted[j];
          if ((x < y) == ((i & run) == 0)) { s.sorted[i] = y; s.sorted[j] = x; }
        }
        if (apart > 64 || (apart == 1 && run > 64)) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      }
  }
  __syncthreads();
}

// ------------------------------------------------------------------------------------------ a row
struct Past {                                    // a running sum, on from `base`, passes a number or reaches it
  double target;
  bool   reach;
  uint64_t base = 0;
  __device__ __forceinline__ bool operator()(uint64_t s) const { const double x = (double)(base + s); return reach ? x >= target : x > target; }
};

template <class T> struct Row {
  static constexpr int N = 16 / sizeof(T);       // logits to a vector
  const T *x;                                    // of the first vector, at or before the row's first logit
  int lead, V, vectors;
  __device__ __forceinline__ Row(const T *row, int vocab) {
    lead = (int)((uintptr_t)row % 16 / sizeof(T));
    x = row - lead;
    V = vocab;
    vectors = (lead + V + N - 1) / N;
  }
  __device__ __forceinline__ int index(int v, int i) const { return v * N + i - lead; }
  __device__ __forceinline__ float at(int index) const { return Io<T>::ld(x, (size_t)(index + lead)); }
  // vector v as it is stored; what is not the row's is not read, and NaN
  __device__ __forceinline__ uint4 load(int v) const {
    uint4 w = make_uint4(~0u, ~0u, ~0u, ~0u);
    if (v > 0 && v < vectors - 1) w = *reinterpret_cast<const uint4 *>(x + (int64_t)v * N);
    else if (v < vectors) {
      uint32_t u[4] = {~0u, ~0u, ~0u, ~0u};
#pragma unroll
      for (int i = 0; i < N; i++) {
        const bool in = index(v, i) >= 0 && index(v, i) < V;
        if (in) {
          if constexpr (N == 4) u[i] = __float_as_uint(at(index(v, i)));
          else {
            const uint32_t half = __float_as_uint(at(index(v, i))) >> 16;
            u[i / 2] = i & 1 ? (u[i / 2] & 0xffffu) | half << 16 : (u[i / 2] & 0xffff0000u) | half;
          }
        }
      }
      w = make_uint4(u[0], u[1], u[2], u[3]);
    }
    return w;
  }
  static __device__ __forceinline__ float logit(const uint4 &w, int i) {
    const uint32_t u = (N == 4 ? i : i / 2) == 0 ? w.x : (N == 4 ? i : i / 2) == 1 ? w.y : (N == 4 ? i : i / 2) == 2 ? w.z : w.w;
    return N == 4 ? __uint_as_float(u) : __uint_as_float(i & 1 ? u & 0xffff0000u : u << 16);
  }
  // f(vector, its number) for all of them, U loads under way at a time
  template <int U, class F>
  __device__ __forceinline__ void each(F f) const {
    for (int v0 = threadIdx.x; v0 < vectors; v0 += THREADS * U) {
      uint4 w[U];
#pragma unroll
      for (int j = 0; j < U; j++) w[j] = load(v0 + j * THREADS);
#pragma unroll
      for (int j = 0; j < U; j++) if (v0 + j * THREADS < vectors) f(w[j], v0 + j * THREADS);
    }
  }
  // f(logit, index) for the ones above -infinity for which `hit` holds, which are few: the loop over them is there once
  template <class Hit, class F>
  __device__ __forceinline__ void hits(Hit hit, F f) const {
    constexpr int U = 4;
    for (int v0 = threadIdx.x; v0 < vectors; v0 += THREADS * U) {
      uint4 w[U];
#pragma unroll
      for (int j = 0; j < U; j++) w[j] = load(v0 + j * THREADS);
      uint32_t bits = 0;
#pragma unroll
      for (int j = 0; j < U; j++)
#pragma unroll
        for (int i = 0; i < N; i++) { const float l = logit(w[j], i); bits |= l > -INFINITY && hit(l) ? 1u << (j * N + i) : 0u; }
      while (bits) {
        const int b = __builtin_ctz(bits);
        const int n = index(v0 + b / N * THREADS, b % N);
        f(at(n), n);
        bits &= bits - 1;
      }
    }
  }
};

// weights against `top` at a temperature, as whole numbers; or 1 each
struct Weight {
  float top;
  double factor;                                 // 256 log2(e) / temperature
  const double *steps;
  bool one;
  __device__ __forceinline__ uint64_t operator()(float l) const {
    const double y = ((double)l - (double)top) * factor;
    const bool some = y > -44.0 * STEPS;         // (NaN: both are infinite)
    constexpr double ROUND = 0x1.8p52;
    const double whole = y + ROUND;
    const int n = (int)(uint32_t)__builtin_bit_cast(uint64_t, whole);
    const double g = (y - (whole - ROUND)) * (0.693147180559945309417 / STEPS);
    const float h = (float)g;
    const double e = fma(g * g, (double)fmaf(h, fmaf(h, 1.0f / 24, 1.0f / 6), 0.5f), g);
    const double step = steps[n & (STEPS - 1)], w = fma(step, e, step);
    const uint64_t scaled = __builtin_bit_cast(uint64_t, w) + ((uint64_t)(int64_t)((n >> 8) + 43) << 52);
    const uint64_t units = __builtin_bit_cast(uint64_t, __builtin_bit_cast(double, scaled) + 0x1p52) - __builtin_bit_cast(uint64_t, 0x1p52);
    const uint64_t weight = some ? units : l == top ? (uint64_t)UNIT : 0;
    return one ? 1 : weight;
  }
};

// Which of the bins between `high` and `low` a logit falls into: never an earlier one for a smaller logit.  A row's own bins are of one width, over `most`
// at most; those of a bin are of one number of floats, so that they end as single ones whatever the logits are.
struct Bins {
  float high, scale;
  int   shift;                                   // -1: of one width
  __device__ __forceinline__ Bins(float low, float high_, float most) : high(high_), shift(-1) {
    const float range = fminf(high_ - low, most);
    scale = range > 0.f && range < INFINITY ? fminf((BINS - 1) / range, 3.402823466e38f) : 0.f;
  }
  __device__ __forceinline__ Bins(float low, float high_) : high(high_), scale(0.f) {
    const uint32_t range = order_of(high_) - order_of(low);
    shift = max(0, 32 - __clz((int)range) - 11);
  }
  __device__ __forceinline__ int operator()(float l) const {
    if (shift >= 0) return min((int)((order_of(high) - order_of(l)) >> shift), BINS - 1);
    const float at = (high - l) * scale;
    return at < (float)(BINS - 1) ? (int)at : BINS - 1;       // (0 x infinity: the last)
  }
};
static_assert(BINS == 1 << 11, "the shift of a bin's bins");

// s.bins[level] to running sums; the sum of all
__device__ __forceinline__ uint64_t sum_bins(Shared &s, int level) {
  uint64_t x[EACH], sum = 0, all;
#pragma unroll
  for (int i = 0; i < EACH; i++) { x[i] = s.bins[level][EACH * threadIdx.x + i]; sum += x[i]; }
  uint64_t upto = block_before(sum, s, all);
#pragma unroll
  for (int i = 0; i < EACH; i++) { upto += x[i]; s.bins[level][EACH * threadIdx.x + i] = upto; }
  __syncthreads();
  return all;
}
// Where in s.bins[level] a running sum, on from `base`, passes: the bin into s.found, the sum before it into s.found_before.
__device__ __forceinline__ void find_bin(Shared &s, int level, uint64_t base, const Past &past) {
#pragma unroll
  for (int i = 0; i < EACH; i++) {
    const int b = EACH * threadIdx.x + i;
    const uint64_t before = base + (b ? s.bins[level][b - 1] : 0);
    if (!past(before) && past(base + s.bins[level][b])) { s.found = b; s.found_before = before; }
  }
  __syncthreads();
}

struct Found {
  float    logit;
  int      index;                                // -1: one of several equal ones, whose running sums go on from `before`
  uint64_t upto, before;                         // the running sums with it and, of equal ones, without any of them
};

template <class T>
__global__ __launch_bounds__(THREADS) void k_sample(SampleArgs a) {
  constexpr int N = Row<T>::N;
  __shared__ Shared s;
  const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
  const int64_t r = blockIdx.x;
  const Row<T> row((const T *)a.logits + r * a.ld, a.vocab);
  const float temperature = a.temperature ? a.temperature[r] : 1.f;
  const int k = a.top_k ? a.top_k[r] : 0;
  const float p = a.top_p ? a.top_p[r] : 0.f, least_p = a.min_p ? a.min_p[r] : 0.f, u = a.uniform[r];
  auto answer = [&](int token, float logprob) {
    if (t == 0) { a.tokens[r] = token; if (a.logprobs) a.logprobs[r] = logprob; }
  };
  float top = -INFINITY, low = INFINITY;         // this thread's, then the row's
  if (!(temperature > 0.f)) {
    int first = 0;
    row.template each<4>([&](const uint4 &w, int v) {
#pragma unroll
      for (int i = 0; i < N; i++) { const float l = Row<T>::logit(w, i); const bool more = l > top; top = more ? l : top; first = more ? row.index(v, i) : first; }
    });
    // the larger, then the lower index: the largest entry
    uint64_t best = top > -INFINITY ? entry_of(top, first) : 0;
#pragma unroll
    for (int o = 32; o; o >>= 1) { const uint64_t x = __shfl_xor(best, o); best = x > best ? x : best; }
    if (lane == 0) s.part[wave] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; w++) best = s.part[w] > best ? s.part[w] : best;
    answer(best ? entry_index(best) : 0, best ? 0.f : NAN);
    return;
  }
  if (t < STEPS) s.steps[t] = exp2((double)t / STEPS);
  if (t == 0) s.found = 0;
  row.template each<4>([&](const uint4 &w, int) {
#pragma unroll
    for (int i = 0; i < N; i++) { const float l = Row<T>::logit(w, i); top = fmaxf(top, l); low = l > -INFINITY ? fminf(low, l) : low; }
  });
  const float mine = top;
  block_bounds(low, top, s);
  if (top == -INFINITY) { answer(0, NAN); return; }

  Weight weight{top, STEPS * 1.44269504088896340736 / (double)temperature, s.steps, false};
  const bool nucleus = p > 0.f && p < 1.f;
  // a weight of at least min_p
  const double drop = least_p > 0.f && temperature < INFINITY ? (double)temperature * log((double)fminf(least_p, 1.f)) : -INFINITY;
  auto enough = [&](float l) { return l == top || (double)l - (double)top >= drop; };
  const double draw = fmin(fmax((double)u, 0.0), 1.0);
  auto finish = [&](float l, int token, uint64_t all) {
    answer(token, (float)((l == top ? 0.0 : ((double)l - (double)top) / (double)temperature) - log((double)all / UNIT)));
  };
  // the number that the walk has to pass: where rounding, or a number of 1, leaves nothing beyond it, the last that weighs something
  auto walk = [&](uint64_t all) { const double target = draw * (double)all; return (double)all > target ? Past{target, false} : Past{(double)all, true}; };
  auto list = [&](float l, int index) {
    const int at = atomicAdd(&s.listed, 1);
    if (at < LIST) s.list[at] = entry_of(l, index);
  };

  const bool cut = k > 0 && k < row.V;
  if (cut && k <= FEW) {
    // At least k logits are in the bins (of the threads' maxima) up to the one in which the k-th largest of the maxima lies: those are the candidates.
    float lowest = mine > -INFINITY ? mine : INFINITY, dummy = mine;
    block_bounds(lowest, dummy, s);
    const Bins bin(lowest, top, INFINITY);
    for (int i = t; i < BINS; i += THREADS) s.bins[0][i] = 0;
    __syncthreads();
    if (mine > -INFINITY) atomicAdd((unsigned long long *)&s.bins[0][bin(mine)], 1ull);
    if (t == 0) { s.listed = 0; s.found = BINS - 1; }
    __syncthreads();
    const bool every = sum_bins(s, 0) < (uint64_t)k;               // fewer maxima than that: all of the row are candidates
    find_bin(s, 0, 0, Past{(double)k, true});
    const int last = every ? BINS - 1 : same(s.found);
    row.hits([&](float l) { return bin(l) <= last; }, list);
    __syncthreads();
    const int n = same(s.listed);
    if (n <= LIST) {
      sort_list(s, n);
      const uint32_t kth = n > k ? (uint32_t)(same(s.sorted[k - 1]) >> 32) : 0u;
      uint64_t e[EACH], w[EACH], sum = 0, all;
#pragma unroll
      for (int i = 0; i < EACH; i++) {
        const int at = EACH * t + i;
        e[i] = at < n ? s.sorted[at] : 0;
        const uint64_t x = weight(entry_logit(e[i]));
        w[i] = at < n && (uint32_t)(e[i] >> 32) >= kth ? x : 0;
        sum += w[i];
      }
      uint64_t before = block_before(sum, s, all);
      const Past end{nucleus ? (double)p * (double)all : INFINITY, true};
      uint64_t number = 0;
      sum = 0;
#pragma unroll
      for (int i = 0; i < EACH; i++) {
        const bool stays = !end(before) && enough(entry_logit(e[i]));
        before += w[i];
        w[i] = stays ? w[i] : 0;
        number += w[i] != 0;
      }
      if (!nucleus) {                            // by index: the list again with the index first and the place in the order behind it
        uint64_t at = block_before(number, s, number);
#pragma unroll
        for (int i = 0; i < EACH; i++) {
          if (w[i]) s.list[at++] = (uint64_t)(uint32_t)e[i] << 32 | (uint32_t)(EACH * t + i);
          s.bins[0][EACH * t + i] = e[i];        // (what was sorted by logit is needed once more)
          s.bins[1][EACH * t + i] = w[i];
        }
        sort_list(s, (int)number);
#pragma unroll
        for (int i = 0; i < EACH; i++) {
          const int j = EACH * t + i;
          const uint32_t place = j < (int)number ? (uint32_t)s.sorted[j] : 0u;
          e[i] = s.bins[0][place];
          w[i] = j < (int)number ? s.bins[1][place] : 0;
        }
      }
#pragma unroll
      for (int i = 0; i < EACH; i++) sum += w[i];
      before = block_before(sum, s, all);
      const Past past = walk(all);
#pragma unroll
      for (int i = 0; i < EACH; i++) {
        if (!past(before) && past(before + w[i])) s.found_before = e[i];
        before += w[i];
      }
      __syncthreads();
      const uint64_t drawn = same(s.found_before);
      finish(entry_logit(drawn), entry_index(drawn), all);
      return;
    }
  }

  // Descents, from the largest down: to the k-th largest, to where the nucleus ends, to the token.
  float bound = low;                             // what top_k leaves is not below it
  uint64_t all = 0;
  Past past{0.0, true};
  Found f{top, 0, 0, 0};
  enum { KTH, END, TOKEN, NONE };
  int goal = cut ? KTH : nucleus ? END : NONE;
  Bins bin(low, top, INFINITY);
  for (int turn = 0; turn < 3 && goal != NONE; turn++) {
    float least = bound, most = top;
    // (a row's own bins and at most three times those of a bin: 2^32 floats are 2^11 times 2^21, 2^10, 1.  Both loops are bounded whatever the sums are, and
    // every wave takes the same turns: all of them read what decides from the same places between the same two barriers.)
    uint64_t base = 0, of_enough = 0;
    for (int level = 0; level < 5; level++) {
      const int l1 = level ? 1 : 0;
      if (level || goal != TOKEN) {              // (the token's are those of the nucleus)
        weight.one = goal == KTH;
        bin = level ? Bins(least, most) : Bins(bound, top, goal == KTH ? INFINITY : 31.f * temperature);
        __syncthreads();
        for (int i = t; i < BINS; i += THREADS) s.bins[l1][i] = 0;
        __syncthreads();
        uint64_t sum = 0;
        row.template each<2>([&](const uint4 &w, int) {
#pragma unroll
          for (int i = 0; i < N; i++) {
            const float l = Row<T>::logit(w, i);
            if (l >= least && l <= most) {       // (not NaN, and above -infinity like those)
              const uint64_t x = weight(l);
              sum += enough(l) ? x : 0;
              if (x) atomicAdd((unsigned long long *)&s.bins[l1][bin(l)], (unsigned long long)x);
            }
          }
        });
        __syncthreads();
        const uint64_t total = sum_bins(s, l1);
        if (!level) {
          if (goal == KTH && total <= (uint64_t)k) break;            // nothing to cut: f is the largest, set right below
          past = Past{goal == KTH ? (double)k : (double)p * (double)total, true};
          of_enough = block_sum(sum, s);
        }
      }
      __syncthreads();
      if (t == 0) s.listed = 0;
      find_bin(s, l1, base, past);
      const int b = same(s.found);
      base = same(s.found_before);
      float lo = INFINITY, hi = -INFINITY;
      row.hits([&](float l) { return l >= least && l <= most && bin(l) == b; }, [&](float l, int index) {
        lo = fminf(lo, l);
        hi = fmaxf(hi, l);
        list(l, index);
      });
      block_bounds(lo, hi, s);
      const int n = same(s.listed);
      if (n <= LIST) {
        sort_list(s, n);
        uint64_t w[EACH], sum = 0, dummy;
#pragma unroll
        for (int i = 0; i < EACH; i++) {
          const int e = EACH * t + i;
          const uint64_t x = weight(entry_logit(e < n ? s.sorted[e] : 0));
          w[i] = e < n ? x : 0;
          sum += w[i];
        }
        uint64_t before = base + block_before(sum, s, dummy);
#pragma unroll
        for (int i = 0; i < EACH; i++) {
          if (!past(before) && past(before + w[i])) { s.found = EACH * t + i; s.found_before = before + w[i]; }
          before += w[i];
        }
        __syncthreads();
        const uint64_t e = same(s.sorted[same(s.found)]);
        f = Found{entry_logit(e), entry_index(e), same(s.found_before), 0};
        break;
      }
      if (lo == hi) {                            // equal ones: how many of them it takes
        const uint64_t w = same(weight(lo));
        uint32_t few = 1, many = (uint32_t)n;
        for (int i = 0; i < 20 && few < many; i++) {
          const uint32_t middle = few + (many - few) / 2;
          if (past(base + middle * w)) many = middle; else few = middle + 1;
        }
        f = Found{lo, -1, base + few * w, base};
        break;
      }
      least = lo;
      most = hi;
    }
    if (goal == KTH) {
      bound = past.target > 0.0 ? f.logit : low;
      past = Past{0.0, true};
      goal = nucleus ? END : NONE;
    } else if (goal == END) {
      all = enough(f.logit) ? f.upto : of_enough;
      past = walk(all);
      bin = Bins(bound, top, 31.f * temperature);
      goal = TOKEN;
    } else goal = NONE;
  }
  weight.one = false;
  if (nucleus && f.index >= 0) { finish(f.logit, f.index, all); return; }

  // By index: all that is kept where there is no nucleus, or the equal ones among which the token is.
  const bool equal = nucleus;
  const float from = equal ? f.logit : bound, to = equal ? f.logit : top;
  auto term = [&](float l) {
    const uint64_t x = weight(l);
    return l >= from && l <= to && enough(l) ? x : 0;
  };
  const int runs = (row.vectors + 63) / 64;
  __syncthreads();
  for (int n0 = wave; n0 < runs; n0 += 2 * WAVES) {
    uint4 w[2];
#pragma unroll
    for (int j = 0; j < 2; j++) w[j] = row.load((n0 + j * WAVES) * 64 + lane);
#pragma unroll
    for (int j = 0; j < 2; j++) {
      uint64_t sum = 0;
#pragma unroll
      for (int i = 0; i < N; i++) {
        const float l = Row<T>::logit(w[j], i);
        if (l >= from && l <= to && enough(l)) sum += weight(l);
      }
#pragma unroll
      for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
      if (lane == 0 && n0 + j * WAVES < runs) s.runs[n0 + j * WAVES] = sum;
    }
  }
  __syncthreads();
  const int each = (runs + THREADS - 1) / THREADS, r0 = t * each;
  uint64_t sum = 0, total;
  for (int i = 0; i < each; i++) sum += r0 + i < runs ? s.runs[r0 + i] : 0;
  uint64_t before = block_before(sum, s, total);
  if (equal) past.base = f.before;
  else {
    all = total;
    past = walk(all);
  }
  for (int i = 0; i < each; i++) {
    const uint64_t x = r0 + i < runs ? s.runs[r0 + i] : 0;
    if (!past(before) && past(before + x)) { s.found = r0 + i; s.found_before = before; }
    before += x;
  }
  __syncthreads();
  if (wave == 0) {                               // the run again
    const int v = same(s.found) * 64 + lane;
    const uint4 w = row.load(v);
    uint64_t x[N], mass = 0;
#pragma unroll
    for (int i = 0; i < N; i++) { x[i] = term(Row<T>::logit(w, i)); mass += x[i]; }
    uint64_t upto = s.found_before + wave_running(mass) - mass;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const bool here = !past(upto) && past(upto + x[i]);
      upto += x[i];
      if (here) {
        const int token = row.index(v, i);
        const float l = Row<T>::logit(w, i);
        a.tokens[r] = token;
        if (a.logprobs) a.logprobs[r] = (float)((l == top ? 0.0 : ((double)l - (double)top) / (double)temperature) - log((double)all / UNIT));
      }
    }
  }
}

}  // namespace

extern "C" int32_t ah_sample(const AhSample *d) {
  AH_ARG(d, "ah_sample: null argument");
  AH_ARG(d->dtype == AH_F32 || d->dtype == AH_BF16, "ah_sample: logits of f32 or bf16, got dtype %d", d->dtype);
  AH_ARG(d->vocab >= 1 && d->vocab <= MAX_VOCAB, "ah_sample: a vocabulary of %d is outside 1 .. %d", d->vocab, MAX_VOCAB);
  AH_ARG(d->rows >= 0 && d->rows <= INT32_MAX && d->ld >= d->vocab, "ah_sample: %lld rows of %d, %lld apart", (long long)d->rows, d->vocab, (long long)d->ld);
  AH_ARG(d->rows == 0 || (d->logits && d->uniform && d->tokens), "ah_sample: logits, uniform or tokens is null");
  AH_ARG(d->logits % (d->dtype == AH_F32 ? 4 : 2) == 0 && d->temperature % 4 == 0 && d->top_k % 4 == 0 && d->top_p % 4 == 0 && d->min_p % 4 == 0 &&
             d->uniform % 4 == 0 && d->tokens % 4 == 0 && d->logprobs % 4 == 0, "ah_sample: an address that is no multiple of its element's size");
  AH_REQUIRE_READY();
  if (d->rows == 0) return AH_OK;
  const SampleArgs a{dp<void>(d->logits), dp<float>(d->temperature), dp<float>(d->top_p), dp<float>(d->min_p), dp<float>(d->uniform), dp<int32_t>(d->top_k),
                     dp<int32_t>(d->tokens), dp<float>(d->logprobs), d->ld, d->vocab};
  launch_kernel(d->dtype == AH_F32 ? k_sample<float> : k_sample<uint16_t>, dim3((unsigned)d->rows), dim3(THREADS), 0, a);
  AH_LAUNCH_CHECK();
  return AH_OK;
}
