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

// (512 threads: with 1024 the 128 registers that each then has do not hold a row's state)
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
struct Found { float logit; int index; uint64_t upto; };     // upto: the running sum with it

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
  // vector v, NaN for what is not the row's (which is not read)
  __device__ __forceinline__ void load(int v, float (&l)[N]) const {
    if (v > 0 && v < vectors - 1) {
      const uint4 w = *reinterpret_cast<const uint4 *>(x + (int64_t)v * N);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < N; i++) l[i] = N == 4 ? __uint_as_float(u[i]) : __uint_as_float(i & 1 ? u[i / 2] & 0xffff0000u : u[i / 2] << 16);
    } else {
#pragma unroll
      for (int i = 0; i < N; i++) {
        const int index = v * N + i - lead;
        l[i] = NAN;
        if (index >= 0 && index < V) l[i] = Io<T>::ld(x, (size_t)(index + lead));
      }
    }
  }
  // f(logit, index) for every logit above -infinity, U vectors under way at a time
  template <int U, class F>
  __device__ __forceinline__ void each(F f) const {
    for (int v0 = threadIdx.x; v0 < vectors; v0 += THREADS * U) {
      float l[U][N];
#pragma unroll
      for (int j = 0; j < U; j++) if (v0 + j * THREADS < vectors) load(v0 + j * THREADS, l[j]);
#pragma unroll
      for (int j = 0; j < U; j++) if (v0 + j * THREADS < vectors)
#pragma unroll
        for (int i = 0; i < N; i++) if (l[j][i] > -INFINITY) f(l[j][i], (v0 + j * THREADS) * N + i - lead);
    }
  }
};

// weights against `top` at a temperature
struct Weight {
  float top;
  double factor;                                 // 256 log2(e) / temperature
  const double *steps;
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
    return some ? units : l == top ? (uint64_t)UNIT : 0;
  }
};

// The first by index at which the running sum of term(logit, index) passes; there is one.
template <class T, class Term>
__device__ __forceinline__ Found across(const Row<T> &row, Shared &s, Term term, Past past) {
  constexpr int N = Row<T>::N;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, runs = (row.vectors + 63) / 64;
  __syncthreads();
  for (int r = wave; r < runs; r += WAVES) {
    uint64_t sum = 0;
    const int v = r * 64 + lane;
    if (v < row.vectors) {
      float l[N];
      row.load(v, l);
#pragma unroll
      for (int i = 0; i < N; i++) if (l[i] > -INFINITY) sum += term(l[i], v * N + i - row.lead);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) s.runs[r] = sum;
  }
  __syncthreads();
  const int each = (runs + THREADS - 1) / THREADS, r0 = threadIdx.x * each;
  uint64_t sum = 0, all;
  for (int i = 0; i < each; i++) sum += r0 + i < runs ? s.runs[r0 + i] : 0;
  uint64_t before = block_before(sum, s, all);
  for (int i = 0; i < each; i++) {
    const uint64_t x = r0 + i < runs ? s.runs[r0 + i] : 0;
    if (!past(before) && past(before + x)) { s.found = r0 + i; s.found_before = before; }
    before += x;
  }
  __syncthreads();
  Found f{0.f, 0, 0};
  const int v = same(s.found) * 64 + lane;       // every wave does the same
  const uint64_t start = same(s.found_before);
  float l[N];
  uint64_t w[N];
  sum = 0;
#pragma unroll
  for (int i = 0; i < N; i++) { l[i] = NAN; w[i] = 0; }
  if (v < row.vectors) row.load(v, l);
#pragma unroll
  for (int i = 0; i < N; i++) { if (l[i] > -INFINITY) w[i] = term(l[i], v * N + i - row.lead); sum += w[i]; }
  uint64_t upto = start + wave_running(sum) - sum;
  bool here = false;
#pragma unroll
  for (int i = 0; i < N; i++) {
    if (!past(upto) && past(upto + w[i])) { here = true; f = Found{l[i], v * N + i - row.lead, past.base + upto + w[i]}; }
    upto += w[i];
  }
  const uint64_t who = __ballot(here);
  const int from = who ? __builtin_ctzll(who) : 0;
  return Found{same(__shfl(f.logit, from)), same(__shfl(f.index, from)), same((uint64_t)__shfl(f.upto, from))};
}

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

// Running sums of term(logit) over the bins, of the logits between `low` and `high`, into s.bins[level]; the sum of all
template <class T, class Term>
__device__ __forceinline__ uint64_t fill_bins(const Row<T> &row, Shared &s, int level, const Bins &bin, float low, float high, Term term) {
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += THREADS) s.bins[level][i] = 0;
  __syncthreads();
  row.template each<2>([&](float l, int) {
    if (l >= low && l <= high) {
      const uint64_t w = term(l);
      if (w) atomicAdd((unsigned long long *)&s.bins[level][bin(l)], (unsigned long long)w);
    }
  });
  __syncthreads();
  return sum_bins(s, level);
}

// The first, from the largest down, at which the running sum of term(logit) passes; there is one.  s.bins[0] has the running sums of the logits between
// `low` and `high` in `bin`.
template <class T, class Term>
__device__ __forceinline__ Found descend(const Row<T> &row, Shared &s, Bins bin, float low, float high, Term term, Past past) {
  uint64_t base = 0;
  __syncthreads();
  // (the row's own bins, and at most three times those of a bin: 2^32 floats are 2^11 times 2^21, 2^10, 1.  Bounded as it stands, whatever the sums
  // are: every wave takes the same turns, since all of them read what decides from the same places between the same two barriers.)
  for (int cut = 0; cut < 5; cut++) {
    const int level = cut ? 1 : 0;
    if (threadIdx.x == 0) s.listed = 0;
    find_bin(s, level, base, past);
    const int b = same(s.found);
    base = same(s.found_before);
    float least = INFINITY, most = -INFINITY;
    row.template each<4>([&](float l, int index) {
      if (l >= low && l <= high && bin(l) == b) {
        least = fminf(least, l);
        most = fmaxf(most, l);
        const int at = atomicAdd(&s.listed, 1);
        if (at < LIST) s.list[at] = entry_of(l, index);
      }
    });
    block_bounds(least, most, s);
    const int n = same(s.listed);
    if (n <= LIST) {
      sort_list(s, n);
      uint64_t w[EACH], sum = 0, all;
#pragma unroll
      for (int i = 0; i < EACH; i++) { const int e = EACH * threadIdx.x + i; w[i] = e < n ? term(entry_logit(s.sorted[e])) : 0; sum += w[i]; }
      uint64_t before = base + block_before(sum, s, all);
#pragma unroll
      for (int i = 0; i < EACH; i++) {
        if (!past(before) && past(before + w[i])) { s.found = EACH * threadIdx.x + i; s.found_before = before + w[i]; }
        before += w[i];
      }
      __syncthreads();
      const uint64_t e = same(s.sorted[same(s.found)]);
      return Found{entry_logit(e), entry_index(e), same(s.found_before)};
    }
    if (least == most) {                         // equal ones: the first by index
      const uint64_t w = term(least);
      return across(row, s, [&](float l, int) { return l == least ? w : 0; }, Past{past.target, past.reach, base});
    }
    low = least;
    high = most;
    bin = Bins(low, high);
    fill_bins(row, s, 1, bin, low, high, term);
  }
  return Found{NAN, 0, base};                    // (not reached)
}

template <class T>
__global__ __launch_bounds__(THREADS) void k_sample(SampleArgs a) {
  __shared__ Shared s;
  const int t = threadIdx.x;
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
    row.template each<4>([&](float l, int index) { if (l > top) { top = l; first = index; } });
    // the larger, then the lower index: the largest entry
    uint64_t best = top > -INFINITY ? entry_of(top, first) : 0;
#pragma unroll
    for (int o = 32; o; o >>= 1) { const uint64_t x = __shfl_xor(best, o); best = x > best ? x : best; }
    if ((t & 63) == 0) s.part[t >> 6] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; w++) best = s.part[w] > best ? s.part[w] : best;
    answer(best ? entry_index(best) : 0, best ? 0.f : NAN);
    return;
  }
  row.template each<4>([&](float l, int) { top = fmaxf(top, l); low = fminf(low, l); });
  const float mine = top;
  block_bounds(low, top, s);
  if (top == -INFINITY) { answer(0, NAN); return; }
  if (t < STEPS) s.steps[t] = exp2((double)t / STEPS);
  if (t == 0) s.found = 0;

  const Weight weight{top, STEPS * 1.44269504088896340736 / (double)temperature, s.steps};
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

  float bound = low;                             // what top_k leaves is not below it
  if (k > 0 && k < row.V) {
    if (k <= FEW) {
      // At least k logits are in the bins (of the threads' maxima) up to the one in which the k-th largest of the maxima lies: those are the candidates.
      float lowest = mine > -INFINITY ? mine : INFINITY, dummy = mine;
      block_bounds(lowest, dummy, s);
      const Bins bin(lowest, top, INFINITY);
      for (int i = t; i < BINS; i += THREADS) s.bins[0][i] = 0;
      __syncthreads();
      if (mine > -INFINITY) atomicAdd((unsigned long long *)&s.bins[0][bin(mine)], 1ull);
      if (t == 0) { s.listed = 0; s.found = BINS - 1; }
      __syncthreads();
      const bool every = sum_bins(s, 0) < (uint64_t)k;             // fewer maxima than that: all of the row are candidates
      find_bin(s, 0, 0, Past{(double)k, true});
      const int last = every ? BINS - 1 : same(s.found);
      row.template each<4>([&](float l, int index) {
        if (bin(l) <= last) {
          const int at = atomicAdd(&s.listed, 1);
          if (at < LIST) s.list[at] = entry_of(l, index);
        }
      });
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
          w[i] = at < n && (uint32_t)(e[i] >> 32) >= kth ? weight(entry_logit(e[i])) : 0;
          sum += w[i];
        }
        uint64_t before = block_before(sum, s, all);
        const Past end{nucleus ? (double)p * (double)all : INFINITY, true};
        uint64_t number = 0;
#pragma unroll
        for (int i = 0; i < EACH; i++) {
          const bool stays = !end(before) && enough(entry_logit(e[i]));
          before += w[i];
          w[i] = stays ? w[i] : 0;
          number += w[i] != 0;
        }
        if (!nucleus) {                          // by index: the list again with the index first and the place in the order behind it
          uint64_t at = block_before(number, s, number);
#pragma unroll
          for (int i = 0; i < EACH; i++) {
            if (w[i]) s.list[at++] = (uint64_t)(uint32_t)e[i] << 32 | (uint32_t)(EACH * t + i);
            s.bins[0][EACH * t + i] = e[i];      // (what was sorted by logit is needed once more)
          }
          sort_list(s, (int)number);
#pragma unroll
          for (int i = 0; i < EACH; i++) {
            const int j = EACH * t + i;
            e[i] = j < (int)number ? s.bins[0][(uint32_t)s.sorted[j]] : 0;
            w[i] = j < (int)number ? weight(entry_logit(e[i])) : 0;
          }
        }
        sum = 0;
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
    const Bins bin(low, top, INFINITY);
    const auto one = [](float) { return (uint64_t)1; };
    if (fill_bins(row, s, 0, bin, low, top, one) > (uint64_t)k) bound = descend(row, s, bin, low, top, one, Past{(double)k, true}).logit;
  }
  if (nucleus) {
    const Bins bin(bound, top, 31.f * temperature);
    uint64_t sum = 0;
    const uint64_t of_all = fill_bins(row, s, 0, bin, bound, top, [&](float l) {
      const uint64_t w = weight(l);
      if (enough(l)) sum += w;
      return w;
    });
    const uint64_t of_enough = block_sum(sum, s);
    Past past{(double)p * (double)of_all, true};
    uint64_t all = 0;
    Found f;
    for (int end = 1; end >= 0; end--) {         // where the nucleus ends, then the token
      f = descend(row, s, bin, bound, top, weight, past);
      if (end) {
        all = enough(f.logit) ? f.upto : of_enough;
        past = walk(all);
      }
    }
    finish(f.logit, f.index, all);
    return;
  }
  const auto term = [&](float l, int) { return l >= bound && enough(l) ? weight(l) : 0; };
  __syncthreads();
  uint64_t sum = 0;
  row.template each<2>([&](float l, int index) { sum += term(l, index); });
  const uint64_t all = block_sum(sum, s);
  const Found token = across(row, s, term, walk(all));
  finish(token.logit, token.index, all);
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
