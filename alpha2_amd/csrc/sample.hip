// The next token of every row of logits from a given random number (ah_sample, include/alpha_hip.h).
//
// A workgroup to a row.  Every question asked of a row (which is the k-th largest, where does a mass end, which token does the number fall on) is
// "the first, from the largest down, at which a running sum passes a number", and is answered by descending into bins of the logit: the masses (or
// counts) of 2048 bins between the row's bounds are added up in LDS, the bin that holds the answer is found by a scan, and its members are
// gathered, sorted and scanned; if they are too many, the bin is cut again between its own bounds, and if they are all equal the answer is one of them by
// index.  Where no nucleus is asked for the walk is by index: sums of runs of 64 vectors, a scan over those, and the one run again.
// With a small top_k all of that happens in the list of the few candidates that the threads' maxima leave.
//
// Bound by one workgroup's passes over its row, from the second on out of the caches, and by what a pass does with a logit: a weight takes a dozen 64-bit
// operations, a bin an addition in LDS.  One row of 50304, top_k 40, 15 us; largest alone 6.5, by index without cuts 24, nucleus 35.  20 rows of 4096, nucleus,
// 16 us.  160 rows of 131072 in bf16: largest 13 us, by index 52, nucleus 84, all of it mixed 100 (the 42 MB alone 9).  20 of 300, by index, 6.8.
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

constexpr int BINS = 2048, LIST = 2048, STEPS = 256, MOST_WAVES = 16;
static_assert(BINS == LIST, "as many bins as entries to a thread");
constexpr int MAX_VOCAB = 1 << 20;              // sums of as many weights of 2^43 stay below 2^63
constexpr double UNIT = 0x1p43;
// A top_k up to this goes through the maxima of 512 threads or more, which leave about k candidates: of 300 logits the first 40 take 9.6 us, by the bins' counts
// 12.7; of 4096 9.5 and 14.4; of 50304 15.7 and 33.
constexpr int FEW = 256;
// Rows past this have 1024 threads: 20 of 8192, nucleus, 17.6 us, with 1024 threads 18.1; of 12000, 21.2 and 19.8; of 32768, 33 and 28; of 4096, 16.3 and 17.5.
constexpr int LONG = 8192;

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
  uint64_t list[2][LIST], sorted[LIST];
  uint64_t runs[RUNS];                           // sums of 64 vectors of four (or eight) logits
  double   steps[STEPS];                         // 2^(i / 256)
  uint64_t part[MOST_WAVES];
  float    low[MOST_WAVES], high[MOST_WAVES];
  uint64_t found_before, found_entry, answer, kept;
  int      found, listed[2];
};
static_assert(sizeof(Shared) <= 160 * 1024, "a workgroup's LDS");

// ------------------------------------------------------------------------------------------ a workgroup's sums
// What every lane has read from the same place, told the compiler: branches on it, with barriers behind them, are branches of the whole wave.
__device__ __forceinline__ int same(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ float same(float v) { return __uint_as_float((uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(v))); }
__device__ __forceinline__ uint64_t same(uint64_t v) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
}
// What the lanes hold up to this one, by DPP: a step is two moves and an addition, where __shfl_up is two trips through LDS
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t plus_moved(uint64_t v) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xf, false);
  return v + ((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ uint64_t wave_running(uint64_t v) {
  v = plus_moved<0x111, 0xf>(v);                 // one, two, four, eight to the right in rows of 16
  v = plus_moved<0x112, 0xf>(v);
  v = plus_moved<0x114, 0xf>(v);
  v = plus_moved<0x118, 0xf>(v);
  v = plus_moved<0x142, 0xa>(v);                 // the last of a row to the next one, of two rows to the next two
  return plus_moved<0x143, 0xc>(v);
}
__device__ __forceinline__ uint64_t wave_lane(uint64_t v, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
// the sum over the threads before this one, and over all: the waves' sums are added up in the 16 lanes of every row
template <int THREADS>
__device__ __forceinline__ uint64_t block_before(uint64_t v, Shared &s, uint64_t &all) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const uint64_t upto = wave_running(v);
  __syncthreads();
  if (lane == 63) s.part[wave] = upto;
  __syncthreads();
  uint64_t waves = (lane & 15) < THREADS / 64 ? s.part[lane & 15] : 0;
  waves = plus_moved<0x111, 0xf>(waves);
  waves = plus_moved<0x112, 0xf>(waves);
  waves = plus_moved<0x114, 0xf>(waves);
  waves = plus_moved<0x118, 0xf>(waves);
  all = wave_lane(waves, 63);
  const uint64_t before = wave ? wave_lane(waves, wave - 1) : 0;
  return before + upto - v;
}
template <int THREADS>
__device__ __forceinline__ uint64_t block_sum(uint64_t v, Shared &s) {
  uint64_t all;
  block_before<THREADS>(v, s, all);
  return all;
}
template <int THREADS>
__device__ __forceinline__ void block_bounds(float &low, float &high, Shared &s) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  low = -wave_max(-low);
  high = wave_max(high);
  __syncthreads();
  if (lane == 0) { s.low[wave] = low; s.high[wave] = high; }
  __syncthreads();
  low = same(-wave_max(-s.low[lane & (THREADS / 64 - 1)]));
  high = same(wave_max(s.high[lane & (THREADS / 64 - 1)]));
}

// The n entries of a list in order, into `sorted`.  Up to 256 by counting the larger ones of each, 2 to 16 threads to an entry; more by exchanges,
// whose steps between neighbours of 128 need no barrier (20 rows of 4096, top_k 40: 9.5 us, by exchanges 18; nucleus, which sorts twice, 16 and 34).
template <int THREADS>
__device__ __forceinline__ void sort_list(Shared &s, const uint64_t *list, int n) {
  const int t = threadIdx.x;
  __syncthreads();
  if (n <= 256) {
    const int most = THREADS == 512 ? 3 : 4, shift = n <= 64 ? most : n <= 128 ? most - 1 : most - 2, i = t >> shift;
    const uint64_t mine = i < n ? list[i] : 0;
    uint32_t larger = 0;
    for (int j = t & ((1 << shift) - 1); j < n; j += 1 << shift) larger += list[j] > mine;
    larger += lane_xor<1>(larger);
    if (shift > 1) larger += lane_xor<2>(larger);
    if (shift > 2) larger += lane_xor<4>(larger);
    if (shift > 3) larger += lane_xor<8>(larger);
    if (i < n && (t & ((1 << shift) - 1)) == 0) s.sorted[larger] = mine;
  } else {
    int size = 512;
    while (size < n) size <<= 1;
    for (int i = t; i < size; i += THREADS) s.sorted[i] = i < n ? list[i] : 0;
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
template <class T, int THREADS> struct Row {
  static constexpr int N = 16 / sizeof(T);       // logits to a vector
  // The logits before the first whole 16 bytes and behind the last are vectors of one each, so that no other memory is read; all are in the order of the indices.
  const T *x;
  int V, head, whole, vectors;
  __device__ __forceinline__ Row(const T *row, int vocab) {
    x = row;
    V = vocab;
    head = min((int)((16 - (uintptr_t)row % 16) % 16 / sizeof(T)), V);
    whole = (V - head) / N;
    vectors = V - whole * (N - 1);
  }
  __device__ __forceinline__ int index(int v, int i) const {
    const int n = v - head;
    return v < head ? v : n < whole ? head + n * N + i : v + whole * (N - 1);
  }
  __device__ __forceinline__ float at(int index) const { return Io<T>::ld(x, (size_t)index); }
  // vector v as it is stored; NaN where there is no logit
  __device__ __forceinline__ uint4 load(int v) const {
    uint4 w = make_uint4(~0u, ~0u, ~0u, ~0u);
    if (v >= head && v - head < whole) w = *reinterpret_cast<const uint4 *>(x + head + (int64_t)(v - head) * N);
    else if (v < vectors) w.x = N == 4 ? __float_as_uint(at(index(v, 0))) : __float_as_uint(at(index(v, 0))) >> 16 | 0xffff0000u;
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
  // f(logit, index) for the ones in either interval, which are few: a vector is looked into where it has one
  template <class F>
  __device__ __forceinline__ void hits(float lo, float hi, float lo2, float hi2, F f) const {
    constexpr int U = 16 / N;
    const bool two = lo2 <= hi2;
    for (int v0 = threadIdx.x; v0 < vectors; v0 += THREADS * U) {
      uint4 w[U];
#pragma unroll
      for (int j = 0; j < U; j++) w[j] = load(v0 + j * THREADS);
      bool some = false;
#pragma unroll
      for (int j = 0; j < U; j++)
#pragma unroll
        for (int i = 0; i < N; i++) { const float l = logit(w[j], i); some |= l == __builtin_amdgcn_fmed3f(l, lo, hi); }
      if (two)
#pragma unroll
        for (int j = 0; j < U; j++)
#pragma unroll
          for (int i = 0; i < N; i++) { const float l = logit(w[j], i); some |= l == __builtin_amdgcn_fmed3f(l, lo2, hi2); }
      if (some) {
        uint32_t bits = 0;
#pragma unroll
        for (int j = 0; j < U; j++)
#pragma unroll
          for (int i = 0; i < N; i++) { const float l = logit(w[j], i); bits |= (l >= lo && l <= hi) || (l >= lo2 && l <= hi2) ? 1u << (j * N + i) : 0u; }
        while (bits) {
          const int b = __builtin_ctz(bits);
          const int n = index(v0 + b / N * THREADS, b % N);
          f(at(n), n);
          bits &= bits - 1;
        }
      }
    }
  }
};

// weights against `top` at a temperature, as whole numbers; or 1 each
struct Weight {
  float top;
  double factor;                                 // 256 log2(e) / temperature
  const double *steps;
  uint64_t each;                                 // 0, or what each of them counts
  __device__ __forceinline__ uint64_t operator()(float l) const {
    if (each) return each;
    // y = below * factor.  Written with fma and not with y: a compiler that fuses the two in one of this function's many places and not in another would give a
    // logit two weights, and running sums that no total agrees with.
    const double below = (double)l - (double)top;
    const bool some = below * factor > -44.0 * STEPS;                // (not NaN)
    constexpr double ROUND = 0x1.8p52;
    const double whole = fma(below, factor, ROUND);
    const int n = (int)(uint32_t)__builtin_bit_cast(uint64_t, whole);
    const double g = fma(below, factor, -(whole - ROUND)) * (0.693147180559945309417 / STEPS);
    const float h = (float)g;
    const double e = fma(g * g, (double)fmaf(h, fmaf(h, 1.0f / 24, 1.0f / 6), 0.5f), g);
    const double step = steps[n & (STEPS - 1)], w = fma(step, e, step);
    const uint64_t scaled = __builtin_bit_cast(uint64_t, w) + ((uint64_t)(uint32_t)((n >> 8) + 43) << 52);
    const uint64_t units = __builtin_bit_cast(uint64_t, __builtin_bit_cast(double, scaled) + 0x1p52) & ((1ull << 52) - 1);
    return some ? units : 0;
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
  // logits of bin b lie between these (and, by rounding, others at the ends)
  __device__ __forceinline__ void around(int b, float low, float &lo, float &hi) const {
    if (shift >= 0) {
      hi = of_order(order_of(high) - ((uint32_t)b << shift));
      const uint64_t end = ((uint64_t)(b + 1) << shift) - 1, span = order_of(high) - order_of(low);
      lo = of_order(order_of(high) - (uint32_t)(end < span ? end : span));
      return;
    }
    const float wide = 1.0f / scale, slack = 4e-7f * (fabsf(high) + (b + 1) * wide);      // several roundings of each of the two
    lo = high - (b + 1) * wide - slack;
    hi = fminf(high, high - b * wide + slack);
    if (b == BINS - 1 || !(lo >= low)) lo = low;
    if (!(hi >= low)) hi = high;                 // (no width: every bin is the first or the last)
  }
};
static_assert(BINS == 1 << 11, "the shift of a bin's bins");
// Is there only one bf16 number among those between lo and hi that fall into bin b?  Rows of bf16 have thousands of equal logits.
__device__ __forceinline__ bool one_of_bin(const Bins &bin, int b, float lo, float hi, float &only) {
  const uint32_t first = order_of(hi) >> 16, last = order_of(lo) >> 16;
  if (first - last > 6) return false;
  int different = 0;
  only = 0.f;
#pragma unroll 1
  for (uint32_t o = first; o + 1 > last; o--) {
    const float x = __uint_as_float((o & 0x8000u ? o ^ 0x8000u : o ^ 0xffffu) << 16) + 0.f;
    const bool in = x >= lo && x <= hi && bin(x) == b && !(different && x == only);
    only = in ? x : only;
    different += in;
  }
  return different == 1;
}

// s.bins[level] to running sums; the sum of all
template <int THREADS>
__device__ __forceinline__ uint64_t sum_bins(Shared &s, int level) {
  constexpr int EACH = BINS / THREADS;
  uint64_t x[EACH], sum = 0, all;
#pragma unroll
  for (int i = 0; i < EACH; i++) { x[i] = s.bins[level][EACH * threadIdx.x + i]; sum += x[i]; }
  uint64_t upto = block_before<THREADS>(sum, s, all);
#pragma unroll
  for (int i = 0; i < EACH; i++) { upto += x[i]; s.bins[level][EACH * threadIdx.x + i] = upto; }
  __syncthreads();
  return all;
}
// Where in s.bins[level] running sums, on from `base`, reach `mark`: the bin into s.found, the sum before it into s.found_before.
template <int THREADS>
__device__ __forceinline__ void find_bin(Shared &s, int level, uint64_t base, uint64_t mark) {
  constexpr int EACH = BINS / THREADS;
#pragma unroll
  for (int i = 0; i < EACH; i++) {
    const int b = EACH * threadIdx.x + i;
    const uint64_t before = base + (b ? s.bins[level][b - 1] : 0), upto = base + s.bins[level][b];
    if (before < mark && upto >= mark) { s.found = b; s.found_before = before; }
  }
  __syncthreads();
}

struct Found {
  float    logit;
  int      index;                                // -1: one of several equal ones, whose running sums go on from `before`
  uint64_t upto, before;                         // the running sums with it and, of equal ones, without any of them
};

template <class T, int THREADS>
__global__ __launch_bounds__(THREADS) void k_sample(SampleArgs a) {
  constexpr int WAVES = THREADS / 64, EACH = LIST / THREADS, N = Row<T, THREADS>::N, UNDER_WAY = 2;
  __shared__ Shared s;
  const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
  const int64_t r = blockIdx.x;
  const Row<T, THREADS> row((const T *)a.logits + r * a.ld, a.vocab);
  auto logit = [](const uint4 &w, int i) { return Row<T, THREADS>::logit(w, i); };
  const float temperature = a.temperature ? a.temperature[r] : 1.f;
  const int k = a.top_k ? a.top_k[r] : 0;
  const float p = a.top_p ? a.top_p[r] : 0.f, least_p = a.min_p ? a.min_p[r] : 0.f, u = a.uniform[r];
  auto answer = [&](int token, float logprob) { a.tokens[r] = token; if (a.logprobs) a.logprobs[r] = logprob; };      // by one thread
  float top = -INFINITY, low = INFINITY;         // this thread's, then the row's
  if (!(temperature > 0.f)) {
    int first = 0;
    row.template each<4>([&](const uint4 &w, int v) {
#pragma unroll
      for (int i = 0; i < N; i++) { const float l = logit(w, i); const bool more = l > top; top = more ? l : top; first = more ? row.index(v, i) : first; }
    });
    // the larger, then the lower index: the largest entry
    uint64_t best = top > -INFINITY ? entry_of(top, first) : 0;
#pragma unroll
    for (int o = 32; o; o >>= 1) { const uint64_t x = __shfl_xor(best, o); best = x > best ? x : best; }
    if (lane == 0) s.part[wave] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; w++) best = s.part[w] > best ? s.part[w] : best;
    if (t == 0) answer(best ? entry_index(best) : 0, best ? 0.f : NAN);
    return;
  }
  if (t < STEPS) s.steps[t] = exp2((double)t / STEPS);
  if (t == 0) { s.found = 0; s.listed[0] = s.listed[1] = 0; s.answer = 0; s.kept = 0; }
  row.template each<4>([&](const uint4 &w, int) {
#pragma unroll
    for (int i = 0; i < N; i++) { const float l = logit(w, i); top = fmaxf(top, l); low = l > -INFINITY ? fminf(low, l) : low; }
  });
  const float mine = top;
  block_bounds<THREADS>(low, top, s);
  if (top == -INFINITY) { if (t == 0) answer(0, NAN); return; }

  // An infinite largest: there is nothing but those, and each weighs 1.
  const bool infinite = top == INFINITY;
  float bound = infinite ? top : low;            // what top_k leaves is not below it
  Weight weight{top, STEPS * 1.44269504088896340736 / (double)temperature, s.steps, infinite ? (uint64_t)UNIT : 0};
  const uint64_t unit = weight.each;
  const bool nucleus = p > 0.f && p < 1.f, cut = k > 0 && k < row.V, some_drop = least_p > 0.f && temperature < INFINITY;
  // a weight of at least min_p
  const double drop = some_drop ? (double)temperature * log((double)fminf(least_p, 1.f)) : -INFINITY;
  auto enough = [&](float l) { return !some_drop || l == top || (double)l - (double)top >= drop; };
  // The sums that running sums have to reach: the nucleus's, and the token's, which passes the given number; where rounding, or a number of 1, leaves nothing
  // beyond it, that is the last that weighs something.
  auto nucleus_mark = [&](uint64_t all) { const uint64_t m = (uint64_t)ceil((double)p * (double)all); return m < 1 ? 1 : m > all ? all : m; };
  auto token_mark = [&](uint64_t all) { const uint64_t m = (uint64_t)(fmin(fmax((double)u, 0.0), 1.0) * (double)all); return m < all ? m + 1 : all; };
  // what one thread finds: the token and the sum of what is kept
  auto finish = [&](uint64_t entry, uint64_t all) { s.answer = entry; s.kept = all; };
  auto list = [&](int which, float l, int index) {
    const int at = atomicAdd(&s.listed[which], 1);
    if (at < LIST) s.list[which][at] = entry_of(l, index);
  };

  auto choose = [&] {
    if (cut && k <= FEW) {
      // At least k logits are in the bins (of the threads' maxima) up to the one in which the k-th largest of the maxima lies: those are the candidates.
      float lowest = mine > -INFINITY ? mine : INFINITY, dummy = mine;
      block_bounds<THREADS>(lowest, dummy, s);
      const Bins bin(lowest, top, INFINITY);
      for (int i = t; i < BINS; i += THREADS) s.bins[0][i] = 0;
      __syncthreads();
      if (mine > -INFINITY) atomicAdd((unsigned long long *)&s.bins[0][bin(mine)], 1ull);
      __syncthreads();
      const bool every = sum_bins<THREADS>(s, 0) < (uint64_t)k;  // fewer maxima than that: all of the row are candidates
      find_bin<THREADS>(s, 0, 0, (uint64_t)k);
      const int last = every ? BINS - 1 : same(s.found);
      float lo = bound, hi;
      if (last < BINS - 1) bin.around(last, bound, lo, hi);      // (the last bin has no end)
      row.hits(lo, top, INFINITY, -INFINITY, [&](float l, int index) { if (bin(l) <= last) list(0, l, index); });
      __syncthreads();
      const int n = same(s.listed[0]);
      if (n <= LIST) {
        sort_list<THREADS>(s, s.list[0], n);
        const uint32_t kth = n > k ? (uint32_t)(same(s.sorted[k - 1]) >> 32) : 0u, lowest = max(kth, order_of(bound));
        if (n <= 64) {                           // a wave alone (9.5 us; by all of them, with their barriers, 11.6)
          if (wave) return;
          const uint64_t e = lane < n ? s.sorted[lane] : 0;
          const float l = entry_logit(e);
          const uint64_t x = weight(l);
          uint64_t w = lane < n && (uint32_t)(e >> 32) >= lowest ? x : 0, upto = wave_running(w), all = wave_lane(upto, 63);
          w = (!nucleus || upto - w < nucleus_mark(all)) && enough(l) ? w : 0;
          upto = wave_running(w);
          all = wave_lane(upto, 63);
          if (!nucleus) {                        // by index
            s.bins[0][lane] = (uint32_t)e;
            s.bins[1][lane] = w;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            upto = 0;
            for (int j = 0; j < n; j++) { const uint64_t other = s.bins[0][j], more = s.bins[1][j]; upto += other >= (uint32_t)e ? more : 0; }
          }
          const uint64_t mark = token_mark(all);
          if (upto - w < mark && upto >= mark && w) finish(e, all);
          return;
        }
        uint64_t e[EACH], w[EACH], sum = 0, all;
#pragma unroll
        for (int i = 0; i < EACH; i++) {
          const int at = EACH * t + i;
          e[i] = at < n ? s.sorted[at] : 0;
          const uint64_t x = weight(entry_logit(e[i]));
          w[i] = at < n && (uint32_t)(e[i] >> 32) >= lowest ? x : 0;
          sum += w[i];
        }
        uint64_t before = block_before<THREADS>(sum, s, all), number = 0;
        const uint64_t end = nucleus ? nucleus_mark(all) : ~0ull;
        sum = 0;
#pragma unroll
        for (int i = 0; i < EACH; i++) {
          const bool stays = before < end && enough(entry_logit(e[i]));
          before += w[i];
          w[i] = stays ? w[i] : 0;
          number += w[i] != 0;
        }
        if (!nucleus) {                          // by index: the list again with the index first and the place in the order behind it
          uint64_t at = block_before<THREADS>(number, s, number);
#pragma unroll
          for (int i = 0; i < EACH; i++) {
            if (w[i]) s.list[0][at++] = (uint64_t)(uint32_t)e[i] << 32 | (uint32_t)(EACH * t + i);
            s.bins[0][EACH * t + i] = e[i];      // (what was sorted by logit is needed once more)
            s.bins[1][EACH * t + i] = w[i];
          }
          sort_list<THREADS>(s, s.list[0], (int)number);
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
        before = block_before<THREADS>(sum, s, all);
        const uint64_t mark = token_mark(all);
#pragma unroll
        for (int i = 0; i < EACH; i++) {
          if (before < mark && before + w[i] >= mark) finish(e[i], all);
          before += w[i];
        }
        return;
      }
    }

    // Descents, from the largest down: to the k-th largest, to where the nucleus ends, to the token.
    uint64_t all = 0, mark = (uint64_t)k;
    Found f{bound, 0, 0, 0};
    enum { KTH, END, TOKEN, NONE };
    int goal = cut ? KTH : nucleus ? END : NONE;
    Bins bin(bound, top, INFINITY);
    // The row's own bins whose members are in the two lists: the one the nucleus ends in and, so that the row need not be gone over again, the one the
    // token is in if the nucleus ends with that bin.
    int have[2] = {-1, -1}, members[2] = {0, 0};
    for (int turn = 0; turn < 3 && goal != NONE; turn++) {
      float least = bound, most = top;
      // (a row's own bins and at most three times those of a bin: 2^32 floats are 2^11 times 2^21, 2^10, 1.  Both loops are bounded whatever the sums are, and
      // every wave takes the same turns: all of them read what decides from the same places between the same two barriers.)
      uint64_t base = 0, of_enough = 0;
      for (int level = 0; level < 5; level++) {
        const int l1 = level ? 1 : 0;
        if (level || goal != TOKEN) {            // (the token's are those of the nucleus)
          weight.each = goal == KTH ? 1 : unit;
          bin = level ? Bins(least, most) : Bins(bound, top, goal == KTH ? INFINITY : 31.f * temperature);
          __syncthreads();
          for (int i = t; i < BINS; i += THREADS) s.bins[l1][i] = 0;
          __syncthreads();
          uint64_t sum = 0;
          row.template each<UNDER_WAY>([&](const uint4 &w, int) {
            uint64_t x[N];                       // (all of a vector's at once, so that they are under way side by side)
#pragma unroll
            for (int i = 0; i < N; i++) {
              const float l = logit(w, i);
              const uint64_t y = weight(l);
              x[i] = l >= least && l <= most ? y : 0;                // (not NaN, and above -infinity like those)
            }
            if (some_drop)
#pragma unroll
              for (int i = 0; i < N; i++) sum += enough(logit(w, i)) ? x[i] : 0;
#pragma unroll
            for (int i = 0; i < N; i++) if (x[i]) atomicAdd((unsigned long long *)&s.bins[l1][bin(logit(w, i))], (unsigned long long)x[i]);
          });
          __syncthreads();
          const uint64_t total = sum_bins<THREADS>(s, l1);
          if (!level) {
            if (goal == KTH && total <= (uint64_t)k) break;          // nothing to cut: f is the lowest
            if (goal == END) mark = nucleus_mark(total);
            of_enough = some_drop && goal == END ? block_sum<THREADS>(sum, s) : total;
          }
        }
        __syncthreads();
        if (t == 0 && (level || goal != TOKEN)) s.listed[0] = s.listed[1] = 0;
        find_bin<THREADS>(s, l1, base, mark);
        const int b = same(s.found);
        base = same(s.found_before);
        int which = 0, n = 0;
        float lo, hi, value = 0.f;
        bin.around(b, least, lo, hi);
        bool equal = N == 8 && one_of_bin(bin, b, lo, hi, value);
        const bool listed = !equal && !level && goal == TOKEN && (b == have[0] || b == have[1]);
        if (equal) {
        } else if (listed) {
          which = b == have[0] ? 0 : 1;
          n = members[which];
        } else {
          int too = -1;
          float lo2 = INFINITY, hi2 = -INFINITY;
          if (!level && goal == END) {
            const uint64_t then = token_mark(same(s.bins[0][b]));
            __syncthreads();
            find_bin<THREADS>(s, 0, 0, then);
            too = same(s.found);
            if (too != b) bin.around(too, least, lo2, hi2);
            if (N == 8 && too != b && one_of_bin(bin, too, lo2, hi2, value)) { too = b; lo2 = INFINITY; hi2 = -INFINITY; }
          } else if (!level && goal == TOKEN) {  // (neither list: the first is made anew)
            __syncthreads();
            if (t == 0) s.listed[0] = 0;
            __syncthreads();
          }
          row.hits(lo, hi, lo2, hi2, [&](float l, int index) {
            const int at = bin(l);
            if (at == b || at == too) list(at == b ? 0 : 1, l, index);
          });
          __syncthreads();
          n = same(s.listed[0]);
          if (!level && goal == END) {
            have[0] = b;
            members[0] = n;
            have[1] = too == b ? -1 : too;
            members[1] = same(s.listed[1]);
          } else if (goal == END) have[0] = -1;
        }
        if (!equal && n <= LIST) {
          if (!(listed && which == 0)) sort_list<THREADS>(s, s.list[which], n);      // (the nucleus's is sorted)
          uint64_t w[EACH], sum = 0, dummy;
#pragma unroll
          for (int i = 0; i < EACH; i++) {
            const int e = EACH * t + i;
            const uint64_t x = weight(entry_logit(e < n ? s.sorted[e] : 0));
            w[i] = e < n ? x : 0;
            sum += w[i];
          }
          uint64_t before = base + block_before<THREADS>(sum, s, dummy);
#pragma unroll
          for (int i = 0; i < EACH; i++) {
            if (before < mark && before + w[i] >= mark) {
              const uint64_t e = s.sorted[EACH * t + i];
              if (goal == TOKEN) finish(e, all);
              s.found_entry = e;
              s.found_before = before + w[i];
            }
            before += w[i];
          }
          if (goal == TOKEN) return;
          __syncthreads();
          const uint64_t e = same(s.found_entry);
          f = Found{entry_logit(e), entry_index(e), same(s.found_before), 0};
          break;
        }
        if (!equal) {
          const float from = lo, to = hi;
          lo = INFINITY;
          hi = -INFINITY;
          row.hits(from, to, INFINITY, -INFINITY, [&](float l, int) {
            const bool in = bin(l) == b;
            lo = in ? fminf(lo, l) : lo;
            hi = in ? fmaxf(hi, l) : hi;
          });
          block_bounds<THREADS>(lo, hi, s);
          equal = lo == hi;
          value = lo;
        }
        if (equal) {                             // how many of them it takes
          const uint64_t w = same(weight(value));
          uint32_t few = 1, many = (uint32_t)row.V;
          for (int i = 0; i < 20 && few < many; i++) {
            const uint32_t middle = few + (many - few) / 2;
            if (base + middle * w >= mark) many = middle; else few = middle + 1;
          }
          f = Found{value, -1, base + few * w, base};
          break;
        }
        least = lo;
        most = hi;
      }
      if (goal == KTH) {
        bound = f.logit;
        goal = nucleus ? END : NONE;
      } else if (goal == END) {
        all = enough(f.logit) ? f.upto : of_enough;
        mark = token_mark(all);
        bin = Bins(bound, top, 31.f * temperature);
        goal = TOKEN;
      } else goal = NONE;
    }
    weight.each = unit;

    // By index: all that is kept where there is no nucleus, or the equal ones among which the token is.
    const float from = nucleus ? f.logit : bound, to = nucleus ? f.logit : top;
    const int runs = (row.vectors + 63) / 64;
    __syncthreads();
    for (int n0 = wave; n0 < runs; n0 += 2 * WAVES) {
      uint4 w[2];
#pragma unroll
      for (int j = 0; j < 2; j++) w[j] = row.load((n0 + j * WAVES) * 64 + lane);
#pragma unroll
      for (int j = 0; j < 2; j++) {
        uint64_t sum = 0;
        bool some = false;
#pragma unroll
        for (int i = 0; i < N; i++) { const float l = logit(w[j], i); some |= l >= from && l <= to && enough(l); }
        if (__any(some)) {
#pragma unroll
          for (int i = 0; i < N; i++) {
            const float l = logit(w[j], i);
            const uint64_t x = weight(l);
            sum += l >= from && l <= to && enough(l) ? x : 0;
          }
        }
        sum = wave_running(sum);
        if (lane == 63 && n0 + j * WAVES < runs) s.runs[n0 + j * WAVES] = sum;
      }
    }
    __syncthreads();
    const int each = (runs + THREADS - 1) / THREADS, r0 = t * each;
    uint64_t sum = 0, total;
    for (int i = 0; i < each; i++) sum += r0 + i < runs ? s.runs[r0 + i] : 0;
    uint64_t before = block_before<THREADS>(sum, s, total);
    if (!nucleus) {
      all = total;
      mark = token_mark(all);
    } else mark -= f.before;
    for (int i = 0; i < each; i++) {
      const uint64_t x = r0 + i < runs ? s.runs[r0 + i] : 0;
      if (before < mark && before + x >= mark) { s.found = r0 + i; s.found_before = before; }
      before += x;
    }
    __syncthreads();
    if (wave) return;
    const int v = same(s.found) * 64 + lane;     // the run again
    const uint4 w = row.load(v);
    uint64_t x[N], mass = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float l = logit(w, i);
      const uint64_t y = weight(l);
      x[i] = l >= from && l <= to && enough(l) ? y : 0;
      mass += x[i];
    }
    uint64_t upto = s.found_before + wave_running(mass) - mass;
    int token = -1;
    float l = 0.f;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const bool here = upto < mark && upto + x[i] >= mark;
      upto += x[i];
      token = here ? row.index(v, i) : token;
      l = here ? logit(w, i) : l;
    }
    if (token >= 0) finish(entry_of(l, token), all);
  };
  choose();
  __syncthreads();
  if (t == 0) {
    const float l = entry_logit(s.answer);
    answer(entry_index(s.answer), (float)((l == top ? 0.0 : ((double)l - (double)top) / (double)temperature) - log((double)s.kept / UNIT)));
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
  if (d->vocab > LONG) launch_kernel(d->dtype == AH_F32 ? k_sample<float, 1024> : k_sample<uint16_t, 1024>, dim3((unsigned)d->rows), dim3(1024), 0, a);
  else launch_kernel(d->dtype == AH_F32 ? k_sample<float, 512> : k_sample<uint16_t, 512>, dim3((unsigned)d->rows), dim3(512), 0, a);
  AH_LAUNCH_CHECK();
  return AH_OK;
}
