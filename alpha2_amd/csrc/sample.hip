// The next token of every row of logits from a given random number (include/alpha_hip.h has the definition).
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

constexpr int THREADS = 1024, WAVES = THREADS / 64;
// A weight exp((l - largest) / t) is at most 1 and counts as a whole number of 2^-43: sums of 2^20 of them stay below 2^63, are the same in
// every order, and are off by at most 2^-44 a term, far less than a number of 24 bits resolves.
constexpr int MAX_VOCAB = 1 << 20;
constexpr double UNIT = 0x1p43;

// f32 -> whole numbers of the same order, -0 as 0, NaN as 0 below everything
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x != x ? 0u : b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
constexpr uint32_t LOWEST = 0x007fffffu;        // that of -infinity

__device__ __forceinline__ uint64_t wave_total(uint64_t v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ uint64_t block_total(uint64_t v, uint64_t *shared) {
  v = wave_total(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
  for (int w = 0; w < WAVES; w++) v += shared[w];
  return v;
}

// A workgroup to a row.  Every question (the k-th largest, where a mass is reached) is a search by halves over the logits' order or over the
// index, a pass over the row for each half.
template <class T>
__global__ __launch_bounds__(THREADS) void k_sample(SampleArgs a) {
  __shared__ uint64_t shared[WAVES];
  const int row = blockIdx.x, t = threadIdx.x, V = a.vocab;
  const T *x = (const T *)a.logits + row * a.ld;
  auto order_at = [&](int i) { return order_of(Io<T>::ld(x, i)); };
  auto over = [&](auto term) {                  // the sum of term(index) over the row
    uint64_t s = 0;
    for (int i = t; i < V; i += THREADS) s += term(i);
    return block_total(s, shared);
  };
  // the largest number in (lo, hi] for which `holds`, which it does below some number and not above; lo if it does nowhere
  auto last_of = [&](uint32_t lo, uint32_t hi, auto holds) {
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo - 1) / 2 + 1;
      if (holds(mid)) lo = mid; else hi = mid - 1;
    }
    return lo;
  };
  const uint32_t top = last_of(LOWEST, 0xffffffffu, [&](uint32_t o) { return over([&](int i) { return (uint64_t)(order_at(i) >= o); }) > 0; });
  if (top == LOWEST) {
    if (t == 0) { a.tokens[row] = 0; if (a.logprobs) a.logprobs[row] = NAN; }
    return;
  }
  // the first index at which a running sum of term(index) passes `target`
  auto first_past = [&](auto term, double target) {
    return (int)last_of(0u, (uint32_t)V - 1, [&](uint32_t n) { return !((double)over([&](int i) { return i < (int)n ? term(i) : 0u; }) > target); });
  };
  const float temperature = a.temperature ? a.temperature[row] : 1.f;
  if (!(temperature > 0.f)) {
    const int token = first_past([&](int i) { return (uint64_t)(order_at(i) == top); }, 0.5);
    if (t == 0) { a.tokens[row] = token; if (a.logprobs) a.logprobs[row] = 0.f; }
    return;
  }
  const int k = a.top_k ? a.top_k[row] : 0;
  const float p = a.top_p ? a.top_p[row] : 0.f, m = a.min_p ? a.min_p[row] : 0.f, u = a.uniform[row];
  const float largest = __uint_as_float((top >> 31) ? top ^ 0x80000000u : ~top);
  auto exponent = [&](float l) { return l == largest ? 0.0 : ((double)l - (double)largest) / (double)temperature; };
  auto weight = [&](int i) {
    const float l = Io<T>::ld(x, i);
    return l > -INFINITY ? exp(exponent(l)) : 0.0;
  };
  auto mass = [&](int i) { return (uint64_t)rint(weight(i) * UNIT); };

  // what is kept: orders above `bound`, and those equal to it up to index `until`
  uint32_t bound = LOWEST + 1;
  int until = V - 1;
  auto kept = [&](int i) { const uint32_t o = order_at(i); return o > bound || (o == bound && i <= until); };
  if (k > 0 && k < V)
    bound = last_of(bound, top, [&](uint32_t o) { return over([&](int i) { return (uint64_t)(order_at(i) >= o); }) >= (uint64_t)k; });
  // from the largest down (equal ones by index), the first at which the running mass of what is kept passes `target` (or reaches it)
  auto descend = [&](double target, bool reach, uint32_t &order, int &index) {
    auto past = [&](uint64_t s) { return reach ? (double)s >= target : (double)s > target; };
    order = last_of(bound, top, [&](uint32_t o) { return past(over([&](int i) { return order_at(i) >= o && kept(i) ? mass(i) : 0u; })); });
    const uint64_t above = over([&](int i) { return order_at(i) > order && kept(i) ? mass(i) : 0u; });
    index = (int)last_of(0u, (uint32_t)V - 1, [&](uint32_t n) { return !past(above + over([&](int i) { return i < (int)n && order_at(i) == order && kept(i) ? mass(i) : 0u; })); });
  };
  const bool nucleus = p > 0.f && p < 1.f;
  if (nucleus) {
    const uint64_t all = over([&](int i) { return kept(i) ? mass(i) : 0u; });
    uint32_t order;
    int index;
    descend((double)p * (double)all, true, order, index);
    bound = order;
    until = index;
  }
  if (m > 0.f) {
    const double least = (double)fminf(m, 1.f);
    const uint32_t o = last_of(bound, top, [&](uint32_t o) {
      return o <= bound || exp(exponent(__uint_as_float((o >> 31) ? o ^ 0x80000000u : ~o))) < least;
    });
    // orders up to o weigh too little (o itself too, unless it is the bound and weighs enough)
    const bool bound_stays = exp(exponent(__uint_as_float((bound >> 31) ? bound ^ 0x80000000u : ~bound))) >= least;
    if (!(o == bound && bound_stays)) { bound = o + 1; until = V - 1; }
  }
  const uint64_t all = over([&](int i) { return kept(i) ? mass(i) : 0u; });
  const double target = fmin(fmax((double)u, 0.0), 1.0) * (double)all;
  int token;
  if ((double)all > target) {
    uint32_t order;
    if (nucleus) descend(target, false, order, token);
    else token = first_past([&](int i) { return kept(i) ? mass(i) : 0u; }, target);
  } else {                                      // the last that is kept and weighs something
    const auto left = [&](int i) { return kept(i) && mass(i) > 0; };
    const uint32_t order = nucleus ? last_of(bound, top, [&](uint32_t o) { return over([&](int i) { return (uint64_t)(left(i) && order_at(i) < o); }) == 0; }) : 0u;
    token = (int)last_of(0u, (uint32_t)V - 1, [&](uint32_t n) {
      return over([&](int i) { return (uint64_t)(i >= (int)n && left(i) && (!nucleus || order_at(i) == order)); }) > 0;
    });
  }
  if (t == 0) {
    a.tokens[row] = token;
    if (a.logprobs) a.logprobs[row] = (float)(exponent(Io<T>::ld(x, token)) - log((double)all / UNIT));
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
