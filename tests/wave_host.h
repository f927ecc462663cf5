// A workgroup of a kernel's own source on the CPU: a fiber to a thread, which gives way where it waits for its wave or its workgroup.  Each exchange between
// lanes is two meetings of the wave.  If nobody can go on, run() says so.
#pragma once
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <ucontext.h>
#include <bit>
#include <functional>
#include <vector>
#define __device__
#define __global__
#define __forceinline__ inline
#define __shared__ static
#define __launch_bounds__(...)
#define __host__
struct uint4 { uint32_t x, y, z, w; };
struct Dim { unsigned x; };
inline uint4 make_uint4(uint32_t x, uint32_t y, uint32_t z, uint32_t w) { return {x, y, z, w}; }
static thread_local Dim threadIdx, blockIdx;
namespace host {
struct Meeting { int here = 0, need = 0; uint64_t round = 0; };
struct Fiber { ucontext_t c; std::vector<char> stack; Meeting *at = nullptr; uint64_t round = 0; bool done = false; };
static ucontext_t boss;
static std::vector<Fiber> fibers;
static std::vector<Meeting> waves;
static Meeting block;
static int now;
static std::vector<uint64_t> box;          // what the lanes exchange
static std::function<void()> body;
inline void meet(Meeting &m) {
  Fiber &f = fibers[now];
  if (++m.here == m.need) { m.here = 0; m.round++; return; }
  f.at = &m; f.round = m.round;
  swapcontext(&f.c, &boss);
}
inline void meet_wave() { meet(waves[threadIdx.x / 64]); }
static void enter() { body(); fibers[now].done = true; swapcontext(&fibers[now].c, &boss); }
inline bool run(int threads, std::function<void()> f) {
  body = f;
  fibers = std::vector<Fiber>(threads);
  waves = std::vector<Meeting>(threads / 64);
  box.assign(threads, 0);
  for (auto &w : waves) w.need = 64;
  block = Meeting{}; block.need = threads;
  for (auto &x : fibers) {
    x.stack.resize(64 << 10);
    getcontext(&x.c);
    x.c.uc_stack.ss_sp = x.stack.data(); x.c.uc_stack.ss_size = x.stack.size(); x.c.uc_link = &boss;
    makecontext(&x.c, enter, 0);
  }
  for (;;) {
    int moved = 0, left = 0;
    for (int i = 0; i < threads; i++) {
      Fiber &x = fibers[i];
      if (x.done) continue;
      left++;
      if (x.at && x.at->round == x.round) continue;
      x.at = nullptr;
      now = i; threadIdx.x = i;
      swapcontext(&boss, &x.c);
      moved++;
    }
    if (!left) return true;
    if (!moved) return false;
  }
}
template <class V> inline V exchange(V v, int from) {
  static_assert(sizeof(V) <= 8);
  uint64_t raw = 0; memcpy(&raw, &v, sizeof(V));
  const int me = threadIdx.x;
  box[me] = raw; meet_wave();
  raw = box[me / 64 * 64 + from]; meet_wave();
  threadIdx.x = me;
  memcpy(&v, &raw, sizeof(V));
  return v;
}
}
#define __syncthreads() host::meet(host::block)
#define __builtin_amdgcn_fence(a, b) host::meet_wave()
template <class V> inline V __shfl(V v, int from) { return host::exchange(v, from & 63); }
template <class V> inline V __shfl_xor(V v, int o) { return host::exchange(v, (threadIdx.x & 63) ^ o); }
template <class V> inline V __shfl_up(V v, int o) { const int l = threadIdx.x & 63; return host::exchange(v, l >= o ? l - o : l); }
inline int __builtin_amdgcn_readfirstlane(int v) { return __shfl(v, 0); }
inline uint64_t __ballot(bool b) { uint64_t r = 0; const int me = threadIdx.x; host::box[me] = b; host::meet_wave(); for (int i = 0; i < 64; i++) r |= host::box[me / 64 * 64 + i] << i; host::meet_wave(); return r; }
inline int __builtin_amdgcn_readlane(int v, int from) { return __shfl(v, from); }
inline int __builtin_amdgcn_update_dpp(int old, int v, int ctrl, int rows, int, bool) {
  const int lane = threadIdx.x & 63, row = lane / 16;
  const int from = ctrl >= 0x111 && ctrl <= 0x11f ? (lane % 16 >= (ctrl & 15) ? lane - (ctrl & 15) : -1) : ctrl == 0x142 ? row * 16 - 1 : ctrl == 0x143 ? 31 : -1;
  const int got = __shfl(v, from < 0 ? 0 : from);
  return from >= 0 && (rows >> row & 1) ? got : old;
}
inline bool __any(bool b) { return __ballot(b) != 0; }
inline float __builtin_amdgcn_fmed3f(float a, float b, float c) { return a != a || b != b || c != c ? fminf(fminf(a, b), c) : fmaxf(fminf(a, b), fminf(fmaxf(a, b), c)); }
template <int O> inline uint32_t lane_xor(uint32_t v) { return __shfl_xor(v, O); }
inline float wave_max(float v) { for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o)); return v; }
inline uint32_t __float_as_uint(float f) { return std::bit_cast<uint32_t>(f); }
inline float __uint_as_float(uint32_t u) { return std::bit_cast<float>(u); }
inline int __clz(int x) { return x ? __builtin_clz((unsigned)x) : 32; }
template <class V, class W> inline V atomicAdd(V *p, W v) { const V o = *p; *p += (V)v; return o; }
inline float unsafeAtomicAdd(float *p, float v) { const float o = *p; *p += v; return o; }
#define __builtin_amdgcn_exp2f exp2f
template <class T> T max(T a, T b) { return a > b ? a : b; }
template <class T> T min(T a, T b) { return a < b ? a : b; }
template <class T> struct Io;
template <> struct Io<float> { static float ld(const float *p, size_t i) { return p[i]; } };
template <> struct Io<uint16_t> { static float ld(const uint16_t *p, size_t i) { return std::bit_cast<float>((uint32_t)p[i] << 16); } };
namespace ah {}
