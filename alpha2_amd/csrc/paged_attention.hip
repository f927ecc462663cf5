// Attention of new tokens over keys and values in pages (ah_paged_attention, include/alpha_hip.h).
//
// Mathematics.  For a new token with limit n (the positions it sees, 0 .. n - 1):
//   x_j = scale q.k_j (capped: cap tanh(x_j / cap)),  o = sum_j e^(x_j - m) v_j / sum_j e^(x_j - m),  lse = m + log sum_j e^(x_j - m)
// in one pass over j with the running maximum m, sum l and product o, all in fp32; where the positions are cut into parts, each part leaves
// its (m, l, o) and a second kernel joins them: m = max m_i, l = sum l_i e^(m_i - m), o = sum o_i e^(m_i - m).
// bf16 pages: a weight e^(x_j - m) is rounded to bf16 for the product with v_j, which is what the matrix instructions take (as in attention_bf16.hip; fp32 products would be
// at an eighth of their rate), and goes into l as it was.  Outputs are 2.2e-3 off 64 bits (root mean square, relative), 1.7e-3 of them by their own rounding.
//
// Work.  The heads that share keys are rows of one matrix: a COLUMN is a (new token, head of the group), column i of a sequence token
// i / group, head i % group.  A workgroup takes one unit: TILE columns of a sequence, one kv head, one part of the positions.  Which unit that is
// follows from starts and lens on the device (find_unit), so the lengths need not be known on the host and a captured launch follows them.  Where tiles are few the positions
// are cut (parts as long as the launch's work over the workgroups wanted, those of a sequence as long as each other), so that contexts of any lengths end together; where the
// tiles alone are as many as the GPU takes at once, nothing is, however much longer than the others one context is (attend).
//
// Two kernels for each type; both compute every case, which is taken is a matter of speed (ah_paged_attention):
//   keys   16 columns; the four waves take tiles of positions in turn and are joined in LDS.  For one or a few new tokens a sequence, where the
//          launch is bound by reading the pages once: 16 columns are the fewest that the matrix instructions take, most of them idle for one token.
//   rows   bf16: 128 columns, the waves own 32 each and stream the same positions through LDS; fp32: 32 columns, otherwise as keys.  For chunks and
//          prompts, bound by the matrix and vector pipes.
//
// Masked places.  A position past a column's limit has its score replaced by -infinity, whatever it was.  Its value would still meet a weight of 0
// in the matrix product, and 0 x infinity is NaN; so rows past the part's end are zeros, and where some columns see a row that others do
// not (tiles on the diagonal) values that are not finite are taken as 0 in the product and added, as they are, to the columns that see them, behind the loop.
// A page that the table has wrong reads as NaN keys and zero values: whoever sees it gets NaN, nobody else.
#include "attention_bf16_tiles.h"
#include "paged.h"

using namespace ah;

namespace {

struct Plan {
  int32_t target;             // units that the positions of all tiles are cut into, about; 0: no cutting
  int32_t least;              // positions of a part, at least
  int32_t whole;              // a sequence of as many is not cut
  float  *parts;              // what the units of tiles with more than one part leave: see part_at
};
struct AttendArgs {
  PagedCache c;
  Plan plan;
  const void *k, *v, *q;
  void *o;
  float *lse;
  int64_t q_st, q_sh, o_st, o_sh;
  int32_t heads, kv_heads, group, head_dim;
  float scale, cap;
};

struct Unit {
  Sequence s;
  int32_t seq, tile;          // -1: no such unit
  int32_t part, parts;        // parts that hold positions which a column of the tile sees (at least one)
  int32_t span;               // positions of a part, at most: the launch's
  int32_t own;                // and this sequence's, whose parts are as long as each other
  int32_t first;              // the tile's first unit
  // the positions that column `i` of the sequence sees
  __device__ __forceinline__ int limit(int i, int group) const { return s.len - s.count + i / group + 1; }
};
template <int TILE>
__device__ __forceinline__ int tiles_of(const Sequence &s, int group) { return (int)(((int64_t)s.count * group + TILE - 1) / TILE); }

__device__ __forceinline__ int parts_of(int positions, int span) { return positions <= span ? 1 : (positions - 1) / span + 1; }
__device__ __forceinline__ int parts_of(const Sequence &s, const PagedCache &c, const Plan &plan, int span) {
  const int reach = min(s.len, c.capacity);
  return reach <= plan.whole ? 1 : parts_of(reach, span);
}

// Unit `index` of the launch, or (by_tile) tile `index`, by a whole wave; the same for all its lanes.  A lane looks at a sequence, and every workgroup at all of
// them: what that takes grows with the square of their number.  A token each after 64 positions, 8 heads of 64 on 1: 192 sequences 7.5 us, 1024 19, 4096 146, 16384 1900
// (their bytes 0.8, 4, 16 and 65).
template <int TILE>
__device__ __forceinline__ Unit find_unit(const PagedCache &c, const Plan &plan, int group, int index, bool by_tile) {
  const int lane = threadIdx.x & 63;
  auto sequence = [&](int s) { return s < c.seqs ? sequence_of(c.starts[s], c.starts[s + 1], c.lens[s], c.rows) : Sequence{0, 0, 0}; };
  Unit u{};
  u.seq = -1;
  u.span = INT32_MAX;
  Sequence mine = sequence(lane);
  if (plan.target > 0) {
    double work = 0;
    for (int s0 = 0; s0 < c.seqs; s0 += 64) {
      const Sequence s = s0 ? sequence(s0 + lane) : mine;
      work += (double)tiles_of<TILE>(s, group) * min(s.len, c.capacity);
    }
    if (c.seqs > 1) work = wave_sum_d(work);
    else work = __shfl(work, 0);
    const double span = fmax(ceil(work / plan.target), (double)plan.least);
    u.span = span < 2147483584.0 ? ((int)span + 63) / 64 * 64 : INT32_MAX;
  }
  int base = 0;
  for (int s0 = 0; s0 < c.seqs; s0 += 64) {
    if (s0) mine = sequence(s0 + lane);
    const int tiles = tiles_of<TILE>(mine, group), parts = parts_of(mine, c, plan, u.span);
    int count = by_tile ? tiles : tiles * parts, upto = count;
    if (c.seqs > 1)
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) { const int x = __shfl_up(upto, o); upto += lane >= o ? x : 0; }
    const uint64_t past = __ballot(base + upto > index);
    if (past) {
      const int at = __builtin_ctzll(past);
      const int before = base + __shfl(upto - count, at), p = __shfl(parts, at), n = __shfl(tiles, at);
      u.s = Sequence{__shfl(mine.first, at), __shfl(mine.count, at), __shfl(mine.len, at)};
      u.seq = s0 + at;
      const int local = index - before, t = by_tile ? local : local / p;
      u.tile = n - 1 - t;                                            // the last tiles of a prompt, which see most, come first
      u.part = by_tile ? 0 : local - t * p;
      u.first = by_tile ? 0 : before + t * p;
      const int last = min((u.tile + 1) * TILE, u.s.count * group) - 1;
      const int seen = min(u.limit(last, group), c.capacity);
      const int reach = min(u.s.len, c.capacity);
      u.own = p > 1 ? ((reach - 1) / p + 64) / 64 * 64 : INT32_MAX;  // (at most span, a multiple of 64 as well)
      u.parts = parts_of(seen, u.own);
      // (by tile, the units before it are those of all tiles before it)
      if (by_tile) u.first = t * p;
      break;
    }
    base += __shfl(upto, 63);
  }
  // all lanes hold the same: scalars from here on
  auto scalar = [](int &v) { v = __builtin_amdgcn_readfirstlane(v); };
  scalar(u.s.first); scalar(u.s.count); scalar(u.s.len);
  scalar(u.seq); scalar(u.tile); scalar(u.part); scalar(u.parts); scalar(u.span); scalar(u.own); scalar(u.first);
  return u;
}

// Where a unit's part is kept: TILE columns of D products, then TILE maxima, then TILE sums
template <int TILE, int D>
__device__ __forceinline__ float *part_at(const Plan &p, int64_t slot) { return p.parts + slot * (TILE * (D + 2)); }

// ------------------------------------------------------------------------------------------ pages
constexpr int64_t NO_PAGE = -1, NO_ROW = -2;         // a position whose page does not exist; one past the end
// the table's entry for a position (0 where there is none to read)
__device__ __forceinline__ int32_t page_entry(const PagedCache &c, const int32_t *__restrict__ table, int position, int end) {
  return position < end ? table[quotient((uint32_t)position, c.page_rows)] : 0;
}
__device__ __forceinline__ int64_t place_of(const PagedCache &c, int32_t page, int position, int end) {
  const uint32_t row = (uint32_t)position - quotient((uint32_t)position, c.page_rows) * c.page_rows.divisor;
  const int64_t at = page_place(c, page, row);
  return position < end ? at : NO_ROW;
}
constexpr uint32_t NAN_PAIR = 0x7fc07fc0u;
__device__ __forceinline__ u32x4 piece_or(const uint16_t *base, int64_t place, int feature, bool inside, uint32_t missing) {
  const uint32_t other = place == NO_PAGE && inside ? missing : 0u;
  u32x4 x = {other, other, other, other};
  if (place >= 0 && inside) x = *reinterpret_cast<const u32x4 *>(base + place + feature);
  return x;
}

// ------------------------------------------------------------------------------------------ values that are not finite, bf16
__device__ __forceinline__ bool has_special(bf16x8 v) {
  const u32x4 w = __builtin_bit_cast(u32x4, v);
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) any |= (w[i] & 0x7f807f80u) + 0x00800080u;
  return (any & 0x80008000u) != 0;
}
__device__ __forceinline__ bf16x8 finite_of(bf16x8 v) {             // 0 in their place
  u32x4 w = __builtin_bit_cast(u32x4, v);
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t low = (w[i] & 0x7f80u) == 0x7f80u ? 0u : 0xffffu, high = (w[i] & 0x7f800000u) == 0x7f800000u ? 0u : 0xffff0000u;
    w[i] &= low | high;
  }
  return __builtin_bit_cast(bf16x8, w);
}
__device__ __forceinline__ float special_of(float v, bool seen) { return seen && !(fabsf(v) < INFINITY) ? v : 0.f; }
// The same address, as far as the compiler knows another one: what the seldom taken path reads from LDS is not kept in registers for the usual one.
__device__ __forceinline__ const char *apart(const char *p) {
  int offset = 0;
  asm volatile("" : "+v"(offset));
  return p + offset;
}
// the four values from `feature` on at a place, those that are not finite; 0 for the others
__device__ __forceinline__ void special4(const uint16_t *v, float (&x)[4], bool seen) {
  const uint2 w = *reinterpret_cast<const uint2 *>(v);
  x[0] = special_of(__uint_as_float(w.x << 16), seen); x[1] = special_of(__uint_as_float(w.x & 0xffff0000u), seen);
  x[2] = special_of(__uint_as_float(w.y << 16), seen); x[3] = special_of(__uint_as_float(w.y & 0xffff0000u), seen);
}

// ------------------------------------------------------------------------------------------ joining
// The finished column: o and lse, or one unit's part of them.  m in units of `natural` (its logarithm's base), l the sum of weights.
__device__ __forceinline__ float column_sum(float l, int limit, int reach) { return limit > reach ? NAN : l; }      // a position that no table entry names
template <class T> __device__ __forceinline__ void store4(T *p, float a, float b, float c, float d);
template <> __device__ __forceinline__ void store4<float>(float *p, float a, float b, float c, float d) { *reinterpret_cast<float4 *>(p) = make_float4(a, b, c, d); }
template <> __device__ __forceinline__ void store4<uint16_t>(uint16_t *p, float a, float b, float c, float d) {
  *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16x2(a, b), pack_bf16x2(c, d));
}
constexpr float LN2 = 0.693147180559945309f;

// Joins the parts of a tile: a thread to four features of a column.  Few columns can have many parts: there four waves share them, each its own sum with its
// own running maximum, and are joined in LDS; a workgroup has 64 such fours.  A tile of rows has many columns, and a workgroup 256 fours of it.
// One sequence of 32768, 8 kv heads of 128, in 96 parts: 35 us with attention, one wave to 64 fours 45; four of 8192, 32 columns each in a tile of 128: 39 us where a
// workgroup of 256 threads joins a whole tile 63.
constexpr int join_ways(int tile) { return tile <= 32 ? 4 : 1; }
constexpr int join_slices(int tile, int d) { return tile * d / 4 * join_ways(tile) / 256; }
template <class T, int TILE, int D>
__global__ __launch_bounds__(256) void k_paged_join(AttendArgs a) {
  constexpr int SLICES = join_slices(TILE, D), WAYS = join_ways(TILE), ITEMS = 256 / WAYS;
  __shared__ float4 products[WAYS][ITEMS];
  __shared__ float tops[WAYS][ITEMS], sums[WAYS][ITEMS];
  const int index = blockIdx.x / SLICES, head = index % a.kv_heads, slice = blockIdx.x % SLICES;
  // the units of the tiles before this one have to be known: find_unit by tile gives those of the sequence, the others are added up here
  const Unit u = find_unit<TILE>(a.c, a.plan, a.group, index / a.kv_heads, true);
  if (u.seq < 0 || u.parts == 1) return;
  const int columns = u.s.count * a.group;
  if (u.tile * TILE + slice * ITEMS / (D / 4) >= columns) return;          // (all of the workgroup)
  const int way = threadIdx.x / ITEMS, item = threadIdx.x % ITEMS, e = slice * ITEMS + item, col = e / (D / 4), f = e % (D / 4) * 4, i = u.tile * TILE + col;
  int before = 0;
  for (int s0 = 0; s0 < u.seq; s0 += 64) {
    const int s = s0 + (threadIdx.x & 63);
    if (s < u.seq) {
      const Sequence x = sequence_of(a.c.starts[s], a.c.starts[s + 1], a.c.lens[s], a.c.rows);
      before += tiles_of<TILE>(x, a.group) * parts_of(x, a.c, a.plan, u.span);
    }
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) before += __shfl_xor(before, o);
  const int64_t first = before + u.first;
  const bool some = i < columns && f < a.head_dim;
  const int64_t pitch = (int64_t)a.kv_heads * (TILE * (D + 2));
  const float *part = part_at<TILE, D>(a.plan, first * a.kv_heads + head), *stats = part + TILE * D + col;
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto join = [&](float more_m, float more_l, const float4 &x) {
    const float top = fmaxf(m, more_m), shift = top == -INFINITY ? 0.f : top, keep = exp2_fast(m - shift), w = exp2_fast(more_m - shift);
    l = fmaf(more_l, w, l * keep);
    o.x = fmaf(x.x, w, o.x * keep); o.y = fmaf(x.y, w, o.y * keep); o.z = fmaf(x.z, w, o.z * keep); o.w = fmaf(x.w, w, o.w * keep);
    m = top;
  };
  if (some)
#pragma unroll 4
    for (int p = way; p < u.parts; p += WAYS) join(stats[p * pitch], stats[p * pitch + TILE], *reinterpret_cast<const float4 *>(part + p * pitch + col * D + f));
  if constexpr (WAYS > 1) {
    products[way][item] = o;
    tops[way][item] = m;
    sums[way][item] = l;
    __syncthreads();
    if (way) return;
#pragma unroll
    for (int w = 1; w < WAYS; w++) join(tops[w][item], sums[w][item], products[w][item]);
  }
  if (!some) return;
  l = column_sum(l, u.limit(i, a.group), a.c.capacity);
  const int64_t row = u.s.first + i / a.group, h = (int64_t)head * a.group + i % a.group;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  store4<T>((T *)a.o + row * a.o_st + h * a.o_sh + f, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  if (f == 0 && a.lse) a.lse[row * a.heads + h] = l == 0.f ? -INFINITY : fmaf(m, LN2, logf(l));
}

// ------------------------------------------------------------------------------------------ the cap
// tanh as in attention.hip (where the polynomial's origin and both errors stand): up to 0.625, and beyond.  A last place of the cap is one of the score, whatever
// the score is, if tanh is 1 - 2 / (e^(2 x) + 1) throughout: the bf16 kernels take that up to FIXED_MAX_CAP, where it is 4e-6, and this above.  Chunks of 1024 in
// 8192, 32 heads of 128 on 8: the one 341 us, the other 432; 16 heads of 64, 144 and 188; a token each of 16 sequences of 8192, 122 and 123, of 8 of 1000, 13.5 and 13.9.
constexpr float TANH_SMALL = 0.625f;
__device__ __forceinline__ float tanh_small(float x) {
  const float z = x * x;
  float p = -0.005704985465854406f;
  p = fmaf(p, z, 0.02063908614218235f);
  p = fmaf(p, z, -0.05373971536755562f);
  p = fmaf(p, z, 0.13331441581249237f);
  p = fmaf(p, z, -0.3333328068256378f);
  return fmaf(x * z, p, x);
}
__device__ __forceinline__ float tanh_large(float x) { return copysignf(fmaf(-2.0f, rcp_fast(exp2_fast(fabsf(x) * (2.0f * LOG2E)) + 1.0f), 1.0f), x); }
__device__ __forceinline__ float tanh_any(float x) { return fabsf(x) < TANH_SMALL ? tanh_small(x) : tanh_large(x); }

// ------------------------------------------------------------------------------------------ keys, bf16
// v_mfma_f32_16x16x32_bf16: S^T[32 positions, 16 columns] = K Q^T in two halves of 16, a lane holding positions 16 i + 4 g + r (g = lane / 16, r < 4) of column
// lane % 16.  Those are, as they lie, the B operand of O^T[16 features, 16 columns] += V^T P^T when its slot 8 g + 4 i + r is taken to mean that
// position; the A operand is read from V's tile in the same order (ds_read_b64_tr_b16 of four rows).  K goes from the pages straight into its operand's
// registers (16 rows of 64 bytes to an instruction), V through LDS that is the wave's own, so that no wave waits for another before the end.
// Bound by the pages: a token each of 24 sequences of up to 24000 positions, 32 heads of 128 on 8, 246 us, 5.0 TB/s; of one sequence of 777, 12 heads of 64, by the
// loads that wait for each other (lengths, table, page) and the two launches: 10.1 us, 7.2 and 3.7 of them in the kernels.
template <int D> struct KeysTile {
  static constexpr int PITCH = D + 16, V_BYTES = 32 * PITCH * 2, O_PITCH = D + 4, O_BYTES = 16 * O_PITCH * 4;
  static constexpr int WAVE_BYTES = V_BYTES > O_BYTES ? V_BYTES : O_BYTES;
};

template <int D, int MODE>                       // 0: no cap; 1: one up to FIXED_MAX_CAP; 2: a larger one
__global__ __launch_bounds__(256, 2) void k_paged_keys_bf16(AttendArgs a) {
  using G = KeysTile<D>;
  constexpr int KS = D / 32, DB = D / 16, NV = D / 16, TILE = 16;
  __shared__ __attribute__((aligned(16))) char own[4 * G::WAVE_BYTES];
  __shared__ float tops[4][TILE], sums[4][TILE];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int head = blockIdx.x % a.kv_heads;
  const Unit u = find_unit<TILE>(a.c, a.plan, a.group, blockIdx.x / a.kv_heads, false);
  if (u.seq < 0 || (u.part > 0 && u.part >= u.parts)) return;
  const int columns = u.s.count * a.group, i = u.tile * TILE + col, last = min((u.tile + 1) * TILE, columns) - 1;
  const int limit = i < columns ? u.limit(i, a.group) : 0;
  const int least = u.limit(u.tile * TILE, a.group);                 // every column sees the positions before this one
  const int begin = u.parts > 1 ? u.part * u.own : 0;
  const int seen = min(u.limit(last, a.group), a.c.capacity), end = u.parts > 1 ? min(begin + u.own, seen) : seen;
  const uint16_t *K = (const uint16_t *)a.k + head * a.c.head_stride, *V = (const uint16_t *)a.v + head * a.c.head_stride;
  const int32_t *table = a.c.table + (int64_t)u.seq * a.c.table_pages;
  uint16_t *tile = (uint16_t *)(own + wave * G::WAVE_BYTES);

  bf16x8 q[KS];
  {
    const int64_t row = u.s.first + i / a.group, h = (int64_t)head * a.group + i % a.group;
    const uint16_t *p = (const uint16_t *)a.q + row * a.q_st + h * a.q_sh;
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
      u32x4 x = {0u, 0u, 0u, 0u};
      if (i < columns && ks * 32 + g * 8 < a.head_dim) x = *reinterpret_cast<const u32x4 *>(p + ks * 32 + g * 8);
      q[ks] = __builtin_bit_cast(bf16x8, x);
    }
  }
  // MODE 1: e^(2 x / cap) = 2^(c1 s), and the score in base 2 is c2 - 2 c2 / (that + 1); 2: it is c2 tanh(c1 s); 0: c1 s
  const float c1 = MODE == 1 ? 2.0f * a.scale * LOG2E / a.cap : MODE == 2 ? a.scale / a.cap : a.scale * LOG2E, c2 = a.cap * LOG2E;
  f32x4 o[DB];
#pragma unroll
  for (int d = 0; d < DB; d++) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  bool specials = false;

  u32x4 kr[2][KS], vr[NV];
  auto load = [&](int32_t page, int base) {        // a tile's rows: lane r (and r + 32) looks after position base + r
    const int64_t place = place_of(a.c, page, base + (lane & 31), end);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int64_t at = __shfl(place, 16 * h + col);
#pragma unroll
      for (int ks = 0; ks < KS; ks++) kr[h][ks] = piece_or(K, at, ks * 32 + g * 8, ks * 32 + g * 8 < a.head_dim, NAN_PAIR);
    }
#pragma unroll
    for (int n = 0; n < NV; n++) {
      const int c = lane + 64 * n, f = c % (D / 8) * 8;
      vr[n] = piece_or(V, __shfl(place, c / (D / 8)), f, f < a.head_dim, 0u);
    }
  };
  const int stride = 4 * 32;
  int base = begin + wave * 32;
  int32_t page = page_entry(a.c, table, base + (lane & 31), end), next = page_entry(a.c, table, base + stride + (lane & 31), end);
  if (base < end) load(page, base);
  for (; base < end; base += stride) {
    bf16x8 k[2][KS];
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int ks = 0; ks < KS; ks++) k[h][ks] = __builtin_bit_cast(bf16x8, kr[h][ks]);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");           // the tile's last reads are done
#pragma unroll
    for (int n = 0; n < NV; n++) {
      const int c = lane + 64 * n;
      *reinterpret_cast<u32x4 *>(tile + c / (D / 8) * G::PITCH + c % (D / 8) * 8) = vr[n];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (base + stride < end) {
      page = next;
      next = page_entry(a.c, table, base + 2 * stride + (lane & 31), end);
      load(page, base + stride);
    }
    f32x4 s[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      s[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ks++) s[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[h][ks], q[ks], s[h], 0, 0, 0);
    }
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int r = 0; r < 4; r++) s[h][r] = MODE == 1 ? fmaf(-2.0f * c2, rcp_fast(exp2_fast(s[h][r] * c1) + 1.0f), c2) : MODE == 2 ? c2 * tanh_any(s[h][r] * c1) : s[h][r] * c1;
    const bool edge = base + 32 > min(least, end);
    if (edge) {
      keep_branch();
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int r = 0; r < 4; r++) s[h][r] = base + 16 * h + 4 * g + r < min(limit, end) ? s[h][r] : -INFINITY;
    }
    float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    top = max_lane<16>(max_lane<32>(top));
    if (__any(top > m)) {
      const float larger = fmaxf(m, top), keep = exp2_fast(m - (larger == -INFINITY ? 0.f : larger));
      l *= keep;
#pragma unroll
      for (int d = 0; d < DB; d++)
#pragma unroll
        for (int r = 0; r < 4; r++) o[d][r] *= keep;
      m = larger;
    }
    const float shift = m == -INFINITY ? 0.f : m;
    bf16x8 p;
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const float w = exp2_fast(s[h][r] - shift);
        l += w;
        p[4 * h + r] = (__bf16)w;
      }
    auto values = [&](const uint16_t *from, int d) {
      const uint16_t *at = from + (4 * g + (col >> 2)) * G::PITCH + 16 * d + 4 * (col & 3);
      const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_v4 *)at), hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_v4 *)(at + 16 * G::PITCH));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    bool special = false;
    if (edge && least < end) {                                       // some columns see less than others
      keep_branch();
#pragma unroll 1
      for (int d = 0; d < DB; d++) special |= has_special(values((const uint16_t *)apart((const char *)tile), d));
      special = __any(special);
      specials |= special;
    }
    if (!special) {
#pragma unroll
      for (int d = 0; d < DB; d++) o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(values(tile, d), p, o[d], 0, 0, 0);
    } else {
      const uint16_t *again = (const uint16_t *)apart((const char *)tile);
#pragma unroll
      for (int d = 0; d < DB; d++) o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(finite_of(values(again, d)), p, o[d], 0, 0, 0);
    }
  }
  if (specials) {
    keep_branch();
    for (int b = begin + wave * 32; b < end; b += stride)
      for (int kv = b; b + 32 > least && kv < min(b + 32, end); kv++) {
        const int64_t at = position_place(a.c, u.seq, kv);
        if (at < 0) continue;
#pragma unroll
        for (int d = 0; d < DB; d++) {
          if (16 * d + 4 * g >= a.head_dim) continue;
          float x[4];
          special4(V + at + 16 * d + 4 * g, x, kv < limit);
#pragma unroll
          for (int r = 0; r < 4; r++) o[d][r] += x[r];
        }
      }
  }

  // the four waves: weights relative to the largest of their maxima
  l = add_lane<16>(add_lane<32>(l));
  if (g == 0) { tops[wave][col] = m; sums[wave][col] = l; }
  __syncthreads();
  {
    const float top = fmaxf(fmaxf(tops[0][col], tops[1][col]), fmaxf(tops[2][col], tops[3][col]));
    const float w = exp2_fast(m - (top == -INFINITY ? 0.f : top));
    float *mine = (float *)(own + wave * G::WAVE_BYTES) + col * G::O_PITCH + 4 * g;
#pragma unroll
    for (int d = 0; d < DB; d++) *reinterpret_cast<float4 *>(mine + 16 * d) = make_float4(o[d][0] * w, o[d][1] * w, o[d][2] * w, o[d][3] * w);
  }
  __syncthreads();
  float *part = part_at<TILE, D>(a.plan, ((int64_t)u.first + u.part) * a.kv_heads + head);
  for (int e = threadIdx.x; e < TILE * D / 4; e += 256) {
    const int c = e / (D / 4), f = e % (D / 4) * 4, ci = u.tile * TILE + c;
    if (ci >= columns || f >= a.head_dim) continue;
    const float top = fmaxf(fmaxf(tops[0][c], tops[1][c]), fmaxf(tops[2][c], tops[3][c])), shift = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const float4 y = *reinterpret_cast<const float4 *>((const float *)(own + w * G::WAVE_BYTES) + c * G::O_PITCH + f);
      sum = fmaf(sums[w][c], exp2_fast(tops[w][c] - shift), sum);
      x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
    }
    if (u.parts > 1) {
      *reinterpret_cast<float4 *>(part + c * D + f) = x;
      if (f == 0) { part[TILE * D + c] = top; part[TILE * D + TILE + c] = sum; }
    } else {
      sum = column_sum(sum, u.limit(ci, a.group), a.c.capacity);
      const int64_t row = u.s.first + ci / a.group, h = (int64_t)head * a.group + ci % a.group;
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;
      store4<uint16_t>((uint16_t *)a.o + row * a.o_st + h * a.o_sh + f, x.x * inv, x.y * inv, x.z * inv, x.w * inv);
      if (f == 0 && a.lse) a.lse[row * a.heads + h] = sum == 0.f ? -INFINITY : fmaf(top, LN2, logf(sum));
    }
  }
}

// ------------------------------------------------------------------------------------------ rows, bf16
// Four waves of 32 columns on v_mfma_f32_32x32x16_bf16 (operands as in attention_bf16.hip), K and V in LDS in tiles of 64 positions, two of them in turn,
// one barrier to a tile.  The tiles come by global_load_lds, 16 bytes to a lane from wherever its position's page lies, past the registers; what does not
// exist is fetched from rows of zeros or NaN.  A wave's 1 KB lands in lane order, so rows cannot be padded: the 16-byte pieces of a row are permuted instead
// (by the lane that fetches them), so that 16 rows' same piece and four rows' same 64 bytes each meet all 64 banks.
// The two tiles are arrays of their own, and the loop is written out for both: an LDS read that may touch what a load under way writes waits for it, and
// the compiler keeps them apart by the array.  Both halves of a tile's scores are taken together, so that the values (whose reads wait all the same) come
// late.  Two sequences, chunks of 2048 and 1200 behind 14336 and 5058 positions, 32 heads of 128 on 8: 702 us, 890 TFLOP/s of the 1218 that a large product
// reaches; before page and row were the wave's, 746; one array and a half at a time, 791; the values' finite form chosen in the loop and not in LDS, 989.  Bound by the vector
// instructions of the softmax and by waiting between them and the matrix ones, two waves to a SIMD.
// MODE 0: no cap; 1: a cap up to 40, whose softmax takes the cap itself for the maximum (attention_bf16.hip); 2: a larger cap.
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) const void glb_void;
__device__ __attribute__((aligned(16))) const uint32_t nothing[3][4] = {{0u, 0u, 0u, 0u}, {NAN_PAIR, NAN_PAIR, NAN_PAIR, NAN_PAIR}, {0x7fc00000u, 0x7fc00000u, 0x7fc00000u, 0x7fc00000u}};      // (bf16, fp32)

template <int D> struct RowsTile {
  static constexpr int PIECES = D / 8, ROW = 2 * D, BYTES = ST * ROW;         // 16-byte pieces of a row, bytes
  static constexpr int LOADS = ST * PIECES / 256;                             // of a wave for K, and for V
  static __device__ __forceinline__ int turned(int row) {                     // what a row's piece numbers are XORed with
    if constexpr (PIECES == 16) return (row & 3) << 2 | (row >> 2 & 3);
    else if constexpr (PIECES == 8) return (row >> 1 & 1) << 2 | (row >> 2 & 3);
    else return row >> 2 & 3;
  }
};

template <int D, int MODE, bool WHOLE>
__global__ __launch_bounds__(256, 2) void k_paged_rows_bf16(AttendArgs a) {
  using G = RowsTile<D>;
  constexpr int DB = D / 32, KS = D / 16, TILE = 128, N = G::LOADS;
  constexpr bool CAPPED = MODE == 1;
  __shared__ __attribute__((aligned(1024))) char Ks0[G::BYTES], Vs0[G::BYTES], Ks1[G::BYTES], Vs1[G::BYTES];
  __shared__ int specials;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, lr = lane & 31, lk = lane >> 5;
  const int head = blockIdx.x % a.kv_heads;
  const Unit u = find_unit<TILE>(a.c, a.plan, a.group, blockIdx.x / a.kv_heads, false);
  if (u.seq < 0 || (u.part > 0 && u.part >= u.parts)) return;
  const int columns = u.s.count * a.group, i0 = u.tile * TILE + wave * 32, i = i0 + lr;
  const int last = min((u.tile + 1) * TILE, columns) - 1, wave_last = min(i0 + 31, columns - 1);
  const int begin = u.parts > 1 ? u.part * u.own : 0;
  const int seen = min(u.limit(last, a.group), a.c.capacity), end = u.parts > 1 ? min(begin + u.own, seen) : seen;
  const int wave_end = wave_last < i0 ? 0 : min(u.limit(wave_last, a.group), end), least = u.limit(min(i0, columns - 1), a.group);
  const int limit = i < columns ? min(u.limit(i, a.group), end) : 0;          // positions that the column sees of these
  const uint16_t *K = (const uint16_t *)a.k + head * a.c.head_stride, *V = (const uint16_t *)a.v + head * a.c.head_stride;
  const int32_t *table = a.c.table + (int64_t)u.seq * a.c.table_pages;
  // MODE 0: the score in base 2 is c1 s, c1 > 0 (a negative scale turns q's sign; a masked s, -infinity, times a scale of 0 would be NaN).  1: e^(2 x / cap) = 2^(c1 s), the score is c2 - 2 c2 / (that + 1);
  // 2: c2 tanh(c1 s)
  const float c1 = MODE == 1 ? 2.0f * a.scale * LOG2E / a.cap : MODE == 2 ? a.scale / a.cap : fmaxf(fabsf(a.scale) * LOG2E, 0x1p-126f), c2 = a.cap * LOG2E;
  const float ic2 = MODE == 1 ? -1.0f / (2.0f * c2) : 0.f;                    // and 2^(-2 c2 r) with -2 c2 r = 1 / ((e + 1) ic2)
  const float slope = MODE ? 1.f : c1;

  bf16x8 qf[KS];
  const int64_t row = u.s.first + i / a.group, h = (int64_t)head * a.group + i % a.group;
#pragma unroll
  for (int ks = 0; ks < KS; ks++) {
    u32x4 x = {0u, 0u, 0u, 0u};
    if (i < columns && ks * 16 + lk * 8 < a.head_dim) x = *reinterpret_cast<const u32x4 *>((const uint16_t *)a.q + row * a.q_st + h * a.q_sh + ks * 16 + lk * 8);
    if (MODE == 0 && a.scale < 0.f) x ^= u32x4{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
    qf[ks] = __builtin_bit_cast(bf16x8, x);
  }
  f32x16 o[DB];
#pragma unroll
  for (int d = 0; d < DB; d++)
#pragma unroll
    for (int e = 0; e < 16; e++) o[d][e] = 0.f;
  float m = CAPPED ? c2 : -INFINITY, l = 0.f;
  if (threadIdx.x == 0) specials = 0;
  const int all_see = u.limit(u.tile * TILE, a.group);                        // every column of the workgroup sees the positions before this one

  // What this lane fetches: piece `lane % PIECES`, as it lands, of row base + its_row(n).  Positions past the end look at the last one's entry, so that nothing
  // here branches: page and row in 16-byte pieces, one multiplication each, and the row of zeros or NaN where they name no place.
  // WHOLE: pages of a multiple of 64 positions hold whole tiles (which begin at multiples of 64): page and row are the wave's, and a lane has only its place
  // in the tile to add.
  auto its_row = [&](int n) { return (wave * N + n) * (64 / G::PIECES) + lane / G::PIECES; };
  uint32_t entry[N], line[N], tile_entry = 0, tile_line = 0;
  uint64_t in_tile[N];
#pragma unroll
  for (int n = 0; n < N; n++) in_tile[n] = ((uint64_t)(uint32_t)its_row(n) * a.c.row_pieces + (uint32_t)(lane % G::PIECES ^ G::turned(its_row(n)))) * 16;
  auto entries = [&](int base) {
    if (WHOLE) {
      const uint32_t p = (uint32_t)min(base, end - 1), page = quotient(p, a.c.page_rows);
      tile_entry = (uint32_t)table[page];
      tile_line = p - page * a.c.page_rows.divisor;
      return;
    }
#pragma unroll
    for (int n = 0; n < N; n++) {
      const uint32_t p = (uint32_t)min(base + its_row(n), end - 1), page = quotient(p, a.c.page_rows);
      entry[n] = (uint32_t)table[page];
      line[n] = p - page * a.c.page_rows.divisor;
    }
  };
  const uint32_t pages = (uint32_t)a.c.pages;
  auto load = [&](char *kt, char *vt, int base) {
    if (WHOLE && base + ST <= end && tile_entry < pages) {
      const uint64_t at = ((uint64_t)tile_entry * a.c.page_pieces + (uint64_t)tile_line * a.c.row_pieces) * 16;
#pragma unroll
      for (int n = 0; n < N; n++) {
        __builtin_amdgcn_global_load_lds((glb_void *)((const char *)K + at + in_tile[n]), (lds_void *)(kt + (wave * N + n) * 1024), 16, 0, 0);
        __builtin_amdgcn_global_load_lds((glb_void *)((const char *)V + at + in_tile[n]), (lds_void *)(vt + (wave * N + n) * 1024), 16, 0, 0);
      }
      return;
    }
#pragma unroll
    for (int n = 0; n < N; n++) {
      const int r = its_row(n);
      const uint32_t its_entry = WHOLE ? tile_entry : entry[n], its_line = WHOLE ? tile_line + r : line[n];
      const uint32_t piece = (uint32_t)(lane % G::PIECES ^ G::turned(r));
      const uint64_t at = (uint64_t)its_entry * a.c.page_pieces + ((uint64_t)its_line * a.c.row_pieces + piece);
      const bool wanted = base + r < end && (int)piece * 8 < a.head_dim, there = its_entry < pages;
      const uint16_t *k = (const uint16_t *)nothing[0], *v = k;
      k = wanted ? there ? K + at * 8 : (const uint16_t *)nothing[1] : k;
      v = wanted && there ? V + at * 8 : v;
      __builtin_amdgcn_global_load_lds((glb_void *)k, (lds_void *)(kt + (wave * N + n) * 1024), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((glb_void *)v, (lds_void *)(vt + (wave * N + n) * 1024), 16, 0, 0);
    }
  };
  const int k_turned = G::turned(lr);
  auto keys = [&](const char *tile, int sub, int ks) {             // A operand: row sub + lr, features 16 ks + 8 lk ..
    return *reinterpret_cast<const bf16x8 *>(tile + (sub + lr) * G::ROW + ((2 * ks + lk) ^ k_turned) * 16);
  };
  const int vj = lane & 15, vg = lane >> 4, v_row = 4 * (vg >> 1) + (vj >> 2), v_piece = 2 * (vg & 1) + (vj >> 1 & 1);
  const int v_turned = G::turned(v_row), v_turned8 = G::turned(v_row + 8);
  auto values = [&](const char *tile, int sub, int m_, int d) {    // A operand: feature 32 d + lane % 32, k-slot i row sub + 16 m + 8 (i / 4) + 4 lk + i % 4
    const char *at = tile + (sub + 16 * m_ + v_row) * G::ROW + (vj & 1) * 8;
    const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_v4 *)(at + ((4 * d + v_piece) ^ v_turned) * 16));
    const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_v4 *)(at + 8 * G::ROW + ((4 * d + v_piece) ^ v_turned8) * 16));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  if (begin < end) {
    entries(begin);
    load(Ks0, Vs0, begin);
    entries(begin + ST);
  }
  auto step = [&](char *kt, char *vt, char *next_kt, char *next_vt, int base) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");               // this tile is there, for all behind the barrier
    __syncthreads();
    if (base + ST < end) {
      load(next_kt, next_vt, base + ST);
      entries(base + 2 * ST);
    }
    if (base + ST > all_see && all_see < end) {
      bool some = false;
#pragma unroll
      for (int e = 0; e < G::BYTES; e += 256 * 16) {
        bf16x8 *at = reinterpret_cast<bf16x8 *>(vt + e + threadIdx.x * 16);
        const bool special = has_special(*at);
        if (special) *at = finite_of(*at);
        some |= special;
      }
      if (some) specials = 1;
      __syncthreads();
    }
    if (base >= wave_end) return;                                  // (the same for the wave) nothing for its columns
    f32x16 s[2];
#pragma unroll
    for (int b = 0; b < 2; b++) {
#pragma unroll
      for (int e = 0; e < 16; e++) s[b][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ks++) s[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(keys(kt, 32 * b, ks), qf[ks], s[b], 0, 0, 0);
    }
    const bool edge = base + ST > min(least, end);
    if (MODE == 1) {
#pragma unroll
      for (int b = 0; b < 2; b++)
#pragma unroll
        for (int e = 0; e < 16; e++) s[b][e] = exp2_fast(rcp_fast(fmaf(exp2_fast(s[b][e] * c1), ic2, ic2)));
      if (edge) {
        keep_branch();
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
          for (int e = 0; e < 16; e++) s[b][e] = base + 32 * b + 8 * (e >> 2) + 4 * lk + (e & 3) < limit ? s[b][e] : 0.f;
      }
    } else {
      if (MODE == 2) {
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
          for (int e = 0; e < 16; e++) s[b][e] = c2 * tanh_any(s[b][e] * c1);
      }
      if (edge) {
        keep_branch();
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
          for (int e = 0; e < 16; e++) s[b][e] = base + 32 * b + 8 * (e >> 2) + 4 * lk + (e & 3) < limit ? s[b][e] : -INFINITY;
      }
      float top = s[0][0];
#pragma unroll
      for (int b = 0; b < 2; b++)
#pragma unroll
        for (int e = 0; e < 16; e++) top = fmaxf(top, s[b][e]);
      top = max_lane<32>(top);
      if (__any(top > m)) {
        const float larger = fmaxf(m, top), keep = exp2_fast((m - (larger == -INFINITY ? 0.f : larger)) * slope);
        l *= keep;
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
          for (int e = 0; e < 16; e++) o[d][e] *= keep;
        m = larger;
      }
      const float shift = (m == -INFINITY ? 0.f : -m) * slope;
#pragma unroll
      for (int b = 0; b < 2; b++)
#pragma unroll
        for (int e = 0; e < 16; e++) s[b][e] = exp2_fast(fmaf(s[b][e], slope, shift));
    }
#pragma unroll
    for (int b = 0; b < 2; b++) {
      const bf16x8 p0 = acc_to_b(s[b], 0), p1 = acc_to_b(s[b], 1);
#pragma unroll
      for (int e = 0; e < 16; e++) l += s[b][e];
#pragma unroll
      for (int d = 0; d < DB; d++) {
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(values(vt, 32 * b, 0, d), p0, o[d], 0, 0, 0);
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(values(vt, 32 * b, 1, d), p1, o[d], 0, 0, 0);
      }
    }
  };
  for (int base = begin; base < end; base += 2 * ST) {
    step(Ks0, Vs0, Ks1, Vs1, base);
    if (base + ST < end) step(Ks1, Vs1, Ks0, Vs0, base + ST);
  }
  __syncthreads();
  if (specials) {
    keep_branch();
    for (int kv = all_see > begin ? begin + (all_see - begin) / ST * ST : begin; kv < wave_end; kv++) {
      const int64_t at = position_place(a.c, u.seq, kv);
      if (at < 0) continue;
#pragma unroll
      for (int d = 0; d < DB; d++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          asm volatile("" ::: "memory");                           // (one after the other: few registers)
          if (32 * d + 8 * j + 4 * lk >= a.head_dim) continue;
          float x[4];
          special4(V + at + 32 * d + 8 * j + 4 * lk, x, kv < limit);
#pragma unroll
          for (int r = 0; r < 4; r++) o[d][4 * j + r] += x[r];
        }
    }
  }
  l = add_lane<32>(l);
  if (CAPPED && l == 0.f) m = -INFINITY;
  if (MODE == 0 && m > -INFINITY) m *= c1;                           // (to base 2)
  if (i >= columns) return;
  if (u.parts > 1) {
    float *part = part_at<TILE, D>(a.plan, ((int64_t)u.first + u.part) * a.kv_heads + head);
    const int c = wave * 32 + lr;
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
      for (int j = 0; j < 4; j++)
        *reinterpret_cast<float4 *>(part + c * D + 32 * d + 8 * j + 4 * lk) = make_float4(o[d][4 * j], o[d][4 * j + 1], o[d][4 * j + 2], o[d][4 * j + 3]);
    if (lk == 0) { part[TILE * D + c] = m; part[TILE * D + TILE + c] = l; }
    return;
  }
  l = column_sum(l, u.limit(i, a.group), a.c.capacity);
  store_rows<D, true>((uint16_t *)a.o + row * a.o_st + h * a.o_sh, o, l == 0.f ? 0.f : 1.0f / l, lane, a.head_dim);
  if (lk == 0 && a.lse) a.lse[row * a.heads + h] = l == 0.f ? -INFINITY : fmaf(m, LN2, logf(l));
}

// ------------------------------------------------------------------------------------------ fp32
// v_mfma_f32_16x16x4_f32, nothing through LDS before the end: a tile is 16 positions, S^T[16 positions, 16 columns] = K Q^T, whose slot g of
// instruction (j, c) is taken to mean feature 16 j + 4 g + c, so that both operands are 16-byte loads; a lane then holds positions 4 g + r of column
// lane % 16, the B operand of O^T += V^T P^T whose slot g of instruction r means that position, and the A operand's row n of block (h, c) is taken
// to mean feature W (16 h + n) + c with W = min(4, D / 16), so that V's pieces are 16-byte loads (8 at D = 32) of whole rows too.
// The waves take tiles in turn and are joined, for NC = 1 block of columns (keys) and for 2 (rows): no wave waits for another before the end, and
// each piece of a page is read once by a workgroup.  With 32 columns to a wave, each streaming all positions, a batch of prompts of 12 heads of 64
// took 254 us; with the positions cut, 168, and with one block as long, but chunks of 512 in 4096 positions, 16 heads of 64: 398 us, two 369 (88 TFLOP/s of
// the 154 that fp32 products reach; the exponentials and the loads' addresses are in the way); heads of 128: 1144 and 972.  As it stands, lengths and
// wave numbers in scalar registers: 148, 344 (94 TFLOP/s), 796; the matrix pipes are busy half of the time.  One token each: a batch of 20 of up to 512
// positions, 8 heads of 48, 14 us, the loads that wait for each other; 40 of 5000, 32 heads of 128 on 8, 286 us, 5.7 TB/s (with one workgroup to a compute unit, which 256 registers and more would mean, 4 of 8192 take
// 63 us, not 55).
template <int D, int NC>
__global__ __launch_bounds__(256, D <= 64 || NC == 1 ? 2 : 1) void k_paged_f32(AttendArgs a) {
  constexpr int KQ = D / 16, W = D >= 64 ? 4 : 2, VH = D / (16 * W), DB = D / 16, TILE = 16 * NC, O_PITCH = D + 4;
  __shared__ __attribute__((aligned(16))) float joined[4 * TILE * O_PITCH];
  __shared__ float tops[4][TILE], sums[4][TILE];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int head = blockIdx.x % a.kv_heads;
  const Unit u = find_unit<TILE>(a.c, a.plan, a.group, blockIdx.x / a.kv_heads, false);
  if (u.seq < 0 || (u.part > 0 && u.part >= u.parts)) return;
  const int columns = u.s.count * a.group, i0 = u.tile * TILE;
  const int last = min((u.tile + 1) * TILE, columns) - 1;
  const int begin = u.parts > 1 ? u.part * u.own : 0;
  const int seen = min(u.limit(last, a.group), a.c.capacity), end = u.parts > 1 ? min(begin + u.own, seen) : seen;
  const int least = u.limit(i0, a.group);
  const float *K = (const float *)a.k + head * a.c.head_stride, *V = (const float *)a.v + head * a.c.head_stride;
  const int32_t *table = a.c.table + (int64_t)u.seq * a.c.table_pages;
  const float factor = a.cap > 0.f ? a.scale / a.cap : a.scale;

  int limit[NC];
  f32x4 q[NC][KQ], o[NC][DB];
  float m[NC], l[NC];
#pragma unroll
  for (int n = 0; n < NC; n++) {
    const int i = i0 + 16 * n + col;
    limit[n] = i < columns ? min(u.limit(i, a.group), end) : 0;
    const float *p = (const float *)a.q + (u.s.first + (int64_t)(i / a.group)) * a.q_st + ((int64_t)head * a.group + i % a.group) * a.q_sh;
#pragma unroll
    for (int j = 0; j < KQ; j++) {
      q[n][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (i < columns && 16 * j + 4 * g < a.head_dim) q[n][j] = *reinterpret_cast<const f32x4 *>(p + 16 * j + 4 * g);
    }
#pragma unroll
    for (int d = 0; d < DB; d++) o[n][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    m[n] = -INFINITY;
    l[n] = 0.f;
  }

  bool specials = false;
  f32x4 kr[KQ];
  float vr[4][VH][W];
  // Lane l looks after position base + l % 16: the table's entry (past the end, the last one's) and the row in its page; no branches, as in the rows' kernel.
  const uint32_t pages = (uint32_t)a.c.pages;
  auto entry_at = [&](int base, uint32_t &line) {
    const uint32_t p = (uint32_t)max(0, min(base + col, end - 1)), page = quotient(p, a.c.page_rows);
    line = p - page * a.c.page_rows.divisor;
    return end > 0 ? (uint32_t)table[page] : 0u;
  };
  auto load = [&](uint32_t page, uint32_t line, int base) {
    const uint64_t at = (uint64_t)page * a.c.page_pieces + (uint64_t)line * a.c.row_pieces;
    const bool wanted = base + col < end, there = page < pages;
    const float *k = wanted && there ? K + at * 4 : (const float *)nothing[wanted ? 2 : 0];
    const uint64_t place = wanted && there ? at : ~0ull;
#pragma unroll
    for (int j = 0; j < KQ; j++) {
      const bool inside = 16 * j + 4 * g < a.head_dim;
      const float *p = wanted && there ? k + 16 * j + 4 * g : k;
      kr[j] = *reinterpret_cast<const f32x4 *>(inside ? p : (const float *)nothing[0]);
    }
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const uint64_t row = __shfl(place, 4 * g + r);
#pragma unroll
      for (int h = 0; h < VH; h++) {
        const int f = W * (16 * h + col);
        typedef __attribute__((ext_vector_type(W))) float piece;
        const piece x = *reinterpret_cast<const piece *>(row != ~0ull && f < a.head_dim ? V + row * 4 + f : (const float *)nothing[0]);
#pragma unroll
        for (int c = 0; c < W; c++) vr[r][h][c] = x[c];
      }
    }
  };
  int base = begin + wave * 16;
  uint32_t line, next_line, next = entry_at(base + 64, next_line);
  {
    const uint32_t first = entry_at(base, line);
    if (base < end) load(first, line, base);
  }
  for (; base < end; base += 64) {
    f32x4 k[KQ];
    float v[4][VH][W];
#pragma unroll
    for (int j = 0; j < KQ; j++) k[j] = kr[j];
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
      for (int h = 0; h < VH; h++)
#pragma unroll
        for (int c = 0; c < W; c++) v[r][h][c] = vr[r][h][c];
    if (base + 64 < end) {
      const uint32_t page = next;
      line = next_line;
      next = entry_at(base + 128, next_line);
      load(page, line, base + 64);
    }
    const bool edge = base + 16 > min(least, end);
    bool special = false;
    if (edge && least < end) {                        // some columns see less than others
      keep_branch();
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int h = 0; h < VH; h++)
#pragma unroll
          for (int c = 0; c < W; c++) special |= !(fabsf(v[r][h][c]) < INFINITY);
      if (__any(special)) {
        specials = true;
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
          for (int h = 0; h < VH; h++)
#pragma unroll
            for (int c = 0; c < W; c++) v[r][h][c] = fabsf(v[r][h][c]) < INFINITY ? v[r][h][c] : 0.f;
      }
    }
#pragma unroll
    for (int n = 0; n < NC; n++) {
      f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < KQ; j++)
#pragma unroll
        for (int c = 0; c < 4; c++) s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[j][c], q[n][j][c], s, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; r++) s[r] *= factor;
      if (a.cap > 0.f) {
        const f32x4 x = s;
        const float most = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
#pragma unroll
        for (int r = 0; r < 4; r++) s[r] = a.cap * tanh_small(x[r]);
        if (__any(!(most < TANH_SMALL))) {            // (scores are seldom near the cap)
          keep_branch();
#pragma unroll
          for (int r = 0; r < 4; r++) s[r] = fabsf(x[r]) < TANH_SMALL ? s[r] : a.cap * tanh_large(x[r]);
        }
      }
      if (edge) {
        keep_branch();
#pragma unroll
        for (int r = 0; r < 4; r++) s[r] = base + 4 * g + r < limit[n] ? s[r] : -INFINITY;
      }
      float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
      top = max_lane<16>(max_lane<32>(top));
      if (__any(top > m[n])) {
        const float larger = fmaxf(m[n], top), keep = exp2_fast((m[n] - (larger == -INFINITY ? 0.f : larger)) * LOG2E);
        l[n] *= keep;
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
          for (int r = 0; r < 4; r++) o[n][d][r] *= keep;
        m[n] = larger;
      }
      const float shift = m[n] == -INFINITY ? 0.f : m[n];
#pragma unroll
      for (int r = 0; r < 4; r++) { s[r] = exp2_fast((s[r] - shift) * LOG2E); l[n] += s[r]; }
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int h = 0; h < VH; h++)
#pragma unroll
          for (int c = 0; c < W; c++) o[n][W * h + c] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[r][h][c], s[r], o[n][W * h + c], 0, 0, 0);
    }
  }
  if (specials) {
    keep_branch();
    for (int b = begin + wave * 16; b < end; b += 64)
      for (int kv = b; b + 16 > least && kv < min(b + 16, end); kv++) {
        const int64_t at = position_place(a.c, u.seq, kv);
        if (at < 0) continue;
#pragma unroll
        for (int h = 0; h < VH; h++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            const int f = W * (16 * h + 4 * g + r);
            if (f >= a.head_dim) continue;
#pragma unroll
            for (int c = 0; c < W; c++) {
              const float x = V[at + f + c];
#pragma unroll
              for (int n = 0; n < NC; n++) o[n][W * h + c][r] += special_of(x, kv < limit[n]);
            }
          }
      }
  }
  // a lane has features W (16 h + 4 g + r) + c of its column in element r of block W h + c
#pragma unroll
  for (int n = 0; n < NC; n++) {
    const float mine = add_lane<16>(add_lane<32>(l[n]));
    if (g == 0) { tops[wave][16 * n + col] = m[n]; sums[wave][16 * n + col] = mine; }
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NC; n++) {
    const int c0 = 16 * n + col;
    const float top = fmaxf(fmaxf(tops[0][c0], tops[1][c0]), fmaxf(tops[2][c0], tops[3][c0]));
    const float w = exp2_fast((m[n] - (top == -INFINITY ? 0.f : top)) * LOG2E);
    float *to = joined + (wave * TILE + c0) * O_PITCH;
#pragma unroll
    for (int h = 0; h < VH; h++)
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int c = 0; c < W; c++) to[W * (16 * h + 4 * g + r) + c] = o[n][W * h + c][r] * w;
  }
  __syncthreads();
  float *part = part_at<TILE, D>(a.plan, ((int64_t)u.first + u.part) * a.kv_heads + head);
  for (int e = threadIdx.x; e < TILE * D / 4; e += 256) {
    const int c = e / (D / 4), f = e % (D / 4) * 4, ci = u.tile * TILE + c;
    if (ci >= columns || f >= a.head_dim) continue;
    const float top = fmaxf(fmaxf(tops[0][c], tops[1][c]), fmaxf(tops[2][c], tops[3][c])), shift = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const float4 y = *reinterpret_cast<const float4 *>(joined + (w * TILE + c) * O_PITCH + f);
      sum = fmaf(sums[w][c], exp2_fast((tops[w][c] - shift) * LOG2E), sum);
      x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
    }
    if (u.parts > 1) {
      *reinterpret_cast<float4 *>(part + c * D + f) = x;
      if (f == 0) { part[TILE * D + c] = top * LOG2E; part[TILE * D + TILE + c] = sum; }
    } else {
      sum = column_sum(sum, u.limit(ci, a.group), a.c.capacity);
      const int64_t row = u.s.first + ci / a.group, h = (int64_t)head * a.group + ci % a.group;
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;
      store4<float>((float *)a.o + row * a.o_st + h * a.o_sh + f, x.x * inv, x.y * inv, x.z * inv, x.w * inv);
      if (f == 0 && a.lse) a.lse[row * a.heads + h] = sum == 0.f ? -INFINITY : top + logf(sum);
    }
  }
}
// ------------------------------------------------------------------------------------------ launches
// Parts go through the library's scratch (64 MB from ah_init on, ordered with everything else on the main stream), of which a launch takes at most this.
constexpr int64_t PART_BYTES = int64_t(60) << 20;

// TILE columns to a unit: how many workgroups, and how many of them the positions are cut for.  Two workgroups fit a compute unit; where the tiles alone
// are as many, nothing is cut (64 sequences of 1024, 8 kv heads of 128, bf16: 44 us, 53 us cut), and the join is not launched either where the table
// cannot name more positions than a part has.  That rule sees no lengths: 63 sequences of 500 beside one of 24000, the same heads, take 477 us, the one by itself 29, and 47
// beside it, which are cut, 53; 15 of 300 beside one of 32768, 32 kv heads, 656 us, the one by itself 109.  Otherwise about `wanted` units are cut: more of them even out ragged sequences, fewer are fewer to join.
template <class T, int TILE, int D, class Kernel>
int32_t attend(AttendArgs a, Kernel kernel, int64_t wanted, int32_t least, int32_t whole) {
  // of one kv head, at most: every sequence with new tokens may end inside a tile
  const int64_t ends = a.c.seqs < a.c.rows ? a.c.seqs : a.c.rows, tiles = ((int64_t)a.c.rows * a.group + ends * (TILE - 1)) / TILE;
  const int64_t slot = (int64_t)TILE * (D + 2) * sizeof(float) * a.kv_heads;
  const int64_t cus = num_cus();
  int64_t target = 0;
  if (tiles * a.kv_heads < 2 * cus && a.c.capacity > whole) {
    target = cdiv(wanted, a.kv_heads);
    if ((tiles + target) * slot > PART_BYTES) target = PART_BYTES / slot - tiles;
    if (target < 1) target = 0;
  }
  if (target > 0) {
    a.plan.target = (int32_t)target;
    a.plan.least = least;
    a.plan.whole = whole;
    a.plan.parts = (float *)scratch((size_t)((tiles + target) * slot));
    if (!a.plan.parts) return fail(AH_ERR_OOM, "ah_paged_attention: no scratch for the parts of long sequences");
  }
  // parts are as many as positions over the launch's own length of a part, which is at least work / target, and at least `least`; and the rest of each
  const int64_t parts = cdiv(a.c.capacity, least), units = target == 0 ? tiles : tiles * parts < tiles + target ? tiles * parts : tiles + target;
  const int64_t grid = units * a.kv_heads;
  if (grid > INT32_MAX) return fail(AH_ERR_UNSUPPORTED, "ah_paged_attention: %lld workgroups", (long long)grid);
  launch_kernel(kernel, dim3((unsigned)grid), dim3(256), 0, a);
  AH_LAUNCH_CHECK();
  if (target > 0) {
    launch_kernel(k_paged_join<T, TILE, D>, dim3((unsigned)(tiles * a.kv_heads * join_slices(TILE, D))), dim3(256), 0, a);
    AH_LAUNCH_CHECK();
  }
  return AH_OK;
}
template <int D>
int32_t attend_sized(const AttendArgs &a, bool bf16_pages) {
  // Columns of a sequence, in the mean.  At 32 the two are even (bf16, 4 x 8192 positions, 8 kv heads of 128: 40 and 39 us; fp32, 4 x 1024, 12 of 64: 19.0
  // and 19.6); at 48, 60 and 44 us; at 256, 182 and 74.  The other way, 16 columns: 35 and 39 us.
  // The mean is the launch's, so a prompt beside single tokens may go through tiles of 16 columns, or they through its own.  bf16, 8 heads of 128, 63 tokens after 500 positions
  // and a prompt of 1900 (keys) 73 us, of 2048 (rows) 78, in two calls 25 and 38; on 32 heads, 41 (400 new, keys), 44 (600, rows) and 82 (2048), in two 26 and 22, 33, 66.
  // Sequences without new tokens count: a chunk of 2048 in 8192 positions, 8 heads of 128, 86 us, beside 62 idle ones, with fewer parts, 215, beside 63 (keys) 291.
  const bool rows = (int64_t)a.c.rows * a.group > (int64_t)32 * a.c.seqs;
  const int64_t cus = num_cus();
  // Units wanted, of keys: three to a compute unit, 246 us at 24 ragged sequences of up to 24000 positions (8 kv heads of 128, bf16), two, 276, four, 245; at
  // four equal ones of 8192, 36, 31 and 36.
  // fp32 heads of more than 64, two workgroups to a compute unit as well: 4 of 8192 (8 kv heads) 61 us with three, 55 with four, 3 of 24000 (16) 226 and 203.
  // A part has 256 positions at least, and what has no more than 512 is not cut: 500 positions of 12 heads of 64, bf16, 8.7 us, in two parts, which have to be
  // joined, 10.0; 1000 in four, 10.1, in two 12.4.  fp32 heads of more than 64 are slower to get through: 500 whole, 20.9, in two parts 17.0.
  // Rows, whose units are longer, are cut down to 128: 12 tokens after 500 (8 kv heads of 128), 13.9 us against 18.7 with 256.
  if (bf16_pages) {
    if (!rows) return attend<uint16_t, 16, D>(a, a.cap > FIXED_MAX_CAP ? k_paged_keys_bf16<D, 2> : a.cap > 0.f ? k_paged_keys_bf16<D, 1> : k_paged_keys_bf16<D, 0>, 3 * cus, 256, 512);
    // Tiles inside a page are fetched by the wave's address where a row has 16 pieces and more: chunks of 2048 and 1200, 32 heads of 128, in pages of 64
    // positions 702 us, position by position 760; heads of 64, the same; of 32, 33 and 31.
    constexpr bool MANY = D > 64;
    if (MANY && a.c.page_rows.divisor % ST == 0 && a.head_dim == D)
      return attend<uint16_t, 128, D>(a, a.cap > FIXED_MAX_CAP ? k_paged_rows_bf16<D, 2, MANY> : a.cap > 0.f ? k_paged_rows_bf16<D, 1, MANY> : k_paged_rows_bf16<D, 0, MANY>, 2 * cus, 128, 128);
    return attend<uint16_t, 128, D>(a, a.cap > FIXED_MAX_CAP ? k_paged_rows_bf16<D, 2, false> : a.cap > 0.f ? k_paged_rows_bf16<D, 1, false> : k_paged_rows_bf16<D, 0, false>,
                                    2 * cus, 128, 128);
  }
  if (!rows) return attend<float, 16, D>(a, k_paged_f32<D, 1>, (D <= 64 ? 3 : 4) * cus, 256, D <= 64 ? 512 : 256);
  return attend<float, 32, D>(a, k_paged_f32<D, 2>, 3 * cus, 256, D <= 64 ? 512 : 256);
}

}  // namespace

extern "C" int32_t ah_paged_attention(const AhPages *p, const AhPagedAttention *d) {
  AH_ARG(d, "ah_paged_attention: no queries");
  AttendArgs a{};
  if (const int32_t rc = paged_cache("ah_paged_attention", p, d->rows, &a.c)) return rc;
  const int64_t piece = p->dtype == AH_F32 ? 4 : 8;
  AH_ARG(d->heads >= p->kv_heads && d->heads <= 65535 && d->heads % p->kv_heads == 0, "ah_paged_attention: %d heads are no multiple of the pages' %d", d->heads, p->kv_heads);
  AH_ARG((int64_t)d->rows * (d->heads / p->kv_heads) <= INT32_MAX / 2, "ah_paged_attention: %d rows of %d heads to a kv head", d->rows, d->heads / p->kv_heads);
  AH_ARG(d->q_st % piece == 0 && d->q_sh % piece == 0 && d->o_st % piece == 0 && d->o_sh % piece == 0 && aligned16(d->q) && aligned16(d->o) && d->lse % 4 == 0,
         "ah_paged_attention: q and o of whole 16 bytes to a row and head");
  AH_ARG(d->soft_cap >= 0.f && d->soft_cap < INFINITY && d->scale == d->scale, "ah_paged_attention: soft_cap %g, scale %g", d->soft_cap, d->scale);
  AH_ARG(d->rows == 0 || p->seqs == 0 || (d->q && d->o), "ah_paged_attention: q or o is null");
  AH_REQUIRE_READY();
  if (d->rows == 0 || p->seqs == 0) return AH_OK;
  a.k = dp<void>(p->k); a.v = dp<void>(p->v); a.q = dp<void>(d->q); a.o = dp<void>(d->o); a.lse = dp<float>(d->lse);
  a.q_st = d->q_st; a.q_sh = d->q_sh; a.o_st = d->o_st; a.o_sh = d->o_sh;
  a.heads = d->heads; a.kv_heads = p->kv_heads; a.group = d->heads / p->kv_heads; a.head_dim = p->head_dim;
  a.scale = d->scale;
  a.cap = d->soft_cap < 0x1p40f ? d->soft_cap : 0.f;                 // (a score would have to pass 2^28 for such a cap to move it by its last place)
  // Under a cap of 2^-40 scores are 0 to the last place of their exponential; a smaller one's reciprocal may be infinite, and 0 times that NaN.
  if (a.cap > 0.f && a.cap < 0x1p-40f) a.cap = 0x1p-40f;
  const bool bf16_pages = p->dtype == AH_BF16;
  return p->head_dim <= 32 ? attend_sized<32>(a, bf16_pages) : p->head_dim <= 64 ? attend_sized<64>(a, bf16_pages) : attend_sized<128>(a, bf16_pages);
}
