// Keys and values in pages: appending those of new tokens (ah_paged_append, include/alpha_hip.h).
#include "common.h"
#include "paged.h"

using namespace ah;

namespace ah {

int32_t paged_cache(const char *who, const AhPages *p, int32_t rows, PagedCache *out) {
  AH_ARG(p, "%s: no pages", who);
  AH_ARG(p->dtype == AH_F32 || p->dtype == AH_BF16, "%s: pages of f32 or bf16, got dtype %d", who, p->dtype);
  AH_ARG(p->kv_heads >= 1 && p->kv_heads <= 65535, "%s: kv_heads %d is outside 1 .. 65535", who, p->kv_heads);
  AH_ARG(p->head_dim >= 8 && p->head_dim <= 128 && p->head_dim % 8 == 0, "%s: head_dim %d is no multiple of 8 from 8 to 128", who, p->head_dim);
  AH_ARG(p->page_rows >= 1 && p->page_rows <= 65536, "%s: page_rows %d is outside 1 .. 65536", who, p->page_rows);
  AH_ARG(p->seqs >= 0 && p->seqs <= 1 << 20 && p->table_pages >= 0 && p->pages >= 0 && p->pages <= INT32_MAX, "%s: %d sequences of %d pages, of %lld", who,
         p->seqs, p->table_pages, (long long)p->pages);
  AH_ARG(rows >= 0, "%s: %d rows", who, rows);
  const int64_t piece = p->dtype == AH_F32 ? 4 : 8;
  AH_ARG(p->page_stride % piece == 0 && p->row_stride % piece == 0 && p->head_stride % piece == 0, "%s: page strides of whole 16 bytes, got %lld, %lld, %lld", who,
         (long long)p->page_stride, (long long)p->row_stride, (long long)p->head_stride);
  AH_ARG(p->page_stride >= 0 && p->row_stride >= 0 && p->head_stride >= 0, "%s: page strides are not negative", who);
  AH_ARG(p->page_stride / piece <= INT32_MAX && p->row_stride / piece <= INT32_MAX && p->head_stride / piece <= INT32_MAX, "%s: page strides of 2^31 times 16 bytes and more", who);
  AH_ARG(aligned16(p->k) && aligned16(p->v) && p->table % 4 == 0 && p->starts % 4 == 0 && p->lens % 4 == 0, "%s: pages that are not 16-byte aligned", who);
  if (rows > 0 && p->seqs > 0)
    AH_ARG(p->starts && p->lens && ((p->k && p->v && p->table) || p->pages == 0 || p->table_pages == 0), "%s: a null page array, table, starts or lens", who);
  const int64_t capacity = p->pages == 0 ? 0 : (int64_t)p->table_pages * p->page_rows;
  *out = PagedCache{dp<const int32_t>(p->table), dp<const int32_t>(p->starts), dp<const int32_t>(p->lens), p->pages, p->page_stride, p->row_stride, p->head_stride,
                    (uint32_t)(p->page_stride / piece), (uint32_t)(p->row_stride / piece), quotient_by((uint32_t)p->page_rows), p->seqs, p->table_pages, rows, (int32_t)(capacity < MOST_POSITIONS ? capacity : MOST_POSITIONS)};
  return AH_OK;
}

}  // namespace ah

namespace {

// ------------------------------------------------------------------------------------------ append
// A workgroup takes a few rows.  Its first wave finds out where they go, all at once: three loads one after the other (the starts, the length and the starts
// of each row's sequence, the table's entry), whatever the rows.  Then every thread takes 16-byte pieces of heads, a pair of them where the turned features
// of a pair lie half a rotation apart.  Bound by those loads where there are few rows (one token 2.9 us, 192 of 32 heads of 128 on 8, turned, 4.7) and by
// memory where there are many: 18779 tokens of 16 heads of 128 on 4, fp32, read and written in 103 us, 4.5 TB/s (a copy of as much: 4.7), 9220 of 12 heads of 64,
// bf16, in 11 us, 5.2 TB/s.  1024 pieces to a workgroup: twice as many 109 us, half as many 107; two pieces of a thread under way at once 117.  Every workgroup looks through all
// starts: a token each of 1024 sequences 7.6 us, of 4096 21, of 16384 200.
constexpr int MOST_ROWS = 16;

struct AppendArgs {
  PagedCache c;
  void *k_pages, *v_pages;
  const void *q, *k, *v;
  void *rotated;
  const float *rotary;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, r_st, r_sh;
  int32_t heads, kv_heads, head_dim, rot, rot_rows;
  int32_t group;              // rows of a workgroup
  Quotient of_row;            // items of a row: those of the turned heads, q before k, then those of v
  Quotient of_turned;         // items of a turned head
  Quotient of_head;           // 16-byte pieces of a head
};
// How the turned heads are cut into items.  NONE: no rotation; HALVES: a piece of each half of the rotation, and the pieces behind it; NEIGHBOURS: pieces; ODD:
// two features, where the halves are no whole pieces, by loads and stores of one: 18779 tokens of 16 heads of 128 on 4, 60 of 128 turned, fp32 152 us, bf16 114 (64
// turned, HALVES, 98 and 63; bytes 99 and 50).
enum { NONE, HALVES, NEIGHBOURS, ODD };

template <class T> struct Piece;
template <> struct Piece<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const float *p, float (&x)[4]) { const float4 w = *reinterpret_cast<const float4 *>(p); x[0] = w.x; x[1] = w.y; x[2] = w.z; x[3] = w.w; }
  static __device__ __forceinline__ void put(float *p, const float (&x)[4]) { *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]); }
};
template <> struct Piece<uint16_t> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint16_t *p, float (&x)[8]) {
    const uint4 w = *reinterpret_cast<const uint4 *>(p);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) { x[2 * i] = __uint_as_float(u[i] << 16); x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
  }
  static __device__ __forceinline__ void put(uint16_t *p, const float (&x)[8]) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
  }
};
__device__ __forceinline__ void turn(float &a, float &b, float cosine, float sine) {
  const float x = a;
  a = fmaf(x, cosine, -(b * sine));
  b = fmaf(b, cosine, x * sine);
}

template <class T, int MODE>
__global__ __launch_bounds__(256) void k_paged_append(AppendArgs a) {
  constexpr int N = Piece<T>::N;
  __shared__ int64_t places[MOST_ROWS];         // elements from the start of the pages, negative: nowhere
  __shared__ int32_t positions[MOST_ROWS];      // INT32_MIN: a row of no sequence
  const int first = blockIdx.x * a.group, rows = min(a.group, a.c.rows - first);
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    int before = 0;                             // lane r: starts at or before row first + r
    for (int s0 = 0; s0 < a.c.seqs; s0 += 64) {
      const int start = s0 + lane < a.c.seqs ? a.c.starts[s0 + lane] : INT32_MAX;
      for (int r = 0; r < rows; r++) {
        const int n = __popcll(__ballot(start <= first + r));
        before += lane == r ? n : 0;
      }
    }
    if (lane < rows) {
      int64_t place = -1;
      int32_t position = INT32_MIN;
      if (before > 0) {
        const int seq = before - 1, row = first + lane;
        const Sequence s = sequence_of(a.c.starts[seq], a.c.starts[seq + 1], a.c.lens[seq], a.c.rows);
        if (row >= s.first && row < s.first + s.count) {
          position = s.len - s.count + (row - s.first);
          place = position_place(a.c, seq, position);
        }
      }
      places[lane] = place;
      positions[lane] = position;
    }
  }
  __syncthreads();
  const int half = a.rot / 2;
  const uint32_t turned = MODE == NONE ? 0u : (uint32_t)(a.heads + a.kv_heads) * a.of_turned.divisor;
  for (uint32_t i = threadIdx.x; i < (uint32_t)rows * a.of_row.divisor; i += 256) {
    const uint32_t r = quotient(i, a.of_row), item = i - r * a.of_row.divisor;
    const int64_t place = places[r], row = first + r;
    const int32_t position = positions[r];
    if (position == INT32_MIN) continue;
    if (MODE != NONE && item < turned) {
      const uint32_t h = quotient(item, a.of_turned), part = item - h * a.of_turned.divisor;
      const bool is_q = (int)h < a.heads;
      if (!is_q && place < 0) continue;
      const int kh = (int)h - a.heads;
      const T *src = is_q ? (const T *)a.q + row * a.q_st + h * a.q_sh : (const T *)a.k + row * a.k_st + kh * a.k_sh;
      T *dst = is_q ? (T *)a.rotated + row * a.r_st + h * a.r_sh : (T *)a.k_pages + place + kh * a.c.head_stride;
      const bool known = position >= 0 && position < a.rot_rows;
      const float *table = a.rotary + (known ? (int64_t)position * a.rot : 0);
      if constexpr (MODE == HALVES) {
        const int f = (int)part * N;
        if (f < half) {
          float x[N], y[N];
          Piece<T>::get(src + f, x);
          Piece<T>::get(src + f + half, y);
#pragma unroll
          for (int e = 0; e < N; e += 4) {
            float4 c = make_float4(NAN, NAN, NAN, NAN), s = c;
            if (known) { c = *reinterpret_cast<const float4 *>(table + f + e); s = *reinterpret_cast<const float4 *>(table + half + f + e); }
            turn(x[e], y[e], c.x, s.x); turn(x[e + 1], y[e + 1], c.y, s.y); turn(x[e + 2], y[e + 2], c.z, s.z); turn(x[e + 3], y[e + 3], c.w, s.w);
          }
          Piece<T>::put(dst + f, x);
          Piece<T>::put(dst + f + half, y);
        } else *reinterpret_cast<uint4 *>(dst + f + half) = *reinterpret_cast<const uint4 *>(src + f + half);
      } else if constexpr (MODE == NEIGHBOURS) {
        const int f = (int)part * N;
        if (f < a.rot) {
          float x[N];
          Piece<T>::get(src + f, x);
#pragma unroll
          for (int e = 0; e < N; e += 2)
            if (f + e < a.rot) turn(x[e], x[e + 1], known ? table[(f + e) / 2] : NAN, known ? table[half + (f + e) / 2] : NAN);
          Piece<T>::put(dst + f, x);
        } else *reinterpret_cast<uint4 *>(dst + f) = *reinterpret_cast<const uint4 *>(src + f);
      } else {
        const int p = (int)part, f = p < half ? p : 2 * p, g = p < half ? p + half : 2 * p + 1;
        if (p < half) {
          float x = Io<T>::ld(src, f), y = Io<T>::ld(src, g);
          turn(x, y, known ? table[p] : NAN, known ? table[half + p] : NAN);
          Io<T>::st(dst, f, x);
          Io<T>::st(dst, g, y);
        } else { dst[f] = src[f]; dst[g] = src[g]; }
      }
    } else if (place >= 0) {
      const uint32_t rest = item - turned, h = quotient(rest, a.of_head), f = (rest - h * a.of_head.divisor) * N;
      const bool is_k = MODE == NONE && (int)h < a.kv_heads;
      const int kh = MODE == NONE && !is_k ? (int)h - a.kv_heads : (int)h;
      const T *src = is_k ? (const T *)a.k + row * a.k_st + kh * a.k_sh : (const T *)a.v + row * a.v_st + kh * a.v_sh;
      T *dst = (T *)(is_k ? a.k_pages : a.v_pages) + place + kh * a.c.head_stride;
      *reinterpret_cast<uint4 *>(dst + f) = *reinterpret_cast<const uint4 *>(src + f);
    }
  }
}
template <class T>
int32_t append(AppendArgs &a, bool neighbours) {
  constexpr int N = Piece<T>::N;
  const uint32_t pieces = (uint32_t)(a.head_dim / N), half = (uint32_t)(a.rot / 2);
  const int mode = a.rot == 0 ? NONE : neighbours ? NEIGHBOURS : half % N == 0 ? HALVES : ODD;
  a.of_head = quotient_by(pieces);
  a.of_turned = quotient_by(mode == HALVES ? pieces - half / N : mode == ODD ? (uint32_t)a.head_dim / 2 : pieces);
  const int64_t items = mode == NONE ? (int64_t)2 * a.kv_heads * pieces
                                     : (int64_t)(a.heads + a.kv_heads) * a.of_turned.divisor + (int64_t)a.kv_heads * pieces;
  if (items > INT32_MAX / MOST_ROWS) return fail(AH_ERR_UNSUPPORTED, "ah_paged_append: %lld pieces to a row", (long long)items);
  a.of_row = quotient_by((uint32_t)items);
  const int64_t want = cdiv(1024, items), fill = cdiv(a.c.rows, (int64_t)4 * num_cus());
  a.group = (int32_t)(want < fill ? want : fill);
  if (a.group > MOST_ROWS) a.group = MOST_ROWS;
  const dim3 grid((unsigned)cdiv(a.c.rows, a.group));
  if (mode == NONE) launch_kernel(k_paged_append<T, NONE>, grid, dim3(256), 0, a);
  else if (mode == HALVES) launch_kernel(k_paged_append<T, HALVES>, grid, dim3(256), 0, a);
  else if (mode == NEIGHBOURS) launch_kernel(k_paged_append<T, NEIGHBOURS>, grid, dim3(256), 0, a);
  else launch_kernel(k_paged_append<T, ODD>, grid, dim3(256), 0, a);
  AH_LAUNCH_CHECK();
  return AH_OK;
}

}  // namespace

extern "C" {

int32_t ah_paged_append(const AhPages *p, const AhPagedAppend *d) {
  AH_ARG(d, "ah_paged_append: no new tokens");
  AppendArgs a{};
  if (const int32_t rc = paged_cache("ah_paged_append", p, d->rows, &a.c)) return rc;
  const int64_t piece = p->dtype == AH_F32 ? 4 : 8;
  AH_ARG(d->rot_dim >= 0 && d->rot_dim % 2 == 0 && d->rot_dim <= p->head_dim, "ah_paged_append: rot_dim %d is not even or past head_dim %d", d->rot_dim, p->head_dim);
  AH_ARG(d->k_st % piece == 0 && d->k_sh % piece == 0 && d->v_st % piece == 0 && d->v_sh % piece == 0 && aligned16(d->k) && aligned16(d->v),
         "ah_paged_append: k and v of whole 16 bytes to a row and head");
  if (d->rot_dim > 0) {
    AH_ARG(d->heads >= 0 && d->heads <= 65535 && d->rot_rows >= 0, "ah_paged_append: %d heads, %d positions of the rotation", d->heads, d->rot_rows);
    AH_ARG(d->q_st % piece == 0 && d->q_sh % piece == 0 && d->r_st % piece == 0 && d->r_sh % piece == 0 && aligned16(d->q) && aligned16(d->rotated) && aligned16(d->rotary),
           "ah_paged_append: q and rotated of whole 16 bytes to a row and head");
  } else
    AH_ARG(!d->q && !d->rotated && !d->rotary, "ah_paged_append: q, rotated and rotary are for a rotation (rot_dim > 0)");
  if (d->rows > 0 && p->seqs > 0) {
    AH_ARG(d->k && d->v, "ah_paged_append: k or v is null");
    AH_ARG(d->rot_dim == 0 || ((d->heads == 0 || (d->q && d->rotated)) && (d->rotary || d->rot_rows == 0)), "ah_paged_append: q, rotated or rotary is null");
  }
  AH_REQUIRE_READY();
  if (d->rows == 0 || p->seqs == 0) return AH_OK;
  a.k_pages = dp<void>(p->k); a.v_pages = dp<void>(p->v);
  a.q = dp<void>(d->q); a.k = dp<void>(d->k); a.v = dp<void>(d->v);
  a.rotated = dp<void>(d->rotated); a.rotary = dp<float>(d->rotary);
  a.q_st = d->q_st; a.q_sh = d->q_sh; a.k_st = d->k_st; a.k_sh = d->k_sh; a.v_st = d->v_st; a.v_sh = d->v_sh; a.r_st = d->r_st; a.r_sh = d->r_sh;
  a.heads = d->rot_dim > 0 ? d->heads : 0; a.kv_heads = p->kv_heads; a.head_dim = p->head_dim;
  a.rot = d->rot_dim; a.rot_rows = d->rot_rows;
  return p->dtype == AH_F32 ? append<float>(a, d->rot_neighbours != 0) : append<uint16_t>(a, d->rot_neighbours != 0);
}

}  // extern "C"
