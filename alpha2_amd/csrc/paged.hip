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
  AH_ARG(aligned16(p->k) && aligned16(p->v) && p->table % 4 == 0 && p->starts % 4 == 0 && p->lens % 4 == 0, "%s: pages that are not 16-byte aligned", who);
  if (rows > 0 && p->seqs > 0)
    AH_ARG(p->starts && p->lens && ((p->k && p->v && p->table) || p->pages == 0 || p->table_pages == 0), "%s: a null page array, table, starts or lens", who);
  const int64_t capacity = p->pages == 0 ? 0 : (int64_t)p->table_pages * p->page_rows;
  *out = PagedCache{dp<const int32_t>(p->table), dp<const int32_t>(p->starts), dp<const int32_t>(p->lens), p->pages, p->page_stride, p->row_stride, p->head_stride,
                    quotient_by((uint32_t)p->page_rows), p->seqs, p->table_pages, rows, (int32_t)(capacity < MOST_POSITIONS ? capacity : MOST_POSITIONS)};
  return AH_OK;
}

}  // namespace ah

namespace {

// The sequence that new row `row` belongs to, by a whole wave: the last one that starts at or before it; -1: none.  `position`: its
// position in it, negative where the sequence has fewer positions than new tokens.
__device__ __forceinline__ int sequence_at(const PagedCache &c, int row, int &position) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int s0 = 0; s0 < c.seqs; s0 += 64) {
    const int s = s0 + lane;
    before += __popcll(__ballot(s < c.seqs && c.starts[s < c.seqs ? s : 0] <= row));
  }
  if (before == 0) return -1;
  const Sequence s = sequence_of(c.starts[before - 1], c.starts[before], c.lens[before - 1], c.rows);
  position = s.len - s.count + (row - s.first);
  return row >= s.first && row < s.first + s.count ? before - 1 : -1;
}

// ------------------------------------------------------------------------------------------ append
struct AppendArgs {
  PagedCache c;
  void *k_pages, *v_pages;
  const void *q, *k, *v;
  void *rotated;
  const float *rotary;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, r_st, r_sh;
  int32_t heads, kv_heads, head_dim, rot, rot_rows, neighbours;
};

// A wave to a row, a feature to a lane.
template <class T>
__global__ __launch_bounds__(64) void k_paged_append(AppendArgs a) {
  const int row = blockIdx.x, lane = threadIdx.x;
  int position;
  const int seq = sequence_at(a.c, row, position);
  if (seq < 0) return;
  const int64_t place = position_place(a.c, seq, position);
  const int half = a.rot / 2;
  for (int h = 0; h < a.heads + 2 * a.kv_heads; h++) {
    const bool is_q = h < a.heads, is_k = !is_q && h < a.heads + a.kv_heads;
    if (is_q ? a.rot == 0 : place < 0) continue;
    const int kh = is_k ? h - a.heads : h - a.heads - a.kv_heads;
    const T *src = is_q ? (const T *)a.q + row * a.q_st + h * a.q_sh : is_k ? (const T *)a.k + row * a.k_st + kh * a.k_sh : (const T *)a.v + row * a.v_st + kh * a.v_sh;
    T *dst = is_q ? (T *)a.rotated + row * a.r_st + h * a.r_sh : (T *)(is_k ? a.k_pages : a.v_pages) + place + kh * a.c.head_stride;
    const int rot = is_q || is_k ? a.rot : 0;
    for (int i = lane; i < rot / 2; i += 64) {
      const int f0 = a.neighbours ? 2 * i : i, f1 = a.neighbours ? 2 * i + 1 : i + half;
      float cosine = NAN, sine = NAN;
      if (position >= 0 && position < a.rot_rows) { cosine = a.rotary[(int64_t)position * a.rot + i]; sine = a.rotary[(int64_t)position * a.rot + half + i]; }
      const float x = Io<T>::ld(src, f0), y = Io<T>::ld(src, f1);
      Io<T>::st(dst, f0, x * cosine - y * sine);
      Io<T>::st(dst, f1, y * cosine + x * sine);
    }
    for (int f = rot + lane; f < a.head_dim; f += 64) dst[f] = src[f];
  }
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
  a.rot = d->rot_dim; a.rot_rows = d->rot_rows; a.neighbours = d->rot_neighbours != 0;
  launch_kernel(p->dtype == AH_F32 ? k_paged_append<float> : k_paged_append<uint16_t>, dim3((unsigned)d->rows), dim3(64), 0, a);
  AH_LAUNCH_CHECK();
  return AH_OK;
}

}  // extern "C"
