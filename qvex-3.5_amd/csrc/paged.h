// The paged KV cache as its kernels see it: a page's element, a sequence's rows,
// and the checks that the entry points share (include/qvex.h has the layout).
#pragma once
#include <math.h>

#include "qvex_common.h"

namespace {

// Positions and row counts stay below this, so that their sums fit an int.
constexpr int KV_LIMIT = 1 << 30;

struct KvPages {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  int n_pages, shift, Hkv;       // page = 1 << shift positions
};

struct KvRows {
  const int32_t* table;
  const int32_t* pos;
  const int32_t* cu;
  long stride;
  int width, L, T;
};

// Rows [first, first + n) of sequence b, the first of them at position `pos`.
struct KvSeq {
  int first, n, pos;
  __device__ __forceinline__ KvSeq(const KvRows& r, int b) {
    first = b * r.L;
    int end = first + r.L;
    if (r.cu) {
      first = min(max(r.cu[b], 0), r.T);
      end = min(max(r.cu[b + 1], first), r.T);
    }
    n = end - first;
    pos = min(max(r.pos[b], -KV_LIMIT), KV_LIMIT);
  }
};

// The slot (page * Hkv + head) * page size + slot of position p, or -1 where none is.
__device__ __forceinline__ long kv_slot(const KvPages& c, const KvRows& r, int b, int head, int p) {
  if (p < 0 || (p >> c.shift) >= r.width) return -1;
  const int page = r.table[b * r.stride + (p >> c.shift)];
  if (page < 0 || page >= c.n_pages) return -1;
  return (((long)page * c.Hkv + head) << c.shift) + (p & ((1 << c.shift) - 1));
}

constexpr int kv_bytes(int format) { return format == QVEX_KV_BF16 ? 2 : 1; }

// Checks the two structs; on success *pc and *rc are what the kernels take.
inline int kv_check(const char* fn, const qvex_kv_pages* p, const qvex_kv_rows* r, KvPages* pc, KvRows* rc) {
  QVEX_CHECK_ARG(p && r, "%s: null pages or rows", fn);
  QVEX_CHECK_ARG(p->format == QVEX_KV_BF16 || p->format == QVEX_KV_INT8 || p->format == QVEX_KV_FP8,
                 "%s: format=%d is none of bf16 (0), int8 (1), fp8 (2)", fn, p->format);
  QVEX_CHECK_ARG(p->D == 128 || p->D == 256, "%s: D=%d (128 or 256 supported)", fn, p->D);
  QVEX_CHECK_ARG(p->page >= 16 && p->page <= 1024 && (p->page & (p->page - 1)) == 0,
                 "%s: page=%d must be a power of two, 16..1024", fn, p->page);
  QVEX_CHECK_ARG(p->n_pages >= 1 && p->Hkv >= 1 && p->Hkv <= 1024 && (int64_t)p->n_pages * p->Hkv * p->page < 1LL << 31,
                 "%s: n_pages=%d Hkv=%d (1..1024; page * n_pages * Hkv below 2^31)", fn, p->n_pages, p->Hkv);
  QVEX_CHECK_ARG(p->k && p->v && qvex_aligned(p->k, 16) && qvex_aligned(p->v, 16),
                 "%s: the pages of K and V must be 16-byte aligned, not null", fn);
  QVEX_CHECK_ARG(p->format == QVEX_KV_BF16 || (p->k_scales && p->v_scales && qvex_aligned(p->k_scales, 16) &&
                                               qvex_aligned(p->v_scales, 16)),
                 "%s: an 8-bit format needs scales, 16-byte aligned", fn);
  QVEX_CHECK_ARG(r->B >= 1 && r->B <= 65535 && r->L >= 1 && r->T >= 0 && r->T <= KV_LIMIT / 4,
                 "%s: B=%d (1..65535) L=%d T=%d", fn, r->B, r->L, r->T);
  QVEX_CHECK_ARG(r->cu || (long)r->B * r->L == r->T, "%s: without row offsets T=%d must be B*L = %ld", fn, r->T,
                 (long)r->B * r->L);
  QVEX_CHECK_ARG(r->table && r->pos, "%s: null table or positions", fn);
  QVEX_CHECK_ARG(r->table_width >= 1 && (long)r->table_width * p->page <= KV_LIMIT && r->table_stride >= 0 &&
                     (r->B == 1 || r->table_stride >= r->table_width),
                 "%s: table_width=%d table_stride=%ld", fn, r->table_width, r->table_stride);
  int shift = 0;
  while ((1 << shift) < p->page) ++shift;
  *pc = KvPages{(uint8_t*)p->k, (uint8_t*)p->v, p->k_scales, p->v_scales, p->n_pages, shift, p->Hkv};
  *rc = KvRows{r->table, r->pos, r->cu, r->table_stride, r->table_width, r->L, r->T};
  return QVEX_OK;
}

}  // namespace
