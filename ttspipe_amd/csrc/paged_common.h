// The paged key-value cache as its kernels see it (paged_rows.hip,
// paged_attn.hip, paged_evict.hip).
//
// K and V pools are [pages][n_kv][page_size][head_dim] by strides; row b of
// the table names the pages of sequence b, and slot j of the sequence is row
// j % page_size of its page j / page_size. A table entry outside [0, pages) is
// a hole: nothing is read or written through it. Every index that comes from
// device memory (table entries, slots, sequences, positions) is checked here
// before it becomes an address.
#pragma once

#define TTSP_HIP_TYPES_ONLY
#include "../../include/ttsp_hip.h"
#include "ttsp_common.h"

namespace ttsp {

// Workgroups of 256 threads a launch may have (its threads are counted in 32 bits).
constexpr long long PG_MAX_GRID = 0xffffff;

// ttsp_paged_cache with the page size as a shift (the kernels' argument).
struct Paged {
  uint16_t* K;
  uint16_t* V;
  long long k_page, k_head, k_row, v_page, v_head, v_row;  // strides, elements
  const int* table;
  long long table_stride;
  int seqs, cols, pages, shift, nkv;
  float* scores;
  int* slot_pos;
  long long score_seq, score_head, pos_seq, pos_head;

  __host__ __device__ int cap() const { return cols << shift; }  // (paged_args bounds it)
  // The page of sequence b that holds slot j (0 <= j < cap), -1: a hole.
  __host__ __device__ __forceinline__ int page(int b, int j) const {
    const int p = table[b * table_stride + (j >> shift)];
    return (unsigned)p < (unsigned)pages ? p : -1;
  }
  // The rows of sequence b, 0 .. slots[b], cut to the table; 0: none.
  __host__ __device__ __forceinline__ int rows(long long slot) const {
    return slot < 0 ? 0 : slot < cap() ? (int)slot + 1 : cap();
  }
};

// v plus the lower lanes' v, by shifts within the rows of 16 lanes and two row
// broadcasts (lanes without a source add 0).
__device__ __forceinline__ uint32_t lane_prefix(uint32_t v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
  return v;
}

// Whether the `cap` words of every (sequence, kv head) lie apart by these strides.
// (A workgroup adds to its own words, or moves them, while others do to theirs.)
inline bool words_apart(long long seq, long long head, int seqs, int nkv, long long cap) {
  if (seq < (seqs > 1 ? cap : 0) || head < (nkv > 1 ? cap : 0)) return false;
  return seqs == 1 || nkv == 1 || (seq - cap) / (nkv - 1) >= head || (head - cap) / (seqs - 1) >= seq;
}

// The kernels' form of `c` for head dim `hd`-wide rows; false where the fields
// do not describe a cache these kernels take (the caller returns
// hipErrorInvalidValue). Rows are read and written 16 bytes at a time.
inline bool paged_args(const ttsp_paged_cache* c, Paged* p) {
  if (!c || !c->K || !c->V || !c->table || (uintptr_t)c->K % 16 || (uintptr_t)c->V % 16 || (uintptr_t)c->table % 4)
    return false;
  const long long strides[] = {c->k_page, c->k_head, c->k_row, c->v_page, c->v_head, c->v_row};
  for (long long s : strides)
    if (s < 0 || s % 8) return false;
  if (c->k_row > TTSP_PAGED_MAX_ROW_STRIDE || c->v_row > TTSP_PAGED_MAX_ROW_STRIDE) return false;
  if (c->n_kv < 1 || c->n_kv > 4096 || c->pages < 1 || c->seqs < 1 || c->seqs > 65535 || c->cols < 1 ||
      c->table_stride < c->cols || c->page_size < 16 || c->page_size > 4096 || (c->page_size & (c->page_size - 1)))
    return false;
  if ((c->head_dim != 64 && c->head_dim != 128) || (c->dtype != DT_F16 && c->dtype != DT_BF16)) return false;
  const long long cap = (long long)c->cols * c->page_size;
  if (cap > TTSP_PAGED_MAX_SLOTS) return false;
  if (c->scores && ((uintptr_t)c->scores % 4 || !words_apart(c->score_seq, c->score_head, c->seqs, c->n_kv, cap)))
    return false;
  if (c->slot_pos && ((uintptr_t)c->slot_pos % 4 || !words_apart(c->pos_seq, c->pos_head, c->seqs, c->n_kv, cap)))
    return false;
  *p = Paged{(uint16_t*)c->K, (uint16_t*)c->V, c->k_page, c->k_head, c->k_row, c->v_page, c->v_head, c->v_row,
             c->table, c->table_stride, c->seqs, c->cols, c->pages, __builtin_ctz((unsigned)c->page_size), c->n_kv,
             c->scores, c->slot_pos, c->score_seq, c->score_head, c->pos_seq, c->pos_head};
  return true;
}

}  // namespace ttsp
