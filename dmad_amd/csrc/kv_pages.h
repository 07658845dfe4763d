// Pages of a key-value cache, and where a sequence's slot lies. Host code can
// include this too: the bounds that keep the kernels inside the pool are all here.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define DMAD_HD __host__ __device__ __forceinline__
#else
#define DMAD_HD inline
#endif

namespace dmad {

struct KvSlot {
  int page, slot;  // page < 0: the slot is on no page
};

// k, v: [num_pages][heads][P][D] by strides (elements), one row of the table per
// sequence. An id outside the pool marks a page that holds nothing: nothing is
// read from or written to it.
struct KvPages {
  void* k;
  void* v;
  int64_t k_sp, k_sh, k_sl;  // strides of a page, a head, a slot
  int64_t v_sp, v_sh, v_sl;
  const int32_t* table;  // [B] rows of M page ids
  int64_t table_stride;
  int32_t* lengths;   // [B] slots in use
  int32_t* seen;      // [B] tokens appended so far
  float* weight;      // [num_pages][heads][P], or null
  int32_t* position;  // [num_pages][heads][P], or null (both or none)
  int num_pages, heads, P, M, B;
  uint32_t p_mul;  // s / P = (s p_mul) >> (32 + p_shift) for s < 2^26 (set_pages)
  int p_shift;

  // Page size and pages per sequence, P M <= 2^26. With 2^l >= P the multiplier
  // ceil(2^sh / P) at sh = max(32, 26 + l) is off by less than P / 2^sh, which
  // times s < 2^26 stays below 1 / P: the quotient is exact.
  inline void set_pages(int page_size, int pages) {
    P = page_size;
    M = pages;
    int l = 0;
    while (((int64_t)1 << l) < page_size) ++l;
    const int sh = l < 6 ? 32 : 26 + l;
    p_mul = (uint32_t)((((uint64_t)1 << sh) + page_size - 1) / page_size);
    p_shift = sh - 32;
  }
  DMAD_HD int capacity() const { return M * P; }
  // Slots of sequence b, whatever its length says.
  DMAD_HD int length(int b) const {
    const int n = lengths[b], cap = M * P;
    return n < 0 ? 0 : n < cap ? n : cap;
  }
  // Slot s of sequence b; s may be any number.
  DMAD_HD KvSlot locate(int b, int s) const {
    if ((unsigned)s >= (unsigned)(M * P)) return KvSlot{-1, 0};
    const int entry = (int)((uint32_t)(((uint64_t)(uint32_t)s * p_mul) >> 32) >> p_shift);
    const int page = table[b * table_stride + entry];
    if ((unsigned)page >= (unsigned)num_pages) return KvSlot{-1, 0};
    return KvSlot{page, s - entry * P};
  }
  // Index into weight and position, and offsets (elements) into k and v.
  DMAD_HD int64_t index(KvSlot at, int head) const { return ((int64_t)at.page * heads + head) * P + at.slot; }
  DMAD_HD int64_t k_offset(KvSlot at, int head) const { return at.page * k_sp + head * k_sh + at.slot * k_sl; }
  DMAD_HD int64_t v_offset(KvSlot at, int head) const { return at.page * v_sp + head * v_sh + at.slot * v_sl; }
};

// Slots of the S new tokens of a sequence that holds n of `capacity`: token i's,
// or -1 where it does not fit; and the length afterwards. n + i may not overflow.
DMAD_HD int kv_append_slot(int n, int i, int capacity) { return i < capacity - n ? n + i : -1; }
DMAD_HD int kv_append_length(int n, int S, int capacity) { return S < capacity - n ? n + S : capacity; }

}  // namespace dmad
