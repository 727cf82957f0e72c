// kv_dest.h - where a token's key / value rows lie in the paged cache: the block-table and slot forms of
// the stores.
#pragma once

#include "device.h"

namespace mas {
namespace {

// Resolves token t's (page, entry). Returns false when the token is skipped. Args holds the destination's
// fields: slots, or batch_indices, positions, kv_indices, num_indices, kv_indptr and batch; num_pages,
// page_size and err.
template <bool kSlotForm, class Args>
__device__ __forceinline__ bool resolve(const Args& a, int64_t t, int64_t* page, int64_t* entry) {
  if constexpr (kSlotForm) {
    const int64_t slot = a.slots[t];
    if (slot < 0) return false;
    const int64_t pg = slot / a.page_size;
    if (pg >= a.num_pages) {
      report(a.err, MAS_ERRBIT_SLOT);
      return false;
    }
    *page = pg;
    *entry = slot - pg * a.page_size;
    return true;
  } else {
    // Both per-token indices are loaded before either is checked, so the two loads overlap.
    const int64_t b = a.batch_indices[t];
    const int64_t p = a.positions[t];
    const bool b_ok = b >= 0 && b < a.batch;
    if (!b_ok || p < 0) {
      report(a.err, b_ok ? MAS_ERRBIT_POSITION : MAS_ERRBIT_BATCH);
      return false;
    }
    const int64_t first = a.kv_indptr[b];
    const int64_t end = a.kv_indptr[b + 1];
    const int64_t idx = first + p / a.page_size;
    if (idx < 0 || idx >= a.num_indices || idx >= end) {
      report(a.err, MAS_ERRBIT_PAGE);
      return false;
    }
    const int64_t pg = a.kv_indices[idx];
    if (pg < 0 || pg >= a.num_pages) {
      report(a.err, MAS_ERRBIT_PAGE);
      return false;
    }
    *page = pg;
    *entry = p % a.page_size;
    return true;
  }
}

}  // namespace
}  // namespace mas
