// paged_dev.cuh -- device helpers of the paged-cache kernels: which sequence a
// packed row belongs to, where a position's slot is, 16-bit conversions.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "kernels.h"

namespace rpgc {
namespace paged {

constexpr int kStatusDropped = 1, kStatusTimeout = 2;  // RPGC_PAGED_*

// First packed row of sequence s (s == n_seqs: past the last), kept inside
// [0, n_tokens] whatever cu holds.
RPGC_DEV int64_t seq_row(const PagedSeqs& b, int s) {
  if (!b.cu) return s;
  const int64_t r = b.cu[s];
  return r < 0 ? 0 : (r > b.n_tokens ? b.n_tokens : r);
}

// Cache positions a sequence's table reaches.
RPGC_DEV int64_t table_reach(const PagedView& kv, const PagedSeqs& b) {
  return (int64_t)b.max_pages << kv.page_shift;
}

// Page of position t, or -1 where it is not there.
RPGC_DEV int32_t page_of(const PagedView& kv, const PagedSeqs& b, int s, int64_t t) {
  const int64_t j = t >> kv.page_shift;
  if (j >= b.max_pages) return -1;
  const int32_t p = b.table[(int64_t)s * b.table_stride + j];
  return (uint32_t)p < (uint32_t)kv.n_pages ? p : -1;
}

// Two values of a 16-bit pair as floats, and back (round to nearest even).
template <bool BF>
RPGC_DEV float2 unpack2(uint32_t w) {
  if (BF) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool BF>
RPGC_DEV uint32_t pack2(float a, float b) {
  if (BF) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The sequence whose rows hold packed row r, or -1: the last s with
// seq_row(s) <= r, found by the whole warp 32 candidates at a time.
RPGC_DEV int seq_of_row(const PagedSeqs& b, int64_t r, int lane) {
  if (!b.cu) return r < b.n_seqs ? (int)r : -1;
  int lo = 0, n = b.n_seqs;  // the answer is in [lo, lo + n)
  if (r < seq_row(b, 0)) return -1;
  while (n > 1) {
    const int step = (n + 31) / 32, c = lo + lane * step;
    const bool le = lane * step < n && seq_row(b, c) <= r;
    const uint32_t m = __ballot_sync(0xffffffffu, le);
    const int top = 31 - __clz(m | 1u);
    n = min(step, n - top * step);
    lo += top * step;
  }
  return r < seq_row(b, lo + 1) ? lo : -1;
}

}  // namespace paged
}  // namespace rpgc
