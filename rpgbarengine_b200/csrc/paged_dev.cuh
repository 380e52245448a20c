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

// What a call has to say goes to its status word or, where it has none, to this
// one (each kernel's file has its own), which rpgc_paged_status reads.
static __device__ int32_t g_status;
RPGC_DEV void report(int32_t* status, int32_t bit) { atomicOr(status ? status : &g_status, bit); }

// Host: the bits of this file's word on the current device, which starts again at 0.
static inline cudaError_t take_bits(int32_t* bits) {
  int32_t b = 0, zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&b, g_status, sizeof b);
  if (e == cudaSuccess && b) e = cudaMemcpyToSymbol(g_status, &zero, sizeof zero);
  *bits |= b;
  return e;
}

// max that carries NaN
RPGC_DEV float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
RPGC_DEV float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

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

// Attention of packed row r (of sequence s) and query head h by one warp, from
// the visible keys alone: 32 keys a step, lane l scoring key l, then every
// lane adding the keys' values for its own dims; fp32 throughout.  Half hf of
// the row is written (-1: all of it).  For the rare rows that the tiles' arithmetic
// cannot give: 0.12 ms per 1000 positions.
template <int HD, bool BF>
RPGC_DEV void attn_row(const PagedAttnArgs& a, int s, int64_t r, int h, int hf, int lane) {
  constexpr int E = HD / 32;
  const int kh = h / (a.n_heads / a.kv.n_kv);
  const int64_t r0 = seq_row(a.b, s), r1 = seq_row(a.b, s + 1);
  const int64_t len = a.b.table ? (int64_t)a.b.kv_lens[s] : r1 - r0;
  int64_t end = len - (r1 - r0) + (r - r0) + 1;  // keys [0, end)
  if (a.b.table) end = min(end, table_reach(a.kv, a.b));
  const uint4* qp =
      reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + r * a.q_tok + h * a.q_head);
  float m = -INFINITY, l = 0.0f, o[E];
#pragma unroll
  for (int i = 0; i < E; ++i) o[i] = 0.0f;
  const int64_t mask = (1 << a.kv.page_shift) - 1;
  for (int64_t t0 = 0; t0 < end; t0 += 32) {
    const int64_t t = t0 + lane;
    bool ok = t < end;
    int64_t ko = 0, vo = 0;
    if (ok) {
      if (a.b.table) {
        const int32_t p = page_of(a.kv, a.b, s, t);
        ok = p >= 0;
        ko = (int64_t)p * a.kv.k_page + (t & mask) * a.kv.k_pos;
        vo = (int64_t)p * a.kv.v_page + (t & mask) * a.kv.v_pos;
      } else {
        ko = (r0 + t) * a.kv.k_pos;
        vo = (r0 + t) * a.kv.v_pos;
      }
    }
    float sc = -INFINITY;
    if (ok) {
      const uint4* kp = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.kv.k) + ko + kh * a.kv.k_head);
      sc = 0.0f;
#pragma unroll 4
      for (int i = 0; i < HD / 8; ++i) {
        const uint4 u = kp[i], v = qp[i];
        const uint32_t ws[4] = {u.x, u.y, u.z, u.w}, qs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = unpack2<BF>(ws[j]), q = unpack2<BF>(qs[j]);
          sc += q.x * f.x + q.y * f.y;
        }
      }
      sc *= a.scale;
    }
    const uint32_t live = __ballot_sync(0xffffffffu, ok);
    if (!live) continue;
    const float mn = fmaxf(m, warp_max(sc));
    const float base = mn == -INFINITY ? 0.0f : mn;
    const float corr = expf(m - base), p = ok ? expf(sc - base) : 0.0f;
    m = mn;
    l = l * corr + warp_sum(p);
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] *= corr;
#pragma unroll 8
    for (int j = 0; j < 32; ++j) {
      const bool on = live >> j & 1;
      const float pj = __shfl_sync(0xffffffffu, p, j);
      const int64_t vj = __shfl_sync(0xffffffffu, vo, j);
      const uint16_t* vp = static_cast<const uint16_t*>(a.kv.v) + vj + kh * a.kv.v_head + E * lane;
#pragma unroll
      for (int i = 0; i < E; i += 2) {
        const float2 f = unpack2<BF>(on ? *reinterpret_cast<const uint32_t*>(vp + i) : 0u);
        o[i] += pj * f.x;
        o[i + 1] += pj * f.y;
      }
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (hf >= 0 && lane >> 4 != hf) return;
  uint16_t* op = static_cast<uint16_t*>(a.out) + (r * a.n_heads + h) * HD + E * lane;
#pragma unroll
  for (int i = 0; i < E; i += 2) *reinterpret_cast<uint32_t*>(op + i) = pack2<BF>(o[i] * inv, o[i + 1] * inv);
}

}  // namespace paged
}  // namespace rpgc
