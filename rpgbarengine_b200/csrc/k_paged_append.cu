// k_paged_append.cu -- QK-norm + RoPE + write of new tokens into the pages of
// the KV cache.
//
// Reference: QK-norm before RoPE (src/qwen3.cc:141-152), half-split RoPE
// (src/kernels.h:108-120), the cache write (src/kv_cache.cc:5-33); the
// reference's cache has no pages.
#include <cuda_runtime.h>

#include "paged_dev.cuh"

namespace rpgc {
namespace {

using namespace paged;

// ----------------------------------------------------------------- append
// One warp per (token, head), q heads first, then k, then v: lane l holds
// dims E*l .. E*l + E - 1 (E = HD / 32), so the rotation's partner dim
// (d +- HD/2) is in lane l ^ 16.
enum { kInF32 = 0, kInF16 = 1, kInBF16 = 2 };

template <int IN, int E>
RPGC_DEV void load_row(const void* base, int64_t off, int lane, float* x) {
  if (IN == kInF32) {
    const float* p = static_cast<const float*>(base) + off + E * lane;
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const float2 f = *reinterpret_cast<const float2*>(p + i);
      x[i] = f.x;
      x[i + 1] = f.y;
    }
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(base) + off + E * lane;
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const float2 f = unpack2<IN == kInBF16>(*reinterpret_cast<const uint32_t*>(p + i));
      x[i] = f.x;
      x[i + 1] = f.y;
    }
  }
}

template <int HD, int IN, bool BF>
__global__ void __launch_bounds__(256) append_kernel(const PagedAppendArgs a) {
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31;
  const int heads = a.n_heads + 2 * a.kv.n_kv;
  const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (w >= a.b.n_tokens * heads) return;  // whole warps
  const int64_t r = w / heads;
  const int h = (int)(w % heads);
  const int s = seq_of_row(a.b, r, lane);
  if (s < 0) return;
  const int64_t r0 = seq_row(a.b, s), r1 = seq_row(a.b, s + 1);
  const int64_t pos = (int64_t)a.b.kv_lens[s] - (r1 - r0) + (r - r0);
  const int32_t page = pos >= 0 ? page_of(a.kv, a.b, s, pos) : -1;
  const bool drop = page < 0 || (a.rope && pos >= a.rope_rows);
  const bool isq = h < a.n_heads, isk = !isq && h < a.n_heads + a.kv.n_kv;
  if (drop && lane == 0 && a.b.status) atomicOr(a.b.status, kStatusDropped);
  float x[E];
  if (isq) {
    load_row<IN, E>(a.q, r * a.q_tok + h * a.q_head, lane, x);
  } else if (isk) {
    load_row<IN, E>(a.k, r * a.k_tok + (h - a.n_heads) * a.k_head, lane, x);
  } else {
    load_row<IN, E>(a.v, r * a.v_tok + (h - a.n_heads - a.kv.n_kv) * a.v_head, lane, x);
  }
  if (isq || isk) {
    const float* g = isq ? a.q_norm : a.k_norm;
    if (g) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < E; ++i) ss += x[i] * x[i];
      const float f = 1.0f / sqrtf(warp_sum(ss) / (float)HD + a.eps);
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = x[i] * f * g[E * lane + i];
    }
    if (a.rope && !drop) {
      const float* cs = a.rope + pos * HD;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float y = __shfl_xor_sync(0xffffffffu, x[i], 16);
        const int j = (E * lane + i) & (HD / 2 - 1);
        const float c = cs[j], sn = cs[HD / 2 + j];
        x[i] = lane < 16 ? x[i] * c - y * sn : x[i] * c + y * sn;
      }
    }
  }
  uint16_t* dst;
  if (isq) {
    dst = static_cast<uint16_t*>(a.q_out) + (r * a.n_heads + h) * HD;
    if (drop)
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = 0.0f;
  } else {
    if (drop) return;
    const int64_t slot = pos & ((1 << a.kv.page_shift) - 1);
    if (isk) {
      dst = static_cast<uint16_t*>(const_cast<void*>(a.kv.k)) + page * a.kv.k_page + slot * a.kv.k_pos +
            (h - a.n_heads) * a.kv.k_head;
    } else {
      dst = static_cast<uint16_t*>(const_cast<void*>(a.kv.v)) + page * a.kv.v_page + slot * a.kv.v_pos +
            (h - a.n_heads - a.kv.n_kv) * a.kv.v_head;
    }
  }
#pragma unroll
  for (int i = 0; i < E; i += 2) *reinterpret_cast<uint32_t*>(dst + E * lane + i) = pack2<BF>(x[i], x[i + 1]);
}

template <int HD, int IN>
cudaError_t append_go(const PagedAppendArgs& a, cudaStream_t s) {
  const int64_t warps = a.b.n_tokens * (a.n_heads + 2 * a.kv.n_kv);
  const dim3 grid((unsigned)((warps + 7) / 8));
  if (a.kv.bf16) append_kernel<HD, IN, true><<<grid, 256, 0, s>>>(a);
  else append_kernel<HD, IN, false><<<grid, 256, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t paged_append_launch(const PagedAppendArgs& a, cudaStream_t s) {
  if (!a.b.n_tokens) return cudaSuccess;
  cudaError_t e;
  const int in = a.in_type == kF32 ? kInF32 : a.in_type == kF16 ? kInF16 : kInBF16;
  if (a.kv.hd == 128)
    e = in == kInF32 ? append_go<128, kInF32>(a, s) : in == kInF16 ? append_go<128, kInF16>(a, s) : append_go<128, kInBF16>(a, s);
  else
    e = in == kInF32 ? append_go<64, kInF32>(a, s) : in == kInF16 ? append_go<64, kInF16>(a, s) : append_go<64, kInBF16>(a, s);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

}  // namespace rpgc
