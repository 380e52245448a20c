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

// One warp per token and kHeads heads (q heads first, then k, then v): lane l
// holds dims E*l .. E*l + E - 1 (E = HD / 32), so the rotation's partner dim
// (d +- HD/2) is in lane l ^ 16.  Bound by memory: every input row is loaded
// before the token's position and page are looked up, so that a warp has
// kHeads rows in flight behind one chain of dependent reads (length -> page
// and rope row).
constexpr int kHeads = 4;
enum { kInF32 = 0, kInF16 = 1, kInBF16 = 2 };

template <int IN, int E>
RPGC_DEV void load_row(const void* base, int64_t off, int lane, float* x) {
  if (IN == kInF32) {
    const float* p = static_cast<const float*>(base) + off + E * lane;
    if (E == 4) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(p));
      x[0] = f.x, x[1] = f.y, x[E - 2] = f.z, x[E - 1] = f.w;
    } else {
      const float2 f = __ldg(reinterpret_cast<const float2*>(p));
      x[0] = f.x, x[1] = f.y;
    }
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(base) + off + E * lane;
    uint32_t w[2];
    if (E == 4) {
      const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = u.x, w[1] = u.y;
    } else {
      w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    }
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const float2 f = unpack2<IN == kInBF16>(w[i]);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
}

template <int HD, int IN, bool BF>
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ PagedAppendArgs a) {
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31, kv = a.kv.n_kv, heads = a.n_heads + 2 * kv;
  const int h0 = ((int)blockIdx.y * ((int)blockDim.x >> 5) + ((int)threadIdx.x >> 5)) * kHeads;
  // launched as a programmatic dependent: its inputs come from earlier kernels
  grid_dep_wait();
  grid_dep_launch();
  if (h0 >= heads) return;  // whole warps
  const int64_t r = blockIdx.x;
  float x[kHeads][E];
#pragma unroll
  for (int j = 0; j < kHeads; ++j) {
    const int h = h0 + j;
    if (h < a.n_heads) load_row<IN, E>(a.q, r * a.q_tok + h * a.q_head, lane, x[j]);
    else if (h < a.n_heads + kv) load_row<IN, E>(a.k, r * a.k_tok + (h - a.n_heads) * a.k_head, lane, x[j]);
    else if (h < heads) load_row<IN, E>(a.v, r * a.v_tok + (h - a.n_heads - kv) * a.v_head, lane, x[j]);
  }
  const int s = seq_of_row(a.b, r, lane);
  if (s < 0) return;
  const int64_t r0 = seq_row(a.b, s), r1 = seq_row(a.b, s + 1);
  const int64_t pos = (int64_t)a.b.kv_lens[s] - (r1 - r0) + (r - r0);
  const int32_t page = pos >= 0 ? page_of(a.kv, a.b, s, pos) : -1;
  const bool drop = page < 0 || (a.rope && pos >= a.rope_rows);
  if (drop && h0 == 0 && lane == 0 && a.b.status) atomicOr(a.b.status, kStatusDropped);
  float c[E], sn[E];
  const bool turn = a.rope && !drop;
  if (turn) {
    const float* cs = a.rope + pos * HD + ((E * lane) & (HD / 2 - 1));
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const float2 f = __ldg(reinterpret_cast<const float2*>(cs + i)), g = __ldg(reinterpret_cast<const float2*>(cs + HD / 2 + i));
      c[i] = f.x, c[i + 1] = f.y;
      sn[i] = lane < 16 ? -g.x : g.x, sn[i + 1] = lane < 16 ? -g.y : g.y;
    }
  }
  const int64_t slot = pos & ((1 << a.kv.page_shift) - 1);
#pragma unroll
  for (int j = 0; j < kHeads; ++j) {
    const int h = h0 + j;
    if (h >= heads) break;  // whole warps
    const bool isq = h < a.n_heads, isk = !isq && h < a.n_heads + kv;
    if (isq || isk) {
      const float* g = isq ? a.q_norm : a.k_norm;
      if (g) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) ss += x[j][i] * x[j][i];
        const float f = 1.0f / sqrtf(warp_sum(ss) / (float)HD + a.eps);
#pragma unroll
        for (int i = 0; i < E; ++i) x[j][i] = x[j][i] * f * __ldg(g + E * lane + i);
      }
      if (turn)
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const float y = __shfl_xor_sync(0xffffffffu, x[j][i], 16);
          x[j][i] = x[j][i] * c[i] + y * sn[i];
        }
    }
    uint16_t* dst;
    if (isq) {
      dst = static_cast<uint16_t*>(a.q_out) + (r * a.n_heads + h) * HD;
      if (drop)
#pragma unroll
        for (int i = 0; i < E; ++i) x[j][i] = 0.0f;
    } else if (drop) {
      break;
    } else if (isk) {
      dst = static_cast<uint16_t*>(const_cast<void*>(a.kv.k)) + page * a.kv.k_page + slot * a.kv.k_pos + (h - a.n_heads) * a.kv.k_head;
    } else {
      dst = static_cast<uint16_t*>(const_cast<void*>(a.kv.v)) + page * a.kv.v_page + slot * a.kv.v_pos +
            (h - a.n_heads - kv) * a.kv.v_head;
    }
    if (E == 4)
      *reinterpret_cast<uint2*>(dst + E * lane) = make_uint2(pack2<BF>(x[j][0], x[j][1]), pack2<BF>(x[j][E - 2], x[j][E - 1]));
    else
      *reinterpret_cast<uint32_t*>(dst + E * lane) = pack2<BF>(x[j][0], x[j][1]);
  }
}

template <int HD, int IN>
cudaError_t append_go(const PagedAppendArgs& a, cudaStream_t s) {
  const int groups = (a.n_heads + 2 * a.kv.n_kv + kHeads - 1) / kHeads, rows = (groups + 7) / 8;
  const dim3 grid((unsigned)a.b.n_tokens, (unsigned)rows), block(32u * (unsigned)((groups + rows - 1) / rows));
  return a.kv.bf16 ? launch_pdl(append_kernel<HD, IN, true>, grid, block, 0, s, a) : launch_pdl(append_kernel<HD, IN, false>, grid, block, 0, s, a);
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
