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

// E values of a row, from this lane's first.
template <int IN, int E>
RPGC_DEV void load_row(const uint8_t* p, float* x) {
  if (IN == kInF32) {
    if (E == 4) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(p));
      x[0] = f.x, x[1] = f.y, x[E - 2] = f.z, x[E - 1] = f.w;
    } else {
      const float2 f = __ldg(reinterpret_cast<const float2*>(p));
      x[0] = f.x, x[1] = f.y;
    }
  } else {
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
  constexpr int E = HD / 32, kIn = IN == kInF32 ? 4 : 2;
  const int lane = threadIdx.x & 31, kv = a.kv.n_kv, nk = a.n_heads + kv, heads = nk + kv;
  const int h0 = ((int)blockIdx.y * ((int)blockDim.x >> 5) + ((int)threadIdx.x >> 5)) * kHeads;
  // launched as a programmatic dependent: its inputs come from earlier kernels
  grid_dep_wait();
  grid_dep_launch();
  if (h0 >= heads) return;  // whole warps
  const int64_t r = blockIdx.x;
  const int nh = min(kHeads, heads - h0);
  float x[kHeads][E];
#pragma unroll
  for (int j = 0; j < kHeads; ++j) {
    const int h = h0 + j;
    const bool isq = h < a.n_heads, isk = h < nk;
    const void* base = isq ? a.q : isk ? a.k : a.v;
    const int64_t off = isq ? r * a.q_tok + h * a.q_head : isk ? r * a.k_tok + (h - a.n_heads) * a.k_head : r * a.v_tok + (h - nk) * a.v_head;
    if (j < nh) load_row<IN, E>(static_cast<const uint8_t*>(base) + (off + E * lane) * kIn, x[j]);
  }
  const int s = seq_of_row(a.b, r, lane);
  if (s < 0) return;
  const int64_t r0 = seq_row(a.b, s), r1 = seq_row(a.b, s + 1);
  const int64_t pos = (int64_t)__ldg(a.b.kv_lens + s) - (r1 - r0) + (r - r0);
  const int32_t page = pos >= 0 ? page_of(a.kv, a.b, s, pos) : -1;
  const bool drop = page < 0 || (a.rope && pos >= a.rope_rows);
  if (drop && h0 == 0 && lane == 0 && a.b.status) atomicOr(a.b.status, kStatusDropped);
  const bool turn = a.rope && !drop;
  float c[E], sn[E], g[2][E];  // gains of q and of k
#pragma unroll
  for (int i = 0; i < E; ++i) c[i] = 1.0f, sn[i] = 0.0f, g[0][i] = g[1][i] = 1.0f;
  if (turn) {
    const uint8_t* cs = reinterpret_cast<const uint8_t*>(a.rope + pos * HD + ((E * lane) & (HD / 2 - 1)));
    load_row<kInF32, E>(cs, c);
    load_row<kInF32, E>(cs + HD * 2, sn);
#pragma unroll
    for (int i = 0; i < E; ++i) sn[i] = lane < 16 ? -sn[i] : sn[i];
  }
  if (a.q_norm && h0 < a.n_heads) load_row<kInF32, E>(reinterpret_cast<const uint8_t*>(a.q_norm + E * lane), g[0]);
  if (a.k_norm && h0 + nh > a.n_heads) load_row<kInF32, E>(reinterpret_cast<const uint8_t*>(a.k_norm + E * lane), g[1]);
  const int64_t slot = pos & ((1 << a.kv.page_shift) - 1);
  uint16_t* qd = static_cast<uint16_t*>(a.q_out) + r * a.n_heads * HD + E * lane;
  uint16_t* kd = static_cast<uint16_t*>(const_cast<void*>(a.kv.k)) + page * a.kv.k_page + slot * a.kv.k_pos + E * lane;
  uint16_t* vd = static_cast<uint16_t*>(const_cast<void*>(a.kv.v)) + page * a.kv.v_page + slot * a.kv.v_pos + E * lane;
#pragma unroll
  for (int j = 0; j < kHeads; ++j) {
    if (j >= nh) break;  // whole warps
    const int h = h0 + j;
    const bool isq = h < a.n_heads, isk = h < nk;
    if (isk && (isq ? a.q_norm : a.k_norm)) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < E; ++i) ss += x[j][i] * x[j][i];
      const float f = rsqrtf(warp_sum(ss) * (1.0f / HD) + a.eps);  // (2 ulp: far below the 16-bit rounding)
#pragma unroll
      for (int i = 0; i < E; ++i) x[j][i] = x[j][i] * f * (isq ? g[0][i] : g[1][i]);
    }
    if (isk && turn)
#pragma unroll
      for (int i = 0; i < E; ++i) x[j][i] = x[j][i] * c[i] + __shfl_xor_sync(0xffffffffu, x[j][i], 16) * sn[i];
    if (drop) {  // no place in the cache; q's row is zeros
      if (!isq) break;
#pragma unroll
      for (int i = 0; i < E; ++i) x[j][i] = 0.0f;
    }
    uint16_t* dst = isq ? qd + h * HD : isk ? kd + (h - a.n_heads) * a.kv.k_head : vd + (h - nk) * a.kv.v_head;
    if (E == 4)
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<BF>(x[j][0], x[j][1]), pack2<BF>(x[j][E - 2], x[j][E - 1]));
    else
      *reinterpret_cast<uint32_t*>(dst) = pack2<BF>(x[j][0], x[j][1]);
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
