// k_paged_append.cu -- QK-norm + RoPE + write of new tokens into the pages of
// the KV cache.
//
// Reference: QK-norm before RoPE (src/qwen3.cc:141-152), half-split RoPE
// (src/kernels.h:108-120), the cache write (src/kv_cache.cc:5-33); the
// reference's cache has no pages.
#include <cuda_runtime.h>

#include "paged_dev.cuh"
#include "paged_tma.cuh"

namespace rpgc {
namespace {

using namespace paged;

// A warp takes one token and kSteps x 32 / (HD / 8) of its heads (q heads first,
// then k, then v): HD / 8 lanes hold a row, each with 4 dims of its first half and
// the 4 dims they rotate with, so the rotation needs no exchange and a row's
// sum of squares few.  Bound by memory as long as instructions are few: with a
// row over the whole warp and the rotation through shuffles the kernel issued
// twice as many and took 1.5 times as long.  Every input row is loaded before
// the token's position and page are looked up (one chain of dependent reads).
// Steps a warp: one where all warps run at once all the same, kAtOnce of them an
// SM, so that only the latency counts (64 tokens of 32 + 2 x 8 heads of 128, fp32:
// 2.8 us, 3.1 with two; 128 tokens fp16 3.0 and 3.4 with three; 192 tokens, 31 warps
// an SM, 4.1 and 3.6); else two of fp32 (4096 tokens: one 33.0 us, two 28.9, three
// 32.3 for the registers they take) and three of 16-bit rows (two 26.4, three 24.6,
// four 25.4).  So 4096 fp32 tokens take 28.9 us, 153 MB, 5.3 TB/s, and 12114 ragged
// tokens of 12 + 2 x 4 heads of 64, fp16, 16.9 us, 65 MB, 3.9 TB/s (bound by the
// latency of its warps).
constexpr int kAtOnce = 24;
enum { kInF32 = 0, kInF16 = 1, kInBF16 = 2 };

// Four consecutive values as they are read, and as floats.  16-bit ones stay as
// they are until they are used: half the registers and with that more warps (13
// to 18 % faster).  (__ldcg, not __ldg: the kernel before may still be writing
// the inputs when this one is launched.)
template <int IN>
struct Four {
  uint2 u;
  RPGC_DEV void load(const void* base, int64_t off) {
    u = __ldcg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + off));
  }
  RPGC_DEV void get(float* x) const {
    const float2 f = unpack2<IN == kInBF16>(u.x), g = unpack2<IN == kInBF16>(u.y);
    x[0] = f.x, x[1] = f.y, x[2] = g.x, x[3] = g.y;
  }
};
template <>
struct Four<kInF32> {
  float4 f;
  RPGC_DEV void load(const void* base, int64_t off) {
    f = __ldcg(reinterpret_cast<const float4*>(static_cast<const float*>(base) + off));
  }
  RPGC_DEV void get(float* x) const { x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w; }
};

// The same of tables that stay as they are: gains and rope rows.
RPGC_DEV void table4(const float* p, float* x) {
  const float4 f = __ldg(reinterpret_cast<const float4*>(p));
  x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
}

template <int HD, int IN, bool BF, int kSteps>
__global__ void __launch_bounds__(128) append_kernel(const __grid_constant__ PagedAppendArgs a) {
  constexpr int kLanes = HD / 8, kRows = 32 / kLanes, kHalf = HD / 2;
  const int lane = threadIdx.x & 31, kv = a.kv.n_kv, nk = a.n_heads + kv, heads = nk + kv;
  const int w = (int)blockIdx.y * ((int)blockDim.x >> 5) + ((int)threadIdx.x >> 5);
  const int h0 = w * kSteps * kRows, hl = h0 + lane / kLanes, d = 4 * (lane % kLanes);
  // launched as a programmatic dependent: its inputs come from earlier kernels
  grid_dep_wait();
  grid_dep_launch();
  if (h0 >= heads) return;  // whole warps
  const int64_t r = blockIdx.x;
  Four<IN> in[kSteps][2] = {};  // dims d .. d + 3, then kHalf + d ..
#pragma unroll
  for (int j = 0; j < kSteps; ++j) {
    const int h = hl + j * kRows;
    const bool isq = h < a.n_heads, isk = h < nk;
    const void* base = isq ? a.q : isk ? a.k : a.v;
    const int64_t off = (isq ? r * a.q_tok + h * a.q_head : isk ? r * a.k_tok + (h - a.n_heads) * a.k_head : r * a.v_tok + (h - nk) * a.v_head) + d;
    if (h < heads) {
      in[j][0].load(base, off);
      in[j][1].load(base, off + kHalf);
    }
  }
  const int s = seq_of_row(a.b, r, lane);
  if (s < 0) {  // no sequence's row: zeros for q, nothing for the cache
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      const int h = hl + j * kRows;
      if (h >= a.n_heads) break;
      uint16_t* dst = static_cast<uint16_t*>(a.q_out) + (r * a.n_heads + h) * HD + d;
      *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(dst + kHalf) = make_uint2(0u, 0u);
    }
    return;
  }
  const int64_t r0 = seq_row(a.b, s), r1 = seq_row(a.b, s + 1);
  const int64_t pos = (int64_t)a.b.kv_lens[s] - (r1 - r0) + (r - r0);
  // (the two look-ups that pos leads to run beside each other)
  float c[4] = {}, sn[4] = {};
  if (a.rope && pos >= 0 && pos < a.rope_rows) {
    table4(a.rope + pos * HD + d, c);
    table4(a.rope + pos * HD + kHalf + d, sn);
  }
  const int32_t page = pos >= 0 ? page_of(a.kv, a.b, s, pos) : -1;
  const bool drop = page < 0 || (a.rope && pos >= a.rope_rows);
  if (drop && h0 == 0 && lane == 0) report(a.b.status, kStatusDropped);
  const bool turn = a.rope && !drop, norm = a.k_norm != nullptr;
  const int64_t slot = pos & ((1 << a.kv.page_shift) - 1);
  uint16_t* qd = static_cast<uint16_t*>(a.q_out) + r * a.n_heads * HD + d;
  uint16_t* kd = static_cast<uint16_t*>(const_cast<void*>(a.kv.k)) + page * a.kv.k_page + slot * a.kv.k_pos + d;
  uint16_t* vd = static_cast<uint16_t*>(const_cast<void*>(a.kv.v)) + page * a.kv.v_page + slot * a.kv.v_pos + d;
#pragma unroll
  for (int j = 0; j < kSteps; ++j) {
    const int hs = h0 + j * kRows, h = hl + j * kRows;  // the step's first head; this lane's
    if (hs >= heads) break;                             // whole warps
    const bool isq = h < a.n_heads, isk = h < nk;
    float x[8];
    in[j][0].get(x);
    in[j][1].get(x + 4);
    if (hs < nk) {  // (a step's rows may be of two kinds: v's keep their values)
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = x[i];
      if (norm) {
        float ss = 0.0f, g[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += y[i] * y[i];
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float f = rsqrtf(ss * (1.0f / HD) + a.eps);  // (2 ulp: far below the 16-bit rounding)
        const float* gain = isq ? a.q_norm : a.k_norm;
        table4(gain + d, g);
        table4(gain + kHalf + d, g + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = y[i] * f * g[i];
      }
      if (turn)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float u = y[i], v = y[i + 4];
          y[i] = u * c[i] - v * sn[i];
          y[i + 4] = v * c[i] + u * sn[i];
        }
      if (isk)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = y[i];
    }
    if (h >= heads || (drop && !isq)) continue;
    if (drop)  // no place in the cache: q's row is zeros
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.0f;
    uint16_t* dst = isq ? qd + h * HD : isk ? kd + (h - a.n_heads) * a.kv.k_head : vd + (h - nk) * a.kv.v_head;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<BF>(x[0], x[1]), pack2<BF>(x[2], x[3]));
    *reinterpret_cast<uint2*>(dst + kHalf) = make_uint2(pack2<BF>(x[4], x[5]), pack2<BF>(x[6], x[7]));
  }
}

template <int HD, int IN, int kSteps>
cudaError_t append_steps(const PagedAppendArgs& a, cudaStream_t s) {
  const int per = kSteps * 256 / HD;  // heads of a warp
  const int groups = (a.n_heads + 2 * a.kv.n_kv + per - 1) / per, rows = (groups + 3) / 4;  // blocks of at most 4 warps: 5 % faster than of 8
  const dim3 grid((unsigned)a.b.n_tokens, (unsigned)rows), block(32u * (unsigned)((groups + rows - 1) / rows));
  return a.kv.bf16 ? launch_pdl(append_kernel<HD, IN, true, kSteps>, grid, block, 0, s, a)
                   : launch_pdl(append_kernel<HD, IN, false, kSteps>, grid, block, 0, s, a);
}

template <int HD, int IN>
cudaError_t append_go(const PagedAppendArgs& a, cudaStream_t s) {
  int dev = 0;
  cudaGetDevice(&dev);
  const int64_t warps = (a.n_heads + 2 * a.kv.n_kv + 256 / HD - 1) / (256 / HD) * a.b.n_tokens;
  if (warps <= (int64_t)kAtOnce * sm_count(dev)) return append_steps<HD, IN, 1>(a, s);
  return append_steps<HD, IN, IN == kInF32 ? 2 : 3>(a, s);
}

}  // namespace

cudaError_t paged_append_status(int32_t* bits) { return take_bits(bits); }

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
