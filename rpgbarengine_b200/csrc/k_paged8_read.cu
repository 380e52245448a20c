// k_paged8_read.cu -- positions of the 8-bit paged cache back into 16-bit pages.
//
// value = scale * code, rounded once.  Bound by memory: 2 HD + 8 bytes in and 4 HD out
// for a position and kv head.  A unit is 16 positions of one kv head (K and V): pages
// begin at multiples of 16 positions on both sides, so a unit lies in one page each.
// The units of all sequences form one list, cut into equal ranges, one a warp; a warp
// has a unit's 4 KB (heads of 128) in flight at once.
//
// Measured: 32 k positions of 8 heads of 128 in 16 sequences 43.8 us (217 MB, 5.0 TB/s), two
// thirds of the bytes written, which sets the pace: filling 151 MB alone takes 41 us.  256
// positions 4.4 us, latency of the look-ups.  Rows in 8-byte parts, so that a warp's stores are whole lines,
// and the next unit's pages looked up ahead: 43.4 and 4.9 us, not kept.
#include <cuda_runtime.h>

#include "paged8_dev.cuh"
#include "paged_tma.cuh"

namespace rpgc {
namespace {

using namespace paged;

constexpr int kSpan = 16;  // positions of a unit
constexpr int kWarps = 4;  // of a block

RPGC_DEV int64_t scan_sum(int64_t v, int lane) {  // inclusive sums over the lanes
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}

RPGC_DEV int32_t length_of(const PagedReadArgs& a, int s) {
  return s < a.b.n_seqs ? (int32_t)min((int64_t)max(0, a.b.kv_lens[s]), table_reach(a.kv, a.b)) : 0;
}
RPGC_DEV int64_t spans_of(const PagedReadArgs& a, int s) { return ((int64_t)length_of(a, s) + kSpan - 1) / kSpan * a.kv.n_kv; }

template <int HD, bool BF>
__global__ void __launch_bounds__(kWarps * 32) read_kernel(const __grid_constant__ PagedReadArgs a) {
  constexpr int kLanes = HD / 16;        // lanes of a row, 16 codes each
  constexpr int kRows = 32 / kLanes;     // rows of a step
  constexpr int kSteps = kSpan / kRows;  // steps of K's (or V's) rows
  const int lane = threadIdx.x & 31;
  grid_dep_wait();
  grid_dep_launch();
  // every warp finds its range by itself: each lane adds up a run of sequences, then
  // the run that holds the range's first unit is looked through
  const int run = (a.b.n_seqs + 31) / 32;
  int64_t sum = 0;
  for (int i = 0; i < run; ++i) sum += spans_of(a, lane * run + i);
  int64_t upto = scan_sum(sum, lane);
  const int64_t total = __shfl_sync(0xffffffffu, upto, 31), warps = (int64_t)gridDim.x * kWarps,
                me = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  int64_t u = me * total / warps;
  const int64_t stop = (me + 1) * total / warps;
  if (u >= stop) return;
  const int src = __ffs(__ballot_sync(0xffffffffu, upto > u)) - 1;
  int64_t first = __shfl_sync(0xffffffffu, upto - sum, src);  // unit where sequence s begins
  int s = src * run;
  for (;; s += 32) {
    const int64_t mine = spans_of(a, s + lane);
    upto = scan_sum(mine, lane);
    const uint32_t in = __ballot_sync(0xffffffffu, first + upto > u);
    if (in) {
      const int at = __ffs(in) - 1;
      first += __shfl_sync(0xffffffffu, upto - mine, at);
      s += at;
      break;
    }
    first += __shfl_sync(0xffffffffu, upto, 31);
  }
  const int row = lane / kLanes, d = 16 * (lane % kLanes);
  int32_t len = length_of(a, s);
  for (; u < stop; ++u) {
    while (u - first >= ((int64_t)len + kSpan - 1) / kSpan * a.kv.n_kv) {  // (a later unit exists: a later sequence has one)
      first += ((int64_t)len + kSpan - 1) / kSpan * a.kv.n_kv;
      len = length_of(a, ++s);
    }
    const int kh = (int)((u - first) % a.kv.n_kv);
    const int32_t t0 = (int32_t)((u - first) / a.kv.n_kv) * kSpan, n = min(kSpan, len - t0);
    const int32_t page = page_of(a.kv, a.b, s, t0);
    if (page < 0) continue;
    const int32_t j = t0 >> a.to.page_shift;
    const int32_t to = j < a.to_max ? a.to_table[s * a.to_stride + j] : -1;
    if ((uint32_t)to >= (uint32_t)a.to.n_pages) {
      if (lane == 0 && kh == 0) report(a.b.status, kStatusDropped);
      continue;
    }
    const int64_t slot = t0 & ((1 << a.kv.page_shift) - 1), to_slot = t0 & ((1 << a.to.page_shift) - 1);
    const uint8_t* kp = static_cast<const uint8_t*>(a.kv.k) + page * a.kv.k_page + slot * a.kv.k_pos + kh * a.kv.k_head + d;
    const uint8_t* vp = static_cast<const uint8_t*>(a.kv.v) + page * a.kv.v_page + slot * a.kv.v_pos + kh * a.kv.v_head + d;
    // lanes 0-15: K's scales, 16-31: V's
    const int pos = lane & 15;
    const float sc = pos < n ? __ldcg(a.scales + page * a.sc_page + kh * a.sc_head + slot + pos + (lane < 16 ? 0 : 1 << a.kv.page_shift)) : 0.0f;
    uint4 in[2][kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int p = i * kRows + row;
      in[0][i] = p < n ? __ldcg(reinterpret_cast<const uint4*>(kp + p * a.kv.k_pos)) : make_uint4(0, 0, 0, 0);
      in[1][i] = p < n ? __ldcg(reinterpret_cast<const uint4*>(vp + p * a.kv.v_pos)) : make_uint4(0, 0, 0, 0);
    }
    uint16_t* ko = static_cast<uint16_t*>(const_cast<void*>(a.to.k)) + to * a.to.k_page + to_slot * a.to.k_pos + kh * a.to.k_head + d;
    uint16_t* vo = static_cast<uint16_t*>(const_cast<void*>(a.to.v)) + to * a.to.v_page + to_slot * a.to.v_pos + kh * a.to.v_head + d;
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int p = i * kRows + row;
        const float f = __shfl_sync(0xffffffffu, sc, p + 16 * w);
        const uint32_t c[4] = {in[w][i].x, in[w][i].y, in[w][i].z, in[w][i].w};
        uint32_t o[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 x = float2_lo(c[e]), y = float2_hi(c[e]);
          o[2 * e] = pack2<BF>(x.x * f, x.y * f);
          o[2 * e + 1] = pack2<BF>(y.x * f, y.y * f);
        }
        if (p < n) {
          uint4* dst = reinterpret_cast<uint4*>(w ? vo + p * a.to.v_pos : ko + p * a.to.k_pos);
          dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
          dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
        }
      }
  }
}

}  // namespace

cudaError_t paged_read_status(int32_t* bits) { return take_bits(bits); }

cudaError_t paged_read_launch(const PagedReadArgs& a, cudaStream_t s) {
  if (!a.b.n_seqs) return cudaSuccess;
  int dev = 0;
  cudaGetDevice(&dev);
  const dim3 grid(8u * (unsigned)sm_count(dev)), block(kWarps * 32);
  const cudaError_t e = a.kv.hd == 128 ? (a.to.bf16 ? launch_pdl(read_kernel<128, true>, grid, block, 0, s, a)
                                                    : launch_pdl(read_kernel<128, false>, grid, block, 0, s, a))
                                       : (a.to.bf16 ? launch_pdl(read_kernel<64, true>, grid, block, 0, s, a)
                                                    : launch_pdl(read_kernel<64, false>, grid, block, 0, s, a));
  if (e == cudaSuccess) count_launches(1);
  return e;
}

}  // namespace rpgc
