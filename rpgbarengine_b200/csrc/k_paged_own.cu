// k_paged_own.cu -- attention of one new token per sequence over 8-bit pages, with a
// shared prefix, or both: a warp per sequence and query head, fp32.
#include <cuda_runtime.h>

#include "paged8_dev.cuh"
#include "paged_dev.cuh"
#include "paged_tma.cuh"

namespace rpgc {
namespace {

using namespace paged;

template <int HD, bool BF, bool F8, bool SH>
__global__ void __launch_bounds__(128) rows_kernel(const __grid_constant__ PagedOwnArgs a) {
  grid_dep_wait();
  grid_dep_launch();
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (i < (int64_t)a.b.n_seqs * a.n_heads) own_row<HD, BF, F8, SH>(a, (int32_t)(i / a.n_heads), (int)(i % a.n_heads), threadIdx.x & 31);
}

template <int HD, bool BF>
cudaError_t rows_go(const PagedOwnArgs& a, cudaStream_t s) {
  const dim3 grid((unsigned)(((int64_t)a.b.n_seqs * a.n_heads + 3) / 4)), block(128);
  const cudaError_t e = !a.scales          ? launch_pdl(rows_kernel<HD, BF, false, true>, grid, block, 0, s, a)
                        : a.pre.n_groups ? launch_pdl(rows_kernel<HD, BF, true, true>, grid, block, 0, s, a)
                                         : launch_pdl(rows_kernel<HD, BF, true, false>, grid, block, 0, s, a);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

}  // namespace

int64_t paged_prefix_workspace(int32_t, int32_t, int32_t, int32_t) { return 16; }

cudaError_t paged_own_decode_status(int32_t* bits) { return take_bits(bits); }

cudaError_t paged_own_decode_launch(const PagedOwnArgs& a, cudaStream_t s) {
  if (!a.b.n_tokens) return cudaSuccess;
  if (a.kv.hd == 128) return a.kv.bf16 ? rows_go<128, true>(a, s) : rows_go<128, false>(a, s);
  return a.kv.bf16 ? rows_go<64, true>(a, s) : rows_go<64, false>(a, s);
}

}  // namespace rpgc
