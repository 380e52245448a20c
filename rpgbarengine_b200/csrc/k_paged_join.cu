// k_paged_join.cu -- single-token attention with a shared prefix: the workspace, the
// launches of its three kernels, and the last of them, which joins the sums over the
// pieces of a prefix with those over a sequence's own positions.
//
// Mathematics: out = sum_k 2^(m_k - M) o_k / sum_k 2^(m_k - M) l_k over the pieces k and the
// own positions, M the largest of their references m_k, in fp32.  A row whose result is
// infinite or NaN though its weights are finite is computed again from its definition.
//
// Bound by the sums' bytes, 4 HD + 8 a row and piece, which come from L2; in a kernel of
// its own all rows' chains of look-ups run at once (joined by the CTAs that end the items of
// own positions, 256 sequences x 32 heads in 4 pieces took 22 us).
#include <cuda_runtime.h>

#include "paged8_dev.cuh"
#include "paged_dev.cuh"
#include "paged_tma.cuh"

namespace rpgc {
namespace {

using namespace paged;

constexpr int kWarps = 4;  // of a block
constexpr int kAtOnce = 8; // pieces whose sums are in flight together

// HD / 4 lanes a row, four values each.
template <int HD, bool BF, bool F8>
__global__ void __launch_bounds__(kWarps * 32) join_kernel(const __grid_constant__ PagedOwnArgs a,
                                                           const __grid_constant__ PrefixParts p) {
  constexpr int kLanes = HD / 4, kRows = 32 / kLanes;
  const int lane = threadIdx.x & 31, d = 4 * (lane % kLanes);
  const int64_t rows = (int64_t)a.b.n_seqs * a.n_heads,
                row = ((int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5)) * kRows + lane / kLanes;
  grid_dep_launch();
  const bool in = row < rows;
  const int32_t s = in ? (int32_t)(row / a.n_heads) : 0;
  // (lengths and groups: earlier kernels' than the two that this one follows, and those
  // waited for them before they let this one begin)
  GroupAt at;
  const Sight v = in ? sight_of<true>(a, s, __ldcg(a.b.kv_lens + s), at) : Sight{0, 0, 0};
  grid_dep_wait();
  const int32_t chunk = __ldcg(p.chunk), pieces = v.pre > 0 ? (v.pre - 1) / chunk + 1 : 0;
  float M = -INFINITY, L = 0.0f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (v.len > v.own) {
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.own_ml) + row);
    acc = __ldcg(reinterpret_cast<const float4*>(p.own + row * HD + d));
    M = ml.x;
    L = ml.y;
    if (M == -INFINITY) acc = make_float4(0.f, 0.f, 0.f, 0.f), L = 0.0f;  // (saw nothing: what its sums hold counts for nothing)
  }
  for (int k0 = 0; k0 < pieces; k0 += kAtOnce) {
    float2 ml[kAtOnce];
    float4 o[kAtOnce];
    float top = M;
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int64_t i = row + (k0 + k) * rows;
      ml[k] = make_float2(-INFINITY, 0.0f);
      if (k0 + k < pieces) {
        ml[k] = __ldcg(reinterpret_cast<const float2*>(p.ml) + i);
        o[k] = __ldcg(reinterpret_cast<const float4*>(p.part + i * HD + d));
      }
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) top = fmaxf(top, ml[k].x);
    const float c = M == -INFINITY ? 0.0f : exp2_fast(M - top);
    acc.x *= c, acc.y *= c, acc.z *= c, acc.w *= c;
    L *= c;
    M = top;
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      if (ml[k].x == -INFINITY) continue;
      const float c = exp2_fast(ml[k].x - top);
      acc.x += c * o[k].x;
      acc.y += c * o[k].y;
      acc.z += c * o[k].z;
      acc.w += c * o[k].w;
      L += c * ml[k].y;
    }
  }
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  if (in)
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + row * HD + d) =
        make_uint2(pack2<BF>(acc.x * inv, acc.y * inv), pack2<BF>(acc.z * inv, acc.w * inv));
  const float z = fmaf(acc.x, 0.0f, fmaf(acc.y, 0.0f, fmaf(acc.z, 0.0f, acc.w * 0.0f)));  // NaN: not all finite
  uint32_t again = __ballot_sync(0xffffffffu, in && z != 0.0f && L < INFINITY);
  while (__builtin_expect(again != 0, 0)) {
    const int src = (__ffs(again) - 1) / kLanes * kLanes;
    again &= ~((kLanes == 32 ? 0xffffffffu : (1u << kLanes) - 1u) << src);
    const int64_t r = __shfl_sync(0xffffffffu, row, src);
    own_row<HD, BF, F8, true>(a, (int32_t)(r / a.n_heads), (int)(r % a.n_heads), lane);
  }
}

template <int HD, bool BF>
cudaError_t join_go(const PagedOwnArgs& a, const PrefixParts& p, cudaStream_t s) {
  const int64_t per = kWarps * (128 / HD), rows = (int64_t)a.b.n_seqs * a.n_heads;
  const dim3 grid((unsigned)((rows + per - 1) / per)), block(kWarps * 32);
  return a.scales ? launch_pdl(join_kernel<HD, BF, true>, grid, block, 0, s, a, p)
                  : launch_pdl(join_kernel<HD, BF, false>, grid, block, 0, s, a, p);
}

// Pieces of a prefix that the workspace has room for: fewer for more rows, whose units
// fill the SMs with longer ones (148 SMs, two tiles of 128 rows each, twice over).
constexpr int kPieces = 32;  // (a lane of the plan for each)
int pieces_of(int32_t n_seqs, int32_t n_heads) {
  const int64_t rows = (int64_t)(n_seqs > 0 ? n_seqs : 1) * n_heads, n = 75776 / rows;
  return n < 1 ? 1 : n > kPieces ? kPieces : (int)n;
}

// The workspace: single-token attention's, the length of a piece, the pieces' sums, the
// own positions', then all references and weights.
int64_t front_bytes(int32_t n_heads, int32_t n_kv, int32_t hd) {
  PagedView v{};
  v.n_kv = n_kv;
  v.hd = hd;
  return (paged_decode_workspace(v, n_heads) + 255) / 256 * 256 + 256;
}

}  // namespace

int64_t paged_prefix_workspace(int32_t n_seqs, int32_t n_heads, int32_t n_kv, int32_t hd) {
  return front_bytes(n_heads, n_kv, hd) + (int64_t)(pieces_of(n_seqs, n_heads) + 1) * n_seqs * n_heads * (hd + 2) * 4;
}

cudaError_t paged_prefix_decode_launch(const PagedOwnArgs& a, cudaStream_t s) {
  const int G = a.n_heads / a.kv.n_kv;
  const int64_t rows = (int64_t)a.b.n_seqs * a.n_heads;
  int dev = 0;
  cudaGetDevice(&dev);
  PrefixShape shape;
  shape.T = 128 / G;
  shape.pieces = pieces_of(a.b.n_seqs, a.n_heads);
  // as many CTAs as may have a unit: the others' SMs are free for the next kernel at once
  const int64_t reach = (((int64_t)a.pre.max_pages << a.pre.kv.page_shift) + kPrefixKeys - 1) / kPrefixKeys,
                most = (a.b.n_seqs / (2 * shape.T) + a.pre.n_groups) * a.kv.n_kv * (reach < shape.pieces ? reach : shape.pieces);
  shape.ctas = (int32_t)(most < sm_count(dev) ? most : sm_count(dev));
  uint8_t* w = static_cast<uint8_t*>(a.workspace) + front_bytes(a.n_heads, a.kv.n_kv, a.kv.hd);
  PrefixParts p;
  p.chunk = reinterpret_cast<int32_t*>(w - 256);
  p.part = reinterpret_cast<float*>(w);
  p.own = p.part + shape.pieces * rows * a.kv.hd;
  p.ml = p.own + rows * a.kv.hd;
  p.own_ml = p.ml + 2 * shape.pieces * rows;
  cudaError_t e = paged_prefix_launch(a, p, shape, s);
  if (e == cudaSuccess) e = a.scales ? paged8_decode_prefix_launch(a, p, shape, s) : paged_decode_prefix_launch(a, p, shape, s);
  if (e != cudaSuccess) return e;
  if (a.kv.hd == 128) e = a.kv.bf16 ? join_go<128, true>(a, p, s) : join_go<128, false>(a, p, s);
  else e = a.kv.bf16 ? join_go<64, true>(a, p, s) : join_go<64, false>(a, p, s);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

}  // namespace rpgc
