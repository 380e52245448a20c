// k_paged_join.cu -- single-token attention with a shared prefix: the workspace, the
// launches of its four kernels (or of the one that goes through a small prefix), and the
// last of them, which joins the sums over the pieces of a prefix with those over a
// sequence's own positions.
//
// Mathematics: out = sum_k 2^(m_k - M) o_k / sum_k 2^(m_k - M) l_k over the pieces k and the
// own positions, M the largest of their references m_k, in fp32.  A row whose result is
// infinite or NaN though its weights are finite is computed again from its definition.
//
// Bound by the sums' bytes, 4 HD + 8 a row and piece, which come from L2; in a kernel of
// its own all rows' chains of look-ups run at once (joined by the CTAs that end the items of
// own positions, 256 sequences x 32 heads in 4 pieces took 22 us; here 6 us for 21 MB, and 4 us
// for 64 sequences in two).
#include <cuda_runtime.h>

#include <type_traits>

#include "paged8_dev.cuh"
#include "paged_dev.cuh"
#include "paged_tma.cuh"

namespace rpgc {
namespace {

using namespace paged;

constexpr int kWarps = 4;  // of a block
constexpr int kAtOnce = 5; // pieces whose sums are in flight together

// HD / 4 lanes a row, four values each.
template <int HD, bool BF, bool F8>
__global__ void __launch_bounds__(kWarps * 32, 8) join_kernel(const __grid_constant__ PagedOwnArgs a,
                                                           const __grid_constant__ PrefixParts p) {
  constexpr int kLanes = HD / 4, kRows = 32 / kLanes;
  const int lane = threadIdx.x & 31, d = 4 * (lane % kLanes);
  const int64_t rows = (int64_t)a.b.n_seqs * a.n_heads,
                row = ((int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5)) * kRows + lane / kLanes;
  grid_dep_launch();
  const bool in = row < rows;
  const int32_t s = in ? (int32_t)(row / a.n_heads) : 0;
  grid_dep_wait();
  // (look-ups that all warps share go through L1: thousands of warps at one line of L2 took 6 us)
  PrefixSeq v = {0, 0, 0, 1};
  uint32_t rec = 0;
  const int G = a.n_heads / a.kv.n_kv, h = (int)(row - (int64_t)s * a.n_heads);
  if (in) {
    v = p.seqs[s];
    rec = (uint32_t)p.pieces[(int64_t)s * a.kv.n_kv + h / G];
  }
  float M = -INFINITY, L = 0.0f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  // the sums of `count` pieces, piece k at row at(k) of the arrays that it names
  auto join = [&](int count, auto at) {
    for (int k0 = 0; k0 < count; k0 += kAtOnce) {
      float2 ml[kAtOnce];
      float4 o[kAtOnce];
      float top = M;
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        ml[k] = make_float2(-INFINITY, 0.0f);
        if (k0 + k < count) {
          const float *os, *mls;
          const int64_t i = at(k0 + k, &os, &mls);
          ml[k] = __ldcg(reinterpret_cast<const float2*>(mls) + i);
          o[k] = __ldcg(reinterpret_cast<const float4*>(os + i * HD + d));
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
        if (ml[k].x == -INFINITY) continue;  // (saw nothing: what its sums hold counts for nothing)
        const float c = exp2_fast(ml[k].x - top);
        acc.x += c * o[k].x;
        acc.y += c * o[k].y;
        acc.z += c * o[k].z;
        acc.w += c * o[k].w;
        L += c * ml[k].y;
      }
    }
  };
  // the prefix's pieces, then the own positions' (one, or those of an item that CTAs shared)
  const int pieces = v.pre > 0 ? (v.pre - 1) / v.chunk + 1 : 0, slot = rec & 0xffffu;
  const int own = v.len > v.own ? (rec ? min((int)(rec >> 16), 1024) : 1) : 0;
  join(pieces + own, [&](int k, const float** os, const float** mls) {
    const int j = k - pieces;
    *os = j < 0 ? p.part : rec ? p.slots : p.own;
    *mls = j < 0 ? p.ml : rec ? p.slots_ml : p.own_ml;
    return j < 0 ? row + k * rows : rec ? (int64_t)min(j ? (slot & ~1) + 2 * j : slot, p.n_slots - 1) * G + h % G : row;
  });
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

// Pieces of a prefix: as many as fill the SMs once, a unit (two tiles of rows of a group
// and kv head, a piece) each.  A group with few sequences has a unit of its own for the few.
constexpr int kPieces = 32;  // at most (a piece's sums are written and read again)
int pieces_of(int32_t n_seqs, int32_t n_heads, int32_t n_kv, int32_t n_groups) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) cudaGetLastError();
  const int64_t U = 2 * (128 / (n_heads / n_kv)), rows = (n_seqs + U - 1) / U, units = (rows > n_groups ? rows : n_groups) * n_kv;
  const int64_t n = sm_count(dev) / (units > 0 ? units : 1);
  return n < 1 ? 1 : n > kPieces ? kPieces : (int)n;
}

// Slots of items that several CTAs share: two for each CTA of the kernel before.
int64_t slot_count() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) cudaGetLastError();
  return 2 * 4 * sm_count(dev);
}

// The workspace: single-token attention's (for calls of one kernel), then what the four
// kernels hand on.
struct Places {
  PrefixParts parts;
  int64_t bytes;
};
Places places(uint8_t* base, int32_t n_seqs, int32_t n_heads, int32_t n_kv, int32_t hd, int32_t n_groups) {
  PagedView v{};
  v.n_kv = n_kv;
  v.hd = hd;
  const int64_t rows = (int64_t)n_seqs * n_heads, pieces = pieces_of(n_seqs, n_heads, n_kv, n_groups), slots = slot_count() * (n_heads / n_kv);
  int64_t at = paged_decode_workspace(v, n_heads);
  Places p;
  auto take = [&](auto** to, int64_t n) {
    at += (256 - (int64_t)((reinterpret_cast<uintptr_t>(base) + (uintptr_t)at) & 255)) % 256;  // (the workspace may begin on any 16 bytes)
    *to = reinterpret_cast<std::remove_reference_t<decltype(*to)>>(base + at);
    at += n * (int64_t)sizeof(**to);
  };
  take(&p.parts.starts, slot_count());
  take(&p.parts.seqs, n_seqs);
  take(&p.parts.cum, (int64_t)n_seqs + 1);
  take(&p.parts.pieces, (int64_t)n_seqs * n_kv);
  take(&p.parts.ml, 2 * pieces * rows);
  take(&p.parts.own_ml, 2 * rows);
  take(&p.parts.slots_ml, 2 * slots);
  take(&p.parts.part, pieces * rows * hd);
  take(&p.parts.own, rows * hd);
  take(&p.parts.slots, slots * hd);
  p.parts.n_slots = (int32_t)slot_count();
  p.bytes = at + 256;
  return p;
}

}  // namespace

int64_t paged_prefix_workspace(int32_t n_seqs, int32_t n_heads, int32_t n_kv, int32_t hd) {
  return places(nullptr, n_seqs, n_heads, n_kv, hd, 0).bytes;  // (more groups, fewer pieces)
}

cudaError_t paged_prefix_decode_launch(const PagedOwnArgs& a, cudaStream_t s) {
  if (paged_decode_through_fits(a)) return paged_decode_through_launch(a, s);
  const int G = a.n_heads / a.kv.n_kv;
  int dev = 0;
  cudaGetDevice(&dev);
  PrefixShape shape;
  shape.T = 128 / G;
  shape.pieces = pieces_of(a.b.n_seqs, a.n_heads, a.kv.n_kv, a.pre.n_groups);
  // as many CTAs as may have a unit: the others' SMs are free for the next kernel at once
  const int64_t reach = (((int64_t)a.pre.max_pages << a.pre.kv.page_shift) + kPrefixKeys - 1) / kPrefixKeys,
                most = (a.b.n_seqs / (2 * shape.T) + a.pre.n_groups) * a.kv.n_kv * (reach < shape.pieces ? reach : shape.pieces);
  shape.ctas = (int32_t)(most < sm_count(dev) ? most : sm_count(dev));
  if (a.scales) paged8_decode_prefix_shape(a, &shape);
  else paged_decode_prefix_shape(a, &shape);
  const PrefixParts p = places(static_cast<uint8_t*>(a.workspace), a.b.n_seqs, a.n_heads, a.kv.n_kv, a.kv.hd, a.pre.n_groups).parts;
  cudaError_t e = paged_plan_launch(a, p, shape, s);
  if (e == cudaSuccess) e = paged_prefix_launch(a, p, shape, s);
  if (e == cudaSuccess) e = a.scales ? paged8_decode_prefix_launch(a, p, shape, s) : paged_decode_prefix_launch(a, p, shape, s);
  if (e != cudaSuccess) return e;
  if (a.kv.hd == 128) e = a.kv.bf16 ? join_go<128, true>(a, p, s) : join_go<128, false>(a, p, s);
  else e = a.kv.bf16 ? join_go<64, true>(a, p, s) : join_go<64, false>(a, p, s);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

}  // namespace rpgc
