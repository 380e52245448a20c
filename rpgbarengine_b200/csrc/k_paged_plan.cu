// k_paged_plan.cu -- single-token attention with a shared prefix: who does what.
//
// Lengths, groups and prefixes are device data, so the work is cut on the device, by one
// CTA before the kernels that do it: what each sequence sees, the length of a piece of a
// prefix and each CTA's first unit of rows and positions (k_paged_prefix.cu), each CTA's
// range of the list of own key tiles (paged_decode.cuh).  Each of those kernels' hundreds of
// CTAs finding this by itself took 4 to 15 us, most of it instructions fetched and the same
// few lines of L2 asked for.
#include <cuda_runtime.h>

#include "paged8_dev.cuh"
#include "paged_dev.cuh"
#include "paged_tma.cuh"

namespace rpgc {
namespace {

using namespace paged;

constexpr int kThreads = 1024;
constexpr int kSeqs = 2048;    // sequences whose sums of weights are in shared memory
constexpr int kGroups = 1024;  // groups that are
// What a unit of the prefix kernel costs besides its tiles (its begin and end), in tiles.
constexpr int kUnitCost = 8;
// Bytes (of K and V) that a CTA over own positions copies, four on an SM, while a unit of
// the prefix kernel begins and ends, and while one of its tiles runs: 7 us and 0.85 us at 11 GB/s.
constexpr float kLateFixed = 77000.0f, kLateTile = 9400.0f;

// w places in n equal ranges: where range b begins, and the range that holds place t.
RPGC_DEV int64_t part_begin(int64_t b, int64_t n, int64_t w) { return w < (1 << 21) ? (int64_t)((uint32_t)b * (uint32_t)w / (uint32_t)n) : b * w / n; }
RPGC_DEV int32_t part_of(int64_t t, int64_t n, int64_t w) {
  return w < (1 << 21) ? (int32_t)((((uint32_t)t + 1) * (uint32_t)n - 1) / (uint32_t)w) : (int32_t)(((t + 1) * n - 1) / w);  // (n < 2048)
}

// Inclusive sums over the block; *all: over all of it.  (Every thread calls it.)
RPGC_DEV uint32_t block_scan(uint32_t v, uint32_t* warps, uint32_t* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  __syncthreads();  // (the last call's sums are read)
  if (lane == 31) warps[warp] = v;
  __syncthreads();
  uint32_t x = warps[lane], sum = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += y;
  }
  *all = __shfl_sync(0xffffffffu, sum, 31);
  return v + __shfl_sync(0xffffffffu, sum - x, warp);
}

__global__ void __launch_bounds__(kThreads) plan_kernel(const __grid_constant__ PagedOwnArgs a, const __grid_constant__ PrefixParts p,
                                                        const __grid_constant__ PrefixShape sh) {
  __shared__ int64_t cum_here[kSeqs + 1];
  __shared__ int32_t first[kGroups + 1], len[kGroups];
  __shared__ uint32_t warps[32], units_by[32];
  __shared__ int32_t most, rows, some;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n_seqs = a.b.n_seqs, n_groups = a.pre.n_groups, kv = a.kv.n_kv;
  const int T = sh.T, U = 2 * T;
  if (tid < 32) units_by[tid] = 0;
  if (tid == 0) most = rows = some = 0;
  grid_dep_wait();
  grid_dep_launch();
  const bool few = n_groups <= kGroups;
  Share mine = {0, 0, 0};  // group tid's, where they are few
  if (few) {
    mine = share_of(a, tid);
    if (tid < n_groups) {
      first[tid] = mine.seq;
      len[tid] = a.pre.lens[tid];
    }
    if (tid == 0) first[n_groups] = group_seq(a.pre, n_seqs, n_groups);
  }
  __syncthreads();
  // ------------------------------------------ sequences: what they see, their tiles' weights
  int64_t* cum = n_seqs <= kSeqs ? cum_here : p.cum;
  int64_t carry = 0;
  int32_t with = 0;
  for (int s0 = 0; s0 < n_seqs; s0 += kThreads) {
    const int s = s0 + tid;
    uint32_t w = 0, all;
    if (s < n_seqs) {
      const int32_t n = a.b.kv_lens[s];
      const int32_t g = few ? group_of(n_groups, s, [&](int i) { return first[i]; })
                            : group_of(n_groups, s, [&](int i) { return group_seq(a.pre, n_seqs, i); });
      const PrefixSeq v = sight_of(a, n, g < 0 ? 0 : few ? len[g] : a.pre.lens[g]);
      p.seqs[s] = v;
      if (v.len > v.own) {
        const int64_t T1 = (int64_t)1 << sh.tile_log;
        w = (uint32_t)((v.len + T1 - 1) >> sh.tile_log) - (uint32_t)(v.own >> sh.tile_log) + kItemEnd;
        ++with;
      }
    }
    const uint32_t upto = block_scan(w, warps, &all);
    if (s < n_seqs) cum[s + 1] = carry + upto;
    carry += all;
  }
  if (tid == 0) cum[0] = 0;
  with = __reduce_add_sync(0xffffffffu, with);
  if (lane == 0 && with) atomicAdd(&some, with);
  // --------------------------------------------------------- prefixes: the length of a piece
  for (int g0 = warp * 32; g0 < n_groups; g0 += kThreads) {
    const Share s = few ? mine : share_of(a, g0 + lane);
    const int32_t nt = __reduce_max_sync(0xffffffffu, tiles_of(s)), r = __reduce_max_sync(0xffffffffu, s.end ? s.n : 0);
    if (lane == 0) {
      atomicMax(&most, nt);
      atomicMax(&rows, r);
    }
  }
  __syncthreads();
  // lane k weighs the length that cuts the longest prefix into k + 1 pieces: rounds of units
  // over the CTAs, each a piece's tiles (two for each where a unit has two tiles of rows)
  const int32_t c = max(1, (most + lane) / (lane + 1)), per = rows > T ? 2 : 1;
  for (int g0 = warp * 32; g0 < n_groups; g0 += kThreads) {
    const Share s = few ? mine : share_of(a, g0 + lane);
    const int32_t R = (s.n + U - 1) / U, nt = tiles_of(s);
    uint32_t units = 0;
    for (int i = 0; i < min(32, n_groups - g0); ++i) units += __shfl_sync(0xffffffffu, R, i) * ((__shfl_sync(0xffffffffu, nt, i) + c - 1) / c);
    if (units) atomicAdd(units_by + lane, units * kv);
  }
  __syncthreads();
  const int32_t rounds = (int32_t)((units_by[lane] + sh.ctas - 1) / sh.ctas);
  const float cost = lane < sh.pieces ? (float)rounds * (float)(c * per + kUnitCost) : INFINITY;
  const uint32_t best = __reduce_min_sync(0xffffffffu, __float_as_uint(cost));  // (positive floats in order)
  const int src = __ffs(__ballot_sync(0xffffffffu, __float_as_uint(cost) == best)) - 1;
  const int32_t chunk = __shfl_sync(0xffffffffu, c, src), units = (int32_t)__shfl_sync(0xffffffffu, units_by[lane], src),
                turns = __shfl_sync(0xffffffffu, rounds, src);
  if (tid == 0) *p.head = PrefixHead{chunk, units};
  // ---------------------------------------------------------- the CTAs' first units of prefixes
  if (few) {
    __syncthreads();  // (the groups' first sequences are read no more: their units' sums take the place)
    uint32_t all;
    const uint32_t upto = block_scan(units_of(mine, U, chunk, kv), warps, &all);
    if (tid < n_groups) first[tid + 1] = (int32_t)upto;
    if (tid == 0) first[0] = 0;
    __syncthreads();
  }
  for (int b = tid; b < sh.ctas; b += kThreads) {
    PrefixUnit un;
    un.seq = b >= units ? -1 : -2;
    if (few && b < units) {
      const int32_t g = group_of(n_groups, b, [&](int i) { return first[i]; });
      un = unit_of(share_of(a, g), g, b - first[g], T, chunk, kv);
    }
    p.units[b] = un;
  }
  // ------------------------------------------------------------ ranges of the own tiles' list
  const int64_t total = carry * kv;
  // no more CTAs than there is weight, nor so many pieces of an item that its join is long
  int parts = (int)min(min(total, (int64_t)sh.own_ctas), (int64_t)some * kv * kItemPieces);
  // CTAs whose SMs the prefix kernel holds begin when its units end (the last ones: CTAs
  // begin in order): they get less, by the tiles that the others do meanwhile
  int early = max(0, sh.own_ctas - sh.on_sm * min(units, sh.ctas));
  int64_t theirs = total;
  if (early > 0 && early < parts) {
    const int64_t less = (int64_t)((kLateFixed + kLateTile * (float)min(turns * chunk * per, 1 << 16)) / (float)sh.stage) + 1,
                  each = (total + (parts - early) * less) / parts;
    if (each <= less || each * early >= total) parts = early;
    else theirs = each * early;
  } else {
    early = parts;
  }
  auto begin = [&](int b) { return b <= early ? part_begin(b, early, theirs) : theirs + part_begin(b - early, parts - early, total - theirs); };
  auto find = [&](int64_t place, PrefixStart& r) {  // the item that holds a place; its weight
    int lo = 0, hi = n_seqs - 1;                     // the last sequence that begins at it or before
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (cum[mid] * kv <= place) lo = mid;
      else hi = mid - 1;
    }
    const int64_t w = cum[lo + 1] - cum[lo], in = place - cum[lo] * kv;
    r.seq = lo;
    r.kh = (int32_t)(in / w);
    r.first = cum[lo] * kv + r.kh * w;
    return w;
  };
  for (int b = tid; b < sh.own_ctas; b += kThreads) {
    PrefixStart r;
    r.lo = r.hi = r.first = 0;
    r.seq = r.kh = r.len = r.own = r.tail = r.pad = 0;
    if (b < parts) {
      PrefixStart last;
      r.lo = begin(b);
      r.hi = begin(b + 1);
      if (r.hi > r.lo) {
        const int64_t w = find(r.hi - 1, last), i0 = last.first + kItemEnd, i1 = last.first + w;
        if (i1 > r.hi && i0 >= r.lo && i0 < r.hi) {
          const int64_t t = i1 - 1;
          r.tail = (t < theirs ? part_of(t, early, theirs) : early + part_of(t - theirs, parts - early, total - theirs)) - b + 1;
        }
        find(r.lo, r);
        const PrefixSeq v = p.seqs[r.seq];
        r.len = v.len;
        r.own = v.own;
      }
    }
    p.starts[b] = r;
  }
}

}  // namespace

cudaError_t paged_plan_launch(const PagedOwnArgs& a, const PrefixParts& parts, const PrefixShape& shape, cudaStream_t s) {
  const cudaError_t e = launch_pdl(plan_kernel, dim3(1), dim3(kThreads), 0, s, a, parts, shape);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

}  // namespace rpgc
