// k_paged_plan.cu -- single-token attention with a shared prefix: what each sequence
// sees, and which own key tiles each CTA takes.
//
// Lengths, groups and prefixes are device data, so the work is cut on the device, by one
// CTA before the kernels that do it: each CTA's range of the list of own key tiles
// (paged_decode.cuh) is here.  Each of that kernel's hundreds of CTAs finding its own took 4
// to 15 us, most of it instructions fetched and the same few lines of L2 asked for.  The
// prefix kernel runs beside this one.
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
// Bytes (of K and V) that a CTA over own positions copies, four on an SM, while a unit of
// the prefix kernel begins and ends, and while one of its tiles runs: 7 us and 0.85 us at 11 GB/s.
constexpr float kLateFixed = 77000.0f, kLateTile = 9400.0f;

// w places in n (< 2048) equal ranges: where range b begins, and the range that holds place t.
RPGC_DEV int64_t part_begin(int b, int n, int64_t w) { return w < (1 << 21) ? (int64_t)((uint32_t)b * (uint32_t)w / (uint32_t)n) : b * w / n; }
RPGC_DEV int part_of(int64_t t, int n, int64_t w) {
  return w < (1 << 21) ? (int)((((uint32_t)t + 1) * (uint32_t)n - 1) / (uint32_t)w) : (int)(((t + 1) * n - 1) / w);
}

// Inclusive sums over the block; *all: over all of it.  (Every thread calls it.)
RPGC_DEV uint32_t block_scan(uint32_t v, uint32_t* warps, uint32_t* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
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
  __shared__ int64_t cum_here[kSeqs + 1], begins[kThreads + 1];
  __shared__ int32_t first[kGroups + 1], len[kGroups], weight[kThreads + 1];
  __shared__ uint32_t warps[2][32];
  __shared__ int32_t some, units, longest, pairs;
  const int tid = threadIdx.x, lane = tid & 31, n_seqs = a.b.n_seqs, n_groups = a.pre.n_groups, kv = a.kv.n_kv;
  if (tid == 0) some = units = longest = pairs = 0;
  grid_dep_wait();
  grid_dep_launch();
  const bool few = n_groups <= kGroups;
  int32_t n = tid < n_seqs ? a.b.kv_lens[tid] : 0;
  __syncthreads();
  // the prefix kernel's units, tiles of the longest, whether some have two tiles of rows
  for (int g0 = tid - lane; g0 < n_groups; g0 += kThreads) {
    const Share s = share_of<false>(a, g0 + lane);
    if (few && tid < n_groups) {
      first[tid] = s.seq;
      len[tid] = a.pre.lens[tid];
      if (tid + 1 == n_groups) first[n_groups] = group_seq<false>(a.pre, n_seqs, n_groups);
    }
    const int32_t u = __reduce_add_sync(0xffffffffu, units_of(s, sh.T, sh.pieces, kv)), c = __reduce_max_sync(0xffffffffu, s.end ? chunk_of(tiles_of(s), sh.pieces) : 0),
                  r = __reduce_max_sync(0xffffffffu, s.end ? s.n : 0);
    if (lane == 0) {
      atomicAdd(&units, u);
      atomicMax(&longest, c);
      atomicMax(&pairs, r > sh.T);
    }
  }
  __syncthreads();
  // ------------------------------------------ sequences: what they see, their tiles' weights
  int64_t* cum = n_seqs <= kSeqs ? cum_here : p.cum;
  int64_t carry = 0;
  for (int s0 = 0; s0 < n_seqs; s0 += kThreads) {
    const int s = s0 + tid;
    uint32_t w = 0, all;
    if (s < n_seqs) {
      if (s0) n = a.b.kv_lens[s];
      const int32_t g = few ? group_of(n_groups, s, [&](int i) { return first[i]; })
                            : group_of(n_groups, s, [&](int i) { return group_seq<false>(a.pre, n_seqs, i); });
      const int32_t plen = g < 0 ? 0 : few ? len[g] : a.pre.lens[g];
      PrefixSeq v = sight_of(a, n, plen);
      Share share{0, 0, (int32_t)min((int64_t)max(0, plen), (int64_t)a.pre.max_pages << a.pre.kv.page_shift)};
      v.chunk = chunk_of(tiles_of(share), sh.pieces) * kPrefixKeys;
      p.seqs[s] = v;
      if (v.len > v.own) {
        const int64_t T1 = (int64_t)1 << sh.tile_log;
        w = (uint32_t)((v.len + T1 - 1) >> sh.tile_log) - (uint32_t)(v.own >> sh.tile_log) + kItemEnd;
      }
    }
    const uint32_t has = __ballot_sync(0xffffffffu, w > 0);
    if (lane == 0 && has) atomicAdd(&some, __popc(has));
    const uint32_t upto = block_scan(w, warps[s0 / kThreads & 1], &all);
    if (s < n_seqs) cum[s + 1] = carry + upto;
    carry += all;
  }
  if (tid == 0) cum[0] = 0;
  __syncthreads();
  // ------------------------------------------------------------ ranges of the own tiles' list
  const int64_t total = carry * kv;
  // no more CTAs than there is weight, nor so many pieces of an item that its join is long
  int parts = (int)min(min(total, (int64_t)sh.own_ctas), (int64_t)some * kv * kItemPieces);
  // CTAs whose SMs the prefix kernel holds begin when its units end (the last ones: CTAs
  // begin in order): they get less, by the tiles that the others do meanwhile
  int early = max(0, sh.own_ctas - sh.on_sm * min(units, sh.ctas));
  int64_t theirs = total;
  if (early > 0 && early < parts) {
    const int rounds = (units + sh.ctas - 1) / sh.ctas;
    const int64_t less = (int64_t)((kLateFixed + kLateTile * (float)min(rounds * longest * (pairs ? 2 : 1), 1 << 16)) / (float)sh.stage) + 1,
                  each = (total + (parts - early) * less) / parts;
    if (each <= less || each * early >= total) parts = early;
    else theirs = each * early;
  } else {
    early = parts;
  }
  const int b = tid;  // (no more CTAs than threads)
  PrefixStart r;
  r.lo = r.hi = r.first = 0;
  r.seq = r.kh = r.len = r.own = r.tail = r.pad = 0;
  auto begin = [&](int i) { return i <= early ? part_begin(i, early, theirs) : theirs + part_begin(i - early, parts - early, total - theirs); };
  int32_t w = 0;
  if (b < parts) {
    r.lo = begin(b);
    int lo = 0, hi = n_seqs - 1;  // the last sequence that begins there or before
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (cum[mid] * kv <= r.lo) lo = mid;
      else hi = mid - 1;
    }
    const int64_t at = cum[lo] * kv, in = r.lo - at;
    w = (int32_t)(cum[lo + 1] - cum[lo]);
    r.seq = lo;
    r.kh = in < (int64_t)0x7fffffff ? (int32_t)((uint32_t)in / (uint32_t)w) : (int32_t)(in / w);
    r.first = at + (int64_t)r.kh * w;
    const PrefixSeq v = p.seqs[lo];
    r.len = v.len;
    r.own = v.own;
    begins[b] = r.first;
    weight[b] = w;
  }
  __syncthreads();
  if (b < parts) {
    r.hi = begin(b + 1);
    // the item that goes on past hi is the next CTA's first
    if (b + 1 < parts && begins[b + 1] < r.hi) {
      const int64_t i0 = begins[b + 1] + kItemEnd, t = begins[b + 1] + weight[b + 1] - 1;
      if (i0 >= r.lo && i0 < r.hi)
        r.tail = (t < theirs ? part_of(t, early, theirs) : early + part_of(t - theirs, parts - early, total - theirs)) - b + 1;
    }
  }
  if (b < sh.own_ctas) p.starts[b] = r;
}

}  // namespace

cudaError_t paged_plan_launch(const PagedOwnArgs& a, const PrefixParts& parts, const PrefixShape& shape, cudaStream_t s) {
  if (shape.own_ctas > kThreads) return cudaErrorInvalidValue;
  const cudaError_t e = launch_pdl(plan_kernel, dim3(1), dim3(kThreads), 0, s, a, parts, shape);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

}  // namespace rpgc
