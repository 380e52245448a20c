// k_paged_plan.cu -- single-token attention with a shared prefix: what each sequence
// sees, and which own key tiles each CTA takes.
//
// Lengths, groups and prefixes are device data, so the work is cut on the device, by one
// CTA before the kernels that do it: each CTA's range of the list of own key tiles
// (paged_decode.cuh) is here.  Each of that kernel's hundreds of CTAs finding its own took 4
// to 15 us, most of it instructions fetched and the same few lines of L2 asked for.  This one
// takes 5-6 us, latency all of it, and the prefix kernel runs beside it.
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

// w places in n (< 2048) equal ranges: where range b begins, and the range that holds place
// t.  I: uint32_t where w n is below 2^32, int64_t else.
template <typename I>
RPGC_DEV I part_begin(int b, int n, I w) { return (I)b * w / (I)n; }
template <typename I>
RPGC_DEV int part_of(I t, int n, I w) { return (int)(((t + 1) * (I)n - 1) / w); }

// The list of own tiles in ranges: the first `early` of `parts` have `theirs` of its places.
template <typename I>
struct Ranges {
  I total, theirs;
  int parts, early;
  RPGC_DEV I begin(int b) const {
    return b <= early ? part_begin<I>(b, early, theirs) : theirs + part_begin<I>(b - early, parts - early, total - theirs);
  }
  RPGC_DEV int holder(I t) const {
    return t < theirs ? part_of<I>(t, early, theirs) : early + part_of<I>(t - theirs, parts - early, total - theirs);
  }
};

// Inclusive sums over the block; *all: over all of it.  (Every thread calls it.)
template <typename I>
RPGC_DEV I block_scan(I v, I* warps, I* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const I x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  if (lane == 31) warps[warp] = v;
  __syncthreads();
  I x = warps[lane], sum = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const I y = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += y;
  }
  *all = __shfl_sync(0xffffffffu, sum, 31);
  return v + __shfl_sync(0xffffffffu, sum - x, warp);
}

__global__ void __launch_bounds__(kThreads) plan_kernel(const __grid_constant__ PagedOwnArgs a, const __grid_constant__ PrefixParts p,
                                                        const __grid_constant__ PrefixShape sh) {
  __shared__ uint32_t cum_here[kSeqs + 1];
  __shared__ int2 seen_here[kSeqs];
  __shared__ int64_t begins[kThreads + 1];
  __shared__ int32_t first[kGroups + 1], len[kGroups], weight[kThreads + 1];
  __shared__ uint64_t warps[2][32];
  __shared__ int32_t some, units, longest, pairs;
  const int tid = threadIdx.x, lane = tid & 31, n_seqs = a.b.n_seqs, n_groups = a.pre.n_groups, kv = a.kv.n_kv;
  if (tid == 0) some = units = longest = pairs = 0;
  grid_dep_wait();
  grid_dep_launch();
  const bool few = n_groups <= kGroups;
  int32_t n = tid < n_seqs ? a.b.kv_lens[tid] : 0;
  Share mine{0, 0, 0};  // of the group of the last warps' threads first, so that they are not those of the sequences
  const int g1 = kThreads - 1 - tid;
  if (few) {
    mine = share_of<false>(a, g1);
    if (g1 < n_groups) {
      first[g1] = mine.seq;
      len[g1] = a.pre.lens[g1];
      if (g1 + 1 == n_groups) first[n_groups] = group_seq<false>(a.pre, n_seqs, n_groups);
    }
  }
  __syncthreads();
  // the prefix kernel's units, tiles of the longest, whether some have two tiles of rows
  for (int g0 = kThreads - 32 - (tid - lane); g0 < n_groups; g0 += kThreads) {  // (whole warps)
    const Share s = few ? mine : share_of<false>(a, g0 + 31 - lane);
    const int32_t u = __reduce_add_sync(0xffffffffu, units_of(s, sh.T, sh.pieces, kv)), c = __reduce_max_sync(0xffffffffu, s.end ? chunk_of(tiles_of(s), sh.pieces) : 0),
                  r = __reduce_max_sync(0xffffffffu, s.end ? s.n : 0);
    if (lane == 0) {
      atomicAdd(&units, u);
      atomicMax(&longest, c);
      atomicMax(&pairs, r > sh.T);
    }
  }
  // ------------------------------------------ sequences: what they see, their tiles' weights
  int64_t carry = 0;
  for (int s0 = 0; s0 < n_seqs; s0 += kThreads) {
    const int s = s0 + tid;
    uint32_t w = 0;
    uint64_t upto, all;
    if (s < n_seqs) {
      if (s0) n = a.b.kv_lens[s];
      const int32_t g = few ? group_of(n_groups, s, [&](int i) { return first[i]; })
                            : group_of(n_groups, s, [&](int i) { return group_seq<false>(a.pre, n_seqs, i); });
      const int32_t plen = g < 0 ? 0 : few ? len[g] : a.pre.lens[g];
      PrefixSeq v = sight_of(a, n, plen);
      Share share{0, 0, (int32_t)min((int64_t)max(0, plen), (int64_t)a.pre.max_pages << a.pre.kv.page_shift)};
      v.chunk = chunk_of(tiles_of(share), sh.pieces) * kPrefixKeys;
      p.seqs[s] = v;
      if (s < kSeqs) seen_here[s] = make_int2(v.len, v.own);
      if (v.len > v.own) {
        const int64_t T1 = (int64_t)1 << sh.tile_log;
        w = (uint32_t)((v.len + T1 - 1) >> sh.tile_log) - (uint32_t)(v.own >> sh.tile_log) + kItemEnd;
      }
    }
    const uint32_t has = __ballot_sync(0xffffffffu, w > 0);
    if (lane == 0 && has) atomicAdd(&some, __popc(has));
    uint64_t* sums = warps[s0 / kThreads & 1];
    if (__syncthreads_or(w >> 21)) {
      upto = block_scan<uint64_t>(w, sums, &all);
    } else {  // (1024 of them are below 2^32)
      uint32_t every;
      upto = block_scan<uint32_t>(w, reinterpret_cast<uint32_t*>(sums), &every);
      all = every;
    }
    if (s < n_seqs) {
      p.cum[s + 1] = carry + (int64_t)upto;
      if (s < kSeqs) cum_here[s + 1] = (uint32_t)(carry + (int64_t)upto);
    }
    carry += (int64_t)all;
  }
  if (tid == 0) {
    cum_here[0] = 0;
    p.cum[0] = 0;
  }
  __syncthreads();
  // ------------------------------------------------------------ ranges of the own tiles' list
  const int64_t total = carry * kv;
  const bool here = n_seqs <= kSeqs && carry < (int64_t)1 << 31;  // in shared memory
  // no more CTAs than there is weight, nor so many pieces of an item that its join is long
  int parts = (int)min(min(total, (int64_t)sh.own_ctas), (int64_t)some * kv * kItemPieces);
  // CTAs whose SMs the prefix kernel holds begin when its units end (the last ones: CTAs
  // begin in order): they get less, by the tiles that the others do meanwhile
  int early = max(0, sh.own_ctas - sh.on_sm * min(units, sh.ctas));
  int64_t theirs = total;
  if (early > 0 && early < parts) {
    const float tiles = (float)((units + sh.ctas - 1) / sh.ctas) * (float)(longest * (pairs ? 2 : 1)), less = (kLateFixed + kLateTile * tiles) / (float)sh.stage + 1.0f,
                each = floorf(((float)total + (float)(parts - early) * less) / (float)parts);  // (a share: it need not be exact)
    const int64_t first_ones = (int64_t)each * early;
    if (each <= less || first_ones > total - (parts - early)) parts = early;
    else theirs = first_ones;
  } else {
    early = parts;
  }
  const int b = tid;  // (no more CTAs than threads)
  PrefixStart r;
  r.lo = r.hi = r.first = 0;
  r.seq = r.kh = r.len = r.own = r.tail = r.pad = 0;
  // cum(s): weight of the sequences before s, for one kv head
  auto cut = [&](auto type, auto cum) {
    using I = decltype(type);
    const Ranges<I> in{(I)total, (I)theirs, parts, early};
    if (b < parts) {
      const I place = in.begin(b);
      int lo = 0, hi = n_seqs - 1;  // the last sequence that begins there or before
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if ((I)cum(mid) * (I)kv <= place) lo = mid;
        else hi = mid - 1;
      }
      const I before = (I)cum(lo), w = (I)cum(lo + 1) - before;
      r.lo = (int64_t)place;
      r.seq = lo;
      r.kh = (int32_t)((place - before * (I)kv) / w);
      r.first = (int64_t)(before * (I)kv + (I)r.kh * w);
      begins[b] = r.first;
      weight[b] = (int32_t)w;
      int2 v;
      if (here) {
        v = seen_here[lo];
      } else {
        const PrefixSeq x = p.seqs[lo];
        v = make_int2(x.len, x.own);
      }
      r.len = v.x;
      r.own = v.y;
    }
    __syncthreads();
    if (b < parts) {
      r.hi = (int64_t)in.begin(b + 1);
      // the item that goes on past hi is the next CTA's first
      if (b + 1 < parts && begins[b + 1] < r.hi) {
        const int64_t i0 = begins[b + 1] + kItemEnd, t = begins[b + 1] + weight[b + 1] - 1;
        if (i0 >= r.lo && i0 < r.hi) r.tail = in.holder((I)t) - b + 1;
      }
    }
  };
  if (here && total < (int64_t)1 << 21) cut(uint32_t{}, [&](int i) { return cum_here[i]; });
  else if (here) cut(int64_t{}, [&](int i) { return cum_here[i]; });
  else cut(int64_t{}, [&](int i) { return p.cum[i]; });
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
