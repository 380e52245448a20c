// paged_decode.cuh -- the kernel of attention of one new token per sequence over the
// pages of the KV cache: 16-bit pages (k_paged_decode.cu), 8-bit ones (F8,
// k_paged8_decode.cu), and either behind a shared prefix (SH, k_paged_decode_prefix.cu,
// k_paged8_decode_prefix.cu), whose sums k_paged_prefix.cu has made; or through a small prefix
// and on through 16-bit pages (k_paged_decode_through.cu).
//
// Mathematics: out = sum_t p_t v_t / sum_t p_t with p_t = 2^(c s_t - m),
// s_t = q . k_t, c = scale * log2(e): one pass over the keys with a reference m,
// the maximum of a warp's first keys until a later probability outgrows what 16
// bits hold (2^40 in bf16, 2^15 in fp16), so that most steps look for no
// maximum and rescale nothing.  Reference: AttentionFromCache (src/qwen3.cc:79-117).
//
// Bound: every K and V byte is read once, so HBM is the limit.  The key tiles of
// all (sequence, kv head) items form one list, cut into equal ranges, one per
// CTA: batches of any mix of lengths, and one long sequence as well, give every
// SM the same bytes.  An item that several CTAs share is joined by the last of
// them to finish, from partial results in the workspace, in the order of the
// pieces (the same result whoever is last).
//
// A CTA: two warps walk its range and issue the TMA copies of K and of V into a
// ring (with one warp for both, pages of 16 positions of 64 dims were issued at
// 2.8 TB/s); 4 warps take 16 keys each of every tile: S^T = K Q^T (m16n8k16, the
// kv head's query heads are the N side), P^T turned from the accumulator layout
// into an operand by movmatrix, O^T += V^T P^T.  (mma.sync: at 4 to 16 rows a
// head group has nothing for wider MMAs.)  The warps' sums meet in shared memory
// at an item's end.  A row that comes out infinite or NaN though its weights are
// finite is computed again by one warp in fp32 (attn_row): a weight's second
// 16-bit value may be 0 or negative, and that times a visible infinity is not the
// infinity that the row should have; and weights of up to 2^40 may overflow with
// values that the true weights, at most 1, do not.  Two such CTAs on an SM, 192 KB in flight between them: while
// one ends an item or looks for the next, the other's tiles go on (one CTA of 8
// warps took 1.5 times as long on 128 sequences of 20 positions, 1.08 times on
// 128 of 500).
//
// Measured with 32 query and 8 kv heads of 128, bf16: 128 sequences of 1-8192
// positions 318-327 us (2.17 GB, 6.6-6.8 TB/s), 64 of ~1100 52.6 us (5.5 TB/s; 8 us of it
// are the look-ups before the first tile and the last joins), 128 of 200 28 us
// (3.7 TB/s), one of 4200 10.4 us, one of 33 (16 heads) 4.2 us; 48 sequences with
// 12 heads of 64 in pages of 16, 167 MB, 39-41 us.  Groups of 16 (NT 2, one CTA per SM),
// 64 of ~1090: 32 / 2 heads of 128 28 us (2.5 TB/s), 16 / 1 20.6 us (1.7 TB/s).
//
// 8-bit pages (F8): k_t = dk_t ck_t and v_t = dv_t cv_t, codes c (e4m3) and a scale d for
// each row.  Codes become fp16 operands in registers (exact; two instructions a word), dk
// goes onto the scores, dv onto the weights, q into fp16 by a power of two: scores, weights
// and sums are as exact as over 16-bit pages.  Half the bytes leave half the time for the
// steps of a tile, so a warp has two independent chains of 16 keys (with one: 128 sequences
// of 1-8192 positions 220 us).  Measured, 32 / 8 heads of 128: those 128 sequences 191-211 us
// (1.21 GB, 5.7-6.3 TB/s), one of 4200 10.6 us, one of 33 (16 heads) 4.9; 48 with 12 heads of 64 in
// pages of 16, 92 MB, 37-40 us (2.4 TB/s): 5 us until the first tiles are there, 3 us for each of the
// two shared items of a CTA, and in between 17 KB a tile at 1.6-1.8 k clocks.
//
// Behind a prefix (SH): an item's tiles begin with the one that holds its first own position.
// Planned: ranges and items come from the plan, sums go to the kernel that joins them with the
// prefix's.  Through: the prefix's tiles come before them, by its own table and pool, and the
// item ends as one without a prefix does (64 sequences of ~735 positions behind 256 shared ones
// 41.8 us, where the same pages named by the sequences' own tables take 39.4).
// Tiles that are not seen whole come in copies of 16 rows (planned, and F8).
#pragma once

#include <cuda_runtime.h>

#include <type_traits>

#include "paged8_dev.cuh"
#include "paged_dev.cuh"
#include "paged_tma.cuh"

namespace rpgc {
namespace {

using namespace paged;

constexpr int kJoin = 8;   // pieces of a share whose sums are in flight at once
constexpr int kAhead = 4;  // V operands loaded ahead of the probabilities
constexpr float kLog2e = 1.4426950408889634f;
// SH: behind a prefix.  Planned: ranges by a plan, sums left to the kernel that joins them.
// Through: an item's tiles are its prefix's, then its own, both of 16 bits.
constexpr int kPlanned = 1, kThrough = 2;
constexpr int kThroughGroups = 15;  // (a warp's lanes hold their first sequences and lengths)

// F8: K and V as codes, a byte each.  Many: four small CTAs on an SM.  What ends an item
// and begins the next are chains of dependent steps (q, the first tile's scores, the warps'
// sums: 2500 clocks beside 1200 a tile), and the positions behind a prefix are many short
// items: four chains at once (256 sequences of 1-200 own positions behind 8192 shared ones
// 67.2 us, with two CTAs of 4 warps 73.5; 64 of ~735 behind 256 47.7 either way).
template <int HD, int NT, bool F8 = false, bool Many = false>
struct DShape {
  static constexpr bool kMany = Many && NT == 1;
  static constexpr int kCtas = NT > 1 ? 1 : kMany ? 4 : 2;  // CTAs on an SM (NT 2: over 240 registers a thread leave room for one)
  static constexpr int kWarps = kMany ? 2 : HD == 128 || NT == 1 ? 4 : 8;  // consumer warps
  static constexpr int kLoaders = kMany ? 1 : 2;      // warps that copy K and V, or one K, one V
  static constexpr int kSub = F8 && NT == 1 ? 2 : 1;  // 16 keys of a tile each, or two times 16
  static constexpr int kTile = 16 * kSub * kWarps;    // keys
  static constexpr int kThreads = (kWarps + kLoaders) * 32;
  static constexpr int kPanels = F8 ? 1 : HD / 64;
  static constexpr int kPanel = F8 ? kTile * HD : kTile * 128;
  static constexpr int kHalf = kPanels * kPanel;  // K (or V) of a tile
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kScales = F8 ? kTile * 4 : 0;  // K's (or V's) scales of a tile
  static constexpr int kScaleRoom = 2 * kScales;      // (a TMA copy starts on 128 bytes, one of 16 scales too)
  static constexpr int kHeads = 8 * NT;           // query heads of a kv head, padded
  static constexpr int kPad = HD + 4;             // row of the merge buffer: no bank conflicts
  static constexpr int kMerge = kWarps * kHeads * kPad * 4;  // the warps' sums; later the join's table, 8 bytes per piece and head
  static constexpr int kRest = kMerge + 2 * kWarps * kHeads * 4 + 256;
  // what an SM has, less a kilobyte for each CTA, goes to the ring
  static constexpr int kStages = ((233472 / kCtas - 1024) - kRest) / (kStage + 2 * kScaleRoom);
  static constexpr int kSmem = kStages * (kStage + 2 * kScaleRoom) + kRest;
  static_assert(kStages * 20 + 12 <= 256, "barriers and flags");
};

// Maps that 16-bit pages alone do without: the scales' (8-bit pages), K and V in copies
// of 16 rows for tiles that are not whole.
template <bool F8>
struct MoreMaps {
  CUtensorMap k, v;
};
template <>
struct MoreMaps<true> {
  CUtensorMap k, v, s;
};
struct NoMaps {};
struct PrefixMaps {  // of the prefix's pool
  CUtensorMap k, v;
  int32_t box;  // rows of one copy
};
template <bool F8, int SH>
using MapsOf = std::conditional_t<SH == kThrough, PrefixMaps, std::conditional_t<F8 || SH, MoreMaps<F8>, NoMaps>>;
template <bool F8, int SH>
struct DecodeParams {
  std::conditional_t<F8 || SH, PagedOwnArgs, PagedAttnArgs> a;
  uint32_t* counters;  // [CTAs] pieces that are done of the shared item that begins in a CTA's range
  float* part;         // [2 * CTAs][G][HD] partial sums
  float* part_ml;      // [2 * CTAs][G][2] their reference and weight
  int32_t G;
  int32_t box;         // rows of one TMA copy
  PrefixParts pre;     // kPlanned: own and own_ml are written
};

template <bool BF>
RPGC_DEV void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if (BF)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
RPGC_DEV void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
RPGC_DEV void ldsm4_t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
RPGC_DEV uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// The list of key tiles: sequence by sequence, kv head by kv head.
// Positions [own, len) are what the token of sequence s sees of its pages (own: those
// before are a prefix's, SH).
struct Seen {
  int32_t len, own;
  int32_t pre;  // kThrough: positions of the prefix that it sees
};
// What an item weighs in the list: its key tiles, and the end of an item (the
// warps' sums, a share's join) as kEnd tiles more, at its front.  An item that sees
// nothing weighs nothing.
constexpr int kEnd = kItemEnd;
// Pieces of an item, at most on average: with 8 kv heads of 128, one sequence of 4200
// positions takes 11.6 us in 37 pieces and 10.0 in 18.  Only few long items meet the
// bound, and those of fewer kv heads than 8 lose by it: one sequence of 131072
// positions takes 90 us with 8 kv heads (6.0 TB/s), 81 with 4 (3.3 TB/s) and 89 with one
// (0.76 TB/s, 18 CTAs at work).
constexpr int kPieces = kItemPieces;
template <int T>
RPGC_DEV int64_t tiles_of(const Seen& v) {  // from the tile on that holds its first own position
  return (v.len > v.own ? (v.len + (int64_t)T - 1) / T - v.own / T : 0) + (v.pre + (int64_t)T - 1) / T;
}
template <int T>
RPGC_DEV int64_t weight_of(const Seen& v) {
  return v.len > v.own || v.pre > 0 ? tiles_of<T>(v) + kEnd : 0;
}

// One CTA's range of the list, item by item; every warp walks it by itself.
template <int T, int SH>
struct Walk {
  int64_t total, lo, hi;  // weight of the list; this CTA's range
  int32_t seq, kh;        // the item
  Seen at;                // what it sees
  Seen ahead;             // kPlanned: of the next sequence
  int32_t few;            // kThrough: lane i holds group i's first sequence, lane 16 + i its prefix's length
  int64_t i0, i1;         // its key tiles in the list
  int32_t t0, t1;         // those that are this CTA's, counted from at.own / T
  // where range b of n begins, and the range that holds place t
  RPGC_DEV int64_t begin(int b, int n) const {
    return total < (1 << 23) ? (int64_t)((uint32_t)b * (uint32_t)total / (uint32_t)n) : b * total / n;  // (n < 512)
  }
  RPGC_DEV int holder(int64_t t, int n) const {
    return total < (1 << 23) ? (int)((((uint32_t)t + 1) * (uint32_t)n - 1) / (uint32_t)total) : (int)(((t + 1) * n - 1) / total);
  }
  RPGC_DEV void item(int64_t first) {
    i0 = first + kEnd;
    i1 = first + weight_of<T>(at);
    t0 = (int32_t)(lo > i0 ? lo - i0 : 0);
    t1 = (int32_t)((hi < i1 ? hi : i1) - i0);
  }
  template <typename Args>
  RPGC_DEV void groups(const Args& a, int lane) {
    const int i = lane & 15;
    few = lane < 16 ? (i <= a.pre.n_groups ? group_seq<false>(a.pre, a.b.n_seqs, i) : 0x7fffffff)
                    : (i < a.pre.n_groups ? a.pre.lens[i] : 0);
  }
  // (these two with kThrough: by all lanes of a warp together)
  RPGC_DEV int last_group(int s) const {  // the last group that begins at s or before
    int g = -1;
#pragma unroll
    for (int step = 8; step; step >>= 1) {
      const int32_t first = __shfl_sync(0xffffffffu, few, g + step);
      if (first <= s) g += step;
    }
    return g;
  }
  template <typename Args>
  RPGC_DEV Seen seen(const Args& a, int s) const {
    if constexpr (SH == kThrough) {
      const int32_t n = s < a.b.n_seqs ? a.b.kv_lens[s] : 0;
      const int g = last_group(s);
      const int32_t first = __shfl_sync(0xffffffffu, few, 0), end = __shfl_sync(0xffffffffu, few, min(g + 1, 15)),
                    len = __shfl_sync(0xffffffffu, few, 16 + max(g, 0));
      const PrefixSeq v = sight_of(a, n, first <= s && s < end ? len : 0);
      return {v.len, v.own, v.pre};
    }
    return s < a.b.n_seqs ? Seen{(int32_t)min((int64_t)max(0, a.b.kv_lens[s]), table_reach(a.kv, a.b)), 0, 0} : Seen{0, 0, 0};
  }
  template <typename Args>
  RPGC_DEV bool start(const Args& a, int lane, int ctas, int cta, int* active) {
    const int64_t kv = a.kv.n_kv;
    // each lane adds up a run of sequences; then the run that holds this CTA's
    // first place is looked through 32 sequences at a time
    const int run = (a.b.n_seqs + 31) / 32;
    int64_t sum = 0;
    int32_t some = 0;
    Seen ln = {0, 0, 0};
#pragma unroll 4
    for (int i = 0; i < run; ++i) {
      ln = seen(a, lane * run + i);
      sum += weight_of<T>(ln);
      some += ln.len > 0;
    }
    sum *= kv;
    int64_t upto = scan(sum, lane);
    total = __shfl_sync(0xffffffffu, upto, 31);
    // no more CTAs than there is weight, nor so many that a join is long
    const int64_t items = (int64_t)__reduce_add_sync(0xffffffffu, some) * kv;
    const int parts = (int)min(min(total, (int64_t)ctas), items * kPieces);
    *active = parts;
    if (cta >= parts) return false;
    lo = begin(cta, parts);
    hi = begin(cta + 1, parts);
    const int src = __ffs(__ballot_sync(0xffffffffu, upto > lo)) - 1;
    int64_t before = __shfl_sync(0xffffffffu, upto - sum, src);  // weight of the sequences before s0
#pragma unroll 1
    for (int s0 = src * run;; s0 += 32) {
      if (run > 1 || SH == kThrough) ln = seen(a, s0 + lane);
      else ln.len = __shfl_sync(0xffffffffu, ln.len, (src + lane) & 31);  // (only lane 0's counts: the run is one sequence)
      const int64_t mine = weight_of<T>(ln) * kv;
      upto = scan(mine, lane);
      const uint32_t in = __ballot_sync(0xffffffffu, before + upto > lo);
      if (in) {
        const int i = __ffs(in) - 1;
        const int64_t first = before + __shfl_sync(0xffffffffu, upto - mine, i);
        seq = s0 + i;
        at = {__shfl_sync(0xffffffffu, ln.len, i), 0, 0};
        if constexpr (SH == kThrough) at.own = __shfl_sync(0xffffffffu, ln.own, i), at.pre = __shfl_sync(0xffffffffu, ln.pre, i);
        const int64_t w = weight_of<T>(at), in_seq = lo - first;
        kh = in_seq < (int64_t)0x7fffffff ? (int32_t)((uint32_t)in_seq / (uint32_t)w) : (int32_t)(in_seq / w);
        item(first + kh * w);
        return true;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  // kPlanned: from the plan (through L2: the kernel has not waited for the one before, which
  // waited for the plan)
  RPGC_DEV static Seen planned(const PrefixParts& p, int s, int n_seqs) {
    if (s >= n_seqs) return {0, 0, 0};
    const int2 v = __ldcg(reinterpret_cast<const int2*>(p.seqs + s));
    return {v.x, v.y, 0};
  }
  template <typename Args>
  RPGC_DEV bool start_planned(const Args& a, const PrefixParts& p, int cta, int* tail) {
    const PrefixStart* r = p.starts + cta;
    const longlong2 x = __ldcg(reinterpret_cast<const longlong2*>(r));
    const int4 y = __ldcg(reinterpret_cast<const int4*>(r) + 1), z = __ldcg(reinterpret_cast<const int4*>(r) + 2);
    lo = x.x;
    hi = x.y;
    if (lo >= hi) return false;
    seq = y.z;
    kh = y.w;
    at = {z.x, z.y, 0};
    *tail = z.z;
    ahead = planned(p, seq + 1, a.b.n_seqs);
    item((int64_t)(((uint64_t)(uint32_t)y.y << 32) | (uint32_t)y.x));
    return true;
  }
  RPGC_DEV int64_t scan(int64_t v, int lane) const {  // inclusive sums over the lanes
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += x;
    }
    return v;
  }
  template <typename Args>
  RPGC_DEV bool next(const Args& a, const PrefixParts& p) {
    if (i1 >= hi) return false;
    if (++kh == a.kv.n_kv) {
      kh = 0;
      do {
        ++seq;
        if (SH == kPlanned) at = ahead, ahead = planned(p, seq + 1, a.b.n_seqs);
        else at = seen(a, seq);
      } while (!weight_of<T>(at));  // (a later item exists: i1 < hi <= total)
    }
    item(i1);
    return true;
  }
};

template <int N>
RPGC_DEV void bar_consumers() {
  asm volatile("bar.sync 1, %0;" ::"n"(N) : "memory");
}

template <int HD, bool BF, int NT, bool F8, int SH>
__global__ void __launch_bounds__(DShape<HD, NT, F8, SH == kPlanned>::kThreads, DShape<HD, NT, F8, SH == kPlanned>::kCtas)
    decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                  const __grid_constant__ MapsOf<F8, SH> tm, const __grid_constant__ DecodeParams<F8, SH> p) {
  using S = DShape<HD, NT, F8, SH == kPlanned>;
  constexpr int kStages = S::kStages, kHeads = S::kHeads, kPad = S::kPad, kWarps = S::kWarps, kTile = S::kTile;
  constexpr bool MB = BF && !F8;             // the MMAs' type: bf16, else fp16
  constexpr float kLift = MB ? 0.0f : 6.0f;  // fp16 probabilities carry 2^6: small ones keep their bits
  constexpr float kMost = MB ? 1.0e12f : 32768.0f;  // a probability that needs no new reference
  extern __shared__ __align__(1024) uint8_t ring[];  // (swizzled tiles start on 1024 bytes; the kernel has no other shared memory)
  float* scales = reinterpret_cast<float*>(ring + kStages * S::kStage);  // [stage][K, V][copy][32 at least] (F8)
  float* wo = scales + kStages * 2 * (S::kScaleRoom / 4);            // [warp][head][kPad]
  float* wm = wo + kWarps * kHeads * kPad;                           // [warp][head]
  float* wl = wm + kWarps * kHeads;
  uint64_t* full = reinterpret_cast<uint64_t*>(wl + kWarps * kHeads);
  uint64_t* empty = full + kStages;
  uint32_t* there = reinterpret_cast<uint32_t*>(empty + kStages);  // [kStages] groups of 16 keys that are there
  volatile int32_t* gave_up = reinterpret_cast<volatile int32_t*>(there + kStages);
  int32_t* last = const_cast<int32_t*>(gave_up) + 1;
  uint32_t* again = reinterpret_cast<uint32_t*>(last + 1);  // heads of the item to be computed again
  const auto& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full + i, S::kLoaders);
      mbar_init(empty + i, kWarps);
    }
    *gave_up = 0;
    *again = 0;
    fence_barrier_init();
  }
  if (warp == kWarps && lane < 2) prefetch_map(lane ? &tm_v : &tm_k);
  if constexpr (F8)
    if (warp == kWarps && lane == 2) prefetch_map(&tm.s);
  __syncthreads();
  // launched as a programmatic dependent: nothing that a kernel wrote is read before
  // this.  With a prefix the kernel before is the prefix's, whose results the next one
  // reads, not this, and which let this one begin when all that came earlier had ended: it
  // is waited for at the end, so that this kernel does not end before it.
  if (SH != kPlanned) grid_dep_wait();
  grid_dep_launch();
  auto wait = [&](uint64_t* bar, uint32_t parity) { return wait_for(bar, parity, gave_up, a.b.status); };
  int active;  // CTAs that have a range (kPlanned: pieces of the range's last item)
  Walk<kTile, SH> w;
  if constexpr (SH == kThrough) w.groups(a, lane);
  const bool work = SH == kPlanned ? w.start_planned(a, p.pre, blockIdx.x, &active) : w.start(a, lane, gridDim.x, blockIdx.x, &active);

  if (warp >= kWarps) {  // one warp copies K, the other V (or one both)
    // ---------------------------------------------------------------- loads
    if (!work) {
      if (SH == kPlanned) grid_dep_wait();  // (so that this kernel ends after the prefix's)
      return;
    }
    int st = 0;
    uint32_t ph = 0;
    const int per = kTile / p.box;  // copies per panel
    const int pshift = a.kv.page_shift;
    // kThrough: tiles [t0, t1) of a prefix
    auto load_prefix = [&](const int32_t* tab, int t0, int t1) {
      if constexpr (SH == kThrough) {
        const int box = tm.box, per = kTile / box, shift = a.pre.kv.page_shift, copies = (t1 - t0) * per, v = warp - kWarps;
        auto entry = [&](int c) {
          const int64_t e = ((int64_t)t0 * kTile + (int64_t)c * box) >> shift;
          return c < copies && e < a.pre.max_pages ? tab[e] : -1;
        };
        int32_t ids = entry(lane), ids_next = entry(32 + lane);
        for (int c = 0; c < copies; c += per) {
          if (c && !(c & 31)) {
            ids = ids_next;
            ids_next = entry(c + 32 + lane);
          }
          int32_t page = __shfl_sync(0xffffffffu, ids, (c + lane) & 31);
          const bool ok = (uint32_t)page < (uint32_t)a.pre.kv.n_pages;
          if (!ok) page = a.pre.kv.n_pages;
          const uint32_t have = __ballot_sync(0xffffffffu, lane < per && ok);
          const int at = (int)(((int64_t)t0 * kTile + (int64_t)(c + lane) * box) & ((1 << shift) - 1));
          wait(empty + st, ph ^ 1u);
          if (*gave_up) return;
          if (lane == 0) {
            const int g = box >> 4;
            uint32_t groups = 0;
            for (int i = 0; i < per; ++i)
              if (have >> i & 1u) groups |= ((1u << g) - 1u) << (i * g);
            if (v == 0) there[st] = groups;
            mbar_arrive_expect_tx(full + st, S::kHalf);
          }
          __syncwarp();
          if (lane < per)
#pragma unroll
            for (int h = 0; h < S::kPanels; ++h)
              tma_4d(ring + st * S::kStage + v * S::kHalf + h * S::kPanel + lane * box * 128, v ? &tm.v : &tm.k, 64 * h, w.kh, at, page, full + st);
          if (++st == kStages) st = 0, ph ^= 1u;
        }
      }
    };
    do {
      const int pt = SH == kThrough ? (int)(((uint32_t)w.at.pre + kTile - 1) / kTile) : 0;  // tiles of the prefix
      const int32_t* tab = a.b.table + (int64_t)w.seq * a.b.table_stride;
      const int t0 = max(w.t0 - pt, 0), t1 = w.t1 - pt;
      if constexpr (SH == kThrough)
        if (w.t0 < pt) {
          // (the sequence has a group whatever cu holds, for it sees a prefix)
          load_prefix(a.pre.table + (int64_t)w.last_group(w.seq) * a.pre.table_stride, w.t0, min(w.t1, pt));
          if (*gave_up) break;
        }
      if (t1 <= t0) continue;  // (the range ends in the item's front, or in the prefix)
      // page ids ahead of their use: lane l holds the one of copy l of the next 32
      const int copies = (t1 - t0) * per;
      const int64_t base = (int64_t)(t0 + (SH ? w.at.own / kTile : 0)) * kTile;
      auto entry = [&](int c) {
        const int64_t e = (base + (int64_t)c * p.box) >> pshift;
        return c < copies && e < a.b.max_pages ? (SH == kPlanned ? __ldcg(tab + e) : tab[e]) : -1;
      };
      int32_t ids = entry(lane), ids_next = entry(32 + lane);
      for (int t = t0, c = 0; t < t1; ++t, c += per) {
        if (c && !(c & 31)) {
          ids = ids_next;
          ids_next = entry(c + 32 + lane);
        }
        int32_t page = __shfl_sync(0xffffffffu, ids, (c + lane) & 31);  // (per divides 32: never past the 32)
        const bool ok = (uint32_t)page < (uint32_t)a.kv.n_pages;
        if (!ok) page = a.kv.n_pages;  // past the pool: TMA fills zeros
        const uint32_t have = __ballot_sync(0xffffffffu, lane < per && ok);
        const int at = (int)((base + (int64_t)(c + lane) * p.box) & ((1 << pshift) - 1));
        constexpr int kBoth = 3 - S::kLoaders;  // of K and V, this warp's: from v0 on
        const int v0 = warp - kWarps;
        uint8_t* dst = ring + st * S::kStage;
        if constexpr (F8 || SH == kPlanned) {
          // groups of 16 keys that the token sees; a tile that it does not see whole comes
          // in copies of 16 rows, those alone
          const int64_t tb = base + (int64_t)(t - t0) * kTile;
          const int g0 = SH ? (int)max((int64_t)0, w.at.own - tb) >> 4 : 0, g1 = (int)min((int64_t)kTile, w.at.len - tb + 15) >> 4;
          if (g0 > 0 || g1 < kTile / 16) {
            int32_t fine = __shfl_sync(0xffffffffu, ids, (c + lane * 16 / p.box) & 31);
            const bool in = lane >= g0 && lane < g1, there_is = (uint32_t)fine < (uint32_t)a.kv.n_pages;
            if (!there_is) fine = a.kv.n_pages;
            const uint32_t groups = __ballot_sync(0xffffffffu, in && there_is);
            wait(empty + st, ph ^ 1u);
            if (*gave_up) break;
            if (lane == 0) {
              if (warp == kWarps) there[st] = groups;
              mbar_arrive_expect_tx(full + st, kBoth * ((g1 - g0) * (S::kHalf * 16 / kTile) + S::kScales));
            }
            __syncwarp();
#pragma unroll
            for (int v = v0; v < v0 + kBoth; ++v) {
              if (in) {
                const int at16 = (int)((tb + 16 * lane) & ((1 << pshift) - 1));
#pragma unroll
                for (int h = 0; h < S::kPanels; ++h)
                  tma_4d(dst + v * S::kHalf + h * S::kPanel + lane * 16 * (F8 ? HD : 128), v ? &tm.v : &tm.k, 64 * h, w.kh, at16, fine, full + st);
              }
              if constexpr (F8)
                if (lane < per) tma_4d(scales + (2 * st + v) * (S::kScaleRoom / 4) + lane * max(p.box, 32), &tm.s, at, v, w.kh, page, full + st);
            }
            if (++st == kStages) st = 0, ph ^= 1u;
            continue;
          }
        }
        wait(empty + st, ph ^ 1u);
        if (*gave_up) break;
        if (lane == 0) {
          uint32_t groups = 0;  // a copy of 16, 32, .. rows covers 1, 2, .. groups of 16
          const int g = p.box >> 4;
          for (int i = 0; i < per; ++i)
            if (have >> i & 1u) groups |= ((1u << g) - 1u) << (i * g);
          if (warp == kWarps) there[st] = groups;
          mbar_arrive_expect_tx(full + st, kBoth * (S::kHalf + S::kScales));
        }
        __syncwarp();
        if (lane < per)
#pragma unroll
          for (int v = v0; v < v0 + kBoth; ++v) {
#pragma unroll
            for (int h = 0; h < S::kPanels; ++h)
              tma_4d(dst + v * S::kHalf + h * S::kPanel + lane * p.box * (F8 ? HD : 128), v ? &tm_v : &tm_k, 64 * h, w.kh, at, page, full + st);
            if constexpr (F8) tma_4d(scales + (2 * st + v) * (S::kScaleRoom / 4) + lane * max(p.box, 32), &tm.s, at, v, w.kh, page, full + st);
          }
        if (++st == kStages) st = 0, ph ^= 1u;
      }
      if (*gave_up) break;
    } while (w.next(a, p.pre));
    if (*gave_up)  // copies in flight end before the CTA does
      for (int i = 0; i < kStages; ++i)
        for (int k = 0; k < 1 << 12; ++k)
          if (mbar_try_wait(full + i, ph ^ (i < st ? 0u : 1u))) break;
    if (SH == kPlanned) grid_dep_wait();
    return;
  }

  // ----------------------------------------------------------- attention
  // sequences that see nothing: zeros, their rows dealt over the CTAs
  for (int s = blockIdx.x; SH != kPlanned && s < a.b.n_seqs; s += gridDim.x)
    if (w.seen(a, s).len == 0)
      for (int i = tid; i < a.n_heads * HD / 8; i += kWarps * 32)
        reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + (int64_t)s * a.n_heads * HD)[i] = make_uint4(0, 0, 0, 0);
  if (!work) {
    if (SH == kPlanned) grid_dep_wait();
    return;
  }
  const int gr = lane >> 2, tq = lane & 3, G = p.G;
  const float c = a.scale * kLog2e;
  // ldmatrix rows of this lane in the warp's 16 keys: K as stored, V transposed
  const int mi = lane >> 3, mr = lane & 7;
  const int krow = 16 * warp + mr + 8 * (mi & 1), kc = mi >> 1;
  const int vrow = 16 * warp + mr + 8 * (mi >> 1), vc = mi & 1;
  // F8: 16-byte chunk c of this lane's row in group u of the warp's 16 keys, in tiles of 128- or 64-byte rows
  auto chunk8 = [&](uint32_t base, int u, int c) {
    const int row = 16 * ((S::kSub - 1) * warp + u) + krow;
    return base + row * HD + ((c ^ (HD == 128 ? row & 7 : row >> 1 & 3)) << 4);
  };
  int st = 0;
  uint32_t ph = 0;
  auto put = [&](int h, int d, float M, const float4& acc, float L) {  // four values of the item's row of head h
    if constexpr (SH == kPlanned) {  // its sums, for the kernel that joins all of them (weights are 2^(score - reference))
      const int64_t row = (int64_t)w.seq * a.n_heads + w.kh * G + h;
      __stcg(reinterpret_cast<float4*>(p.pre.own + row * HD + d), acc);
      if (d == 0) __stcg(reinterpret_cast<float2*>(p.pre.own_ml) + row, make_float2(L == L ? M - kLift : 0.0f, L));  // (NaN stays: a score was)
      return;
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    uint16_t* op = static_cast<uint16_t*>(a.out) + ((int64_t)w.seq * a.n_heads + w.kh * G + h) * HD + d;
    *reinterpret_cast<uint2*>(op) = make_uint2(pack2<BF>(acc.x * inv, acc.y * inv), pack2<BF>(acc.z * inv, acc.w * inv));
    const float z = fmaf(acc.x, 0.0f, fmaf(acc.y, 0.0f, fmaf(acc.z, 0.0f, acc.w * 0.0f)));  // NaN: not all finite
    if (__builtin_expect(z != 0.0f && L < INFINITY, 0)) atomicOr(again, 1u << h);
  };
  do {
    const int t0 = w.t0, t1 = w.t1;
    if (t1 <= t0) continue;
    // Q^T as the B operand: head 8 n + gr, dims 16 k + 2 tq (+8)
    uint32_t q[NT][HD / 16][2];
    float cs[NT][2];  // F8: factors from scores to exponents, of heads 8 n + 2 tq (+1)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int h = 8 * n + gr;
      const uint16_t* qp = static_cast<const uint16_t*>(a.q) + (int64_t)w.seq * a.q_tok + (int64_t)(w.kh * G + h) * a.q_head;
      if constexpr (F8) {
        // codes 4 tq .. 4 tq + 3 of a 16-byte chunk are one word of a lane, so Q's dims are
        // taken in that order too.  fp16 as the codes are: a power of two brings the row's
        // largest value to 2^14, and what has fewer than 2^-29 of that loses its bits.
        uint2 raw[HD / 16];
        float top = 0.0f;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          raw[k] = h < G ? __ldcg(reinterpret_cast<const uint2*>(qp + 16 * k + 4 * tq)) : make_uint2(0u, 0u);
          const float2 x = unpack2<BF>(raw[k].x), y = unpack2<BF>(raw[k].y);
          top = fmaxf(fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(y.x), fabsf(y.y)));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int up = top < INFINITY ? min(max(141 - (int)(__float_as_uint(top) >> 23), -100), 100) : 0;
        const float f = __uint_as_float((uint32_t)(127 + up) << 23), back = c * __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const float2 x = unpack2<BF>(raw[k].x), y = unpack2<BF>(raw[k].y);
          q[n][k][0] = pack2<false>(x.x * f, x.y * f);
          q[n][k][1] = pack2<false>(y.x * f, y.y * f);
        }
        cs[n][0] = __shfl_sync(0xffffffffu, back, 8 * tq);
        cs[n][1] = __shfl_sync(0xffffffffu, back, 8 * tq + 4);
        continue;
      }
      qp += 2 * tq;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        const uint32_t *q0 = reinterpret_cast<const uint32_t*>(qp + 16 * k), *q1 = q0 + 4;
        q[n][k][0] = h < G ? (SH == kPlanned ? __ldcg(q0) : *q0) : 0u;
        q[n][k][1] = h < G ? (SH == kPlanned ? __ldcg(q1) : *q1) : 0u;
      }
    }
    float o[NT][HD / 16][4], m[NT][2], l[NT][2];
    float vtop = 0.0f;  // F8: a power of two that no scale of V so far is above; o is in its units
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.0f;
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) o[n][d][0] = o[n][d][1] = o[n][d][2] = o[n][d][3] = 0.0f;
    }
    for (int t = t0; t < t1; ++t) {
      wait(full + st, ph);
      // tile t is kTile positions of the prefix, or of the sequence's own pages from own / kTile on
      const int pt = SH == kThrough ? (int)(((uint32_t)w.at.pre + kTile - 1) / kTile) : 0;
      const bool shared = SH == kThrough && t < pt;
      const int first = (shared ? t : t - pt + (SH ? w.at.own / kTile : 0)) * kTile + 16 * S::kSub * warp;
      const int left = (shared ? w.at.pre : w.at.len) - first;  // keys of this warp's part
      const int skip = SH && !shared ? w.at.own - first : 0;    // those before that the prefix has
      if constexpr (F8) {
        if (left > 0 && skip < 16 * S::kSub) {
          constexpr int kSub = S::kSub, kChains = 2 / kSub;  // two chains of MMAs, so that one's latency hides the other's
          const uint32_t kb = smem_u32(ring + st * S::kStage), vb = kb + S::kHalf, is = there[st] >> kSub * warp;
          float s[kSub][kChains][NT][4];
#pragma unroll
          for (int u = 0; u < kSub; ++u)
#pragma unroll
            for (int n = 0; n < NT * kChains * 4; ++n) (&s[u][0][0][0])[n] = 0.0f;
#pragma unroll
          for (int k = 0; k < HD / 16; k += 2)
#pragma unroll
            for (int u = 0; u < kSub; ++u) {
              uint32_t f[4];
              ldsm4(chunk8(kb, u, k + kc), f);
              const uint32_t x[4] = {half2_lo(f[0]), half2_lo(f[1]), half2_hi(f[0]), half2_hi(f[1])};
              const uint32_t y[4] = {half2_lo(f[2]), half2_lo(f[3]), half2_hi(f[2]), half2_hi(f[3])};
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                mma<MB>(s[u][0][n], x, q[n][k][0], q[n][k][1]);
                mma<MB>(s[u][kChains - 1][n], y, q[n][k + 1][0], q[n][k + 1][1]);
              }
            }
          // the first values (a load brings those of 32 dims) are on their way while the
          // probabilities are made
          constexpr int kLoads = HD / 32, kFirst = kAhead / kSub < kLoads ? kAhead / kSub : kLoads;
          uint32_t v[kSub][kFirst][4];
#pragma unroll
          for (int d = 0; d < kFirst; ++d)
#pragma unroll
            for (int u = 0; u < kSub; ++u) ldsm4_t(chunk8(vb, u, 2 * d + kc), v[u][d]);
          // s: (key gr, head 2 tq), (gr, 2 tq + 1), (gr + 8, 2 tq), (gr + 8, 2 tq + 1)
          bool in[kSub][2];
          float vs[kSub][2];  // V's scales of keys gr, gr + 8 in units of vtop
          const float* ks = scales + 2 * st * (S::kScaleRoom / 4) + (p.box == 16 ? 32 : 16) * kSub * warp + gr;
          bool above = false, fresh = false;
#pragma unroll
          for (int u = 0; u < kSub; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int key = 16 * u + 8 * e + gr;
              in[u][e] = key < left && (!SH || key >= skip) && (is >> u & 1u);
              const float* at = ks + (p.box == 16 ? 32 : 16) * u + 8 * e;
              const float k = at[0] ;
              vs[u][e] = in[u][e] ? at[S::kScaleRoom / 4] : 0.0f;
              above |= vs[u][e] > vtop;
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                  float& y = s[u][0][n][2 * e + j];
                  if (kChains > 1) y += s[u][kChains - 1][n][2 * e + j];
                  y = in[u][e] ? y * k * cs[n][j] : -INFINITY;
                }
            }
          if (__any_sync(0xffffffffu, above)) {
            float t = 0.0f;
#pragma unroll
            for (int u = 0; u < kSub; ++u) t = fmaxf(t, fmaxf(vs[u][0], vs[u][1]));
            t = warp_max(t);
            const float up = __uint_as_float((uint32_t)min(max((int)(__float_as_uint(t) >> 23) + 1, 2), 252) << 23);
            const float f = vtop / up;
            vtop = up;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int d = 0; d < HD / 16; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][d][e] *= f;
          }
          const float down = vtop > 0.0f ? __uint_as_float(0x7f000000u - __float_as_uint(vtop)) : 0.0f;  // 1 / vtop, a power of two
#pragma unroll
          for (int u = 0; u < kSub; ++u) vs[u][0] *= down, vs[u][1] *= down;
#pragma unroll
          for (int n = 0; n < NT; ++n) fresh |= m[n][0] == -INFINITY || m[n][1] == -INFINITY;
          // probabilities by the reference there is; where there is none yet, or one
          // has outgrown it (or is NaN), the maximum becomes it and they are made again;
          // the heads that are not due keep theirs, and with them every bit
          float x[kSub][NT][4];
          bool look = __any_sync(0xffffffffu, fresh);
          uint32_t due = 0;  // heads (columns 8 n + 2 tq + e, bit 2 n + e) that need a reference
#pragma unroll 1
          for (;;) {
            if (look) {
#pragma unroll
              for (int n = 0; n < NT; ++n) due |= (m[n][0] == -INFINITY ? 1u : 0u) << 2 * n | (m[n][1] == -INFINITY ? 2u : 0u) << 2 * n;
              due |= __shfl_xor_sync(0xffffffffu, due, 4);
              due |= __shfl_xor_sync(0xffffffffu, due, 8);
              due |= __shfl_xor_sync(0xffffffffu, due, 16);
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  float t = m[n][e];
#pragma unroll
                  for (int u = 0; u < kSub; ++u) t = fmaxf(t, fmaxf(s[u][0][n][e], s[u][0][n][e + 2]));
                  t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
                  t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
                  t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
                  if (!(due >> (2 * n + e) & 1u)) t = m[n][e];
                  const float f = m[n][e] == -INFINITY ? 0.0f : t == m[n][e] ? 1.0f : exp2_fast(m[n][e] - t);
                  m[n][e] = t;
                  l[n][e] *= f;
#pragma unroll
                  for (int d = 0; d < HD / 16; ++d) {
                    o[n][d][e] *= f;
                    o[n][d][e + 2] *= f;
                  }
                }
            }
            bool grown = false;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float base = (m[n][e & 1] == -INFINITY ? 0.0f : m[n][e & 1]) - kLift;
#pragma unroll
                for (int u = 0; u < kSub; ++u) {
                  x[u][n][e] = exp2_fast(s[u][0][n][e] - base);
                  const bool g = !(x[u][n][e] <= kMost);
                  grown |= g;
                  due |= g ? 1u << (2 * n + (e & 1)) : 0u;
                }
              }
            if (look || !__any_sync(0xffffffffu, grown)) break;
            look = true;
          }
          // each weight, V's scale in it, as two fp16 values, itself rounded and what that
          // left: the memory sets the pace here, so the second product costs nothing
          uint32_t b[kSub][NT][2], b_lo[kSub][NT][2], keep[kSub][2];
#pragma unroll
          for (int u = 0; u < kSub; ++u) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              l[n][0] += x[u][n][0] + x[u][n][2];
              l[n][1] += x[u][n][1] + x[u][n][3];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float w0 = x[u][n][2 * e] * vs[u][e], w1 = x[u][n][2 * e + 1] * vs[u][e];
                const uint32_t hi = pack2<MB>(w0, w1);
                const float2 h = unpack2<MB>(hi);
                b[u][n][e] = transpose8(hi);
                b_lo[u][n][e] = transpose8(pack2<MB>(w0 - h.x, w1 - h.y));
              }
            }
            // keys 2 tq, 2 tq + 1 (and + 8) of the V operand; what the token does not see is
            // cleared, for 0 * NaN is NaN
            keep[u][0] = keep[u][1] = is >> u & 1u ? 0xffffffffu : 0u;
            if (left < 16 * kSub || skip > 0 || !(is >> u & 1u))
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int key = 16 * u + 8 * e + 2 * tq;
                if (!(key < left && key >= skip)) keep[u][e] &= 0xffff0000u;
                if (!(key + 1 < left && key + 1 >= skip)) keep[u][e] &= 0xffffu;
              }
          }
#pragma unroll
          for (int d = 0; d < kLoads; ++d)
#pragma unroll
            for (int u = 0; u < kSub; ++u) {
              uint32_t f[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) f[e] = v[u][d % kFirst][e];
              if (d + kFirst < kLoads) ldsm4_t(chunk8(vb, u, 2 * (d + kFirst) + kc), v[u][d % kFirst]);
              // a word holds dims 2 gr, 2 gr + 1 of keys 2 tq and 2 tq + 1: with the middle bytes
              // changed over its halves are the two keys' codes of one dim.  So row gr of the
              // operand is dim 2 gr, row gr + 8 dim 2 gr + 1.
#pragma unroll
              for (int e = 0; e < 4; ++e) f[e] = __byte_perm(f[e] & keep[u][e & 1], 0u, 0x3120);
              const uint32_t y[4] = {half2_lo(f[0]), half2_hi(f[0]), half2_lo(f[1]), half2_hi(f[1])};
              const uint32_t z[4] = {half2_lo(f[2]), half2_hi(f[2]), half2_lo(f[3]), half2_hi(f[3])};
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                mma<MB>(o[n][2 * d], y, b[u][n][0], b[u][n][1]);
                mma<MB>(o[n][2 * d + 1], z, b[u][n][0], b[u][n][1]);
                mma<MB>(o[n][2 * d], y, b_lo[u][n][0], b_lo[u][n][1]);
                mma<MB>(o[n][2 * d + 1], z, b_lo[u][n][0], b_lo[u][n][1]);
              }
            }
        }
      } else {
        if (left > 0 && skip < 16 && (there[st] >> warp & 1u)) {
          const uint32_t kb = smem_u32(ring + st * S::kStage), vb = kb + S::kHalf;
          // two chains of MMAs, so that one's latency hides the other's
          float s[NT][4], s2[NT][4];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = s2[n][e] = 0.0f;
#pragma unroll
          for (int k = 0; k < HD / 16; ++k) {
            uint32_t f[4];
            ldsm4(kb + (k >> 2) * S::kPanel + krow * 128 + (((2 * (k & 3) + kc) ^ (krow & 7)) << 4), f);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma<MB>(k & 1 ? s2[n] : s[n], f, q[n][k][0], q[n][k][1]);
          }
          // the first values are on their way while the probabilities are made
          uint32_t v[kAhead][4];
          auto load_v = [&](int d, uint32_t* f) {
            ldsm4_t(vb + (d >> 2) * S::kPanel + vrow * 128 + (((2 * (d & 3) + vc) ^ (vrow & 7)) << 4), f);
          };
#pragma unroll
          for (int d = 0; d < kAhead; ++d) load_v(d, v[d]);
          // s: (key gr, head 2 tq), (gr, 2 tq + 1), (gr + 8, 2 tq), (gr + 8, 2 tq + 1)
          const bool in0 = gr < left && gr >= skip, in1 = gr + 8 < left && gr + 8 >= skip;
          bool fresh = false;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = (e < 2 ? in0 : in1) ? (s[n][e] + s2[n][e]) * c : -INFINITY;
            fresh |= m[n][0] == -INFINITY || m[n][1] == -INFINITY;
          }
          // probabilities by the reference there is; where there is none yet, or one
          // has outgrown it (or is NaN), the maximum becomes it and they are made again
          float x[NT][4];
          bool look = __any_sync(0xffffffffu, fresh);
          uint32_t due = 0;  // F8, SH: heads (columns 8 n + 2 tq + e, bit 2 n + e) that need a reference
#pragma unroll 1
          for (;;) {
            if (look) {
              if (SH) {  // the others keep theirs, and with them every bit
#pragma unroll
                for (int n = 0; n < NT; ++n) due |= (m[n][0] == -INFINITY ? 1u : 0u) << 2 * n | (m[n][1] == -INFINITY ? 2u : 0u) << 2 * n;
                due |= __shfl_xor_sync(0xffffffffu, due, 4);
                due |= __shfl_xor_sync(0xffffffffu, due, 8);
                due |= __shfl_xor_sync(0xffffffffu, due, 16);
              }
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  float t = fmaxf(s[n][e], s[n][e + 2]);
                  t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
                  t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
                  t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
                  t = fmaxf(t, m[n][e]);
                  if ((SH) && !(due >> (2 * n + e) & 1u)) t = m[n][e];
                  const float f = m[n][e] == -INFINITY ? 0.0f : (SH) && t == m[n][e] ? 1.0f : exp2_fast(m[n][e] - t);
                  m[n][e] = t;
                  l[n][e] *= f;
#pragma unroll
                  for (int d = 0; d < HD / 16; ++d) {
                    o[n][d][e] *= f;
                    o[n][d][e + 2] *= f;
                  }
                }
            }
            bool grown = false;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                x[n][e] = exp2_fast(s[n][e] - ((m[n][e & 1] == -INFINITY ? 0.0f : m[n][e & 1]) - kLift));
                grown |= !(x[n][e] <= kMost);
                if (SH) due |= !(x[n][e] <= kMost) ? 1u << (2 * n + (e & 1)) : 0u;
              }
            if (look || !__any_sync(0xffffffffu, grown)) break;
            look = true;
          }
          // each probability as two 16-bit values, itself rounded and what that left:
          // the products with V keep 16 bits of it or more.  The memory sets the
          // pace here, so the second product costs nothing; rounded to one value
          // it would be as large an error as the output's own rounding.
          uint32_t b[NT][2], b_lo[NT][2];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            l[n][0] += x[n][0] + x[n][2];
            l[n][1] += x[n][1] + x[n][3];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t hi = pack2<MB>(x[n][2 * e], x[n][2 * e + 1]);
              const float2 h = unpack2<MB>(hi);
              b[n][e] = transpose8(hi);
              b_lo[n][e] = transpose8(pack2<MB>(x[n][2 * e] - h.x, x[n][2 * e + 1] - h.y));
            }
          }
          // keys 2 tq, 2 tq + 1 (and + 8) of the V operand; what lies past the
          // last position is cleared, for 0 * NaN is NaN
          uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
          if (left < 16) {
            keep0 = 2 * tq + 1 < left ? 0xffffffffu : 2 * tq < left ? 0xffffu : 0u;
            keep1 = 2 * tq + 9 < left ? 0xffffffffu : 2 * tq + 8 < left ? 0xffffu : 0u;
          }
          if (SH && skip > 0) {  // (and what the prefix has)
            keep0 &= 2 * tq >= skip ? 0xffffffffu : 2 * tq + 1 >= skip ? 0xffff0000u : 0u;
            keep1 &= 2 * tq + 8 >= skip ? 0xffffffffu : 2 * tq + 9 >= skip ? 0xffff0000u : 0u;
          }
#pragma unroll
          for (int d = 0; d < HD / 16; ++d) {
            uint32_t f[4] = {v[d % kAhead][0], v[d % kAhead][1], v[d % kAhead][2], v[d % kAhead][3]};
            if (d + kAhead < HD / 16) load_v(d + kAhead, v[d % kAhead]);
            f[0] &= keep0;
            f[1] &= keep0;
            f[2] &= keep1;
            f[3] &= keep1;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma<MB>(o[n][d], f, b[n][0], b[n][1]);
              mma<MB>(o[n][d], f, b_lo[n][0], b_lo[n][1]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + st);
      if (++st == kStages) st = 0, ph ^= 1u;
    }
    // ---- the warps' sums meet
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = l[n][e];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        const int h = 8 * n + 2 * tq + e;
        if (gr == 0) {
          wm[warp * kHeads + h] = m[n][e];
          wl[warp * kHeads + h] = x;
        }
        float* row = wo + (warp * kHeads + h) * kPad + (F8 ? 2 * gr : gr);
        if (h < G)
#pragma unroll
          for (int d = 0; d < HD / 16; ++d) {
            row[16 * d] = F8 ? o[n][d][e] * vtop : o[n][d][e];
            row[16 * d + (F8 ? 1 : 8)] = F8 ? o[n][d][e + 2] * vtop : o[n][d][e + 2];
          }
      }
    bar_consumers<kWarps * 32>();
    const bool whole = w.i0 >= w.lo && w.i1 <= w.hi;
    const int slot = 2 * blockIdx.x + (w.lo < w.i0 ? 1 : 0);
    for (int i = tid; i < G * HD / 4; i += kWarps * 32) {
      const int h = i / (HD / 4), d = 4 * (i % (HD / 4));
      float M = -INFINITY;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) M = fmaxf(M, wm[k * kHeads + h]);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float L = 0.0f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        const float mk = wm[k * kHeads + h];
        const float f = mk == -INFINITY ? 0.0f : exp2_fast(mk - M);
        const float4 v = *reinterpret_cast<const float4*>(wo + (k * kHeads + h) * kPad + d);
        acc.x += f * v.x;
        acc.y += f * v.y;
        acc.z += f * v.z;
        acc.w += f * v.w;
        L += f * wl[k * kHeads + h];
      }
      if (whole) {
        put(h, d, M, acc, L);
      } else {
        __stcg(reinterpret_cast<float4*>(p.part + ((int64_t)slot * G + h) * HD + d), acc);
        if (d == 0)
          __stcg(reinterpret_cast<float2*>(p.part_ml) + (int64_t)slot * G + h,
                 SH == kPlanned ? make_float2(L == L ? M - kLift : 0.0f, L) : make_float2(M, L));
      }
    }
    if constexpr (SH == kPlanned) {  // where the item's pieces are: piece 0's slot, piece k in the first slot of the k-th CTA from its own
      if (tid == 0 && w.i0 >= w.lo)
        p.pre.pieces[(int64_t)w.seq * a.kv.n_kv + w.kh] = whole ? 0 : slot | active << 16;
    }
    if (SH != kPlanned && !whole) {
      // ---- the last CTA to finish a shared item joins its pieces
      const int b0 = w.holder(w.i0, active), b1 = w.holder(w.i1 - 1, active);
      bar_consumers<kWarps * 32>();
      if (tid == 0) {
        // (of all the warps' partial results: they are before this by the barrier)
        // (only the last item of a range goes on past it: one counter per CTA, back at 0 after the join)
        if constexpr (F8) {  // (one operation with both orders: one of 4200 positions 10.9 -> 10.6 us)
          uint32_t before;
          asm volatile("atom.acq_rel.gpu.global.inc.u32 %0, [%1], %2;" : "=r"(before) : "l"(p.counters + b0), "r"((uint32_t)(b1 - b0)) : "memory");
          *last = before == (uint32_t)(b1 - b0);
        } else {
          __threadfence();
          *last = atomicInc(p.counters + b0, (uint32_t)(b1 - b0)) == (uint32_t)(b1 - b0);
          __threadfence();
        }
      }
      bar_consumers<kWarps * 32>();
      if (*last) {
        // every piece's (reference, weight) of every head at once, the first rows of
        // partial sums in flight beside them.  Piece k is in its CTA's first slot,
        // but the first piece's CTA may have had an item before.
        const int pieces = b1 - b0 + 1;
        const int front = w.begin(b0, active) < w.i0 ? 1 : 0;
        auto slot_of = [&](int k) { return (int64_t)(2 * (b0 + k) + (k ? 0 : front)); };
        float2* ml = reinterpret_cast<float2*>(wo);  // [piece][head]
        float4 v[kJoin];
        auto fetch = [&](int i, int k0) {
          const float* part = p.part + (i / (HD / 4)) * HD + 4 * (i % (HD / 4));
#pragma unroll
          for (int k = 0; k < kJoin; ++k)
            if (k0 + k < pieces) v[k] = __ldcg(reinterpret_cast<const float4*>(part + slot_of(k0 + k) * G * HD));
        };
        if (tid < G * HD / 4) fetch(tid, 0);
        for (int i = tid; i < pieces * G; i += kWarps * 32)
          ml[i] = __ldcg(reinterpret_cast<const float2*>(p.part_ml) + slot_of(i / G) * G + i % G);
        bar_consumers<kWarps * 32>();
        for (int i = tid; i < G * HD / 4; i += kWarps * 32) {
          const int h = i / (HD / 4), d = 4 * (i % (HD / 4));
          float M = -INFINITY;
          for (int k = 0; k < pieces; ++k) M = fmaxf(M, ml[k * G + h].x);
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
          float L = 0.0f;
          for (int k0 = 0; k0 < pieces; k0 += kJoin) {
            if (k0 || i != tid) fetch(i, k0);
#pragma unroll
            for (int k = 0; k < kJoin; ++k) {
              if (k0 + k >= pieces) break;
              const float2 x = ml[(k0 + k) * G + h];
              const float f = x.x == -INFINITY ? 0.0f : exp2_fast(x.x - M);
              acc.x += f * v[k].x;
              acc.y += f * v[k].y;
              acc.z += f * v[k].z;
              acc.w += f * v[k].w;
              L += f * x.y;
            }
          }
          put(h, d, M, acc, L);
        }
      }
    }
    bar_consumers<kWarps * 32>();  // the merge buffer is free again
    // (attn_row inlined: a kernel that calls takes 0.2 us longer to begin)
    const uint32_t todo = SH == kPlanned ? 0u : *again;
    if (__builtin_expect(todo != 0, 0)) {
      for (int h = warp; h < G; h += kWarps)
        if (todo >> h & 1u) {
          if constexpr (F8 || SH) own_row<HD, BF, F8, SH != 0>(a, w.seq, w.kh * G + h, lane);
          else attn_row<HD, BF>(a, w.seq, w.seq, w.kh * G + h, -1, lane);
        }
      bar_consumers<kWarps * 32>();
      if (tid == 0) *again = 0;
    }
  } while (w.next(a, p.pre));
  if (SH == kPlanned) grid_dep_wait();
}

int device_sms() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) cudaGetLastError();
  return sm_count(dev);
}

// The workspace: counters, one per CTA (two CTAs an SM at most), then the partial
// results.  The counters alone have to be zero when a call begins, so they lie
// where no call of any shape puts anything else.
int64_t counter_bytes() { return ((int64_t)2 * device_sms() * 4 + 255) / 256 * 256; }

// As many CTAs as run at once, and no more than the join's table has room for.
template <int HD, int NT, bool F8>
int decode_ctas(int G) {
  using S = DShape<HD, NT, F8>;
  const int n = device_sms() * S::kCtas, most = S::kMerge / (8 * G);
  return n < most ? n : most;
}

// What the plan has to know of the kernel behind a prefix.
template <int HD, int NT, bool F8>
void own_shape(PrefixShape* s) {
  using S = DShape<HD, NT, F8, true>;
  for (s->tile_log = 0; 1 << s->tile_log < S::kTile;) ++s->tile_log;
  s->stage = S::kStage;
  s->on_sm = S::kCtas;
  s->own_ctas = device_sms() * S::kCtas;
}
template <bool F8>
void own_shape_of(const PagedOwnArgs& a, PrefixShape* s) {
  const bool one = a.n_heads / a.kv.n_kv <= 8;
  if (a.kv.hd == 128) one ? own_shape<128, 1, F8>(s) : own_shape<128, 2, F8>(s);
  else one ? own_shape<64, 1, F8>(s) : own_shape<64, 2, F8>(s);
}

// K or V as codes, and the scales: {position, K or V, kv head, page}.
inline bool make_map8(CUtensorMap* m, const PagedOwnArgs& a, bool v, int box) {
  auto enc = encoder();
  if (!enc) return false;
  const cuuint64_t d[4] = {(cuuint64_t)a.kv.hd, (cuuint64_t)a.kv.n_kv, (cuuint64_t)1 << a.kv.page_shift, (cuuint64_t)a.kv.n_pages};
  const cuuint64_t st[3] = {(cuuint64_t)(v ? a.kv.v_head : a.kv.k_head), (cuuint64_t)(v ? a.kv.v_pos : a.kv.k_pos),
                            (cuuint64_t)(v ? a.kv.v_page : a.kv.k_page)};
  const cuuint32_t b[4] = {(cuuint32_t)a.kv.hd, 1, (cuuint32_t)box, 1}, es[4] = {1, 1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(v ? a.kv.v : a.kv.k), d, st, b, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
             a.kv.hd == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, a.kv.hd == 128 ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_L2_64B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
inline bool make_map_scales(CUtensorMap* m, const PagedOwnArgs& a, int box) {
  auto enc = encoder();
  if (!enc) return false;
  const cuuint64_t size = (cuuint64_t)1 << a.kv.page_shift;
  const cuuint64_t d[4] = {size, 2, (cuuint64_t)a.kv.n_kv, (cuuint64_t)a.kv.n_pages};
  const cuuint64_t st[3] = {size * 4, (cuuint64_t)a.sc_head * 4, (cuuint64_t)a.sc_page * 4};
  const cuuint32_t b[4] = {(cuuint32_t)box, 1, 1, 1}, es[4] = {1, 1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, const_cast<float*>(a.scales), d, st, b, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD, bool BF, int NT, bool F8, int SH, typename Args>
cudaError_t decode_go(const Args& a, const PrefixParts& pre, int own_ctas, cudaStream_t s) {
  using S = DShape<HD, NT, F8, SH == kPlanned>;
  const int ctas = SH == kPlanned ? own_ctas : decode_ctas<HD, NT, F8>(a.n_heads / a.kv.n_kv);
  DecodeParams<F8, SH> p{};
  p.a = a;
  p.G = a.n_heads / a.kv.n_kv;
  p.box = (1 << a.kv.page_shift) < S::kTile ? 1 << a.kv.page_shift : S::kTile;
  p.pre = pre;
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  p.counters = reinterpret_cast<uint32_t*>(ws);
  p.part = reinterpret_cast<float*>(ws + counter_bytes());
  p.part_ml = p.part + (int64_t)2 * ctas * p.G * HD;
  if (SH == kPlanned) {
    p.part = pre.slots;
    p.part_ml = pre.slots_ml;
  }
  CUtensorMap mk, mv;
  MapsOf<F8, SH> more{};
  auto map = [&](CUtensorMap* m, bool v, int box) {
    if constexpr (F8) return make_map8(m, a, v, box);
    else return make_kv_map(m, a, v, box);
  };
  bool made = map(&mk, false, p.box) && map(&mv, true, p.box);
  if constexpr (F8) made = made && make_map_scales(&more.s, a, p.box);
  if constexpr (SH == kThrough) {
    PagedAttnArgs x = a;
    x.kv = a.pre.kv;
    more.box = (1 << x.kv.page_shift) < S::kTile ? 1 << x.kv.page_shift : S::kTile;
    made = made && make_kv_map(&more.k, x, false, more.box) && make_kv_map(&more.v, x, true, more.box);
  } else if constexpr (F8 || SH) {
    made = made && map(&more.k, false, 16) && map(&more.v, true, 16);
  }
  if (!made) return cudaErrorInvalidValue;
  constexpr int smem = S::kSmem;
  static_assert(smem <= 233472 / S::kCtas - 1024, "shared memory of one CTA");
  int dev = 0;
  cudaGetDevice(&dev);
  static bool configured[64] = {false};
  const auto kernel = decode_kernel<HD, BF, NT, F8, SH>;
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const cudaError_t e = launch_pdl(kernel, dim3((unsigned)ctas), dim3(S::kThreads), smem, s, mk, mv, more, p);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

template <bool F8, int SH, typename Args>
cudaError_t decode_any(const Args& a, const PrefixParts& pre, int own_ctas, cudaStream_t s) {
  auto heads = [&](auto hd, auto bf) {
    return a.n_heads / a.kv.n_kv <= 8 ? decode_go<decltype(hd)::value, decltype(bf)::value, 1, F8, SH>(a, pre, own_ctas, s)
                                      : decode_go<decltype(hd)::value, decltype(bf)::value, 2, F8, SH>(a, pre, own_ctas, s);
  };
  using H64 = std::integral_constant<int, 64>;
  using H128 = std::integral_constant<int, 128>;
  if (a.kv.hd == 128) return a.kv.bf16 ? heads(H128{}, std::true_type{}) : heads(H128{}, std::false_type{});
  return a.kv.bf16 ? heads(H64{}, std::true_type{}) : heads(H64{}, std::false_type{});
}

}  // namespace
}  // namespace rpgc
