// k_paged_decode.cu -- attention of one new token per sequence over the pages
// of the KV cache.
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
#include <cuda_runtime.h>

#include "paged_dev.cuh"
#include "paged_tma.cuh"

namespace rpgc {
namespace {

using namespace paged;

constexpr int kJoin = 8;   // pieces of a share whose sums are in flight at once
constexpr int kAhead = 4;  // V operands loaded ahead of the probabilities
constexpr float kLog2e = 1.4426950408889634f;

template <int HD, int NT>
struct DShape {
  static constexpr int kCtas = NT == 1 ? 2 : 1;       // CTAs on an SM (NT 2: over 240 registers a thread leave room for one)
  static constexpr int kTile = HD == 128 || NT == 1 ? 64 : 128;  // keys
  static constexpr int kWarps = kTile / 16;           // consumer warps, 16 keys of a tile each
  static constexpr int kThreads = (kWarps + 2) * 32;
  static constexpr int kPanels = HD / 64;
  static constexpr int kPanel = kTile * 128;
  static constexpr int kHalf = kPanels * kPanel;  // K (or V) of a tile
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kHeads = 8 * NT;           // query heads of a kv head, padded
  static constexpr int kPad = HD + 4;             // row of the merge buffer: no bank conflicts
  static constexpr int kMerge = kWarps * kHeads * kPad * 4;  // the warps' sums; later the join's table, 8 bytes per piece and head
  static constexpr int kRest = kMerge + 2 * kWarps * kHeads * 4 + 256;
  // what an SM has, less a kilobyte for each CTA, goes to the ring
  static constexpr int kStages = ((233472 / kCtas - 1024) - kRest) / kStage;
  static constexpr int kSmem = kStages * kStage + kRest;
  static_assert(kStages * 20 + 12 <= 256, "barriers and flags");
};

struct DecodeParams {
  PagedAttnArgs a;
  uint32_t* counters;  // [CTAs] pieces that are done of the shared item that begins in a CTA's range
  float* part;         // [2 * CTAs][G][HD] partial sums
  float* part_ml;      // [2 * CTAs][G][2] their reference and weight
  int32_t G;
  int32_t box;         // rows of one TMA copy
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
RPGC_DEV int32_t seen(const PagedAttnArgs& a, int s) {  // positions the token of sequence s sees
  const int64_t n = min((int64_t)max(0, a.b.kv_lens[s]), table_reach(a.kv, a.b));
  return (int32_t)n;
}
// What an item weighs in the list: its key tiles, and the end of an item (the
// warps' sums, a share's join) as kEnd tiles more, at its front.  An item that sees
// nothing weighs nothing.
constexpr int kEnd = 3;
// Pieces of an item, at most on average: with 8 kv heads of 128, one sequence of 4200
// positions takes 11.6 us in 37 pieces and 10.0 in 18.  Only few long items meet the
// bound, and those of fewer kv heads than 8 lose by it: one sequence of 131072
// positions takes 90 us with 8 kv heads (6.0 TB/s), 81 with 4 (3.3 TB/s) and 89 with one
// (0.76 TB/s, 18 CTAs at work).
constexpr int kPieces = 18;
template <int T>
RPGC_DEV int64_t weight_of(int32_t n) {
  return n ? (n + (int64_t)T - 1) / T + kEnd : 0;
}

// One CTA's range of the list, item by item; every warp walks it by itself.
template <int T>
struct Walk {
  int64_t total, lo, hi;  // weight of the list; this CTA's range
  int32_t seq, kh, len;   // the item
  int64_t i0, i1;         // its key tiles in the list
  int32_t t0, t1;         // those that are this CTA's
  // where range b of n begins, and the range that holds place t
  RPGC_DEV int64_t begin(int b, int n) const {
    return total < (1 << 23) ? (int64_t)((uint32_t)b * (uint32_t)total / (uint32_t)n) : b * total / n;  // (n < 512)
  }
  RPGC_DEV int holder(int64_t t, int n) const {
    return total < (1 << 23) ? (int)((((uint32_t)t + 1) * (uint32_t)n - 1) / (uint32_t)total) : (int)(((t + 1) * n - 1) / total);
  }
  RPGC_DEV void item(int64_t first) {
    i0 = first + kEnd;
    i1 = first + weight_of<T>(len);
    t0 = (int32_t)(lo > i0 ? lo - i0 : 0);
    t1 = (int32_t)((hi < i1 ? hi : i1) - i0);
  }
  RPGC_DEV bool start(const PagedAttnArgs& a, int lane, int ctas, int cta, int* active) {
    const int64_t kv = a.kv.n_kv;
    // each lane adds up a run of sequences; then the run that holds this CTA's
    // first place is looked through 32 sequences at a time
    const int run = (a.b.n_seqs + 31) / 32;
    int64_t sum = 0;
    int32_t ln = 0, some = 0;
#pragma unroll 4
    for (int i = 0; i < run; ++i) {
      const int s = lane * run + i;
      ln = s < a.b.n_seqs ? seen(a, s) : 0;
      sum += weight_of<T>(ln);
      some += ln > 0;
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
      if (run > 1) ln = s0 + lane < a.b.n_seqs ? seen(a, s0 + lane) : 0;
      else ln = __shfl_sync(0xffffffffu, ln, (src + lane) & 31);  // (only lane 0's counts: the run is one sequence)
      const int64_t mine = weight_of<T>(ln) * kv;
      upto = scan(mine, lane);
      const uint32_t in = __ballot_sync(0xffffffffu, before + upto > lo);
      if (in) {
        const int at = __ffs(in) - 1;
        const int64_t first = before + __shfl_sync(0xffffffffu, upto - mine, at);
        seq = s0 + at;
        len = __shfl_sync(0xffffffffu, ln, at);
        const int64_t w = weight_of<T>(len), in_seq = lo - first;
        kh = in_seq < (int64_t)0x7fffffff ? (int32_t)((uint32_t)in_seq / (uint32_t)w) : (int32_t)(in_seq / w);
        item(first + kh * w);
        return true;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  RPGC_DEV int64_t scan(int64_t v, int lane) const {  // inclusive sums over the lanes
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += x;
    }
    return v;
  }
  RPGC_DEV bool next(const PagedAttnArgs& a) {
    if (i1 >= hi) return false;
    if (++kh == a.kv.n_kv) {
      kh = 0;
      do len = seen(a, ++seq);
      while (!len);  // (a later item exists: i1 < hi <= total)
    }
    item(i1);
    return true;
  }
};

template <int N>
RPGC_DEV void bar_consumers() {
  asm volatile("bar.sync 1, %0;" ::"n"(N) : "memory");
}

template <int HD, bool BF, int NT>
__global__ void __launch_bounds__(DShape<HD, NT>::kThreads, DShape<HD, NT>::kCtas) decode_kernel(const __grid_constant__ CUtensorMap tm_k,
                                                              const __grid_constant__ CUtensorMap tm_v,
                                                              const __grid_constant__ DecodeParams p) {
  using S = DShape<HD, NT>;
  constexpr int kStages = S::kStages, kHeads = S::kHeads, kPad = S::kPad, kWarps = S::kWarps, kTile = S::kTile;
  constexpr float kLift = BF ? 0.0f : 6.0f;  // fp16 probabilities carry 2^6: small ones keep their bits
  constexpr float kMost = BF ? 1.0e12f : 32768.0f;  // a probability that needs no new reference
  extern __shared__ __align__(1024) uint8_t ring[];  // (swizzled tiles start on 1024 bytes; the kernel has no other shared memory)
  float* wo = reinterpret_cast<float*>(ring + kStages * S::kStage);  // [warp][head][kPad]
  float* wm = wo + kWarps * kHeads * kPad;                           // [warp][head]
  float* wl = wm + kWarps * kHeads;
  uint64_t* full = reinterpret_cast<uint64_t*>(wl + kWarps * kHeads);
  uint64_t* empty = full + kStages;
  uint32_t* there = reinterpret_cast<uint32_t*>(empty + kStages);  // [kStages] groups of 16 keys that are there
  volatile int32_t* gave_up = reinterpret_cast<volatile int32_t*>(there + kStages);
  int32_t* last = const_cast<int32_t*>(gave_up) + 1;
  uint32_t* again = reinterpret_cast<uint32_t*>(last + 1);  // heads of the item to be computed again
  const PagedAttnArgs& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full + i, 2);
      mbar_init(empty + i, kWarps);
    }
    *gave_up = 0;
    *again = 0;
    fence_barrier_init();
  }
  if (warp == kWarps && lane < 2) prefetch_map(lane ? &tm_v : &tm_k);
  __syncthreads();
  // launched as a programmatic dependent: nothing that a kernel wrote is read before this
  grid_dep_wait();
  grid_dep_launch();
  auto wait = [&](uint64_t* bar, uint32_t parity) { return wait_for(bar, parity, gave_up, a.b.status); };
  int active;
  Walk<kTile> w;
  const bool work = w.start(a, lane, gridDim.x, blockIdx.x, &active);

  if (warp >= kWarps) {  // one warp copies K, the other V
    // ---------------------------------------------------------------- loads
    if (!work) return;
    int st = 0;
    uint32_t ph = 0;
    const int per = kTile / p.box;  // copies per panel
    const int pshift = a.kv.page_shift;
    do {
      const int32_t* tab = a.b.table + (int64_t)w.seq * a.b.table_stride;
      const int t0 = w.t0, t1 = w.t1;
      if (t1 <= t0) continue;  // (the range ends in the item's front)
      // page ids ahead of their use: lane l holds the one of copy l of the next 32
      const int copies = (t1 - t0) * per;
      const int64_t base = (int64_t)t0 * kTile;
      auto entry = [&](int c) {
        const int64_t e = (base + (int64_t)c * p.box) >> pshift;
        return c < copies && e < a.b.max_pages ? tab[e] : -1;
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
        wait(empty + st, ph ^ 1u);
        if (*gave_up) break;
        if (lane == 0) {
          uint32_t groups = 0;  // a copy of 16, 32, .. rows covers 1, 2, .. groups of 16
          const int g = p.box >> 4;
          for (int i = 0; i < per; ++i)
            if (have >> i & 1u) groups |= ((1u << g) - 1u) << (i * g);
          if (warp == kWarps) there[st] = groups;
          mbar_arrive_expect_tx(full + st, S::kHalf);
        }
        __syncwarp();
        if (lane < per) {
          const int at = (int)((base + (int64_t)(c + lane) * p.box) & ((1 << pshift) - 1));
          const bool v = warp > kWarps;
          uint8_t* dst = ring + st * S::kStage + (v ? S::kHalf : 0) + lane * p.box * 128;
#pragma unroll
          for (int h = 0; h < S::kPanels; ++h) tma_4d(dst + h * S::kPanel, v ? &tm_v : &tm_k, 64 * h, w.kh, at, page, full + st);
        }
        if (++st == kStages) st = 0, ph ^= 1u;
      }
      if (*gave_up) break;
    } while (w.next(a));
    if (*gave_up)  // copies in flight end before the CTA does
      for (int i = 0; i < kStages; ++i)
        for (int k = 0; k < 1 << 12; ++k)
          if (mbar_try_wait(full + i, ph ^ (i < st ? 0u : 1u))) break;
    return;
  }

  // ----------------------------------------------------------- attention
  // sequences that see nothing: zeros, their rows dealt over the CTAs
  for (int s = blockIdx.x; s < a.b.n_seqs; s += gridDim.x)
    if (seen(a, s) == 0)
      for (int i = tid; i < a.n_heads * HD / 8; i += kWarps * 32)
        reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + (int64_t)s * a.n_heads * HD)[i] = make_uint4(0, 0, 0, 0);
  if (!work) return;
  const int gr = lane >> 2, tq = lane & 3, G = p.G;
  const float c = a.scale * kLog2e;
  // ldmatrix rows of this lane in the warp's 16 keys: K as stored, V transposed
  const int mi = lane >> 3, mr = lane & 7;
  const int krow = 16 * warp + mr + 8 * (mi & 1), kc = mi >> 1;
  const int vrow = 16 * warp + mr + 8 * (mi >> 1), vc = mi & 1;
  int st = 0;
  uint32_t ph = 0;
  auto put = [&](int h, int d, const float4& acc, float L) {  // four values of the item's row of head h
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
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int h = 8 * n + gr;
      const uint16_t* qp = static_cast<const uint16_t*>(a.q) + (int64_t)w.seq * a.q_tok + (int64_t)(w.kh * G + h) * a.q_head + 2 * tq;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        q[n][k][0] = h < G ? *reinterpret_cast<const uint32_t*>(qp + 16 * k) : 0u;
        q[n][k][1] = h < G ? *reinterpret_cast<const uint32_t*>(qp + 16 * k + 8) : 0u;
      }
    }
    float o[NT][HD / 16][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.0f;
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) o[n][d][0] = o[n][d][1] = o[n][d][2] = o[n][d][3] = 0.0f;
    }
    for (int t = t0; t < t1; ++t) {
      wait(full + st, ph);
      const int left = w.len - t * kTile - 16 * warp;  // keys of this warp's part
      if (left > 0 && (there[st] >> warp & 1u)) {
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
          for (int n = 0; n < NT; ++n) mma<BF>(k & 1 ? s2[n] : s[n], f, q[n][k][0], q[n][k][1]);
        }
        // the first values are on their way while the probabilities are made
        uint32_t v[kAhead][4];
        auto load_v = [&](int d, uint32_t* f) {
          ldsm4_t(vb + (d >> 2) * S::kPanel + vrow * 128 + (((2 * (d & 3) + vc) ^ (vrow & 7)) << 4), f);
        };
#pragma unroll
        for (int d = 0; d < kAhead; ++d) load_v(d, v[d]);
        // s: (key gr, head 2 tq), (gr, 2 tq + 1), (gr + 8, 2 tq), (gr + 8, 2 tq + 1)
        const bool in0 = gr < left, in1 = gr + 8 < left;
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
#pragma unroll 1
        for (;;) {
          if (look) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float t = fmaxf(s[n][e], s[n][e + 2]);
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
                t = fmaxf(t, m[n][e]);
                const float f = m[n][e] == -INFINITY ? 0.0f : exp2_fast(m[n][e] - t);
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
            const uint32_t hi = pack2<BF>(x[n][2 * e], x[n][2 * e + 1]);
            const float2 h = unpack2<BF>(hi);
            b[n][e] = transpose8(hi);
            b_lo[n][e] = transpose8(pack2<BF>(x[n][2 * e] - h.x, x[n][2 * e + 1] - h.y));
          }
        }
        // keys 2 tq, 2 tq + 1 (and + 8) of the V operand; what lies past the
        // last position is cleared, for 0 * NaN is NaN
        uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
        if (left < 16) {
          keep0 = 2 * tq + 1 < left ? 0xffffffffu : 2 * tq < left ? 0xffffu : 0u;
          keep1 = 2 * tq + 9 < left ? 0xffffffffu : 2 * tq + 8 < left ? 0xffffu : 0u;
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
            mma<BF>(o[n][d], f, b[n][0], b[n][1]);
            mma<BF>(o[n][d], f, b_lo[n][0], b_lo[n][1]);
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
        float* row = wo + (warp * kHeads + h) * kPad + gr;
        if (h < G)
#pragma unroll
          for (int d = 0; d < HD / 16; ++d) {
            row[16 * d] = o[n][d][e];
            row[16 * d + 8] = o[n][d][e + 2];
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
        put(h, d, acc, L);
      } else {
        __stcg(reinterpret_cast<float4*>(p.part + ((int64_t)slot * G + h) * HD + d), acc);
        if (d == 0) __stcg(reinterpret_cast<float2*>(p.part_ml) + (int64_t)slot * G + h, make_float2(M, L));
      }
    }
    if (!whole) {
      // ---- the last CTA to finish a shared item joins its pieces
      const int b0 = w.holder(w.i0, active), b1 = w.holder(w.i1 - 1, active);
      bar_consumers<kWarps * 32>();
      if (tid == 0) {
        __threadfence();  // (of all the warps' partial results: they are before this by the barrier)
        // (only the last item of a range goes on past it: one counter per CTA, back at 0 after the join)
        *last = atomicInc(p.counters + b0, (uint32_t)(b1 - b0)) == (uint32_t)(b1 - b0);
        __threadfence();
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
          put(h, d, acc, L);
        }
      }
    }
    bar_consumers<kWarps * 32>();  // the merge buffer is free again
    // (attn_row inlined: a kernel that calls takes 0.2 us longer to begin)
    const uint32_t todo = *again;
    if (__builtin_expect(todo != 0, 0)) {
      for (int h = warp; h < G; h += kWarps)
        if (todo >> h & 1u) attn_row<HD, BF>(a, w.seq, w.seq, w.kh * G + h, -1, lane);
      bar_consumers<kWarps * 32>();
      if (tid == 0) *again = 0;
    }
  } while (w.next(a));
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
template <int HD, int NT>
int decode_ctas(int G) {
  using S = DShape<HD, NT>;
  const int n = device_sms() * S::kCtas, most = S::kMerge / (8 * G);
  return n < most ? n : most;
}

template <int HD, bool BF, int NT>
cudaError_t decode_go(const PagedAttnArgs& a, cudaStream_t s) {
  const int ctas = decode_ctas<HD, NT>(a.n_heads / a.kv.n_kv);
  DecodeParams p{};
  p.a = a;
  p.G = a.n_heads / a.kv.n_kv;
  p.box = (1 << a.kv.page_shift) < DShape<HD, NT>::kTile ? 1 << a.kv.page_shift : DShape<HD, NT>::kTile;
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  p.counters = reinterpret_cast<uint32_t*>(ws);
  p.part = reinterpret_cast<float*>(ws + counter_bytes());
  p.part_ml = p.part + (int64_t)2 * ctas * p.G * HD;
  CUtensorMap mk, mv;
  const CUtensorMapL2promotion promo = CU_TENSOR_MAP_L2_PROMOTION_L2_256B;
  if (!make_kv_map(&mk, a, false, p.box, promo) || !make_kv_map(&mv, a, true, p.box, promo)) return cudaErrorInvalidValue;
  constexpr int smem = DShape<HD, NT>::kSmem;
  static_assert(smem <= 233472 / DShape<HD, NT>::kCtas - 1024, "shared memory of one CTA");
  int dev = 0;
  cudaGetDevice(&dev);
  static bool configured[64] = {false};
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(decode_kernel<HD, BF, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const cudaError_t e = launch_pdl(decode_kernel<HD, BF, NT>, dim3((unsigned)ctas), dim3(DShape<HD, NT>::kThreads), smem, s, mk, mv, p);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

template <int HD, bool BF>
cudaError_t decode_heads(const PagedAttnArgs& a, cudaStream_t s) {
  return a.n_heads / a.kv.n_kv <= 8 ? decode_go<HD, BF, 1>(a, s) : decode_go<HD, BF, 2>(a, s);
}

}  // namespace

int64_t paged_decode_workspace(const PagedView& kv, int32_t n_heads) {
  const int64_t rows = (int64_t)2 * 2 * device_sms() * (n_heads / kv.n_kv);  // (two items of each CTA)
  return counter_bytes() + rows * (kv.hd + 2) * 4;
}

cudaError_t paged_decode_status(int32_t* bits) { return take_bits(bits); }

cudaError_t paged_decode_launch(const PagedAttnArgs& a, cudaStream_t s) {
  if (!a.b.n_tokens) return cudaSuccess;
  if (a.kv.hd == 128) return a.kv.bf16 ? decode_heads<128, true>(a, s) : decode_heads<128, false>(a, s);
  return a.kv.bf16 ? decode_heads<64, true>(a, s) : decode_heads<64, false>(a, s);
}

}  // namespace rpgc
