// k_prompt.cu -- causal attention of packed prompts on the 5th-generation
// tensor cores (tcgen05, TMEM), K and V packed beside q or in cache pages.
//
// Mathematics: out_i = sum_t p_t v_t / sum_t p_t with p_t = 2^(c s_t - m),
// s_t = q_i . k_t, c = scale * log2(e), over the keys t that row i sees, one
// pass over the keys with a reference m.  m is the maximum of the first key
// tile and stays until a later tile's sum says that its scores have outgrown
// it: fp32 sums and bf16 probabilities have the exponents for 2^40, fp16
// probabilities (which carry another 2^kLift, so that small ones keep their
// 11 bits) for 2^15.  Until then no maximum is taken and nothing is rescaled.
//
// Precision: scores, exponentials, sums and joins in fp32.  P is rounded once to the
// type of V, the only operand that the 16-bit MMA takes: two 16-bit parts, as the
// single-token kernel has them, would be half as many MMAs again on the unit that sets
// the pace.  Each result is within u / 2 (sum p |v| + its own size) for it, u = 2^-8 or
// 2^-11 (relative L2 on normal values: 2.0e-3 to 2.3e-3 in bf16, where the result's
// rounding alone is 1.6e-3; 2.5e-4 and 2.0e-4 in fp16).  l adds the unrounded
// probabilities: their roundings fall both ways and are not correlated with V.
//
// What a row does not see: its score becomes -inf, its weight 0, and it counts for
// nothing whatever it holds, except that 0 times an infinite or NaN V is NaN in an
// MMA.  Rows that come out infinite or NaN though their scores are finite are computed
// again from their visible keys (attn_row), which also settles rows that do see such
// a V.  That is a warp per row and takes 200 to 400 times as long (512 tokens
// 2.4 ms, 2048 tokens 11 ms).
//
// Layout: the G query heads of a kv head share its keys, so a tile of 128 MMA
// rows holds T = 128 / G tokens x G heads; a work unit is two such tiles (A,
// B) of one sequence and kv head, one CTA per SM taking units from a list
// sorted by cost, longest first.  Where that would leave SMs without a unit, a
// unit is one tile of rows, A takes its even key tiles and B the odd ones, and
// their sums meet at the end.  Warps 0-3 / 4-7: softmax of tile A / B, one
// row per thread; warp 8: issues the MMAs; warp 9: TMA; warp 10: finds the
// next unit.  S = Q K^T goes to TMEM (128 fp32 columns per tile); the softmax
// warps read their row, write P over it in 16 bits, and O += P V takes P from
// TMEM and V as it lies in the cache (keys are its rows: an MN-major operand).
// While the softmax of one tile runs, the tensor core works on the other.
//
// TMEM columns: S/P of A 0-127, of B 128-255, O of A 256-, of B 384-.
//
// Bound: per pair of tiles and 128 keys the tensor core needs 2048 clocks and the
// special-function unit as many for the exponentials (an eighth of them go to
// the FMA pipe); a pair takes ~2600, and long prompts run at the board's power
// limit.  Measured with 32 query and 8 kv heads of 128, bf16: 8192 tokens 465-500
// us (1.1-1.18 PFLOP/s), 512 tokens 12.4 us, 16 sequences of ~734 tokens after 256
// cached ones 147-178 us; a key tile's softmax pass takes 1.57 k clocks, a first or a
// masked one 1.05 k more; the end of a unit 0.7 k for its last product and 3.2 k to read,
// scale and store O.  Heads of 64 (the MMAs need half the clocks, the exponentials as
// many): 8192 tokens of 32 and 8 heads 407 us, 676 TFLOP/s.
#include <cuda_runtime.h>

#include "paged_dev.cuh"
#include "paged_tma.cuh"
#include "prompt_dev.cuh"
#include "tc_dev.cuh"

namespace rpgc {
namespace {

using namespace paged;
using namespace tc;

constexpr int kRows = 128;  // MMA rows of a tile
constexpr int kKeys = 128;  // keys of a tile
constexpr int kPThreads = 384;
constexpr int kUnits = 2;   // units in flight between the finder and the other warps
constexpr int kPoly = 1, kPolyOf = 8;  // of every 8 pairs of a row, those on the FMA pipe
constexpr float kLog2e = 1.4426950408889634f;

struct Unit {
  int32_t seq, kh;           // seq < 0: no more work
  int32_t rows[2];           // tokens of tiles A and B
  int32_t tiles[2];          // their key tiles
  int32_t end[2];            // keys [0, end) are seen by some row
  int32_t pos0;              // position of tile A's first token (negative: before the cache)
  int32_t reach;             // positions that exist
  int64_t row0;              // packed row of tile A's first token
  int64_t key0;              // packed K/V: row of key 0
};

template <int HD>
struct Shape {
  static constexpr int kHalves = HD / 64;              // 64-column operand panels
  static constexpr int kPanel = kRows * 128;           // bytes of one
  static constexpr int kQBytes = 2 * kHalves * kPanel; // tiles A and B
  static constexpr int kStage = kHalves * kPanel;      // a K or V tile
  static constexpr int kStages = HD == 128 ? 5 : 10;
  static constexpr int kBars = 1024;                   // barriers and units
  static constexpr int kSmem = 1024 + kQBytes + kStages * kStage + kBars;
};

struct PromptParams {
  PagedAttnArgs a;
  int32_t T;       // tokens of a tile
  int32_t G;       // heads per kv head
  int32_t dual;    // two tiles of rows per unit; else one, its key tiles in turn on A and B
  int32_t box;     // K/V rows of one TMA copy
  int32_t wide;    // out lies on a 32-byte boundary
};

// ---------------------------------------------------------- the unit list
// Token tiles sorted by cost, the number of key tiles their last row sees;
// within one cost by sequence.  Every rank is found from the lengths alone, so
// the list is never written down.
struct SeqLens {
  int32_t n, pre;  // new tokens, positions before them
};
RPGC_DEV SeqLens seq_lens(const PagedSeqs& b, int s) {
  SeqLens q{0, 0};
  if (s < b.n_seqs) {
    q.n = max(0, (int32_t)(seq_row(b, s + 1) - seq_row(b, s)));
    if (b.table) q.pre = max(0, b.kv_lens[s]) - q.n;
  }
  return q;
}
// First tile of the sequence whose cost is at least c (all later ones cost
// more).  c is at most 2^23 + 2^17: positions past 2^30 count as 2^30 here.
RPGC_DEV int32_t first_tile(SeqLens q, int32_t U, int32_t c) {
  const int32_t pre = min(q.pre, 1 << 30), x = kKeys * (c - 1) + 1;
  if (c <= 0) return 0;
  if (pre + q.n < x) return (int32_t)((uint32_t)(q.n + U - 1) / (uint32_t)U);
  return x <= pre ? 0 : (int32_t)((uint32_t)(x - pre - 1) / (uint32_t)U);
}
RPGC_DEV int32_t tiles_at_least(const PagedSeqs& b, SeqLens mine, int32_t U, int32_t c, int lane) {
  int32_t n = (int32_t)((uint32_t)(mine.n + U - 1) / (uint32_t)U) - first_tile(mine, U, c);
  for (int s = lane + 32; s < b.n_seqs; s += 32) {
    const SeqLens q = seq_lens(b, s);
    n += (int32_t)((uint32_t)(q.n + U - 1) / (uint32_t)U) - first_tile(q, U, c);
  }
  return __reduce_add_sync(0xffffffffu, n);
}

// (a call of its own, so that its registers are not the pass's)
template <int HD, bool BF>
__device__ __noinline__ void row_again(const PagedAttnArgs& a, int s, int64_t r, int h, int hf, int lane) {
  attn_row<HD, BF>(a, s, r, h, hf, lane);
}

template <int HD, bool BF>
__global__ void __launch_bounds__(kPThreads, 1) prompt_kernel(const __grid_constant__ CUtensorMap tm_q,
                                                              const __grid_constant__ CUtensorMap tm_k,
                                                              const __grid_constant__ CUtensorMap tm_v,
                                                              const __grid_constant__ PromptParams p) {
  using S = Shape<HD>;
  constexpr int kHalves = S::kHalves, kPanel = S::kPanel, kStages = S::kStages;
  constexpr uint32_t kFmt = BF ? 1u : 0u;
  constexpr uint32_t kIdBase = (1u << 4) | (kFmt << 7) | (kFmt << 10) | ((uint32_t)(kRows >> 4) << 24);
  constexpr uint32_t kIdS = kIdBase | ((uint32_t)(kKeys >> 3) << 17);
  constexpr uint32_t kIdO = kIdBase | ((uint32_t)(HD >> 3) << 17) | (1u << 16);
  constexpr float kLift = BF ? 0.0f : 6.0f;
  constexpr float kMost = BF ? 1.0e12f : 32768.0f;  // sum of a row's 128 probabilities that needs no new reference

  extern __shared__ uint8_t psm_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(psm_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* Qs = sm;
  uint8_t* ring = sm + S::kQBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + kStages * S::kStage);
  uint64_t* full = bars;                   // [kStages] K/V tile landed
  uint64_t* empty = full + kStages;        // [kStages] its MMAs done
  uint64_t* q_full = empty + kStages;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;          // [2] S of tile A / B ready
  uint64_t* p_full = s_full + 2;           // [2] P written, S read
  uint64_t* o_full = p_full + 2;           // [2] last P V of the unit done
  uint64_t* u_full = o_full + 2;           // [kUnits] unit described
  uint64_t* u_empty = u_full + kUnits;     // [kUnits] read by every role
  uint64_t* x_bar = u_empty + kUnits;      // the softmax groups, at the end of a unit of one tile
  uint64_t* done = x_bar + 1;
  Unit* units = reinterpret_cast<Unit*>(done + 1);
  uint32_t* tslot = reinterpret_cast<uint32_t*>(units + kUnits);
  volatile int32_t* gave_up = reinterpret_cast<volatile int32_t*>(tslot + 1);

  const PagedAttnArgs& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const bool paged = a.b.table != nullptr;
  int32_t* status = a.b.status;

  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int g = 0; g < 2; ++g) {
      mbar_init(s_full + g, 1);
      mbar_init(p_full + g, 4);
      mbar_init(o_full + g, 1);
    }
    for (int i = 0; i < kUnits; ++i) {
      mbar_init(u_full + i, 1);
      mbar_init(u_empty + i, 10);
    }
    mbar_init(x_bar, 8);
    mbar_init(done, 1);
    *gave_up = 0;
    fence_barrier_init();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tslot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == 9 && lane < 3) prefetch_map(lane == 0 ? &tm_q : lane == 1 ? &tm_k : &tm_v);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // launched as a programmatic dependent: all of the above runs under the
  // previous kernel's tail, nothing that a kernel wrote is read before this
  grid_dep_wait();
  grid_dep_launch();
  const uint32_t tmem = *tslot;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return wait_for(bar, parity, gave_up, status); };

  // Registers move from the control warps to the softmax warps (8 x 32 x 200 +
  // 4 x 32 x 104 = the launch's 384 x 168), each at the head of its own branch:
  // code that both paths reached would have to fit the smaller share.
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (warp == 10) {
      // ---------------------------------------------------- finds the units
      const int32_t U = p.T * (p.dual ? 2 : 1);
      const SeqLens mine = seq_lens(a.b, lane);
      int32_t cmax = (max(0, min(mine.pre, 1 << 30) + mine.n) + kKeys - 1) / kKeys;
      for (int s = lane + 32; s < a.b.n_seqs; s += 32) {
        const SeqLens q = seq_lens(a.b, s);
        cmax = max(cmax, (max(0, min(q.pre, 1 << 30) + q.n) + kKeys - 1) / kKeys);
      }
      cmax = __reduce_max_sync(0xffffffffu, cmax);
      const int32_t total = tiles_at_least(a.b, mine, U, 0, lane);
      const int64_t units_n = (int64_t)total * a.kv.n_kv;
      // the current cost c: tiles that cost at least c, and more; the sequences from
      // s0 on are still to be looked through, `before` tiles of cost c lie before them
      int32_t c = cmax + 1, at_least = 0, more = 0, s0 = 0, before = 0;
      for (int it = 0;; ++it) {
        // there and back over the CTAs, so that nobody gets the longest of every round
        const int64_t u = (int64_t)it * gridDim.x + ((it & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        if (it >= kUnits) wait(u_empty + it % kUnits, (uint32_t)((it / kUnits) - 1) & 1u);
        Unit un;
        un.seq = -1;
        if (u < units_n) {
          const int32_t k = (int32_t)(u / a.kv.n_kv);  // (never less than the last)
          if (k >= at_least) {  // the largest lower cost that more than k tiles reach
            int32_t lo = 0, hi = c - 1;
            while (lo < hi) {
              const int32_t mid = (lo + hi + 1) >> 1;
              if (tiles_at_least(a.b, mine, U, mid, lane) > k) lo = mid;
              else hi = mid - 1;
            }
            c = lo;
            more = tiles_at_least(a.b, mine, U, c + 1, lane);
            at_least = tiles_at_least(a.b, mine, U, c, lane);
            s0 = before = 0;
          }
          const int32_t r = k - more;  // among the tiles of cost c
          for (; s0 < a.b.n_seqs; s0 += 32) {
            const SeqLens q = s0 ? seq_lens(a.b, s0 + lane) : mine;
            const int32_t f = first_tile(q, U, c), n = first_tile(q, U, c + 1) - f;
            int32_t sum = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const int32_t x = __shfl_up_sync(0xffffffffu, sum, o);
              if (lane >= o) sum += x;
            }
            const uint32_t in = __ballot_sync(0xffffffffu, r - before < sum);
            if (in) {
              const int src = __ffs(in) - 1;
              const int32_t i = __shfl_sync(0xffffffffu, f + r - before - (sum - n), src);
              const int32_t n_new = __shfl_sync(0xffffffffu, q.n, src), pre = __shfl_sync(0xffffffffu, q.pre, src);
              const int32_t t0 = i * U;
              un.seq = s0 + src;
              un.kh = (int32_t)(u % a.kv.n_kv);
              un.key0 = seq_row(a.b, un.seq);
              un.row0 = un.key0 + t0;
              un.pos0 = pre + t0;
              const int64_t reach = paged ? table_reach(a.kv, a.b) : (int64_t)n_new;
              un.reach = (int32_t)min(reach, (int64_t)0x7fffff00);
#pragma unroll
              for (int g = 0; g < 2; ++g) {
                const int32_t first = p.dual ? g * p.T : 0;
                un.rows[g] = max(0, min(p.T, n_new - t0 - first));
                un.end[g] = un.rows[g] ? (int32_t)max((int64_t)0, min((int64_t)un.pos0 + first + un.rows[g], (int64_t)un.reach)) : 0;
                un.tiles[g] = (un.end[g] + kKeys - 1) / kKeys;
              }
              break;
            }
            before += __shfl_sync(0xffffffffu, sum, 31);
          }
        }
        if (lane == 0) {
          units[it % kUnits] = un;
          mbar_arrive(u_full + it % kUnits);
        }
        __syncwarp();
        if (un.seq < 0 || *gave_up) break;
      }
    } else if (warp == 9) {
      // ------------------------------------------------------------ loads
      int st = 0;
      uint32_t ph = 0;
      int nq = 0;
      const int per = kKeys / p.box;  // copies of a tile and panel
      for (int it = 0;; ++it) {
        wait(u_full + it % kUnits, (uint32_t)(it / kUnits) & 1u);
        const Unit un = units[it % kUnits];
        __syncwarp();
        if (lane == 0) mbar_arrive(u_empty + it % kUnits);
        if (un.seq < 0 || *gave_up) break;
        const int nt = max(un.tiles[0], un.tiles[1]);
        if (!nt) continue;
        if (nq) wait(q_empty, (uint32_t)(nq - 1) & 1u);
        ++nq;
        if (lane == 0) {
          const uint32_t bytes = (uint32_t)(p.T * p.G * 128 * kHalves);
          const bool two = p.dual && un.rows[1];
          mbar_arrive_expect_tx(q_full, bytes * (two ? 2 : 1));
#pragma unroll
          for (int g = 0; g < 2; ++g)
            if (g == 0 || two)
#pragma unroll
            for (int h = 0; h < kHalves; ++h)
              tma_3d(Qs + (g * kHalves + h) * kPanel, &tm_q, 64 * h, un.kh * p.G, (int)(un.row0 + g * p.T), q_full);
        }
        for (int j = 0; j < nt; ++j) {
          // lane l: the page of copy l; a page that is not there becomes the one
          // past the last, which TMA fills with zeros
          int page = 0, at = 0;
          if (paged) {
            const int64_t t = (int64_t)j * kKeys + (int64_t)lane * p.box;
            if (lane < per) page = page_of(a.kv, a.b, un.seq, t);
            if (page < 0) page = a.kv.n_pages;
            at = (int)(t & ((1 << a.kv.page_shift) - 1));
          }
          for (int v = 0; v < 2; ++v) {
            wait(empty + st, ph ^ 1u);
            uint8_t* dst = ring + st * S::kStage;
            const CUtensorMap* m = v ? &tm_v : &tm_k;
            if (lane == 0) mbar_arrive_expect_tx(full + st, S::kStage);
            __syncwarp();
            if (lane < per) {
#pragma unroll
              for (int h = 0; h < kHalves; ++h) {
                uint8_t* d = dst + h * kPanel + lane * p.box * 128;
                if (paged) tma_4d(d, m, 64 * h, un.kh, at, page, full + st);
                else tma_3d(d, m, 64 * h, un.kh, (int)un.key0 + j * kKeys, full + st);
              }
            }
            if (++st == kStages) st = 0, ph ^= 1u;
          }
          if (*gave_up) break;
        }
      }
      if (*gave_up) {  // copies in flight end before the CTA does
        for (int i = 0; i < kStages; ++i)
          for (int k = 0; k < 1 << 12; ++k)
            if (mbar_try_wait(full + i, ph ^ (i < st ? 0u : 1u))) break;
      }
    } else if (warp == 8) {
      // ------------------------------------------------------------- MMAs
      uint32_t at = 0;            // the unit's first place in the ring: K tile j at + 2 j, V tile j after it
      uint32_t pp[2] = {0u, 0u};  // parity of p_full
      // One elected lane issues, from descriptors that differ by constants: with
      // anything more to compute between two MMAs the issue, not the tensor
      // core, sets the pace (150 clocks an MMA instead of 64).
      const uint64_t q_desc = sdesc(Qs), k_desc = sdesc(ring), v_desc = vdesc(ring, kPanel);
      int nq = 0;
      auto commit = [&](uint64_t* bar) {
        if (elect_one()) mma_commit(bar);
        __syncwarp();
      };
      auto landed = [&](uint32_t c) {
        wait(full + c % kStages, (c / kStages) & 1u);
        tc_fence_after();
      };
      // S of accumulator g = Q (tile qt) K^T, K at ring place c
      auto issue_s = [&](int g, int qt, uint32_t c) {
        if (elect_one()) {
          const uint64_t q = q_desc + (uint64_t)(qt * kHalves * kPanel / 16), k = k_desc + (uint64_t)(c % kStages * (S::kStage / 16));
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint64_t o = ((kk >> 2) * kPanel + (kk & 3) * 32) / 16;
            mma_f16(tmem + 128u * g, q + o, k + o, kIdS, kk > 0);
          }
          mma_commit(s_full + g);
        }
        __syncwarp();
      };
      // O of accumulator g += P V, V at ring place c, once P is there
      auto issue_pv = [&](int g, uint32_t c, int keys, bool first) {
        wait(p_full + g, pp[g]);
        pp[g] ^= 1u;
        tc_fence_after();
        const int steps = (keys + 15) >> 4;
        if (elect_one()) {
          const uint64_t vd = v_desc + (uint64_t)(c % kStages * (S::kStage / 16));
          const uint32_t o = tmem + 256u + 128u * g, pt = tmem + 128u * g;
          mma_ts(o, pt, vd, kIdO, !first);
          if (steps == 8) {
#pragma unroll
            for (int kk = 1; kk < 8; ++kk) mma_ts(o, pt + 8u * kk, vd + kk * 128, kIdO, 1u);
          } else {
            for (int kk = 1; kk < steps; ++kk) mma_ts(o, pt + 8u * kk, vd + kk * 128, kIdO, 1u);
          }
        }
        __syncwarp();
      };
      // the values past the last position of the last step of 16 keys become zeros
      auto clear_tail = [&](uint32_t c, int keys) {
        if (!(keys & 15)) return;
        uint8_t* v = ring + c % kStages * S::kStage;
        const int stop = (keys + 15) & ~15;
        for (int i = lane; i < (stop - keys) * 8 * kHalves; i += 32) {
          const int h = i / ((stop - keys) * 8), k = i % ((stop - keys) * 8);
          *reinterpret_cast<uint4*>(v + h * kPanel + (keys + (k >> 3)) * 128 + (k & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      };
      for (int it = 0;; ++it) {
        wait(u_full + it % kUnits, (uint32_t)(it / kUnits) & 1u);
        const Unit un = units[it % kUnits];
        __syncwarp();
        if (lane == 0) mbar_arrive(u_empty + it % kUnits);
        if (un.seq < 0 || *gave_up) break;
        const int nt = max(un.tiles[0], un.tiles[1]), end = max(un.end[0], un.end[1]);
        if (!nt) continue;
        wait(q_full, (uint32_t)nq & 1u);
        ++nq;
        if (p.dual) {
          landed(at);
#pragma unroll
          for (int g = 0; g < 2; ++g)
            if (un.tiles[g] > 0) issue_s(g, g, at);
          commit(empty + at % kStages);
          if (nt == 1) commit(q_empty);
          for (int j = 0; j < nt && !*gave_up; ++j) {
            const uint32_t vc = at + 2 * j + 1, kc = vc + 1;
            const bool more = j + 1 < nt;
            landed(vc);
            clear_tail(vc, min(kKeys, end - j * kKeys));
            bool waited = false;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              if (j < un.tiles[g]) {
                issue_pv(g, vc, min(kKeys, un.end[g] - j * kKeys), j == 0);
                if (j + 1 == un.tiles[g]) commit(o_full + g);
              }
              if (j + 1 < un.tiles[g]) {
                if (!waited) landed(kc);
                waited = true;
                issue_s(g, g, kc);
              }
            }
            commit(empty + vc % kStages);
            if (more) commit(empty + kc % kStages);
            if (j + 2 == nt) commit(q_empty);
          }
        } else {
          // one tile of rows: accumulator A takes its even key tiles, B the odd ones
          for (int j = 0; j < 2 && j < nt; ++j) {
            const uint32_t kc = at + 2 * j;
            landed(kc);
            issue_s(j, 0, kc);
            commit(empty + kc % kStages);
          }
          if (nt <= 2) commit(q_empty);
          for (int j = 0; j < nt && !*gave_up; ++j) {
            const uint32_t vc = at + 2 * j + 1, kc = vc + 3;
            const int keys = min(kKeys, end - j * kKeys);
            landed(vc);
            clear_tail(vc, keys);
            if (j & 1) issue_pv(1, vc, keys, j < 2);
            else issue_pv(0, vc, keys, j < 2);
            if (j + 2 >= nt) commit(o_full + (j & 1));
            commit(empty + vc % kStages);
            if (j + 2 < nt) {
              landed(kc);
              issue_s(j & 1, 0, kc);
              commit(empty + kc % kStages);
              if (j + 3 == nt) commit(q_empty);
            }
          }
        }
        at += 2 * nt;
        if (*gave_up) break;
      }
      if (elect_one()) mma_commit(done);
      __syncwarp();
      for (int k = 0; k < 1 << 14; ++k)
        if (mbar_try_wait(done, 0)) break;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // ---------------------------------------------------------- softmax
    const int g = warp >> 2, r = tid & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + 128u * g, to = tmem + lanes + 256u + 128u * g;
    const int tok = r / p.G, head = r - tok * p.G;
    const float c = a.scale * kLog2e;
    const int shift = paged ? min(a.kv.page_shift, 7) : 7, npg = paged ? (shift < 7 ? kKeys >> shift : 1) : 0;
    uint32_t sp = 0, op = 0, op_b = 0, xp = 0;
    const int step = p.dual ? 1 : 2, j0 = p.dual ? 0 : g;  // this group's key tiles
    auto both = [&] {  // the two groups meet
      __syncwarp();
      if (lane == 0) mbar_arrive(x_bar);
      wait(x_bar, xp);
      xp ^= 1u;
    };
    for (int it = 0;; ++it) {
      wait(u_full + it % kUnits, (uint32_t)(it / kUnits) & 1u);
      const Unit* up = units + it % kUnits;
      const int seq = up->seq, rows = up->rows[g], tiles = up->tiles[g];
      if (seq < 0 || *gave_up) break;
      auto release = [&] {  // the unit's description is read no more
        __syncwarp();
        if (lane == 0) mbar_arrive(u_empty + it % kUnits);
      };
      if (!rows) {
        release();
        continue;
      }
      const int off = p.dual ? g * p.T : 0, first = up->pos0 + off, reach = up->reach;
      const bool live = tok < rows;  // (rows past T * G have tok >= T >= rows)
      const int lim = live ? (int)max((int64_t)0, min((int64_t)first + tok + 1, (int64_t)reach)) : 0;
      const int whole = max(0, min(first + 1, reach)) / kKeys;  // key tiles that every row sees whole
      // a row that sees nothing (or is none) has nothing to wait for
      float m = lim > 0 ? -INFINITY : 0.0f, l = 0.0f;
      const int32_t* tab = paged ? a.b.table + (int64_t)seq * a.b.table_stride : nullptr;
      auto entry = [&](int j) {  // page of this lane's part of key tile j
        const int64_t e = (((int64_t)j * kKeys) >> a.kv.page_shift) + lane;
        return lane < npg && e < a.b.max_pages ? tab[e] : 0;
      };
      int32_t pg = paged && j0 < tiles ? entry(j0) : 0;
      for (int j = j0; j < tiles; j += step) {
        uint32_t gone = 0;  // this tile's pages that are not there
        if (paged) {
          gone = __ballot_sync(0xffffffffu, lane < npg && (uint32_t)pg >= (uint32_t)a.kv.n_pages);
          if (j + step < tiles) pg = entry(j + step);
        }
        wait(s_full + g, sp);
        sp ^= 1u;
        tc_fence_after();
        // One pass over the row with the reference it has: the probabilities are
        // made, summed and kept in 16 bits while S stays where it is.  Only where a row
        // has no reference yet, or its sum shows that the scores have outgrown it
        // (or hold NaN: the comparison fails), the row's maximum is looked for
        // first: m becomes it, O and l follow, and the pass is done again.  The other
        // rows of the warp keep theirs, so that what they give does not
        // depend on scores that they do not see.
        if (j >= whole || gone) {
          // scores that the row does not see become -inf where they lie, so that
          // the pass itself has no branches (they made every tile 200 clocks longer)
          const int n = lim - j * kKeys;
#pragma unroll 1
          for (int q = 0; q < 4; ++q) {
            const int k = n - 32 * q;
            uint32_t on = k >= 32 ? 0xffffffffu : k <= 0 ? 0u : (1u << k) - 1u;
            if (gone >> ((32 * q) >> shift) & 1u) on &= 0xffff0000u;
            if (gone >> ((32 * q + 16) >> shift) & 1u) on &= 0x0000ffffu;
            if (__all_sync(0xffffffffu, on == 0xffffffffu)) continue;
            uint32_t x[32];
            tmem_ld32_async(ts + 32u * q, x);
            tmem_landed(x);
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(on >> i & 1u)) x[i] = 0xff800000u;
            tmem_st16_nowait(ts + 32u * q, x);
            tmem_st16_nowait(ts + 32u * q + 16u, x + 16);
          }
          tmem_wait_st();
        }
        uint32_t w[64];
        float tile_sum;
        bool due = m == -INFINITY;  // this row's maximum has to be looked for
#pragma unroll 1
        for (int pass = 0;; ++pass) {
          uint32_t x[2][32];
          if (__any_sync(0xffffffffu, due)) {
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {
              tmem_ld32_async(ts + 32u * q, x[0]);
              tmem_landed(x[0]);
#pragma unroll
              for (int i = 0; i < 32; i += 2)
                mx[(i >> 1) & 3] = max_nan(mx[(i >> 1) & 3], __uint_as_float(x[0][i]), __uint_as_float(x[0][i + 1]));
            }
            const float top = max_nan(max_nan(mx[0], mx[1]), mx[2], mx[3]) * c;
            const float mn = due ? max_nan(m, top) : m;
            const float f = !due ? 1.0f : m == -INFINITY ? 0.0f : exp2_fast(m - mn);
            if (j > j0) {  // O's row: the last P V was done before this S
              l *= f;
#pragma unroll 1
              for (int q = 0; q < HD / 16; ++q) {
                float t[16];
                tmem_ld16(to + 16u * q, t);
#pragma unroll
                for (int i = 0; i < 16; ++i) t[i] *= f;
                tmem_st16_nowait(to + 16u * q, reinterpret_cast<const uint32_t*>(t));
              }
            }
            m = mn;
          }
          const float base = kLift - (m == -INFINITY ? 0.0f : m);
          const uint64_t c2 = pair(c, c), base2 = pair(base, base);
          uint64_t sum[2] = {0ull, 0ull};
          tmem_ld32_async(ts, x[0]);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            tmem_landed(x[q & 1]);
            if (q < 3) tmem_ld32_async(ts + 32u * (q + 1), x[(q + 1) & 1]);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const uint64_t y =
                  fma2(pair(__uint_as_float(x[q & 1][2 * i]), __uint_as_float(x[q & 1][2 * i + 1])), c2, base2);
              float2 e;
              if (i % kPolyOf < kPoly) {
                e = exp2_poly<BF>(y);
              } else {
                const float2 z = unpair(y);
                e = make_float2(exp2_fast(z.x), exp2_fast(z.y));
              }
              sum[i & 1] = add2(sum[i & 1], pair(e.x, e.y));
              w[16 * q + i] = pack2<BF>(e.x, e.y);
            }
          }
          const float2 u = unpair(add2(sum[0], sum[1]));
          tile_sum = u.x + u.y;
          // (rows that see nothing have no say: their queries may be anything)
          // (the second pass settles every row: those without a reference had theirs in the first)
          due = lim > 0 && !(tile_sum <= kMost);
          if (pass || !__any_sync(0xffffffffu, due)) break;
        }
        l += tile_sum;
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_st16_nowait(ts + 16u * q, w + 16 * q);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + g);
        if (*gave_up) break;
      }
      // ------------------------------------------------------- the rows out
      const int64_t row = up->row0 + off + tok;
      const int h = up->kh * p.G + head;
      release();
      // with one tile of rows, each group has half the columns to write
      const int col0 = p.dual ? 0 : HD / 2 * g, cols = p.dual ? HD : HD / 2;
      uint16_t* out = static_cast<uint16_t*>(a.out) + (row * a.n_heads + h) * HD + col0;
      if (!tiles) {
        if (live)
          for (int i = 0; i < cols / 8; ++i) reinterpret_cast<uint4*>(out)[i] = make_uint4(0, 0, 0, 0);
        continue;
      }
      float mine = 1.0f, other = 0.0f;  // weights of this group's sums and of the other's
      if (p.dual) {
        wait(o_full + g, op);
        op ^= 1u;
      } else {
        volatile float2* ml = reinterpret_cast<volatile float2*>(Qs + kHalves * kPanel);  // (tile B's place: there is none)
        ml[g * kRows + r].x = m;
        ml[g * kRows + r].y = l;
        both();
        const float mo = ml[(g ^ 1) * kRows + r].x, lo = ml[(g ^ 1) * kRows + r].y;
        const float top = max_nan(m, mo);
        mine = m == -INFINITY ? 0.0f : exp2_fast(m - top);
        other = mo == -INFINITY ? 0.0f : exp2_fast(mo - top);
        l = l * mine + lo * other;
        m = top;
        wait(o_full, op);
        op ^= 1u;
        if (tiles > 1) {
          wait(o_full + 1, op_b);
          op_b ^= 1u;
        }
      }
      tc_fence_after();
      // a visible score that is NaN or +inf (then m is too) makes the row NaN
      const float inv = l == 0.0f || m == -INFINITY || lim <= 0 ? 0.0f : m < INFINITY ? 1.0f / l : __int_as_float(0x7fffffff);
      mine *= inv;
      other *= inv;
      uint64_t bad[2] = {0ull, 0ull};  // NaN where a value is not finite
      const uint64_t mine2 = pair(mine, mine), other2 = pair(other, other);
      const bool have = p.dual || g < tiles, two = !p.dual && (g ^ 1) < tiles;
      const uint32_t to2 = tmem + lanes + 256u + 128u * (g ^ 1);
#pragma unroll 1
      for (int q = 0; q < cols / 32; ++q) {
        uint64_t t[16];
        if (have) {
          uint32_t x[32];
          tmem_ld32_async(to + col0 + 32u * q, x);
          tmem_landed(x);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint64_t y = pair(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]));
            bad[i & 1] = fma2(y, 0ull, bad[i & 1]);
            t[i] = fma2(y, mine2, 0ull);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) t[i] = 0ull;
        }
        if (two) {
          uint32_t x[32];
          tmem_ld32_async(to2 + col0 + 32u * q, x);
          tmem_landed(x);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint64_t y = pair(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]));
            bad[i & 1] = fma2(y, 0ull, bad[i & 1]);
            t[i] = fma2(y, other2, t[i]);
          }
        }
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float2 z = unpair(t[i]);
          w[i] = pack2<BF>(z.x, z.y);
        }
        if (live)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (p.wide) {
              st_32(out + 32 * q + 16 * i, w + 8 * i);
            } else {
              uint4* o = reinterpret_cast<uint4*>(out + 32 * q + 16 * i);
              o[0] = make_uint4(w[8 * i], w[8 * i + 1], w[8 * i + 2], w[8 * i + 3]);
              o[1] = make_uint4(w[8 * i + 4], w[8 * i + 5], w[8 * i + 6], w[8 * i + 7]);
            }
          }
      }
      tc_fence_before();
      if (!p.dual) both();  // both have read O: the next unit's may go over it
      // 0 * x is NaN for an infinite or NaN x in a place that a row does not
      // see: such rows are computed again from their visible keys alone
      const float2 bad2 = unpair(add2(bad[0], bad[1]));
      uint32_t again = __ballot_sync(0xffffffffu, live && m < INFINITY && !(bad2.x + bad2.y == 0.0f));
      while (again) {
        const int src = __ffs(again) - 1;
        again &= again - 1;
        const int64_t rr = __shfl_sync(0xffffffffu, row, src);
        const int hh = __shfl_sync(0xffffffffu, h, src);
        row_again<HD, BF>(a, seq, rr, hh, p.dual ? -1 : g, lane);
      }
    }
  }
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

template <int HD, bool BF>
cudaError_t prompt_go(const PagedAttnArgs& a, cudaStream_t s) {
  PromptParams p{};
  p.a = a;
  p.G = a.n_heads / a.kv.n_kv;
  p.T = kRows / p.G;
  p.wide = (reinterpret_cast<uintptr_t>(a.out) & 31) == 0;
  int dev = 0;
  cudaGetDevice(&dev);
  const int sms = sm_count(dev);
  const int64_t pairs = (a.b.n_tokens + 2 * p.T - 1) / (2 * p.T);
  p.dual = pairs * a.kv.n_kv >= sms;
  const int U = p.T * (p.dual ? 2 : 1);
  p.box = a.b.table && a.kv.page_shift < 7 ? 1 << a.kv.page_shift : kKeys;
  CUtensorMap mq, mk, mv;
  {
    const int64_t dims[3] = {HD, a.n_heads, a.b.n_tokens}, st[2] = {a.q_head, a.q_tok};
    const int box[3] = {64, p.G, p.T};
    if (!make_map(&mq, a.q, 3, dims, st, box, CU_TENSOR_MAP_L2_PROMOTION_L2_256B)) return cudaErrorInvalidValue;
  }
  if (!make_kv_map(&mk, a, false, p.box) || !make_kv_map(&mv, a, true, p.box)) return cudaErrorInvalidValue;
  constexpr int smem = Shape<HD>::kSmem;
  static_assert(smem <= 232448, "shared memory of one CTA");
  static bool configured[64] = {false};
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(prompt_kernel<HD, BF>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  // the lengths are on the device: at most this many units exist
  const int64_t most = ((a.b.n_tokens + U - 1) / U + a.b.n_seqs) * a.kv.n_kv;
  const dim3 grid((unsigned)(most < sms ? most : sms));
  const cudaError_t e = launch_pdl(prompt_kernel<HD, BF>, grid, dim3(kPThreads), smem, s, mq, mk, mv, p);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

}  // namespace

cudaError_t prompt_attn_status(int32_t* bits) { return take_bits(bits); }

cudaError_t prompt_attn_launch(const PagedAttnArgs& a, cudaStream_t s) {
  if (!a.b.n_tokens) return cudaSuccess;
  if (a.kv.hd == 128) return a.kv.bf16 ? prompt_go<128, true>(a, s) : prompt_go<128, false>(a, s);
  return a.kv.bf16 ? prompt_go<64, true>(a, s) : prompt_go<64, false>(a, s);
}

}  // namespace rpgc
