// k_paged_prefix.cu -- attention of a batch's new tokens over the first positions that
// groups of sequences share: each prefix is read once for all rows of its group, on the
// 5th-generation tensor cores (tcgen05, TMEM).  What it leaves are sums over pieces of the
// prefix; single-token attention over the sequences' own positions joins them
// (paged_decode.cuh).
//
// Mathematics: for a piece J of the positions, sum_{t in J} p_t v_t and l = sum_{t in J} p_t
// with p_t = 2^(c s_t - m), s_t = q . k_t, c = scale * log2(e), and the reference m that they
// go by, fp32.  References, exponentials and masks are the prompt kernel's (k_prompt.cu): no
// running maximum, P rounded once to V's type.  A row that comes out infinite or NaN is
// computed again from its definition where the pieces meet.
//
// Layout: the rows of a group and kv head are its sequences' G query heads, T = 128 / G
// sequences to a tile of 128 MMA rows; a unit is two such tiles (A, B) and a piece of the
// positions, one CTA per SM.  Where a group has no rows left for B, A's even key tiles go
// to accumulator A and the odd ones to B, and their sums meet at the end.  Warps 0-3 / 4-7:
// softmax of A / B, one row per thread; warp 8: MMAs; warp 9: TMA; warp 10: finds the units.
//
// A prefix is cut into as many pieces as fill the SMs once, by the host's count of rows: short
// pieces fill the SMs, but each writes its rows' sums, 4 HD bytes a row, which are read again.
//
// Bound: a pair of tiles and 128 keys need 2048 clocks of the tensor core and as many of the
// special-function unit; a row's scores, softmax and P V follow one another on two accumulators,
// which takes 3050.  Few rows to a group: the prefixes' bytes.  Measured, 32 query and 8 kv heads of 128, bf16:
// 256 sequences over 8192 positions, 128 units of 16 tiles, 41 us (0.84 PFLOP/s; 26 us of it the
// tiles, 4 us from the launch to the first scores, 2 us for the sums out); 64 over 256 positions 12 us beside
// the next kernel, its units' begin and end; six groups of 7 over 100-3000 positions (38 MB) 16 us.
// Not kept: S in two halves of 64 keys, so that scores are there ahead (3970 clocks a pair:
// twice the MMAs, each with as much of Q to read), P handed over in halves (45 us).
#include <cuda_runtime.h>

#include "paged8_dev.cuh"
#include "paged_dev.cuh"
#include "paged_tma.cuh"
#include "prompt_dev.cuh"
#include "tc_dev.cuh"

namespace rpgc {
namespace {

using namespace paged;
using namespace tc;

constexpr int kRows = 128;  // MMA rows of a tile
constexpr int kKeys = kPrefixKeys;  // of a tile
constexpr int kThreads = 384;
constexpr int kUnits = 2;  // units in flight between the finder and the other warps
constexpr int kPoly = 1, kPolyOf = 8;  // of every 8 pairs of a row, those on the FMA pipe
constexpr float kLog2e = 1.4426950408889634f;

struct Unit {
  int32_t seq;          // tile A's first sequence; < 0: no more work
  int32_t kh, group;
  int32_t rows[2];      // sequences of tiles A and B
  int32_t tile, tiles;  // its key tiles
  int32_t end;          // positions of the prefix that exist
  int32_t piece;
};

template <int HD>
struct Shape {
  static constexpr int kHalves = HD / 64;               // 64-column operand panels
  static constexpr int kPanel = kRows * 128;            // bytes of one
  static constexpr int kQBytes = 2 * kHalves * kPanel;  // tiles A and B
  static constexpr int kStage = kHalves * kPanel;       // a K or V tile
  static constexpr int kStages = HD == 128 ? 5 : 10;
  static constexpr int kBars = 1024;                    // barriers and units
  static constexpr int kRefs = 2 * kRows * 8;           // the two accumulators' references and weights
  static constexpr int kSmem = kQBytes + kStages * kStage + kRefs + kBars;
};

struct PrefixParams {
  PagedOwnArgs a;
  int32_t T;       // sequences of a tile
  int32_t G;       // heads per kv head
  int32_t box;     // K/V rows of one TMA copy
  int32_t pieces;  // of a prefix
  PrefixParts parts;
};

template <int HD, bool BF>
__global__ void __launch_bounds__(kThreads, 1) prefix_kernel(const __grid_constant__ CUtensorMap tm_q,
                                                             const __grid_constant__ CUtensorMap tm_k,
                                                             const __grid_constant__ CUtensorMap tm_v,
                                                             const __grid_constant__ PrefixParams p) {
  using S = Shape<HD>;
  constexpr int kHalves = S::kHalves, kPanel = S::kPanel, kStages = S::kStages;
  constexpr uint32_t kFmt = BF ? 1u : 0u;
  constexpr uint32_t kIdBase = (1u << 4) | (kFmt << 7) | (kFmt << 10) | ((uint32_t)(kRows >> 4) << 24);
  constexpr uint32_t kIdS = kIdBase | ((uint32_t)(kKeys >> 3) << 17);
  constexpr uint32_t kIdO = kIdBase | ((uint32_t)(HD >> 3) << 17) | (1u << 16);
  constexpr float kLift = BF ? 0.0f : 6.0f;         // fp16 probabilities carry 2^6: small ones keep their bits
  constexpr float kMost = BF ? 1.0e12f : 32768.0f;  // sum of a row's 128 probabilities that needs no new reference

  extern __shared__ __align__(1024) uint8_t sm[];  // (the kernel has no other shared memory)
  uint8_t* Qs = sm;
  uint8_t* ring = sm + S::kQBytes;
  volatile float2* refs = reinterpret_cast<volatile float2*>(ring + kStages * S::kStage);
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + kStages * S::kStage + S::kRefs);  // [kStages] K/V tile landed
  uint64_t* empty = full + kStages;        // [kStages] its MMAs done
  uint64_t* q_full = empty + kStages;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;          // [2] S of accumulator A / B ready
  uint64_t* p_full = s_full + 2;           // [2] P written, S read
  uint64_t* o_full = p_full + 2;           // [2] last P V of the unit done
  uint64_t* u_full = o_full + 2;           // [kUnits] unit described
  uint64_t* u_empty = u_full + kUnits;     // [kUnits] read by every role
  uint64_t* x_bar = u_empty + kUnits;      // the softmax groups, at the end of a unit of one tile
  uint64_t* done = x_bar + 1;
  Unit* units = reinterpret_cast<Unit*>(done + 1);
  uint32_t* tslot = reinterpret_cast<uint32_t*>(units + kUnits);
  volatile int32_t* gave_up = reinterpret_cast<volatile int32_t*>(tslot + 1);

  const PagedOwnArgs& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
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
  // launched as a programmatic dependent of the plan, which it does not need itself and
  // which let it begin when all that came earlier had ended: it waits for nothing, and what it
  // reads comes from L2, by TMA or __ldcg
  const uint32_t tmem = *tslot;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return wait_for(bar, parity, gave_up, status); };

  // Registers move from the control warps to the softmax warps (8 x 32 x 200 + 4 x 32 x
  // 104 = the launch's 384 x 168; the host checks that it has those)
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (warp == 10) {
      // ---------------------------------------------------- finds the units
      int g0 = 0;          // the groups from g0 on are still to be looked through
      int32_t before = 0;  // units of those before them
      Share s = share_of<true>(a, lane);
      for (int it = 0;; ++it) {
        if (it >= kUnits) wait(u_empty + it % kUnits, (uint32_t)((it / kUnits) - 1) & 1u);
        const int32_t u = it * (int32_t)gridDim.x + (int32_t)blockIdx.x;
        Unit un;
        un.seq = -1;
        while (g0 < a.pre.n_groups) {
          const int32_t mine = units_of(s, p.T, p.pieces, a.kv.n_kv);
          int32_t sum = mine;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int32_t x = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += x;
          }
          const uint32_t in = __ballot_sync(0xffffffffu, u - before < sum);
          if (in) {
            const int src = __ffs(in) - 1;
            const int32_t n = __shfl_sync(0xffffffffu, s.n, src), nt = __shfl_sync(0xffffffffu, tiles_of(s), src), R = (n + 2 * p.T - 1) / (2 * p.T),
                          chunk = chunk_of(nt, p.pieces);
            int32_t w = u - before - __shfl_sync(0xffffffffu, sum - mine, src);
            un.kh = w % a.kv.n_kv;
            w /= a.kv.n_kv;
            const int32_t r = w % R;
            un.piece = w / R;
            un.group = g0 + src;
            un.seq = __shfl_sync(0xffffffffu, s.seq, src) + r * 2 * p.T;
            un.rows[0] = min(p.T, n - r * 2 * p.T);
            un.rows[1] = max(0, min(p.T, n - r * 2 * p.T - p.T));
            un.tile = un.piece * chunk;
            un.tiles = min(chunk, nt - un.tile);
            un.end = __shfl_sync(0xffffffffu, s.end, src);
            break;
          }
          before += __shfl_sync(0xffffffffu, sum, 31);
          g0 += 32;
          s = share_of<true>(a, g0 + lane);
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
      const int per = kKeys / p.box;  // copies of a tile and panel
      const int pshift = a.pre.kv.page_shift;
      for (int it = 0;; ++it) {
        wait(u_full + it % kUnits, (uint32_t)(it / kUnits) & 1u);
        const Unit un = units[it % kUnits];
        __syncwarp();
        if (lane == 0) mbar_arrive(u_empty + it % kUnits);
        if (un.seq < 0 || *gave_up) break;
        if (it) wait(q_empty, (uint32_t)(it - 1) & 1u);
        if (lane == 0) {
          const uint32_t bytes = (uint32_t)(p.T * p.G * 128 * kHalves);
          mbar_arrive_expect_tx(q_full, bytes * (un.rows[1] ? 2 : 1));
#pragma unroll
          for (int g = 0; g < 2; ++g)
            if (un.rows[g])
#pragma unroll
              for (int h = 0; h < kHalves; ++h)
                tma_3d(Qs + (g * kHalves + h) * kPanel, &tm_q, 64 * h, un.kh * p.G, un.seq + g * p.T, q_full);
        }
        const int32_t* tab = a.pre.table + un.group * a.pre.table_stride;
        // lane l: the page of copy l; a page that is not there becomes the one past the
        // last, which TMA fills with zeros
        auto entry = [&](int j) {
          const int64_t t = (int64_t)j * kKeys + (int64_t)lane * p.box, e = t >> pshift;
          return lane < per && e < a.pre.max_pages ? __ldcg(tab + e) : -1;
        };
        int32_t page = entry(un.tile);
        for (int j = un.tile; j < un.tile + un.tiles; ++j) {
          const int at = (int)(((int64_t)j * kKeys + (int64_t)lane * p.box) & ((1 << pshift) - 1));
          if ((uint32_t)page >= (uint32_t)a.pre.kv.n_pages) page = a.pre.kv.n_pages;
          const int32_t next = entry(j + 1);
          for (int v = 0; v < 2; ++v) {
            wait(empty + st, ph ^ 1u);
            uint8_t* dst = ring + st * S::kStage;
            const CUtensorMap* m = v ? &tm_v : &tm_k;
            if (lane == 0) mbar_arrive_expect_tx(full + st, S::kStage);
            __syncwarp();
            if (lane < per)
#pragma unroll
              for (int h = 0; h < kHalves; ++h) tma_4d(dst + h * kPanel + lane * p.box * 128, m, 64 * h, un.kh, at, page, full + st);
            if (++st == kStages) st = 0, ph ^= 1u;
          }
          page = next;
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
      const uint64_t q_desc = sdesc(Qs), k_desc = sdesc(ring), v_desc = vdesc(ring, kPanel);
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
        const int nt = un.tiles, left = un.end - un.tile * kKeys;
        wait(q_full, (uint32_t)it & 1u);
        if (un.rows[1]) {
          landed(at);
          issue_s(0, 0, at);
          issue_s(1, 1, at);
          commit(empty + at % kStages);
          if (nt == 1) commit(q_empty);
          for (int j = 0; j < nt && !*gave_up; ++j) {
            const uint32_t vc = at + 2 * j + 1, kc = vc + 1;
            const bool more = j + 1 < nt;
            const int keys = min(kKeys, left - j * kKeys);
            landed(vc);
            clear_tail(vc, keys);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              issue_pv(g, vc, keys, j == 0);
              if (!more) commit(o_full + g);
              if (more) {
                if (g == 0) landed(kc);
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
            const int keys = min(kKeys, left - j * kKeys);
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
    } else {
      // the kernel over own positions needs the plan and does not wait for this kernel: it
      // may begin when this warp has seen the plan's end
      grid_dep_wait();
      grid_dep_launch();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // ---------------------------------------------------------- softmax
    const int g = warp >> 2, r = tid & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + 128u * g, to = tmem + lanes + 256u + 128u * g, to2 = tmem + lanes + 256u + 128u * (g ^ 1);
    const int tok = r / p.G, head = r - tok * p.G;
    const float c = a.scale * kLog2e;
    const int pshift = a.pre.kv.page_shift, shift = min(pshift, 7), npg = shift < 7 ? kKeys >> shift : 1;
    uint32_t sp = 0, op[2] = {0u, 0u}, xp = 0;  // parities of s_full, o_full, x_bar
    auto both = [&] {  // the two groups meet
      __syncwarp();
      if (lane == 0) mbar_arrive(x_bar);
      wait(x_bar, xp);
      xp ^= 1u;
    };
    for (int it = 0;; ++it) {
      wait(u_full + it % kUnits, (uint32_t)(it / kUnits) & 1u);
      const Unit un = units[it % kUnits];
      __syncwarp();
      if (lane == 0) mbar_arrive(u_empty + it % kUnits);
      if (un.seq < 0 || *gave_up) break;
      const bool dual = un.rows[1] > 0;
      const int step = dual ? 1 : 2, j0 = un.tile + (dual ? 0 : g), j1 = un.tile + un.tiles;  // this group's key tiles
      const int seq = un.seq + (dual ? g * p.T : 0) + tok;
      // a row sees the prefix as far as its sequence goes; one that sees nothing of this
      // piece (or is none) has nothing to wait for and is not written
      const bool in = tok < (dual && g ? un.rows[1] : un.rows[0]);
      const int lim = in ? min(max(0, __ldcg(a.b.kv_lens + seq)), un.end) : 0;
      const bool live = lim > un.tile * kKeys;
      const int whole = (int)(__reduce_min_sync(0xffffffffu, live ? (unsigned)lim : 0x7fffffffu) / kKeys);  // key tiles that every live row sees whole
      float m = live ? -INFINITY : 0.0f, l = 0.0f;
      const int32_t* tab = a.pre.table + un.group * a.pre.table_stride;
      auto entry = [&](int j) {  // page of this lane's part of key tile j
        const int64_t e = (((int64_t)j * kKeys) >> pshift) + lane;
        return lane < npg && e < a.pre.max_pages ? __ldcg(tab + e) : 0;
      };
      int32_t pg = j0 < j1 ? entry(j0) : 0;
      for (int j = j0; j < j1; j += step) {
        const uint32_t gone = __ballot_sync(0xffffffffu, lane < npg && (uint32_t)pg >= (uint32_t)a.pre.kv.n_pages);  // pages that are not there
        if (j + step < j1) pg = entry(j + step);
        wait(s_full + g, sp);
        sp ^= 1u;
        tc_fence_after();
        // One pass over the row with the reference it has (k_prompt.cu); scores that the
        // row does not see become -inf first, where they lie.
        if (j >= whole || gone) {
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
          due = live && !(tile_sum <= kMost);
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
      // ------------------------------------------------------- the sums out
      const int64_t row = ((int64_t)un.piece * a.b.n_seqs + seq) * a.n_heads + un.kh * p.G + head;
      float mine = 1.0f, other = 0.0f;  // weights of this group's sums and of the other's
      if (dual) {
        wait(o_full + g, g ? op[1] : op[0]);
      } else {
        refs[g * kRows + r].x = m;
        refs[g * kRows + r].y = l;
        both();
        const float mo = refs[(g ^ 1) * kRows + r].x, lo = refs[(g ^ 1) * kRows + r].y;
        const float top = max_nan(m, mo);
        mine = m == -INFINITY ? 0.0f : exp2_fast(m - top);
        other = mo == -INFINITY ? 0.0f : exp2_fast(mo - top);
        l = l * mine + lo * other;
        m = top;
        wait(o_full, op[0]);
        if (un.tiles > 1) wait(o_full + 1, op[1]);
      }
      op[0] ^= 1u;
      if (dual || un.tiles > 1) op[1] ^= 1u;
      tc_fence_after();
      // with one tile of rows, each group has half the columns to write
      const int col0 = dual ? 0 : HD / 2 * g, cols = dual ? HD : HD / 2;
      float* out = p.parts.part + row * HD + col0;
      const uint64_t mine2 = pair(mine, mine), other2 = pair(other, other);
      const bool have = dual || g < un.tiles, two = !dual && (g ^ 1) < un.tiles;
#pragma unroll 1
      for (int q = 0; q < cols / 32; ++q) {
        uint32_t x[32];
        if (have) {
          tmem_ld32_async(to + col0 + 32u * q, x);
          tmem_landed(x);
        }
        if (!dual) {
          uint64_t t[16];
#pragma unroll
          for (int i = 0; i < 16; ++i)
            t[i] = have ? mul2(pair(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), mine2) : 0ull;
          if (two) {
            tmem_ld32_async(to2 + col0 + 32u * q, x);
            tmem_landed(x);
#pragma unroll
            for (int i = 0; i < 16; ++i) t[i] = fma2(pair(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), other2, t[i]);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 z = unpair(t[i]);
            x[2 * i] = __float_as_uint(z.x);
            x[2 * i + 1] = __float_as_uint(z.y);
          }
        }
        if (live)
#pragma unroll
          for (int i = 0; i < 4; ++i) st_32(out + 32 * q + 8 * i, x + 8 * i);
      }
      if (live && (dual || g == 0)) {
        // weights are 2^(score - reference); a score that is NaN or +inf makes the row NaN
        const bool fine = m < INFINITY;
        *reinterpret_cast<float2*>(p.parts.ml + row * 2) =
            make_float2(l == 0.0f ? -INFINITY : fine ? m - kLift : 0.0f, fine ? l : __int_as_float(0x7fffffff));
      }
      tc_fence_before();
      if (!dual) both();  // both have read O: the next unit's may go over it
    }
  }
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

template <int HD, bool BF>
cudaError_t prefix_go(const PagedOwnArgs& a, const PrefixParams& given, int ctas, cudaStream_t s) {
  PrefixParams p = given;
  int dev = 0;
  cudaGetDevice(&dev);
  p.box = a.pre.kv.page_shift < 7 ? 1 << a.pre.kv.page_shift : kKeys;
  CUtensorMap mq, mk, mv;
  {
    const int64_t dims[3] = {HD, a.n_heads, a.b.n_seqs}, st[2] = {a.q_head, a.q_tok};
    const int box[3] = {64, p.G, p.T};
    if (!make_map(&mq, a.q, 3, dims, st, box, CU_TENSOR_MAP_L2_PROMOTION_L2_256B)) return cudaErrorInvalidValue;
  }
  PagedAttnArgs over = a;  // the prefix's pages
  over.kv = a.pre.kv;
  if (!make_kv_map(&mk, over, false, p.box) || !make_kv_map(&mv, over, true, p.box)) return cudaErrorInvalidValue;
  constexpr int smem = Shape<HD>::kSmem;
  static_assert(smem <= 232448, "shared memory of one CTA");
  static bool configured[64] = {false};
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    cudaFuncAttributes at;
    cudaError_t e = cudaFuncGetAttributes(&at, prefix_kernel<HD, BF>);
    if (e != cudaSuccess) return e;
    if (at.numRegs != 168) return cudaErrorLaunchOutOfResources;  // setmaxnreg would wait for ever
    e = cudaFuncSetAttribute(prefix_kernel<HD, BF>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const cudaError_t e = launch_pdl(prefix_kernel<HD, BF>, dim3((unsigned)ctas), dim3(kThreads), smem, s, mq, mk, mv, p);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

}  // namespace

cudaError_t paged_prefix_status(int32_t* bits) { return take_bits(bits); }

cudaError_t paged_prefix_launch(const PagedOwnArgs& a, const PrefixParts& parts, const PrefixShape& shape, cudaStream_t s) {
  PrefixParams p{};
  p.a = a;
  p.G = a.n_heads / a.kv.n_kv;
  p.T = shape.T;
  p.parts = parts;
  p.pieces = shape.pieces;
  if (a.kv.hd == 128) return a.kv.bf16 ? prefix_go<128, true>(a, p, shape.ctas, s) : prefix_go<128, false>(a, p, shape.ctas, s);
  return a.kv.bf16 ? prefix_go<64, true>(a, p, shape.ctas, s) : prefix_go<64, false>(a, p, shape.ctas, s);
}

}  // namespace rpgc
