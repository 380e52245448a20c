// paged8_dev.cuh -- device helpers of the 8-bit paged cache (e4m3 codes, a scale for
// each row) and of shared prefixes.
#pragma once

#include <cuda_runtime.h>

#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "paged_dev.cuh"

namespace rpgc {
namespace paged {

// Scale of a row whose largest absolute value is `top` (NaN where one was NaN).
// 2^-126 at least, so that its inverse is finite.
RPGC_DEV float scale_of(float top) {
  return top < INFINITY ? fmaxf(top * (1.0f / 448.0f), 1.17549435e-38f) : __int_as_float(0x7fffffff);
}
// 1 / scale within an ulp.
RPGC_DEV float inverse_of(float scale) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(scale));
  return r;
}

// Four values as codes, rounded to the nearest even (what rounds past 448 becomes 448).
RPGC_DEV uint32_t pack_e4m3(const float* x) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(x[1]), "f"(x[0]));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(x[3]), "f"(x[2]));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

// Codes of the low or high half of a word as two fp16 values (exact).
RPGC_DEV uint32_t half2_lo(uint32_t w) {
  uint32_t r;
  asm("{\n .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %1;\n cvt.rn.f16x2.e4m3x2 %0, lo;\n}" : "=r"(r) : "r"(w));
  return r;
}
RPGC_DEV uint32_t half2_hi(uint32_t w) {
  uint32_t r;
  asm("{\n .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %1;\n cvt.rn.f16x2.e4m3x2 %0, hi;\n}" : "=r"(r) : "r"(w));
  return r;
}
RPGC_DEV float2 float2_lo(uint32_t w) { return unpack2<false>(half2_lo(w)); }
RPGC_DEV float2 float2_hi(uint32_t w) { return unpack2<false>(half2_hi(w)); }

// ------------------------------------------------------- shared prefixes
constexpr int kPrefixKeys = 128;  // keys of a tile of the prefix kernel

// First sequence of group g, kept inside [0, n_seqs] whatever cu holds.  L2: in kernels
// that have not waited for the one before and rely on its wait.
template <bool L2>
RPGC_DEV int32_t group_seq(const PagedPrefix& p, int32_t n_seqs, int g) {
  return min(max(L2 ? __ldcg(p.cu + g) : p.cu[g], 0), n_seqs);
}
// Group of sequence s, or -1: the last g with first(g) <= s, where s is before the next
// one's.
template <typename F>
RPGC_DEV int32_t group_of(int32_t n_groups, int32_t s, F first) {
  int32_t a = 0, b = n_groups;  // it is a - 1 in the end
  while (a < b) {
    const int32_t mid = (a + b) >> 1;
    if (first(mid) <= s) a = mid + 1;
    else b = mid;
  }
  return a > 0 && s < first(a) ? a - 1 : -1;
}
// What the token of a sequence of kv_len positions sees; len: its group's prefix (0: none).
RPGC_DEV PrefixSeq sight_of(const PagedOwnArgs& a, int32_t kv_len, int32_t len) {
  const int32_t n = max(0, kv_len);
  PrefixSeq v;
  v.own = min(n, max(0, len));
  v.pre = (int32_t)min((int64_t)v.own, (int64_t)a.pre.max_pages << a.pre.kv.page_shift);
  v.len = max((int32_t)min((int64_t)n, table_reach(a.kv, a.b)), v.own);
  v.chunk = 0;
  return v;
}

// A group as the prefix kernel sees it.
struct Share {
  int32_t seq, n;  // its sequences
  int32_t end;     // positions that exist, if there is a sequence to see them
};
template <bool L2>
RPGC_DEV Share share_of(const PagedOwnArgs& a, int g) {
  Share s{0, 0, 0};
  if (g < a.pre.n_groups) {
    const int32_t len = L2 ? __ldcg(a.pre.lens + g) : a.pre.lens[g];
    s.seq = group_seq<L2>(a.pre, a.b.n_seqs, g);
    s.n = max(0, group_seq<L2>(a.pre, a.b.n_seqs, g + 1) - s.seq);
    s.end = s.n ? (int32_t)min((int64_t)max(0, len), (int64_t)a.pre.max_pages << a.pre.kv.page_shift) : 0;
  }
  return s;
}
RPGC_DEV int32_t tiles_of(const Share& s) { return (int32_t)(((int64_t)s.end + kPrefixKeys - 1) / kPrefixKeys); }
// Key tiles of a piece: a prefix is cut into `pieces`, or as many as it has tiles.
RPGC_DEV int32_t chunk_of(int32_t tiles, int32_t pieces) { return max(1, (tiles + pieces - 1) / pieces); }
// Units of a group: rows of two tiles x pieces x kv heads.  (n_seqs x kv heads is less
// than 2^31, and pieces are few where it is large.)
RPGC_DEV int32_t units_of(const Share& s, int32_t T, int32_t pieces, int32_t n_kv) {
  const int32_t nt = tiles_of(s), chunk = chunk_of(nt, pieces);
  return (s.n + 2 * T - 1) / (2 * T) * ((nt + chunk - 1) / chunk) * n_kv;
}

// Attention of sequence s's token and query head h by one warp, 32 keys a step, lane
// l scoring key l, fp32 throughout: once over the keys for the largest score and the sum
// of weights, once more with every lane adding the keys' values for its own dims by weights
// that the sum has divided, so that no sum outgrows the values.
template <int HD, bool BF>
struct RowState {
  static constexpr int E = HD / 32;
  float m = -INFINITY, l = 0.0f, inv = 0.0f, o[E] = {};
  // positions [t0, t1) through one row of a table; C8: codes and scales; Values: the second time
  template <bool C8, bool Values>
  RPGC_DEV void keys(const PagedView& kv, const float* scales, int64_t sc_page, int64_t sc_head, const int32_t* table,
                     int32_t max_pages, const uint16_t* q, float scale, int kh, int64_t t0, int64_t t1, int lane) {
    const int64_t mask = (1 << kv.page_shift) - 1;
    for (; t0 < t1; t0 += 32) {
      const int64_t t = t0 + lane, j = t >> kv.page_shift;
      const int32_t page = t < t1 && j < max_pages ? table[j] : -1;
      const bool ok = (uint32_t)page < (uint32_t)kv.n_pages;
      const int64_t slot = t & mask, ko = page * kv.k_page + slot * kv.k_pos + kh * kv.k_head,
                    vo = page * kv.v_page + slot * kv.v_pos + kh * kv.v_head;
      float sc = -INFINITY, vs = 1.0f;
      if (ok) {
        sc = 0.0f;
        const uint32_t* qp = reinterpret_cast<const uint32_t*>(q);
        if (C8) {
          const float* sp = scales + page * sc_page + kh * sc_head + slot;
          vs = sp[mask + 1];
          const uint4* kp = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(kv.k) + ko);
#pragma unroll 2
          for (int i = 0; i < HD / 16; ++i) {
            const uint4 u = kp[i];
            const uint32_t ws[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 a = float2_lo(ws[e]), b = float2_hi(ws[e]), qa = unpack2<BF>(qp[8 * i + 2 * e]),
                           qb = unpack2<BF>(qp[8 * i + 2 * e + 1]);
              sc += qa.x * a.x + qa.y * a.y + (qb.x * b.x + qb.y * b.y);
            }
          }
          sc *= sp[0];
        } else {
          const uint4* kp = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(kv.k) + ko);
#pragma unroll 4
          for (int i = 0; i < HD / 8; ++i) {
            const uint4 u = kp[i];
            const uint32_t ws[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = unpack2<BF>(ws[e]), qf = unpack2<BF>(qp[4 * i + e]);
              sc += qf.x * f.x + qf.y * f.y;
            }
          }
        }
        sc *= scale;
      }
      const uint32_t live = __ballot_sync(0xffffffffu, ok);
      if (!live) continue;
      if (!Values) {
        const float mn = fmaxf(m, warp_max(sc)), base = mn == -INFINITY ? 0.0f : mn;
        l = l * expf(m - base) + warp_sum(ok ? expf(sc - base) : 0.0f);
        m = mn;
        continue;
      }
      const float p = ok ? expf(sc - (m == -INFINITY ? 0.0f : m)) * inv : 0.0f;
      const float pv = p * vs;
#pragma unroll 8
      for (int k = 0; k < 32; ++k) {
        const bool on = live >> k & 1;
        const float pk = __shfl_sync(0xffffffffu, pv, k);
        const int64_t vk = __shfl_sync(0xffffffffu, vo, k);
        float2 f[(E + 1) / 2];
        if (C8) {
          const uint8_t* vp = static_cast<const uint8_t*>(kv.v) + vk + E * lane;
          const uint32_t w = !on ? 0u : E == 4 ? *reinterpret_cast<const uint32_t*>(vp) : *reinterpret_cast<const uint16_t*>(vp);
          f[0] = float2_lo(w);
          if (E == 4) f[E / 4] = float2_hi(w);
        } else {
          const uint16_t* vp = static_cast<const uint16_t*>(kv.v) + vk + E * lane;
#pragma unroll
          for (int i = 0; i < E; i += 2) f[i / 2] = unpack2<BF>(on ? *reinterpret_cast<const uint32_t*>(vp + i) : 0u);
        }
#pragma unroll
        for (int i = 0; i < E; i += 2) {
          o[i] += pk * f[i / 2].x;
          o[i + 1] += pk * f[i / 2].y;
        }
      }
    }
  }
};

template <int HD, bool BF, bool F8, bool SH>
RPGC_DEV void own_row(const PagedOwnArgs& a, int32_t s, int h, int lane) {
  constexpr int E = HD / 32;
  const int kh = h / (a.n_heads / a.kv.n_kv);
  const int32_t g = SH ? group_of(a.pre.n_groups, s, [&](int i) { return group_seq<false>(a.pre, a.b.n_seqs, i); }) : -1;
  const PrefixSeq v = sight_of(a, a.b.kv_lens[s], g >= 0 ? a.pre.lens[g] : 0);
  const uint16_t* q = static_cast<const uint16_t*>(a.q) + s * a.q_tok + h * a.q_head;
  RowState<HD, BF> r;
  auto all = [&](auto values) {
    constexpr bool V = decltype(values)::value;
    if (SH && v.pre > 0)
      r.template keys<false, V>(a.pre.kv, nullptr, 0, 0, a.pre.table + g * a.pre.table_stride, a.pre.max_pages, q, a.scale, kh, 0, v.pre, lane);
    r.template keys<F8, V>(a.kv, a.scales, a.sc_page, a.sc_head, a.b.table + s * a.b.table_stride, a.b.max_pages, q, a.scale, kh, v.own,
                           v.len, lane);
  };
  all(std::false_type{});
  r.inv = r.l == 0.0f ? 0.0f : 1.0f / r.l;
  all(std::true_type{});
  uint16_t* op = static_cast<uint16_t*>(a.out) + ((int64_t)s * a.n_heads + h) * HD + E * lane;
#pragma unroll
  for (int i = 0; i < E; i += 2) *reinterpret_cast<uint32_t*>(op + i) = pack2<BF>(r.o[i], r.o[i + 1]);
}

}  // namespace paged
}  // namespace rpgc
