// paged_tma.cuh -- what the paged-cache attention kernels share around TMA: tensor
// maps over K and V (in pages or packed), the copies, bounded waits.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <mutex>

#include "common.cuh"
#include "kernels.h"
#include "paged_dev.cuh"

namespace rpgc {
namespace paged {

RPGC_DEV void tma_3d(void* dst, const CUtensorMap* m, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
RPGC_DEV void tma_4d(void* dst, const CUtensorMap* m, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}

RPGC_DEV void prefetch_map(const CUtensorMap* m) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
}

RPGC_DEV float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Bounded wait of one role (about ten seconds); after the first that gives up,
// the CTA's other waits end at once and the call's status says so.
constexpr long long kWaitClocks = 20000000000ll;
RPGC_DEV bool wait_for(uint64_t* bar, uint32_t parity, volatile int32_t* gave_up, int32_t* status) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  do {
    // suspended for up to 2 us at a time: a spinning warp would take issue
    // slots from the warps it waits for
    if (mbar_try_wait_sleep(bar, parity, 2000u)) return true;
    if (*gave_up) return false;
  } while (clock64() - t0 < kWaitClocks);
  *gave_up = 1;
  report(status, kStatusTimeout);
  return false;
}

inline PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    cudaDriverEntryPointQueryResult q;
    void* f = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  });
  return fn;
}

// A map of 16-bit values: rows of hd values, `rank` - 1 strides in elements.
inline bool make_map(CUtensorMap* m, const void* base, int rank, const int64_t* dims, const int64_t* strides, const int* box,
                     CUtensorMapL2promotion promo) {
  auto enc = encoder();
  if (!enc) return false;
  cuuint64_t d[4], st[3];
  cuuint32_t b[4], es[4] = {1, 1, 1, 1};
  for (int i = 0; i < rank; ++i) {
    d[i] = (cuuint64_t)dims[i];
    b[i] = (cuuint32_t)box[i];
    if (i) st[i - 1] = (cuuint64_t)strides[i - 1] * 2;
  }
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, (cuuint32_t)rank, const_cast<void*>(base), d, st, b, es,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, promo,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

inline int sm_count(int dev) {
  static int sms[64] = {0};
  if (dev < 0 || dev >= 64) return 148;
  if (!sms[dev]) cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev);
  return sms[dev] > 0 ? sms[dev] : 148;
}

// K or V as TMA sees it, copies of `box` rows: {dim, kv head, position, page},
// or {dim, kv head, row} where K and V are packed.
inline bool make_kv_map(CUtensorMap* m, const PagedAttnArgs& a, bool v, int box,
                        CUtensorMapL2promotion promo = CU_TENSOR_MAP_L2_PROMOTION_L2_256B) {
  const void* base = v ? a.kv.v : a.kv.k;
  const int64_t pos = v ? a.kv.v_pos : a.kv.k_pos, head = v ? a.kv.v_head : a.kv.k_head, page = v ? a.kv.v_page : a.kv.k_page;
  if (!a.b.table) {
    const int64_t dims[3] = {a.kv.hd, a.kv.n_kv, a.b.n_tokens}, st[2] = {head, pos};
    const int b[3] = {64, 1, box};
    return make_map(m, base, 3, dims, st, b, promo);
  }
  const int64_t dims[4] = {a.kv.hd, a.kv.n_kv, int64_t(1) << a.kv.page_shift, a.kv.n_pages}, st[3] = {head, pos, page};
  const int b[4] = {64, 1, box, 1};
  return make_map(m, base, 4, dims, st, b, promo);
}

}  // namespace paged
}  // namespace rpgc
