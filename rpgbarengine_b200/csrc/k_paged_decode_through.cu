// k_paged_decode_through.cu -- single-token attention through a shared prefix's 16-bit pages
// and then the sequence's own, for prefixes that are small (the kernel: paged_decode.cuh).
#include "paged_decode.cuh"

namespace rpgc {

// What the sequences read of a prefix by this kernel, all together and as long as its table
// allows.  Each sequence's copy comes from L2, at 13 TB/s where nothing else is read and nearly
// for nothing beside own positions from HBM; the plan, the prefix's own kernel and the join
// take 6-10 us whatever they read.  Measured with 32 query and 8 kv heads of 128, this against
// those, us: 64 sequences of ~735 own positions behind 256 shared ones (64 MB) 41.8 / 48.5, of
// 1-100 19.0 / 16.4; 8 behind 2048 (64 MB) 14.9 / 19.0, behind 1024 11.9 / 16.0; 2 behind 64 7.7 / 12.2.  At 128 MB it
// depends on the own positions: 64 behind 512 45.0 / 50.6 with ~735 and 23.8 / 17.8 with 1-100.
constexpr int64_t kThroughBytes = 64 << 20;

cudaError_t paged_decode_through_status(int32_t* bits) { return take_bits(bits); }

cudaError_t paged_decode_through_launch(const PagedOwnArgs& a, cudaStream_t s) { return decode_any<false, kThrough>(a, PrefixParts{}, 0, s); }

bool paged_decode_through_fits(const PagedOwnArgs& a) {
  const int64_t bytes = ((int64_t)a.pre.max_pages << a.pre.kv.page_shift) * a.kv.n_kv * a.kv.hd * 4;  // K and V of a prefix
  return !a.scales && a.pre.n_groups <= kThroughGroups && (bytes == 0 || a.b.n_seqs <= kThroughBytes / bytes);
}

}  // namespace rpgc
