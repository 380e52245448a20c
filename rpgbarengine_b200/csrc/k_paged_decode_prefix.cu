// k_paged_decode_prefix.cu -- sums over the sequences' own 16-bit pages behind a shared
// prefix (the kernel: paged_decode.cuh).
#include "paged_decode.cuh"

namespace rpgc {

cudaError_t paged_decode_prefix_status(int32_t* bits) { return take_bits(bits); }

cudaError_t paged_decode_prefix_launch(const PagedOwnArgs& a, const PrefixParts& parts, const PrefixShape& shape, cudaStream_t s) {
  return decode_any<false, kPlanned>(a, parts, shape.own_ctas, s);
}

void paged_decode_prefix_shape(const PagedOwnArgs& a, PrefixShape* shape) { own_shape_of<false>(a, shape); }

}  // namespace rpgc
