// k_paged8_decode_prefix.cu -- sums over the sequences' own 8-bit pages behind a shared
// prefix (the kernel: paged_decode.cuh).
#include "paged_decode.cuh"

namespace rpgc {

cudaError_t paged8_decode_prefix_status(int32_t* bits) { return take_bits(bits); }

cudaError_t paged8_decode_prefix_launch(const PagedOwnArgs& a, const PrefixParts& parts, const PrefixShape& shape, cudaStream_t s) {
  return decode_any<true, kPlanned>(a, parts, shape.own_ctas, s);
}

void paged8_decode_prefix_shape(const PagedOwnArgs& a, PrefixShape* shape) { own_shape_of<true>(a, shape); }

}  // namespace rpgc
