// k_paged_decode_prefix.cu -- attention of one new token per sequence over its own 16-bit pages,
// behind a shared prefix (the kernel: paged_decode.cuh).
#include "paged_decode.cuh"

namespace rpgc {

cudaError_t paged_decode_prefix_status(int32_t* bits) { return take_bits(bits); }

// After paged_prefix_launch on the same stream.
cudaError_t paged_decode_prefix_launch(const PagedOwnArgs& a, cudaStream_t s) {
  int32_t* chunk;
  float *part, *ml;
  paged_prefix_parts(a, &chunk, &part, &ml);
  return decode_any<false, true>(a, PrefixParts{chunk, part, ml}, s);
}

}  // namespace rpgc
