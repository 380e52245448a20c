// k_paged8_decode.cu -- attention of one new token per sequence over 8-bit pages of
// the KV cache (the kernel: paged_decode.cuh).
#include "paged_decode.cuh"

namespace rpgc {

cudaError_t paged8_decode_status(int32_t* bits) { return take_bits(bits); }

cudaError_t paged8_decode_launch(const PagedOwnArgs& a, cudaStream_t s) {
  if (!a.b.n_tokens) return cudaSuccess;
  return decode_any<true, 0>(a, PrefixParts{}, 0, s);
}

}  // namespace rpgc
