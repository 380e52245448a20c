// k_paged_decode.cu -- attention of one new token per sequence over 16-bit pages of
// the KV cache (the kernel: paged_decode.cuh).
#include "paged_decode.cuh"

namespace rpgc {

int64_t paged_decode_workspace(const PagedView& kv, int32_t n_heads) {
  const int64_t rows = (int64_t)2 * 2 * device_sms() * (n_heads / kv.n_kv);  // (two items of each CTA)
  return counter_bytes() + rows * (kv.hd + 2) * 4;
}

cudaError_t paged_decode_status(int32_t* bits) { return take_bits(bits); }

cudaError_t paged_decode_launch(const PagedAttnArgs& a, cudaStream_t s) {
  if (!a.b.n_tokens) return cudaSuccess;
  return decode_any<false, 0>(a, PrefixParts{}, 0, s);
}

}  // namespace rpgc
