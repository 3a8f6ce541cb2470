// The 32-bit forms of the attention over the 8-bit cache, in a file of their own so that they compile beside the others.
#include "kv8_attention.cuh"

namespace rl {
namespace kv8 {
int attention8_f32(const AttnParams8& p, int rows, int blocks, Fit* fit, cudaStream_t stream) {
  return dispatch_attention8<true>(p, rows, blocks, fit, stream);
}
}  // namespace kv8
}  // namespace rl
