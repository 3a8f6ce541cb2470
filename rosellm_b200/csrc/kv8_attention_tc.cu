// The tcgen05 form of the attention over the 8-bit cache, in a file of its own so that it compiles beside the others.
#include "kv8_attention_tc.cuh"

namespace rl {
namespace kv8 {
int attention8_tc(const AttnParams8& p, int blocks, cudaStream_t stream) {
  if (p.head_dim == 64) return launch_attention_tc<64>(p, blocks, stream);
  if (p.head_dim == 128) return launch_attention_tc<128>(p, blocks, stream);
  return -2;
}
}  // namespace kv8
}  // namespace rl
