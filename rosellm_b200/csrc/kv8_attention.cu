// C entry points of the attention over the 8-bit cache, and its bfloat16 forms; the kernels are in kv8_attention.cuh.
#include "kv8_attention.cuh"

namespace rl {
namespace kv8 {
int attention8_tc(const AttnParams8& p, int blocks, cudaStream_t stream);
int attention8_bf16(const AttnParams8& p, int rows, int blocks, Fit* fit, cudaStream_t stream) {
  return dispatch_attention8<false>(p, rows, blocks, fit, stream);
}
}  // namespace kv8
}  // namespace rl

// How many blocks of threads of `rows` rows (8, 16, 32 or 64) stand on an SM at once; 0: sizes that are not taken.
RL_EXPORT int rl_kv8_attention_blocks(int dtype, int rows, int is_tiles, int n_heads, int n_kv_heads, int head_dim) {
  if (n_kv_heads <= 0 || n_heads % n_kv_heads != 0 || (rows != 8 && rows != 16 && rows != 32 && rows != 64)) return 0;
  rl::kv8::AttnParams8 p{};
  p.is_tiles = is_tiles;
  p.n_heads = n_heads;
  p.n_kv_heads = n_kv_heads;
  p.head_dim = head_dim;
  rl::kv8::Fit fit{};
  const int rc = dtype == RL_F32 ? rl::kv8::attention8_f32(p, rows, 0, &fit, nullptr) : rl::kv8::attention8_bf16(p, rows, 0, &fit, nullptr);
  return rc == 0 ? fit.blocks : 0;
}

// items: decoded requests int32 [n_items], or (is_tiles) int32 [n_items][2] = (request, first query) of 64-query tiles.  rows: of a block of
// threads, 8, 16, 32 or 64, or 128 (tcgen05: bfloat16, head sizes 64 and 128, pages of up to 4096 tokens, sms not 0); row_blocks: of an item and key/value head.  sms 0: a block of threads to every unit; else `blocks` of them share all units' tiles
// evenly (sms of them where there is little to do), plan holds n_items * row_blocks + 2 ints, part_o blocks * 2 * rows * head_dim floats and part_ml
// two for every head_dim of those.
RL_EXPORT int rl_kv8_attention(int dtype, const void* q, long q_stride, const void* pool, const float* scales, const int* block_table,
                               int bt_rows, int bt_cols, const int* q_start, const int* kv_len, const int* slots, void* out, long out_stride,
                               const int* items, int n_items, int is_tiles, int n_tokens, int n_heads, int n_kv_heads, int head_dim,
                               int page_size, int n_pages, int window, float scale, int rows, int row_blocks, int sms, int blocks, int* plan,
                               float* part_o, float* part_ml, int* status, cudaStream_t stream) {
  if (n_items <= 0 || n_tokens <= 0) return 0;
  if (head_dim <= 0 || head_dim > 256 || head_dim % 32 != 0) return -2;
  if (n_kv_heads <= 0 || n_heads % n_kv_heads != 0) return -3;
  if (page_size <= 0 || page_size % rl::kv8::BLOCK != 0) return -4;
  if (row_blocks < 1 || sms < 0 || (rows != 8 && rows != 16 && rows != 32 && rows != 64 && rows != 128)) return -5;
  if (rows == 128 && (dtype != RL_BF16 || sms <= 0 || (head_dim != 64 && head_dim != 128) || page_size > 4096)) return -5;
  if (n_kv_heads > 65535 || (long)n_items * row_blocks > 0x7fffffffL / (sms == 0 ? n_kv_heads : 1)) return -6;
  if (sms > 0 && (blocks < 1 || plan == nullptr || part_o == nullptr || part_ml == nullptr)) return -7;
  if (status == nullptr) return -8;
  if (n_pages < 1) return -11;  // (the tcgen05 kernel reads the first page in the place of one that is not there)
  const rl::kv8::AttnParams8 p{q,     q_stride, (const uint8_t*)pool, scales,     block_table, bt_rows,    bt_cols,   q_start, kv_len,
                               slots, out,      out_stride,           items,      is_tiles,    n_tokens,   n_heads,   n_kv_heads, head_dim,
                               page_size, n_pages, window,            scale,      row_blocks,  n_items * row_blocks, sms, 0, plan,
                               part_o, part_ml, 0,                    0,          status};
  const int rc = rows == 128       ? rl::kv8::attention8_tc(p, blocks, stream)
                 : dtype == RL_F32 ? rl::kv8::attention8_f32(p, rows, blocks, nullptr, stream)
                                   : rl::kv8::attention8_bf16(p, rows, blocks, nullptr, stream);
  if (rc != 0) return rc;
  RL_CHECK_LAUNCH();
  return 0;
}
