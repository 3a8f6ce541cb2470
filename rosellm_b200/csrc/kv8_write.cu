// Writing a step's keys and values into the 8-bit cache (kv8.cuh has the format).
//
// One warp takes one (block of 16 tokens, plane, head): the largest finite entry of the step's tokens in the block gives the scale
// that they need; a block that the request began in an earlier step keeps its scale unless the new tokens need a larger one, in which case
// the earlier codes are brought to it (code * old / new, rounded again where it falls below the normal range).  So the
// first token of a request in a step and every token at a multiple of 16 lead a block, and the other tokens have no work of their own.
//
// A token's row is read as pieces of 16 bytes by head dim / 8 lanes, as many rows side by side as fit a warp, and kept in registers
// between the maximum and the codes: the input is read once and the codes written once, which is the floor of the traffic.
// Rows of the cache that the step does not write stay as they are, those behind the last token of a block included.
#include "kv8.cuh"

namespace rl {
namespace kv8 {

struct WriteParams {
  const void* k;
  const void* v;
  long k_stride, v_stride;  // elements between tokens
  uint8_t* pool;
  float* scales;
  const int* block_table;
  int bt_rows, bt_cols;
  const int* positions;
  const int* req_of_token;
  const int* q_start;
  const int* slots;
  int n_tokens, n_reqs, n_kv_heads, page_size, max_pos;
  int n_pages;
  int* status;
};

template <typename T>
struct Piece;  // eight entries of a row
template <>
struct Piece<__nv_bfloat16> {
  uint4 w;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { w = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void clear() { w = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ float get(int i) const {
    const uint32_t u = i < 2 ? w.x : i < 4 ? w.y : i < 6 ? w.z : w.w;
    return __uint_as_float((i & 1) ? (u & 0xFFFF0000u) : (u << 16));
  }
};
template <>
struct Piece<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = reinterpret_cast<const float4*>(p)[0];
    b = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void clear() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ float get(int i) const {
    const float4& f = i < 4 ? a : b;
    return (i & 3) == 0 ? f.x : (i & 3) == 1 ? f.y : (i & 3) == 2 ? f.z : f.w;
  }
};

// group: tokens of a block of threads, 1, 4 or 16 (the entry point's rule); four warps share the blocks that those tokens lead, times
// the planes and heads of blockIdx.y.
template <typename T, int DH>
__global__ __launch_bounds__(128) void kv8_write_kernel(WriteParams p, int group, int planes_per_block) {
  constexpr int LANES = DH / 8, ROWS = 32 / LANES, PASSES = BLOCK / ROWS;  // lanes a row, rows at once, turns a block
  pdl_begin();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t0 = blockIdx.x * group;
  bool leads = false;
  if (lane < group && t0 + lane < p.n_tokens) {
    const int req = p.req_of_token[t0 + lane];
    leads = t0 + lane == p.q_start[req] || p.positions[t0 + lane] % BLOCK == 0;
  }
  const uint32_t leaders = __ballot_sync(0xffffffffu, leads);
  if (leaders == 0u) return;
  const int first_plane = blockIdx.y * planes_per_block;
  const int n_planes = min(planes_per_block, 2 * p.n_kv_heads - first_plane);
  const int row_in_pass = lane / LANES, col = (lane % LANES) * 8;
  const int n_items = __popc(leaders) * n_planes;
  for (int item = warp; item < n_items; item += 4) {
    const int t = t0 + (int)__fns(leaders, 0, item / n_planes + 1);
    const int plane_head = first_plane + item % n_planes;
    const int plane = plane_head >= p.n_kv_heads ? 1 : 0, head = plane_head - plane * p.n_kv_heads;
    const int req = p.req_of_token[t], pos = p.positions[t];
    const int slot = p.slots[req];
    if (slot < 0) continue;  // padding
    const int end = min(p.q_start[req + 1], p.n_tokens), first = p.q_start[req];
    if (pos < 0 || pos >= p.max_pos) {
      if (lane == 0) atomicOr(p.status, RL_STATUS_BAD_POSITION);
      continue;
    }
    const int before = pos % BLOCK;  // rows of the block ahead of this token (earlier tokens, if it is the request's first)
    int n = min(BLOCK - before, end - t);
    if (pos + n > p.max_pos) {
      if (lane == 0) atomicOr(p.status, RL_STATUS_BAD_POSITION);
      n = p.max_pos - pos;
    }
    const int entry = pos / p.page_size;
    const int page = slot < p.bt_rows && entry < p.bt_cols ? p.block_table[(size_t)slot * p.bt_cols + entry] : -1;
    if (page < 0 || page >= p.n_pages) {
      if (lane == 0) atomicOr(p.status, RL_STATUS_BAD_PAGE);
      continue;
    }
    const T* src = (plane ? (const T*)p.v : (const T*)p.k) + (size_t)t * (plane ? p.v_stride : p.k_stride) + (size_t)head * DH + col;
    const long stride = plane ? p.v_stride : p.k_stride;
    const size_t page_head = ((size_t)page * 2 + plane) * p.n_kv_heads + head;
    uint8_t* dst = p.pool + (page_head * p.page_size + pos % p.page_size) * DH + col;  // of the first new token
    float* scale_at = p.scales + page_head * (p.page_size / BLOCK) + pos % p.page_size / BLOCK;
    const bool continued = before != 0 && t == first;
    float s_old = 0.f;
    if (continued) s_old = *scale_at;

    Piece<T> x[PASSES];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int r = i * ROWS + row_in_pass;
      if (row_in_pass < ROWS && r < n)
        x[i].load(src + (size_t)r * stride);
      else
        x[i].clear();
    }
#pragma unroll
    for (int i = 0; i < PASSES; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = fabsf(x[i].get(e));
        top = a <= 3.4e38f ? fmaxf(top, a) : top;
      }
    const float need = scale_for(warp_max(top));
    const float s = continued ? fmaxf(s_old, need) : need;
    const float inv = inverse_of(s);
    if (continued && s > s_old) {
      uint8_t* earlier = dst - (size_t)before * DH;
      const float ratio = s_old * inv;
#pragma unroll 1
      for (int i = 0; i < PASSES; ++i) {
        const int r = i * ROWS + row_in_pass;
        if (row_in_pass < ROWS && r < before) {
          uint2 w = *reinterpret_cast<const uint2*>(earlier + (size_t)r * DH);
          uint32_t out[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t u = h ? w.y : w.x;
            const uint32_t lo = decode2((uint16_t)u), hi = decode2((uint16_t)(u >> 16));
            const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
            out[h] = (uint32_t)encode2(a.x * ratio, a.y * ratio) | ((uint32_t)encode2(b.x * ratio, b.y * ratio) << 16);
          }
          *reinterpret_cast<uint2*>(earlier + (size_t)r * DH) = make_uint2(out[0], out[1]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int r = i * ROWS + row_in_pass;
      if (row_in_pass < ROWS && r < n) {
        uint32_t out[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
          out[h] = (uint32_t)encode2(x[i].get(4 * h) * inv, x[i].get(4 * h + 1) * inv) |
                   ((uint32_t)encode2(x[i].get(4 * h + 2) * inv, x[i].get(4 * h + 3) * inv) << 16);
        *reinterpret_cast<uint2*>(dst + (size_t)r * DH) = make_uint2(out[0], out[1]);
      }
    }
    if (lane == 0) *scale_at = s;
  }
}

template <typename T>
int launch_write(const WriteParams& p, int dh, cudaStream_t stream) {
  // Where most tokens lead a block (decode steps: every one), a block of threads has one token, so that all run side by side; in
  // prompt portions one token in 16 leads, and a block of threads looks at 16 tokens, or 4 where the step is mixed.
  const int group = (long)p.n_tokens >= 32L * p.n_reqs ? 16 : (long)p.n_tokens >= 4L * p.n_reqs ? 4 : 1;
  constexpr int PLANES = 4;  // planes and heads of a block of threads: one a warp for each leading token
  const dim3 grid((p.n_tokens + group - 1) / group, (2 * p.n_kv_heads + PLANES - 1) / PLANES);
  switch (dh) {
#define CASE(D)                                                                            \
  case D:                                                                                  \
    launch_pdl(kv8_write_kernel<T, D>, grid, dim3(128), 0, stream, p, group, (int)PLANES); \
    return 0;
    CASE(32) CASE(64) CASE(96) CASE(128) CASE(160) CASE(192) CASE(224) CASE(256)
#undef CASE
  }
  return -2;
}

}  // namespace kv8
}  // namespace rl

// k, v: rows of n_kv_heads * head_dim entries, 16-byte aligned, strides in elements.  max_pos: the first position that is refused.
// block_table [bt_rows][bt_cols].
RL_EXPORT int rl_kv8_write(int dtype, const void* k, long k_stride, const void* v, long v_stride, void* pool, float* scales,
                           const int* block_table, int bt_rows, int bt_cols, const int* positions, const int* req_of_token,
                           const int* q_start, const int* slots, int n_tokens, int n_reqs, int n_kv_heads, int head_dim,
                           int page_size, int n_pages, int max_pos, int* status, cudaStream_t stream) {
  if (n_tokens <= 0 || n_reqs <= 0) return 0;
  if (head_dim <= 0 || head_dim > 256 || head_dim % 32 != 0) return -2;
  if (page_size <= 0 || page_size % rl::kv8::BLOCK != 0) return -3;
  const int piece = dtype == RL_F32 ? 4 : 8;
  if (k_stride % piece != 0 || v_stride % piece != 0 || (uintptr_t)k % 16 != 0 || (uintptr_t)v % 16 != 0) return -4;
  if (n_kv_heads <= 0 || n_kv_heads > 65535) return -5;
  const rl::kv8::WriteParams p{k, v, k_stride, v_stride, (uint8_t*)pool, scales, block_table, bt_rows, bt_cols, positions, req_of_token,
                               q_start, slots, n_tokens, n_reqs, n_kv_heads, page_size, max_pos, n_pages, status};
  const int rc = dtype == RL_F32 ? rl::kv8::launch_write<float>(p, head_dim, stream)
                                 : rl::kv8::launch_write<__nv_bfloat16>(p, head_dim, stream);
  if (rc != 0) return rc;
  RL_CHECK_LAUNCH();
  return 0;
}
