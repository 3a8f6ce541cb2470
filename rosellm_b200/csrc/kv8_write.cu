// Writing a step's keys and values into the 8-bit cache (kv8.cuh has the format).
//
// One warp takes one (block of 16 tokens, plane, head): the largest finite entry of the step's tokens in the block gives the scale
// that they need; a block that the request began in an earlier step keeps its scale unless the new tokens need a larger one, in which case
// the earlier codes are brought to it (code * old / new, rounded again where it falls below the normal range).  So the
// first token of a request in a step and every token at a multiple of 16 lead a block, and the other tokens have no work of their own.
//
// A token's row is read as pieces of 16 bytes by head dim / 8 lanes, as many rows side by side as fit a warp, and kept in registers
// between the maximum and the codes: the input is read once and the codes written once, which is the floor of the traffic.  What keeps a prompt
// portion from it are latencies: three dependent loads to find a block's place, then the rows, then five shuffles; so a warp has up to four
// blocks on their way (cp.async) while it rounds one.  24 portions, 71 MB: 20 us, 10.9 of traffic.
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

__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}

template <typename T>
struct Piece;  // eight entries of a row
template <>
struct Piece<__nv_bfloat16> {
  uint4 w;
  static constexpr int RUN = 8;  // entries that lie next to one another
  template <int DH>
  static __device__ __forceinline__ void fetch(uint32_t to, const __nv_bfloat16* p) { copy16(to, p); }  // 512 bytes a warp
  template <int DH>
  __device__ __forceinline__ void store(uint8_t* to, float by) const { *reinterpret_cast<uint2*>(to) = make_uint2(codes(0, by), codes(1, by)); }
  __device__ __forceinline__ void load(const uint8_t* at) { w = *reinterpret_cast<const uint4*>(at); }
  __device__ __forceinline__ void clear() { w = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) const {  // two maxima of |entries|; a NaN is passed over
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b & 0x7FFF7FFFu));
    return r;
  }
  __device__ __forceinline__ uint32_t top(uint32_t so_far) const { return larger(larger(larger(larger(so_far, w.x), w.y), w.z), w.w); }
  // infinities become NaN
  static __device__ __forceinline__ uint32_t spoilt(uint32_t u) {
    return u | ((u & 0x7FFFu) == 0x7F80u ? 0x7Fu : 0u) | ((u & 0x7FFF0000u) == 0x7F800000u ? 0x7F0000u : 0u);
  }
  __device__ __forceinline__ void spoil() { w = make_uint4(spoilt(w.x), spoilt(w.y), spoilt(w.z), spoilt(w.w)); }
  // four entries from 4 h on, times a power of two, to their codes (the product is exact where it does not fall below every code)
  __device__ __forceinline__ uint32_t codes(int h, float by) const {
    const uint32_t two = __float_as_uint(by) >> 16 | (__float_as_uint(by) & 0xFFFF0000u);
    uint32_t a, b;
    asm("mul.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(h ? w.z : w.x), "r"(two));
    asm("mul.bf16x2 %0, %1, %2;" : "=r"(b) : "r"(h ? w.w : w.y), "r"(two));
    return (uint32_t)encode2(__uint_as_float(a << 16), __uint_as_float(a & 0xFFFF0000u)) |
           ((uint32_t)encode2(__uint_as_float(b << 16), __uint_as_float(b & 0xFFFF0000u)) << 16);
  }
  static __device__ __forceinline__ float top_of(uint32_t t) { return fmaxf(__uint_as_float(t << 16), __uint_as_float(t & 0xFFFF0000u)); }
};
template <>
struct Piece<float> {
  float4 a, b;
  // Four entries and the four half a row on: eight in a row would take two copies that each touch every sector of 32 bytes (measured: 24 portions
  // of 512, 16 heads of 64, 26.5 us, against 40.0).
  static constexpr int RUN = 4;
  template <int DH>
  static __device__ __forceinline__ void fetch(uint32_t to, const float* p) {
    copy16(to, p);
    copy16(to + 512, p + DH / 2);
  }
  template <int DH>
  __device__ __forceinline__ void store(uint8_t* to, float by) const {
    *reinterpret_cast<uint32_t*>(to) = codes(0, by);
    *reinterpret_cast<uint32_t*>(to + DH / 2) = codes(1, by);
  }
  __device__ __forceinline__ void load(const uint8_t* at) {
    a = *reinterpret_cast<const float4*>(at);
    b = *reinterpret_cast<const float4*>(at + 512);
  }
  __device__ __forceinline__ void clear() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ float get(int i) const {
    const float4& f = i < 4 ? a : b;
    return (i & 3) == 0 ? f.x : (i & 3) == 1 ? f.y : (i & 3) == 2 ? f.z : f.w;
  }
  __device__ __forceinline__ uint32_t top(uint32_t so_far) const {
    float t = __uint_as_float(so_far);
#pragma unroll
    for (int i = 0; i < 8; ++i) t = fmaxf(t, fabsf(get(i)));
    return __float_as_uint(t);
  }
  static __device__ __forceinline__ float spoilt(float f) { return fabsf(f) < CUDART_INF_F ? f : CUDART_NAN_F; }
  __device__ __forceinline__ void spoil() {
    a = make_float4(spoilt(a.x), spoilt(a.y), spoilt(a.z), spoilt(a.w));
    b = make_float4(spoilt(b.x), spoilt(b.y), spoilt(b.z), spoilt(b.w));
  }
  __device__ __forceinline__ uint32_t codes(int h, float by) const {
    return (uint32_t)encode2(get(4 * h) * by, get(4 * h + 1) * by) | ((uint32_t)encode2(get(4 * h + 2) * by, get(4 * h + 3) * by) << 16);
  }
  static __device__ __forceinline__ float top_of(uint32_t t) { return __uint_as_float(t); }
};

template <typename T, int DH>
struct WriteShape {
  static constexpr int LANES = DH / 8, ROWS = 32 / LANES, PASSES = BLOCK / ROWS;  // lanes a row, rows at once, turns a block
  static constexpr int PIECE = 32 * (int)sizeof(Piece<T>), STAGE = PASSES * PIECE;  // bytes of a turn and of a block, of one warp
  static constexpr int STAGES = STAGE <= 4096 ? 4 : STAGE <= 8192 ? 2 : 1;          // blocks that a warp has on their way at once
  // Blocks of threads on an SM; fewer registers cost spills, more cost warps.  Measured, 24 portions of 512, us with 1 / 5 / 8: 16 heads of 64
  // 17.7 / 16.6 / 16.7, 8 of 128 20.2 / 16.7 / 18.2; in 32 bits, 8 of 128, a decode step of 256 with 1 / 4 7.4 / 5.8, 4 of 256 portions 29.1 / 26.7 (2).
  static constexpr int AT_ONCE = STAGE <= 4096 ? 5 : STAGE <= 8192 ? 4 : 2;
};

// group: tokens of a block of threads, 1, 4 or 16; each of its four warps takes `each` planes and heads (the entry point's rules), one after the
// other for every block of tokens that those tokens lead.  What the host's arrays say of a leading token (three loads, each of which needs the
// one before) is looked up once, by a lane for each token.  Each lane copies what it will read itself into a ring in shared memory.
template <typename T, int DH>
__global__ __launch_bounds__(128, WriteShape<T, DH>::AT_ONCE) void kv8_write_kernel(WriteParams p, int group, int each) {
  using S = WriteShape<T, DH>;
  constexpr int LANES = S::LANES, ROWS = S::ROWS, PASSES = S::PASSES, STAGES = S::STAGES, PIECE = S::PIECE;
  extern __shared__ __align__(16) uint8_t smem[];  // [warp][stage][turn][piece]
  pdl_begin();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int across = (2 * p.n_kv_heads + 4 * each - 1) / (4 * each);  // blocks next to one another read, and write, what lies next to one another
  const int t0 = (int)(blockIdx.x / across) * group, plane0 = (int)(blockIdx.x % across) * 4 * each;
  const int first_plane = plane0 + warp, end_plane = min(2 * p.n_kv_heads, plane0 + 4 * each);
  if (first_plane >= end_plane) return;
  uint8_t* ring = smem + warp * min(each, STAGES) * S::STAGE + lane * 16;  // (with fewer planes than stages the last stages are not reached)
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  int my_pos = 0, my_rows = 0, my_page = -1;  // of the token of this lane: its position, the rows it leads, their page
  bool my_first = false;
  if (lane < group && t0 + lane < p.n_tokens) {
    const int t = t0 + lane, req = p.req_of_token[t];
    my_pos = p.positions[t];
    if (req >= 0 && req < p.n_reqs) {
      const int first = p.q_start[req], end = min(p.q_start[req + 1], p.n_tokens), slot = p.slots[req];
      my_first = t == first;
      if ((my_first || my_pos % BLOCK == 0) && t >= first && t < end && slot >= 0) {  // slot < 0: padding
        my_rows = min(BLOCK - (my_pos & (BLOCK - 1)), end - t);
        int bits = 0;
        if (my_pos < 0 || my_pos > p.max_pos - my_rows) {
          bits = RL_STATUS_BAD_POSITION;
          my_rows = my_pos < 0 ? 0 : max(0, p.max_pos - my_pos);
        }
        if (my_rows > 0) {
          const int entry = my_pos / p.page_size;
          my_page = slot < p.bt_rows && entry < p.bt_cols ? p.block_table[(size_t)slot * p.bt_cols + entry] : -1;
          if (my_page < 0 || my_page >= p.n_pages) {
            my_page = -1;
            bits |= RL_STATUS_BAD_PAGE;
          }
        }
        if (bits != 0) atomicOr(p.status, bits);
      }
    }
  }
  const int row_in_pass = lane / LANES, col = (lane % LANES) * Piece<T>::RUN;
  for (uint32_t leaders = __ballot_sync(0xffffffffu, my_rows > 0); leaders != 0u; leaders &= leaders - 1u) {
    const int l = __ffs(leaders) - 1;
    const int n = __shfl_sync(0xffffffffu, my_rows, l), pos = __shfl_sync(0xffffffffu, my_pos, l);
    const int page = __shfl_sync(0xffffffffu, my_page, l);
    const bool is_first = __shfl_sync(0xffffffffu, (int)my_first, l) != 0;
    const int before = pos & (BLOCK - 1);  // rows of the block ahead of this token (earlier tokens, if it is the request's first)
    const bool continued = before != 0 && is_first;
    const int row = pos % p.page_size;
    if (page < 0) continue;
    auto fetch = [&](int plane_head, int stage) {
      if (plane_head < end_plane) {
        const bool is_value = plane_head >= p.n_kv_heads;
        const long stride = is_value ? p.v_stride : p.k_stride;
        const T* src = (is_value ? (const T*)p.v - (size_t)p.n_kv_heads * DH : (const T*)p.k) + (size_t)plane_head * DH + col + (size_t)(t0 + l) * stride;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
          const int r = i * ROWS + row_in_pass;
          if (row_in_pass < ROWS && r < n) Piece<T>::template fetch<DH>(ring_at + stage * S::STAGE + i * PIECE, src + (size_t)r * stride);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) fetch(first_plane + 4 * i, i);
    int stage = 0;
#pragma unroll 1
    for (int plane_head = first_plane; plane_head < end_plane; plane_head += 4) {
      fetch(plane_head + 4 * (STAGES - 1), stage == 0 ? STAGES - 1 : stage - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
      Piece<T> x[PASSES];
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        const int r = i * ROWS + row_in_pass;
        if (row_in_pass < ROWS && r < n)
          x[i].load(ring + stage * S::STAGE + i * PIECE);
        else
          x[i].clear();
      }
      stage = stage + 1 == STAGES ? 0 : stage + 1;
      const size_t page_head = (size_t)page * 2 * p.n_kv_heads + plane_head;
      uint8_t* dst = p.pool + (page_head * p.page_size + row) * DH + col;  // of the first new token
      float* scale_at = p.scales + page_head * (p.page_size / BLOCK) + row / BLOCK;
      const float s_old = continued ? *scale_at : 0.f;
      uint32_t tops = 0;
#pragma unroll
      for (int i = 0; i < PASSES; ++i) tops = x[i].top(tops);
      float top = Piece<T>::top_of(tops);
      if (top == CUDART_INF_F) {  // an infinity: once more, with NaN in its place
        tops = 0;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
          x[i].spoil();
          tops = x[i].top(tops);
        }
        top = Piece<T>::top_of(tops);
      }
      const float s = fmaxf(s_old, scale_for(warp_max(top)));
      const float inv = inverse_of(s);
      if (continued && s > s_old) {
        uint8_t* earlier = dst - (size_t)before * DH - col + (lane % LANES) * 8;
        const float ratio = s_old * inv;
        constexpr int TURN = PASSES < 4 ? PASSES : 4;  // under way at once: this is the longest way through a decode step
#pragma unroll 1
        for (int i0 = 0; i0 < PASSES; i0 += TURN) {
          uint2 was[TURN];
#pragma unroll
          for (int i = 0; i < TURN; ++i) {
            const int r = (i0 + i) * ROWS + row_in_pass;
            if (row_in_pass < ROWS && r < before) was[i] = *reinterpret_cast<const uint2*>(earlier + (size_t)r * DH);
          }
#pragma unroll
          for (int i = 0; i < TURN; ++i) {
            const int r = (i0 + i) * ROWS + row_in_pass;
            if (row_in_pass < ROWS && r < before) {
              uint32_t out[2];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t u = h ? was[i].y : was[i].x;
                const uint32_t lo = decode2((uint16_t)u), hi = decode2((uint16_t)(u >> 16));
                const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                out[h] = (uint32_t)encode2(a.x * ratio, a.y * ratio) | ((uint32_t)encode2(b.x * ratio, b.y * ratio) << 16);
              }
              *reinterpret_cast<uint2*>(earlier + (size_t)r * DH) = make_uint2(out[0], out[1]);
            }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        const int r = i * ROWS + row_in_pass;
        if (row_in_pass < ROWS && r < n) x[i].template store<DH>(dst + (size_t)r * DH, inv);
      }
      if (lane == 0) *scale_at = s;
    }
  }
}

template <typename T, int DH>
int launch_write_at(const WriteParams& p, long blocks, int group, int each, cudaStream_t stream) {
  using S = WriteShape<T, DH>;
  const auto kernel = kv8_write_kernel<T, DH>;
  const int bytes = 4 * (each < S::STAGES ? each : S::STAGES) * S::STAGE;
  if (bytes > 48 << 10 && note_launch(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) != cudaSuccess) return take_launch_error();
  if (each > 1)
    launch_pdl_all_shared(kernel, dim3((unsigned)blocks), dim3(128), bytes, stream, p, group, each);
  else
    launch_pdl(kernel, dim3((unsigned)blocks), dim3(128), bytes, stream, p, group, each);
  return 0;
}

template <typename T>
int launch_write(const WriteParams& p, int dh, cudaStream_t stream) {
  // Where most tokens lead a block (decode steps: every one), a block of threads has one token, so that all run side by side; in
  // prompt portions one token in 16 leads, and a block of threads looks at 16 tokens, or 4 where the step is mixed.
  const int group = (long)p.n_tokens >= 32L * p.n_reqs ? 16 : (long)p.n_tokens >= 4L * p.n_reqs ? 4 : 1;
  // Planes a warp: more share the looking up and the beginning of a block, as long as one or two rounds of blocks are left for the device's 148 SMs.
  // Measured, us with 1 / 2 / 4: 24 portions of 512, 16 heads of 64 (6144 blocks of one) 26.5 / 19.0 / 16.6, 8 of 128 (half as many) 18.9 / 16.8 / 18.5; decode steps
  // of 256, 16 of 64 (2048) 7.7 / 6.5 / 7.0, 8 of 128 in 32 bits (1024) 5.8 / 7.0 / 6.2, of 64, 16 of 64 (512) 3.4 / 3.7 / 4.4.
  const long tokens = (p.n_tokens + group - 1) / group;
  auto blocks_of = [&](int each) { return tokens * ((2 * p.n_kv_heads + 4 * each - 1) / (4 * each)); };
  const int each = blocks_of(4) >= 1480 ? 4 : blocks_of(2) >= 740 ? 2 : 1;
  const long blocks = blocks_of(each);
  if (blocks > 0x7fffffffL) return -6;
  switch (dh) {
#define CASE(D) \
  case D:       \
    return launch_write_at<T, D>(p, blocks, group, each, stream);
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
