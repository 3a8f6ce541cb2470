// Attention over the 8-bit cache on mma.sync (kv8.cuh has the format): the function of attention_kernels.cuh with keys and values
// code * scale.
//
// A block of threads takes up to 16 * WR rows: the queries of one item (a decoded token, or up to 64 queries of a prompt portion) times
// the heads that share one key/value head, so that grouped heads read each key once.  Its four warps are WR along the rows times 4 / WR along the
// keys; the keys of an item may besides be cut into parts over blocks of the grid, whose results a second kernel joins.
//
// No operand passes through shared memory to be rearranged.  In S = Q K^T the inner index may be ordered at will, if Q and K are ordered
// alike: the lane of column n and inner quarter c takes the quarter c of key n's row as it lies, head dim / 4 consecutive bytes, and
// gets from each word the four entries of one step of 16 (Q's fragments are laid out to match, once).  In O = P V the columns may be ordered at
// will: the lane of column n takes the consecutive bytes n * head dim / 8 ... of four keys' rows, and a byte permutation of two rows
// gives the pairs of keys that the operand wants.  Which key is which column of S is free too: columns 2c and 2c+1 are keys c and c+4, so that
// neighbouring lanes read neighbouring rows of V.  Codes become halves by one conversion for two (exact).
//
// Scales: S's 16 columns of a block are multiplied by the block's key scale.  A block of values is one inner step of P V, so its
// probabilities are multiplied by (scale / largest scale so far) * 2^15 before they are rounded to halves (probabilities down to 2^-29 keep
// all of their 11 bits: relative error 2^-11, against 2^-9 of a bfloat16 output), and the output follows the largest scale as it follows the
// maximum.  Q is brought to halves row by row with a power of two that puts its largest entry at 2^14 (a bfloat16 fits exactly,
// within 2^-28 of the row's largest); in 32 bits Q and P are two halves each, a value and what its rounding left, so that products
// are exact to 2^-22.  Sums, maxima and outputs are float32.
#pragma once
#include "kv8.cuh"

namespace rl {
namespace kv8 {

constexpr int TILE_QUERIES = 64;  // queries that an entry of the tile list names

struct AttnParams8 {
  const void* q;       // query of token n, head h: q + n * q_stride + h * head_dim
  long q_stride;       // elements
  const uint8_t* pool;
  const float* scales;
  const int* block_table;
  int bt_rows, bt_cols;
  const int* q_start;  // [requests + 1]
  const int* kv_len;   // [requests] keys the request has
  const int* slots;
  void* out;
  long out_stride;
  const int* items;    // tiles [n][2] (request, first query), or decoded requests [n]
  int is_tiles;
  int n_tokens, n_heads, n_kv_heads, head_dim, page_size, n_pages, window;  // window 0: all keys
  float scale;
  int parts, chunk;    // parts that an item's keys are cut into at most, and keys of a part at least
  int row_blocks;      // blocks of rows of an item and key/value head
  float* part_o;       // [items][kv heads * row blocks][parts][rows][head dim]
  float* part_ml;      // [items][kv heads * row blocks][parts][rows][2]
  int* status;
};

// What a block of threads works on: its rows and the keys that any of them sees.
struct Work {
  int req, head_kv, first_row, rows;  // rows: of the item and key/value head, from first_row on; 0 or less: none
  int token0, pos0;                   // token and position of the item's first query
  int first_block, n_blocks;          // blocks of 16 keys in sight
  int per_part, active;               // blocks of 16 keys of a part; parts that have any
  int slot;
};

template <int RB>
__device__ __forceinline__ Work work_of(const AttnParams8& p, int item, int y) {
  Work w;
  const int group = p.n_heads / p.n_kv_heads;
  w.req = p.is_tiles ? p.items[2 * item] : p.items[item];
  const int t0 = p.is_tiles ? p.items[2 * item + 1] : 0;
  const int qs = p.q_start[w.req], q_len = p.q_start[w.req + 1] - qs, kv_len = p.kv_len[w.req];
  const int n_q = min(p.is_tiles ? TILE_QUERIES : 1, q_len - t0);
  w.head_kv = y / p.row_blocks;
  w.first_row = (y % p.row_blocks) * RB;
  w.rows = min(RB, n_q * group - w.first_row);
  w.token0 = qs + t0;
  w.pos0 = kv_len - q_len + t0;
  w.slot = p.slots[w.req];
  const int q_lo = w.first_row / group, q_hi = w.rows > 0 ? (w.first_row + w.rows - 1) / group : 0;
  if (w.token0 < 0 || w.token0 + q_hi >= p.n_tokens) w.rows = 0;  // a description that does not fit the queries
  const int lo = p.window > 0 ? max(0, w.pos0 + q_lo - p.window + 1) : 0;
  const int hi = w.pos0 + q_hi + 1;
  w.first_block = lo / BLOCK;
  w.n_blocks = hi > lo && w.rows > 0 ? (hi + BLOCK - 1) / BLOCK - w.first_block : 0;
  // parts are of whole tiles of four blocks, so that their number and not the last one's length is what differs
  w.per_part = max((p.chunk + BLOCK - 1) / BLOCK, (w.n_blocks + p.parts - 1) / p.parts);
  w.per_part = (w.per_part + 3) / 4 * 4;
  w.active = (w.n_blocks + w.per_part - 1) / w.per_part;
  return w;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// N words from an address aligned to the largest power of two (up to 16) that divides 4 N bytes.
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * i);
      w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p + 4 * i);
      w[i] = v.x, w[i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = *reinterpret_cast<const uint32_t*>(p + 4 * i);
  }
}

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// What rounding the two halves of `packed` left of lo and hi.
__device__ __forceinline__ uint32_t rest_half(float lo, float hi, uint32_t packed) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&packed));
  return pack_half(lo - f.x, hi - f.y);
}

template <int DH, bool F32>
struct Shapes {
  static constexpr int KSTEPS = DH / 16;            // inner steps of Q K^T
  static constexpr int NT = DH / 8;                 // column tiles of the output
  static constexpr int QPARTS = F32 ? 2 : 1;        // halves of a query entry
  static constexpr int TB = DH <= 128 ? 4 : 2;      // blocks of 16 keys of a warp's tile
  static constexpr bool Q_IN_REGS = KSTEPS * QPARTS <= 8;
};

// The queries of 16 rows as the A fragments of Q K^T, in shared memory: frag[part][step][lane] is that lane's four words.  Row r of the
// fragment is row `first + r` of the work; those at or beyond `rows` are zero.  `factor` [16] gets what a row's scores are multiplied
// by.  Called by a whole warp for rows r0 .. r0 + n - 1 of the 16.
template <int DH, bool F32>
__device__ __forceinline__ void lay_queries(const AttnParams8& p, const Work& w, int first, int r0, int n, uint8_t* frag, float* factor) {
  using S = Shapes<DH, F32>;
  const int lane = threadIdx.x & 31, group = p.n_heads / p.n_kv_heads;
#pragma unroll 4
  for (int r = r0; r < r0 + n; ++r) {
    float x[DH / 32];
    const int row = first + r;  // of the block of rows
    const int i = w.first_row + row, q = i / group, h = w.head_kv * group + i % group;
    const size_t at = (size_t)(w.token0 + q) * p.q_stride + (size_t)h * DH + lane;
#pragma unroll
    for (int k = 0; k < DH / 32; ++k) {
      x[k] = 0.f;
      if (row < w.rows) {
        if constexpr (F32)
          x[k] = reinterpret_cast<const float*>(p.q)[at + 32 * k];
        else
          x[k] = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.q)[at + 32 * k]);
      }
    }
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < DH / 32; ++k) top = fmaxf(top, fabsf(x[k]));
    top = warp_max(top);
    // the power of two that puts the largest entry between 2^14 and 2^15 (kept within the exponents whose inverse is a float)
    const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -110), 126);
    const float up = __uint_as_float((uint32_t)(14 - e + 127) << 23), down = __uint_as_float((uint32_t)(e - 14 + 127) << 23);
    if (lane == 0) factor[r] = down * p.scale * 1.4426950408889634f;
#pragma unroll
    for (int k = 0; k < DH / 32; ++k) {
      const int d = lane + 32 * k, c = d / (DH / 4), j = d % (DH / 4);
      const int place = ((j / 4) * 32 + (r % 8) * 4 + c) * 16 + ((r / 8) + (j % 4 / 2) * 2) * 4 + (j % 2) * 2;
      const float v = x[k] * up;
      const __half hi = __float2half_rn(v);
      *reinterpret_cast<__half*>(frag + place) = hi;
      if constexpr (F32) *reinterpret_cast<__half*>(frag + S::KSTEPS * 512 + place) = __float2half_rn(v - __half2float(hi));
    }
  }
}

// A warp's state over the keys it has seen: 16 rows, of which a lane holds two (lane / 4 and 8 more).
template <int DH>
struct State {
  float o[DH / 8][4];
  float m[2], l[2];  // maximum (in units of log 2) and sum; the sum is over this lane's columns only until the end
  int e;             // o is the sum of p * v / 2^(e - 15); e: exponent of the largest value scale so far
};

// TB blocks of 16 keys at once.  k_at(b), v_at(b): where the codes of block b lie (its 16 rows in a row); ks, vs: scales; ks negative: a
// block that is not there (nothing of it is used; k_at and v_at still name readable memory).  key0: the first key's position.
// whole: every row sees every key.  pos: the lane's two rows' positions.
template <int DH, bool F32, class KAt, class VAt>
__device__ __forceinline__ void take_tile(
    State<DH>& st, const uint4* q_frag,
    const uint4 (&q_regs)[Shapes<DH, F32>::Q_IN_REGS ? Shapes<DH, F32>::KSTEPS * Shapes<DH, F32>::QPARTS : 1], KAt k_at, VAt v_at,
    const float (&ks)[Shapes<DH, F32>::TB], const float (&vs)[Shapes<DH, F32>::TB], const float (&factor)[2], int key0, bool whole,
    const int (&pos)[2], int window) {
  using S = Shapes<DH, F32>;
  constexpr int TB = S::TB;
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  float s[2 * TB][4];
#pragma unroll
  for (int b = 0; b < TB; ++b) {
    uint32_t kw[2][S::KSTEPS];
#pragma unroll
    for (int half = 0; half < 2; ++half) load_words<S::KSTEPS>(k_at(b) + (8 * half + (r >> 1) + 4 * (r & 1)) * DH + c * (DH / 4), kw[half]);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float(&d)[4] = s[2 * b + half];
      d[0] = d[1] = d[2] = d[3] = 0.f;
#pragma unroll
      for (int k = 0; k < S::KSTEPS; ++k) {
        const uint32_t b0 = decode2((uint16_t)kw[half][k]), b1 = decode2((uint16_t)(kw[half][k] >> 16));
#pragma unroll
        for (int qp = 0; qp < S::QPARTS; ++qp) {
          const uint4 a = S::Q_IN_REGS ? q_regs[S::Q_IN_REGS ? qp * S::KSTEPS + k : 0] : q_frag[(qp * S::KSTEPS + k) * 32 + lane];
          mma16816(d, a.x, a.y, a.z, a.w, b0, b1);
        }
      }
    }
  }
  // scores in units of log 2; keys out of a row's sight at minus infinity
  float top[2] = {-CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
  for (int b = 0; b < TB; ++b) {
    const float f[2] = {factor[0] * ks[b], factor[1] * ks[b]};
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float& x = s[2 * b + half][i];
        x *= f[i >> 1];
        if (!whole) {
          const int key = key0 + b * BLOCK + half * 8 + c + 4 * (i & 1);
          if (ks[b] < 0.f || key > pos[i >> 1] || (window > 0 && key <= pos[i >> 1] - window)) x = -CUDART_INF_F;
        }
        top[i >> 1] = fmaxf(top[i >> 1], x);
      }
  }
  int e_new = st.e;
#pragma unroll
  for (int b = 0; b < TB; ++b) e_new = max(e_new, (int)(__float_as_uint(vs[b]) >> 23));
  const float grown = e_new == st.e ? 1.f : e_new - st.e > 126 ? 0.f : __uint_as_float((uint32_t)(127 - (e_new - st.e)) << 23);
  float neg_m[2], turn[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
    top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
    const float m = fmaxf(st.m[i], top[i]);
    const float alpha = m == st.m[i] ? 1.f : ex2(st.m[i] - m);
    neg_m[i] = m == -CUDART_INF_F ? 0.f : -m;
    st.m[i] = m;
    st.l[i] *= alpha;
    turn[i] = alpha * grown;
  }
  if (__any_sync(0xffffffffu, turn[0] != 1.f || turn[1] != 1.f)) {
#pragma unroll
    for (int n = 0; n < S::NT; ++n) {
      st.o[n][0] *= turn[0], st.o[n][1] *= turn[0];
      st.o[n][2] *= turn[1], st.o[n][3] *= turn[1];
    }
  }
  st.e = e_new;
#pragma unroll
  for (int b = 0; b < TB; ++b) {
    // 2^15 times the scale over the largest: the probabilities' factor (zero where the scale is less than 2^-126 of the largest)
    const int down = e_new - (int)(__float_as_uint(vs[b]) >> 23);
    const float f = down > 126 ? 0.f : __uint_as_float((uint32_t)(127 + 15 - down) << 23);
    uint32_t hi[4], lo[4], sees[4];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = ex2(s[2 * b + half][i] + neg_m[i >> 1]);
        st.l[i >> 1] += x;
        w[i] = x * f;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        hi[2 * half + i] = pack_half(w[2 * i], w[2 * i + 1]);
        if constexpr (F32) lo[2 * half + i] = rest_half(w[2 * i], w[2 * i + 1], hi[2 * half + i]);
      }
    }
    uint32_t v[4][DH / 32];
#pragma unroll
    for (int i = 0; i < 4; ++i) load_words<DH / 32>(v_at(b) + (c + 4 * i) * DH + r * (DH / 8), v[i]);
    // Where a row does not see every key, a value that is NaN (of a token it does not see, or of whatever lies behind the last key) must not
    // reach it: 0 * NaN is NaN.  Such codes are counted row by row over the keys that the row does see, and taken out of the product.
    bool nan = false;
    if (!whole) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < DH / 32; ++n) nan |= __vcmpeq4(v[i][n] & 0x7F7F7F7Fu, 0x7F7F7F7Fu) != 0u;
      nan = __any_sync(0xffffffffu, nan);
      if (nan) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            sees[2 * half + i] = (s[2 * b + half][2 * i] == -CUDART_INF_F ? 0u : 0x3C00u) |
                                 (s[2 * b + half][2 * i + 1] == -CUDART_INF_F ? 0u : 0x3C000000u);
      }
    }
#pragma unroll
    for (int n = 0; n < DH / 32; ++n) {
      if (!whole && nan) {
        uint32_t bad[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          bad[i] = __vcmpeq4(v[i][n] & 0x7F7F7F7Fu, 0x7F7F7F7Fu);
          v[i][n] &= ~bad[i];
          bad[i] &= 0x38383838u;  // the code of 1
        }
        const uint32_t x[2] = {__byte_perm(bad[0], bad[1], 0x5140), __byte_perm(bad[0], bad[1], 0x7362)};
        const uint32_t y[2] = {__byte_perm(bad[2], bad[3], 0x5140), __byte_perm(bad[2], bad[3], 0x7362)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float count[4] = {0.f, 0.f, 0.f, 0.f};
          mma16816(count, sees[0], sees[1], sees[2], sees[3], decode2((uint16_t)(x[i >> 1] >> (16 * (i & 1)))),
                   decode2((uint16_t)(y[i >> 1] >> (16 * (i & 1)))));
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (count[j] > 0.f) st.o[4 * n + i][j] = CUDART_NAN_F;
        }
      }
      const uint32_t x[2] = {__byte_perm(v[0][n], v[1][n], 0x5140), __byte_perm(v[0][n], v[1][n], 0x7362)};
      const uint32_t y[2] = {__byte_perm(v[2][n], v[3][n], 0x5140), __byte_perm(v[2][n], v[3][n], 0x7362)};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t b0 = decode2((uint16_t)(x[i >> 1] >> (16 * (i & 1)))), b1 = decode2((uint16_t)(y[i >> 1] >> (16 * (i & 1))));
        mma16816(st.o[4 * n + i], hi[0], hi[1], hi[2], hi[3], b0, b1);
        if constexpr (F32) mma16816(st.o[4 * n + i], lo[0], lo[1], lo[2], lo[3], b0, b1);
      }
    }
  }
}

template <bool F32>
__device__ __forceinline__ void store4(void* out, size_t at, float a, float b, float c, float d) {
  if constexpr (F32)
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + at) = make_float4(a, b, c, d);
  else {
    const __nv_bfloat162 x = __floats2bfloat162_rn(a, b), y = __floats2bfloat162_rn(c, d);
    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(out) + at) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  }
}

// Where row `row` of the work's rows lies in the output.
__device__ __forceinline__ size_t out_at(const AttnParams8& p, const Work& w, int row) {
  const int group = p.n_heads / p.n_kv_heads, i = w.first_row + row;
  return (size_t)(w.token0 + i / group) * p.out_stride + (size_t)(w.head_kv * group + i % group) * p.head_dim;
}

template <int DH, bool F32, int WR>
struct Layout {
  using S = Shapes<DH, F32>;
  static constexpr int RB = 16 * WR, WK = 4 / WR;
  static constexpr int Q_BYTES = S::QPARTS * S::KSTEPS * 512;  // of 16 rows
  static constexpr int FACTOR = WR * Q_BYTES;
  static constexpr int ML = FACTOR + RB * 4;                   // WR 1: [4 warps][16 rows][2]
  static constexpr int O = ML + (WR == 1 ? 512 : 0);           // WR 1: [4 warps][16 rows][DH]
  static constexpr int BYTES = O + (WR == 1 ? 4 * 16 * DH * 4 : 0);
};

// grid: items, key/value heads * row blocks, parts.
template <int DH, bool F32, int WR>
__global__ __launch_bounds__(128) void kv8_attention_kernel(const AttnParams8 p) {
  using S = Shapes<DH, F32>;
  using L = Layout<DH, F32, WR>;
  constexpr int TB = S::TB;
  extern __shared__ __align__(16) uint8_t smem[];
  pdl_begin();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wr = WR == 1 ? 0 : warp, wk = WR == 1 ? warp : 0;
  const int part = blockIdx.z;
  const Work w = work_of<L::RB>(p, blockIdx.x, blockIdx.y);
  if (w.rows <= 0 || part >= max(w.active, 1)) return;
  float* factors = reinterpret_cast<float*>(smem + L::FACTOR);
  if constexpr (WR == 1)
    lay_queries<DH, F32>(p, w, 0, 4 * warp, 4, smem, factors);
  else
    lay_queries<DH, F32>(p, w, 16 * wr, 0, 16, smem + wr * L::Q_BYTES, factors + 16 * wr);
  __syncthreads();
  const int group = p.n_heads / p.n_kv_heads, r = lane >> 2, c = lane & 3;
  const uint4* q_frag = reinterpret_cast<const uint4*>(smem + wr * L::Q_BYTES);
  uint4 q_regs[S::Q_IN_REGS ? S::KSTEPS * S::QPARTS : 1];
  if constexpr (S::Q_IN_REGS) {
#pragma unroll
    for (int i = 0; i < S::KSTEPS * S::QPARTS; ++i) q_regs[i] = q_frag[i * 32 + lane];
  }
  const float factor[2] = {factors[16 * wr + r], factors[16 * wr + r + 8]};
  // rows behind the last one stand where it stands, so that they hide nothing
  const int last = w.rows - 1, row0 = 16 * wr;
  auto position = [&](int row) { return w.pos0 + (w.first_row + min(row, last)) / group; };
  const int pos[2] = {position(row0 + r), position(row0 + r + 8)};
  const int pos_lo = position(row0), pos_hi = position(row0 + 15);

  State<DH> st;
#pragma unroll
  for (int n = 0; n < S::NT; ++n) st.o[n][0] = st.o[n][1] = st.o[n][2] = st.o[n][3] = 0.f;
  st.m[0] = st.m[1] = -CUDART_INF_F;
  st.l[0] = st.l[1] = 0.f;
  st.e = 0;
  const int b0 = w.first_block + part * w.per_part, b1 = min(b0 + w.per_part, w.first_block + w.n_blocks);
  if (row0 <= last) {
    for (int t = b0 + wk * TB; t < b1; t += L::WK * TB) {
      const int key0 = t * BLOCK;
      if (key0 > pos_hi || (p.window > 0 && key0 + TB * BLOCK - 1 <= pos_lo - p.window)) continue;  // nothing in this warp's sight
      // lane b looks up block b: its page, its scales
      int page = -1, sub = 0;
      float sk = -1.f, sv = 0.f;
      if (lane < TB && t + lane < b1) {
        const int key = key0 + lane * BLOCK, entry = key / p.page_size;
        sub = key % p.page_size / BLOCK;
        if (w.slot >= 0 && w.slot < p.bt_rows && entry < p.bt_cols) page = p.block_table[(size_t)w.slot * p.bt_cols + entry];
        if (page < 0 || page >= p.n_pages) {
          atomicOr(p.status, RL_STATUS_BAD_PAGE);
          page = -1;
        } else {
          const size_t at = (((size_t)page * 2) * p.n_kv_heads + w.head_kv) * (p.page_size / BLOCK) + sub;
          sk = p.scales[at];
          sv = p.scales[at + (size_t)p.n_kv_heads * (p.page_size / BLOCK)];
        }
      }
      const bool there = __all_sync(0xffffffffu, lane >= TB || page >= 0);
      const uint8_t* kp[TB];
      float ks[TB], vs[TB];
#pragma unroll
      for (int b = 0; b < TB; ++b) {
        const int pg = max(__shfl_sync(0xffffffffu, page, b), 0), sb = __shfl_sync(0xffffffffu, sub, b);
        kp[b] = p.pool + ((((size_t)pg * 2) * p.n_kv_heads + w.head_kv) * p.page_size + sb * BLOCK) * DH;
        ks[b] = __shfl_sync(0xffffffffu, sk, b);
        vs[b] = __shfl_sync(0xffffffffu, sv, b);
      }
      const bool whole = there && key0 + TB * BLOCK - 1 <= pos_lo && (p.window <= 0 || key0 > pos_hi - p.window);
      const size_t to_values = (size_t)p.n_kv_heads * p.page_size * DH;
      take_tile<DH, F32>(st, q_frag, q_regs, [&](int b) { return kp[b]; }, [&](int b) { return kp[b] + to_values; }, ks, vs, factor, key0, whole,
                         pos, p.window);
    }
  }
  // sums over the four lanes of a row, outputs at their own scale
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    st.l[i] += __shfl_xor_sync(0xffffffffu, st.l[i], 1);
    st.l[i] += __shfl_xor_sync(0xffffffffu, st.l[i], 2);
  }
  const float unit = __uint_as_float((uint32_t)st.e << 23) * 3.0517578125e-05f;  // 2^(e - 127) * 2^-15
  const bool direct = w.active <= 1;
  const size_t part_row = (((size_t)blockIdx.x * gridDim.y + blockIdx.y) * p.parts + part) * L::RB;
  if constexpr (WR == 1) {
    float* ml = reinterpret_cast<float*>(smem + L::ML);
    float* os = reinterpret_cast<float*>(smem + L::O);
    if (c == 0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ml[(warp * 16 + r + 8 * i) * 2] = st.m[i];
        ml[(warp * 16 + r + 8 * i) * 2 + 1] = st.l[i];
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = r + 8 * i;
      if (row > last) continue;
      float m = -CUDART_INF_F;
#pragma unroll
      for (int k = 0; k < 4; ++k) m = fmaxf(m, ml[(k * 16 + row) * 2]);
      const float f = m == -CUDART_INF_F ? 0.f : ex2(st.m[i] - m) * unit;
      float* o = os + (warp * 16 + row) * DH;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < S::NT; n += 4)
          *reinterpret_cast<float4*>(o + (2 * c + h) * S::NT + n) = make_float4(
              st.o[n][2 * i + h] * f, st.o[n + 1][2 * i + h] * f, st.o[n + 2][2 * i + h] * f, st.o[n + 3][2 * i + h] * f);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < w.rows * (DH / 4); i += 128) {
      const int row = i / (DH / 4), d = i % (DH / 4) * 4;
      float m = -CUDART_INF_F, l = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) m = fmaxf(m, ml[(k * 16 + row) * 2]);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float mk = ml[(k * 16 + row) * 2];
        if (mk != -CUDART_INF_F || ml[(k * 16 + row) * 2 + 1] != 0.f) l += ml[(k * 16 + row) * 2 + 1] * ex2(mk - m);
        const float4 a = *reinterpret_cast<const float4*>(os + (k * 16 + row) * DH + d);
        o.x += a.x, o.y += a.y, o.z += a.z, o.w += a.w;
      }
      if (direct) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        store4<F32>(p.out, out_at(p, w, row) + d, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
      } else {
        *reinterpret_cast<float4*>(p.part_o + (part_row + row) * DH + d) = o;
        if (d == 0) *reinterpret_cast<float2*>(p.part_ml + (part_row + row) * 2) = make_float2(m, l);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = row0 + r + 8 * i;
      if (row > last) continue;
      const float f = direct ? (st.l[i] == 0.f ? 0.f : unit / st.l[i]) : unit;
      const size_t at = direct ? out_at(p, w, row) : (part_row + row) * DH;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < S::NT; n += 4) {
          const float x[4] = {st.o[n][2 * i + h] * f, st.o[n + 1][2 * i + h] * f, st.o[n + 2][2 * i + h] * f, st.o[n + 3][2 * i + h] * f};
          if (direct)
            store4<F32>(p.out, at + (2 * c + h) * S::NT + n, x[0], x[1], x[2], x[3]);
          else
            *reinterpret_cast<float4*>(p.part_o + at + (2 * c + h) * S::NT + n) = make_float4(x[0], x[1], x[2], x[3]);
        }
      if (!direct && c == 0) *reinterpret_cast<float2*>(p.part_ml + (part_row + row) * 2) = make_float2(st.m[i], st.l[i]);
    }
  }
}

// Joins the parts of an item's keys, in the order of the keys: m = max m_k, o = sum o_k 2^(m_k - m) / sum l_k 2^(m_k - m).
// grid: items, key/value heads * row blocks.
template <bool F32, int WR>
__global__ __launch_bounds__(128) void kv8_join_kernel(const AttnParams8 p) {
  pdl_begin();
  const Work w = work_of<16 * WR>(p, blockIdx.x, blockIdx.y);
  if (w.rows <= 0 || w.active <= 1) return;
  const size_t first = (((size_t)blockIdx.x * gridDim.y + blockIdx.y) * p.parts) * (16 * WR);
  const int quads = p.head_dim / 4;
  for (int i = threadIdx.x; i < w.rows * quads; i += 128) {
    const int row = i / quads, d = i % quads * 4;
    float m = -CUDART_INF_F, l = 0.f;
    for (int k = 0; k < w.active; ++k) m = fmaxf(m, p.part_ml[(first + (size_t)k * (16 * WR) + row) * 2]);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < w.active; ++k) {
      const size_t at = first + (size_t)k * (16 * WR) + row;
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + at * 2);
      const float f = m == -CUDART_INF_F ? (ml.y == 0.f ? 0.f : ml.y) : ex2(ml.x - m);
      const float4 a = *reinterpret_cast<const float4*>(p.part_o + at * p.head_dim + d);
      l += ml.y * f;
      o.x += a.x * f, o.y += a.y * f, o.z += a.z * f, o.w += a.w * f;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    store4<F32>(p.out, out_at(p, w, row) + d, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  }
}

template <int DH, bool F32, int WR>
int launch_attention(const AttnParams8& p, int n_items, cudaStream_t stream) {
  using L = Layout<DH, F32, WR>;
  const auto kernel = kv8_attention_kernel<DH, F32, WR>;
  if (L::BYTES > 48 * 1024) {
    const int rc = (int)note_launch(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::BYTES));
    if (rc != 0) return take_launch_error();
  }
  const int y = p.n_kv_heads * p.row_blocks;
  launch_pdl(kernel, dim3(n_items, y, p.parts), dim3(128), L::BYTES, stream, p);
  if (p.parts > 1) launch_pdl(kv8_join_kernel<F32, WR>, dim3(n_items, y), dim3(128), 0, stream, p);
  return 0;
}

// Heads of 32 to 256 in steps of 32; wr: 1 or 4 warps along the rows.
template <bool F32>
int dispatch_attention8(const AttnParams8& p, int n_items, int wr, cudaStream_t stream) {
  switch (p.head_dim) {
#define CASE(D) \
  case D:       \
    return wr == 1 ? launch_attention<D, F32, 1>(p, n_items, stream) : launch_attention<D, F32, 4>(p, n_items, stream);
    CASE(32) CASE(64) CASE(96) CASE(128) CASE(160) CASE(192) CASE(224) CASE(256)
#undef CASE
  }
  return -2;
}

int attention8_f32(const AttnParams8& p, int n_items, int wr, cudaStream_t stream);
int attention8_bf16(const AttnParams8& p, int n_items, int wr, cudaStream_t stream);

}  // namespace kv8
}  // namespace rl
