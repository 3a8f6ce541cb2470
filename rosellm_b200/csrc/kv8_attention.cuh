// Attention over the 8-bit cache on mma.sync (kv8.cuh has the format): the function of attention_kernels.cuh with keys and values
// code * scale.
//
// A block of threads takes up to 8 * NR * WR rows: the queries of one item (a decoded token, or up to 64 queries of a prompt portion) times
// the heads that share one key/value head, so that grouped heads read each key once.  Its four warps are WR along the rows times 4 / WR along the
// keys; the keys of an item may besides be cut into parts over blocks of the grid, whose results a second kernel joins.
//
// Keys stand along the long side of the products, S^T = K Q^T and O^T = V^T P^T, so that a decoded token of up to eight heads a group wastes
// none of the 16 rows of an mma.sync and a code is turned into a half once for all rows.  No operand passes through shared memory to be
// rearranged.  The inner index of S may be ordered at will, if Q and K are ordered alike: the lane of key r and inner quarter c takes the
// quarter c of its key's row as it lies, head dim / 4 consecutive bytes, each word of which is one step of 16 (Q's fragments are laid out to match,
// once).  The rows of O^T may be ordered at will: the lane r takes the consecutive bytes r * head dim / 8 ... of four keys' rows, and
// a byte permutation of two rows gives the pairs of keys that the operand wants.  Which key is which row of S^T is free too: rows 2c
// and 2c+1 are keys c and c+4, so that neighbouring lanes read neighbouring rows of V.  P^T is S^T's fragment transposed in registers (movmatrix).
//
// Scales: the 16 keys of a block share a key scale, by which their scores are multiplied.  A block of values is one inner step of P V, so its
// probabilities are multiplied by (scale / largest scale so far) * 2^15 before they are rounded to halves (probabilities down to 2^-29 keep
// all of their 11 bits: relative error 2^-11, against 2^-8 of a bfloat16 output), and the output follows the largest scale as it follows the
// maximum.  Q is brought to halves row by row with a power of two that puts its largest entry at 2^14 (a bfloat16 fits exactly,
// within 2^-28 of the row's largest); in 32 bits Q and P are two halves each, a value and what its rounding left, so that products
// are exact to 2^-22.  Sums, maxima and outputs are float32.
#pragma once
#include "kv8.cuh"
#include "tc_common.cuh"

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
  int ring;            // tiles that the ring holds
  int* status;
};

// What a block of threads works on: its rows and the keys that any of them sees.
struct Work {
  int req, head_kv, first_row, rows;  // rows: of the item and key/value head, from first_row on; 0 or less: none
  int token0, pos0;                   // token and position of the item's first query
  int first_block, n_blocks;          // blocks of 16 keys from one at a multiple of four to the last in sight
  int first_seen;                     // the first in sight
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
  w.first_seen = lo / BLOCK;
  w.first_block = w.first_seen / 4 * 4;
  w.n_blocks = hi > lo && w.rows > 0 ? (hi + BLOCK - 1) / BLOCK - w.first_block : 0;
  // parts are of whole tiles (four blocks, from a multiple of four on), so that a tile lies within a page of 64 tokens or more
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

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// An 8 x 8 matrix of halves, a row of it in four lanes, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
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

template <int DH, bool F32, int NR>
struct Shapes {
  static constexpr int KSTEPS = DH / 16;            // inner steps of K Q^T
  static constexpr int MT = DH / 16;                // row tiles of O^T
  static constexpr int QPARTS = F32 ? 2 : 1;        // halves of a query entry
  static constexpr int TB = DH <= 64 ? 4 : DH <= 128 ? 2 : 1;  // blocks of 16 keys of a tile: 4 to 8 KB of keys and values
  static constexpr bool Q_IN_REGS = KSTEPS * QPARTS * NR <= 16;
  static constexpr int Q_BYTES = NR * QPARTS * KSTEPS * 256;
  static constexpr int AT_ONCE = NR == 1 && DH <= 128 && !F32 ? 3 : NR == 1 || DH <= 160 ? 2 : 1;  // blocks of threads on an SM (registers)
};

// The queries of 8 * NR rows as the B fragments of K Q^T, in shared memory: frag[eight][part][step][lane] is that lane's two words.  Row r of
// the fragment is row `first + r` of the work; those at or beyond `rows` are zero.  `factor` [8 * NR] gets what a row's scores are multiplied
// by.  Called by a whole warp for rows r0 .. r0 + n - 1 of them.
template <int DH, bool F32, int NR>
__device__ __forceinline__ void lay_queries(const AttnParams8& p, const Work& w, int first, int r0, int n, uint8_t* frag, float* factor) {
  using S = Shapes<DH, F32, NR>;
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
      uint8_t* place = frag + ((r / 8 * S::QPARTS) * S::KSTEPS + j / 4) * 256 + ((r % 8) * 4 + c) * 8 + j % 4 * 2;
      const float v = x[k] * up;
      const __half hi = __float2half_rn(v);
      *reinterpret_cast<__half*>(place) = hi;
      if constexpr (F32) *reinterpret_cast<__half*>(place + S::KSTEPS * 256) = __float2half_rn(v - __half2float(hi));
    }
  }
}

// A warp's state over the keys it has seen: 8 * NR rows, of which a lane holds two of each eight (2c and 2c + 1, c = lane % 4).
template <int DH, int NR>
struct State {
  float o[NR][DH / 16][4];  // tile i: entries [0], [1] are dim r * DH / 8 + 2 i of the two rows (r = lane / 4), [2], [3] the dim after it
  float m[NR][2], l[NR][2]; // maximum (in units of log 2) and sum; the sum is over this lane's keys only until the end
  int e;                    // o is the sum of p * v / 2^(e - 127) * 2^15; e: biased exponent of the largest value scale so far
};

// TB blocks of 16 keys at once.  k_at(b), v_at(b): where the codes of block b lie (its 16 rows in a row); ks, vs: scales; ks negative: a
// block that is not there (nothing of it is used; k_at and v_at still name readable memory).  key0: the first key's position.
// whole: every row sees every key.  pos: the lane's rows' positions.
template <int DH, bool F32, int NR, class KAt, class VAt>
__device__ __forceinline__ void take_tile(
    State<DH, NR>& st, const uint2* q_frag,
    const uint2 (&q_regs)[Shapes<DH, F32, NR>::Q_IN_REGS ? Shapes<DH, F32, NR>::KSTEPS * Shapes<DH, F32, NR>::QPARTS * NR : 1], KAt k_at, VAt v_at,
    const float (&ks)[Shapes<DH, F32, NR>::TB], const float (&vs)[Shapes<DH, F32, NR>::TB], const float (&factor)[NR][2], int key0, bool whole,
    const int (&pos)[NR][2], int window) {
  using S = Shapes<DH, F32, NR>;
  constexpr int TB = S::TB;
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int key_row = (r >> 1) + 4 * (r & 1);  // of the block: this lane's first key, and 8 more the second
  float s[TB][NR][4];
  uint32_t kw[TB][2][S::KSTEPS];
#pragma unroll
  for (int b = 0; b < TB; ++b)
#pragma unroll
    for (int half = 0; half < 2; ++half) load_words<S::KSTEPS>(k_at(b) + (8 * half + key_row) * DH + c * (DH / 4), kw[b][half]);
#pragma unroll
  for (int b = 0; b < TB; ++b)
#pragma unroll
    for (int n = 0; n < NR; ++n) s[b][n][0] = s[b][n][1] = s[b][n][2] = s[b][n][3] = 0.f;
#pragma unroll
  for (int k = 0; k < S::KSTEPS; ++k) {
    uint2 q[NR][S::QPARTS];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int qp = 0; qp < S::QPARTS; ++qp)
        q[n][qp] = S::Q_IN_REGS ? q_regs[S::Q_IN_REGS ? (n * S::QPARTS + qp) * S::KSTEPS + k : 0] : q_frag[((n * S::QPARTS + qp) * S::KSTEPS + k) * 32 + lane];
#pragma unroll
    for (int b = 0; b < TB; ++b) {
      const uint32_t a[4] = {decode2((uint16_t)kw[b][0][k]), decode2((uint16_t)kw[b][1][k]), decode2((uint16_t)(kw[b][0][k] >> 16)),
                             decode2((uint16_t)(kw[b][1][k] >> 16))};
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int qp = 0; qp < S::QPARTS; ++qp) mma16816(s[b][n], a, q[n][qp].x, q[n][qp].y);
    }
  }
  // scores in units of log 2; keys out of a row's sight at minus infinity
  float top[NR][2];
#pragma unroll
  for (int n = 0; n < NR; ++n) top[n][0] = top[n][1] = -CUDART_INF_F;
#pragma unroll
  for (int b = 0; b < TB; ++b)
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const float f[2] = {factor[n][0] * ks[b], factor[n][1] * ks[b]};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float& x = s[b][n][i];
        x *= f[i & 1];
        if (!whole) {
          const int key = key0 + b * BLOCK + key_row + 8 * (i >> 1);
          if (ks[b] < 0.f || key > pos[n][i & 1] || (window > 0 && key <= pos[n][i & 1] - window)) x = -CUDART_INF_F;
        }
        top[n][i & 1] = fmaxf(top[n][i & 1], x);
      }
    }
  int e_new = st.e;
#pragma unroll
  for (int b = 0; b < TB; ++b) e_new = max(e_new, (int)(__float_as_uint(vs[b]) >> 23));
  const float grown = e_new == st.e ? 1.f : e_new - st.e > 126 ? 0.f : __uint_as_float((uint32_t)(127 - (e_new - st.e)) << 23);
  float neg_m[NR][2], turn[NR][2];
  bool turns = false;
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float x = top[n][i];
#pragma unroll
      for (int o = 4; o < 32; o *= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
      const float m = fmaxf(st.m[n][i], x);
      const float alpha = m == st.m[n][i] ? 1.f : ex2(st.m[n][i] - m);
      neg_m[n][i] = m == -CUDART_INF_F ? 0.f : -m;
      st.m[n][i] = m;
      st.l[n][i] *= alpha;
      turn[n][i] = alpha * grown;
      turns |= turn[n][i] != 1.f;
    }
  if (__any_sync(0xffffffffu, turns)) {
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int t = 0; t < S::MT; ++t) {
        st.o[n][t][0] *= turn[n][0], st.o[n][t][1] *= turn[n][1];
        st.o[n][t][2] *= turn[n][0], st.o[n][t][3] *= turn[n][1];
      }
  }
  st.e = e_new;
#pragma unroll
  for (int b = 0; b < TB; ++b) {
    uint32_t v[4][DH / 32];  // rows c, c + 4, c + 8, c + 12 of the block: keys 2c, 2c + 1, 2c + 8, 2c + 9 of the fragment
#pragma unroll
    for (int i = 0; i < 4; ++i) load_words<DH / 32>(v_at(b) + (c + 4 * i) * DH + r * (DH / 8), v[i]);
    // 2^15 times the scale over the largest: the probabilities' factor (zero where the scale is less than 2^-126 of the largest)
    const int down = e_new - (int)(__float_as_uint(vs[b]) >> 23);
    const float f = down > 126 ? 0.f : __uint_as_float((uint32_t)(127 + 15 - down) << 23);
    uint32_t hi[NR][2], lo[NR][2];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float x[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          x[i] = ex2(s[b][n][2 * half + i] + neg_m[n][i]);
          st.l[n][i] += x[i];
          x[i] *= f;
        }
        hi[n][half] = pack_half(x[0], x[1]);
        if constexpr (F32) lo[n][half] = transpose8(rest_half(x[0], x[1], hi[n][half]));
        hi[n][half] = transpose8(hi[n][half]);
      }
    // Where a row does not see every key, a value that is NaN (of a token it does not see, or of whatever lies behind the last key) must not
    // reach it: 0 * NaN is NaN.  Such codes are counted row by row over the keys that the row does see, and taken out of the product.
    if (!whole) {
      bool nan = false;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int t = 0; t < DH / 32; ++t) nan |= __vcmpeq4(v[i][t] & 0x7F7F7F7Fu, 0x7F7F7F7Fu) != 0u;
      if (__any_sync(0xffffffffu, nan)) {
        uint32_t sees[NR][2];
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int half = 0; half < 2; ++half)
            sees[n][half] = transpose8((s[b][n][2 * half] == -CUDART_INF_F ? 0u : 0x3C00u) | (s[b][n][2 * half + 1] == -CUDART_INF_F ? 0u : 0x3C000000u));
#pragma unroll
        for (int t = 0; t < DH / 32; ++t) {
          uint32_t bad[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            bad[i] = __vcmpeq4(v[i][t] & 0x7F7F7F7Fu, 0x7F7F7F7Fu);
            v[i][t] &= ~bad[i];
            bad[i] &= 0x38383838u;  // the code of 1
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t x = __byte_perm(bad[0], bad[1], h ? 0x7362 : 0x5140), y = __byte_perm(bad[2], bad[3], h ? 0x7362 : 0x5140);
            const uint32_t a[4] = {decode2((uint16_t)x), decode2((uint16_t)(x >> 16)), decode2((uint16_t)y), decode2((uint16_t)(y >> 16))};
#pragma unroll
            for (int n = 0; n < NR; ++n) {
              float count[4] = {0.f, 0.f, 0.f, 0.f};
              mma16816(count, a, sees[n][0], sees[n][1]);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (count[i] > 0.f) st.o[n][2 * t + h][i] = CUDART_NAN_F;
            }
          }
        }
      }
    }
#pragma unroll
    for (int t = 0; t < DH / 32; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t x = __byte_perm(v[0][t], v[1][t], h ? 0x7362 : 0x5140), y = __byte_perm(v[2][t], v[3][t], h ? 0x7362 : 0x5140);
        const uint32_t a[4] = {decode2((uint16_t)x), decode2((uint16_t)(x >> 16)), decode2((uint16_t)y), decode2((uint16_t)(y >> 16))};
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          mma16816(st.o[n][2 * t + h], a, hi[n][0], hi[n][1]);
          if constexpr (F32) mma16816(st.o[n][2 * t + h], a, lo[n][0], lo[n][1]);
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

// Shared memory: barriers, the work asked for, queries, maxima and sums, outputs on their way to another warp, the ring.
template <int DH, bool F32, int NR, int WR>
struct Layout {
  using S = Shapes<DH, F32, NR>;
  static constexpr int RW = 8 * NR;                            // rows of a warp
  static constexpr int RB = RW * WR, WK = 4 / WR;              // rows of a block, warps along the keys
  static constexpr int MAX_RING = 24;
  static constexpr int FULL = 0, EMPTY = 8 * MAX_RING, ASK_FULL = 16 * MAX_RING, ASK_EMPTY = ASK_FULL + 16, ANSWER = ASK_EMPTY + 16;
  static constexpr int ABORT = ANSWER + 32;
  static constexpr int Q = 512;
  static constexpr int FACTOR = Q + WR * S::Q_BYTES;
  static constexpr int ML = FACTOR + RB * 4;                   // [WK][RB][2]
  static constexpr int O = (ML + (WK > 1 ? WK * RB * 8 : 0) + 15) / 16 * 16;  // [WK / 2][WR][rows of a warp, as its accumulators lie]
  static constexpr int RING = (O + (WK > 1 ? WK / 2 * WR * RW * DH * 4 : 0) + 127) / 128 * 128;
  static constexpr int PLANE = S::TB * BLOCK * DH;             // codes of a tile's keys, and of its values
  static constexpr int SLOT = 2 * PLANE + (S::TB == 4 ? 32 : 16);  // and 2 * TB scales
  static_assert(ABORT + 4 <= Q, "barriers and queries overlap");
};

__device__ __forceinline__ void copy_bulk(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }

// The next block of the grid that has not started yet, taken over by this one: asked for by one thread, answered in shared memory.
__device__ __forceinline__ void ask_for_work(uint32_t answer, uint32_t bar) {
  tc::mbar_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer), "r"(bar) : "memory");
}
__device__ __forceinline__ bool read_answer(uint32_t answer, int (&at)[3]) {
  uint32_t there;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 h;\n\t"
      "ld.shared.b128 h, [%4];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
      "selp.u32 %3, 1, 0, p;\n\t"
      "mov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, %1, %2, _}, h;\n\t}"
      : "=r"(at[0]), "=r"(at[1]), "=r"(at[2]), "=r"(there)
      : "r"(answer)
      : "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the place is written again by the next answer
  return there != 0;
}

// Four warps that compute and one that fetches.  grid: items, key/value heads * row blocks, parts; but a block that is done takes over
// the next one that has not started, and its fetching warp is by then ahead in that one's keys: a block of short contexts
// ends long before its loads have been worth their latency.
//
// The fetching warp copies the codes of a tile by cp.async.bulk (a copy a block and plane, or a plane where the tile lies in one
// page) and its scales by cp.async into a ring of tiles, as many as shared memory has room for beside a second block: about 64 KB an SM have
// to be on their way for the memory's bandwidth.  Pages are looked up and addresses formed for 16 blocks of keys at once, a lane a block and plane: with
// them formed tile by tile the warp took 0.37 us for a tile of 8 KB and was what everything waited for.
template <int DH, bool F32, int NR, int WR>
__global__ __launch_bounds__(160, Shapes<DH, F32, NR>::AT_ONCE) void kv8_attention_kernel(const AttnParams8 p) {
  using S = Shapes<DH, F32, NR>;
  using L = Layout<DH, F32, NR, WR>;
  constexpr int TB = S::TB, WK = L::WK;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t base = tc::smem_u32(smem);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::ABORT);
  const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);
  const uint32_t n_ring = (uint32_t)p.ring;
  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < n_ring; ++i) {
      tc::mbar_init(base + L::FULL + 8 * i, 33);  // each lane's cp.async, and one arrival with the bytes of the bulk copies
      tc::mbar_init(base + L::EMPTY + 8 * i, WR);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(base + L::ASK_FULL + 8 * i, 1);
      tc::mbar_init(base + L::ASK_EMPTY + 8 * i, 4);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncthreads();
  pdl_begin();
  int at[3] = {(int)blockIdx.x, (int)blockIdx.y, (int)blockIdx.z};
  uint32_t slot = 0, phase = 0;  // of the ring, for the next tile (of this warp's, where it computes)

  if (warp == 4) {
    bool ok = true;
    const int page_blocks = p.page_size / BLOCK;
    const bool one_copy = page_blocks % TB == 0;
    uint32_t issued = 0;
    for (uint32_t n = 0; ok; ++n) {
      const uint32_t turn = n & 1u;
      if (n >= 2) ok = tc::mbar_wait_warp(base + L::ASK_EMPTY + 8 * turn, ((n >> 1) & 1u) ^ 1u, abort_flag, p.status);
      if (!ok) break;
      if (lane == 0) ask_for_work(base + L::ANSWER + 16 * turn, base + L::ASK_FULL + 8 * turn);
      __syncwarp();
      const Work w = work_of<L::RB>(p, at[0], at[1]);
      const int part = at[2];
      if (w.rows > 0 && part < w.active) {
        const int b0 = w.first_block + part * w.per_part, b1 = min(b0 + w.per_part, w.first_block + w.n_blocks);
        const bool has_table = w.slot >= 0 && w.slot < p.bt_rows;
        const int* table = p.block_table + (size_t)(has_table ? w.slot : 0) * p.bt_cols;
        // lanes 0 to 15 bring the keys of 16 blocks in a row, the others their values; the pages of the next 16 are looked up meanwhile
        const int plane = lane >> 4, of_batch = lane & 15;
        auto look_up = [&](int b) {  // the page of block b; -1: none, -2: not wanted
          if (b >= b1 || b < w.first_seen) return -2;
          const int entry = b / page_blocks;
          return has_table && entry < p.bt_cols ? table[entry] : -1;
        };
        const uint32_t to_in_slot = (uint32_t)plane * L::PLANE + (uint32_t)(of_batch % TB) * (BLOCK * DH);
        const uint32_t scale_in_slot = 2 * L::PLANE + (uint32_t)(plane * TB + of_batch % TB) * 4;
        int ahead = look_up(b0 + of_batch);
        for (int batch = b0; batch < b1 && ok; batch += 16) {
          int page = ahead;
          ahead = look_up(batch + 16 + of_batch);
          if (page != -2 && (page < 0 || page >= p.n_pages)) {
            atomicOr(p.status, RL_STATUS_BAD_PAGE);
            page = -1;
          }
          const bool there = page >= 0;
          const int sub = (batch + of_batch) % page_blocks;
          const size_t row = ((size_t)(2 * max(page, 0) + plane)) * p.n_kv_heads + w.head_kv;
          const uint8_t* src = p.pool + (row * p.page_size + sub * BLOCK) * DH;
          const float* scale = p.scales + row * page_blocks + sub;
          const uint32_t all_there = __ballot_sync(0xffffffffu, there);
          const int n_tiles = min(16 / TB, (b1 - batch + TB - 1) / TB);
          for (int i = 0; i < n_tiles; ++i) {
            const uint32_t in_tile = (((1u << TB) - 1u) * 0x10001u) << (i * TB);  // the lanes whose blocks the tile has
            const uint32_t bar = base + L::FULL + 8 * slot, to = base + L::RING + slot * L::SLOT;
            const bool merged = one_copy && (all_there & in_tile) == in_tile;
            ok = tc::mbar_wait_warp(base + L::EMPTY + 8 * slot, phase ^ 1u, abort_flag, p.status);
            if (!ok) break;
            const bool mine = (in_tile >> lane) & 1u;
            if (mine && !there) asm volatile("st.shared.f32 [%0], %1;" ::"r"(to + scale_in_slot), "f"(plane == 0 ? -1.f : 0.f) : "memory");
            __syncwarp();
            if (lane == 0) tc::mbar_expect_tx(bar, (uint32_t)__popc(all_there & in_tile) * (BLOCK * DH));
            __syncwarp();
            if (mine && there) {
              asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + scale_in_slot), "l"(scale) : "memory");
              if (!merged)
                copy_bulk(to + to_in_slot, src, BLOCK * DH, bar);
              else if (of_batch % TB == 0)
                copy_bulk(to + to_in_slot, src, L::PLANE, bar);
            }
            asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(bar) : "memory");
            ++issued;
            if (++slot == n_ring) slot = 0, phase ^= 1u;
          }
        }
      }
      // the answer is waited for whatever happens: it is on its way into this block's shared memory
      const bool heard = tc::mbar_wait_warp(base + L::ASK_FULL + 8 * turn, (n >> 1) & 1u, abort_flag, p.status);
      if (!heard) {
        if (lane == 0) tc::mbar_wait_quiet(base + L::ASK_FULL + 8 * turn, (n >> 1) & 1u);
        ok = false;
      }
      if (!ok || !read_answer(base + L::ANSWER + 16 * turn, at)) break;
    }
    if (*abort_flag && lane == 0) {  // copies still in flight must land before the block leaves
      for (uint32_t i = issued > n_ring ? issued - n_ring : 0; i < issued; ++i) tc::mbar_wait_quiet(base + L::FULL + 8 * (i % n_ring), (i / n_ring) & 1u);
    }
    return;
  }

  const int wr = warp % WR, wk = warp / WR;
  const int group = p.n_heads / p.n_kv_heads, r = lane >> 2, c = lane & 3;
  auto meet = [&]() { asm volatile("bar.sync 1, 128;" ::: "memory"); };
  auto step = [&](uint32_t by) {
    slot += by;
    if (slot >= n_ring) slot -= n_ring, phase ^= 1u;
  };
  float* factors = reinterpret_cast<float*>(smem + L::FACTOR) + wr * L::RW;
  const uint2* q_frag = reinterpret_cast<const uint2*>(smem + L::Q + wr * S::Q_BYTES);
  // A warp that gives up a wait goes on through the barriers below without its work: the others meet it there.
  bool ok = true;
  uint32_t place = 0;  // of the ring, for the first tile of the work at hand
  for (uint32_t n = 0;; ++n) {
    const Work w = work_of<L::RB>(p, at[0], at[1]);
    const int part = at[2];
    if (w.rows > 0 && part < max(w.active, 1)) {
      const int last = w.rows - 1, row0 = L::RW * wr;
      lay_queries<DH, F32, NR>(p, w, row0, wk * (L::RW / WK), L::RW / WK, smem + L::Q + wr * S::Q_BYTES, factors);
      if (WK > 1)
        meet();
      else
        __syncwarp();
      uint2 q_regs[S::Q_IN_REGS ? S::KSTEPS * S::QPARTS * NR : 1];
      if constexpr (S::Q_IN_REGS) {
#pragma unroll
        for (int i = 0; i < S::KSTEPS * S::QPARTS * NR; ++i) q_regs[i] = q_frag[i * 32 + lane];
      }
      // rows behind the last one stand where it stands, so that they hide nothing
      auto position = [&](int row) { return w.pos0 + (w.first_row + min(row, last)) / group; };
      State<DH, NR> st;
      float factor[NR][2];
      int pos[NR][2];
#pragma unroll
      for (int j = 0; j < NR; ++j) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          factor[j][i] = factors[8 * j + 2 * c + i];
          pos[j][i] = position(row0 + 8 * j + 2 * c + i);
          st.m[j][i] = -CUDART_INF_F;
          st.l[j][i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < S::MT; ++i) st.o[j][i][0] = st.o[j][i][1] = st.o[j][i][2] = st.o[j][i][3] = 0.f;
      }
      st.e = 0;
      const int pos_lo = position(row0), pos_hi = position(row0 + L::RW - 1);
      const int b0 = w.first_block + part * w.per_part, b1 = min(b0 + w.per_part, w.first_block + w.n_blocks);
      const int n_tiles = part < w.active ? (b1 - b0 + TB - 1) / TB : 0;
      slot = (place + (uint32_t)wk) % n_ring, phase = ((place + (uint32_t)wk) / n_ring) & 1u;
      for (int i = wk; i < n_tiles && ok; i += WK) {
        ok = tc::mbar_wait_warp(base + L::FULL + 8 * slot, phase, abort_flag, p.status);
        if (!ok) break;
        const int key0 = (b0 + i * TB) * BLOCK;
        if (row0 <= last && key0 <= pos_hi && !(p.window > 0 && key0 + TB * BLOCK - 1 <= pos_lo - p.window)) {
          const uint8_t* codes = smem + L::RING + slot * L::SLOT;
          const float* scales = reinterpret_cast<const float*>(codes + 2 * L::PLANE);
          float ks[TB], vs[TB];
          bool there = true;
#pragma unroll
          for (int b = 0; b < TB; ++b) ks[b] = scales[b], vs[b] = scales[TB + b], there = there && ks[b] >= 0.f;
          const bool whole = there && key0 + TB * BLOCK - 1 <= pos_lo && (p.window <= 0 || key0 > pos_hi - p.window);
          take_tile<DH, F32, NR>(st, q_frag, q_regs, [&](int b) { return codes + b * (BLOCK * DH); },
                                 [&](int b) { return codes + L::PLANE + b * (BLOCK * DH); }, ks, vs, factor, key0, whole, pos, p.window);
        }
        __syncwarp();
        if (lane == 0) arrive(base + L::EMPTY + 8 * slot);
        step(WK);
      }
      place += (uint32_t)n_tiles;

      // what brings the output to its own scale, 2^(e - 127) * 2^-15, and to the maximum of all warps; sums over the eight lanes of a row
      const float own_unit = __uint_as_float((uint32_t)st.e << 23) * 3.0517578125e-05f;
      float unit[NR][2], l[NR][2], m[NR][2];
#pragma unroll
      for (int j = 0; j < NR; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          l[j][i] = st.l[j][i], m[j][i] = st.m[j][i], unit[j][i] = own_unit;
#pragma unroll
          for (int o = 4; o < 32; o *= 2) l[j][i] += __shfl_xor_sync(0xffffffffu, l[j][i], o);
        }
      if constexpr (WK > 1) {
        float* ml = reinterpret_cast<float*>(smem + L::ML) + row0 * 2;
        if (r == 0) {
#pragma unroll
          for (int j = 0; j < NR; ++j)
            *reinterpret_cast<float4*>(ml + (wk * L::RB + 8 * j + 2 * c) * 2) = make_float4(m[j][0], l[j][0], m[j][1], l[j][1]);
        }
        meet();
#pragma unroll
        for (int j = 0; j < NR; ++j) {
          float4 x[WK];  // maximum and sum of the two rows, warp by warp
#pragma unroll
          for (int k = 0; k < WK; ++k) x[k] = *reinterpret_cast<const float4*>(ml + (k * L::RB + 8 * j + 2 * c) * 2);
#pragma unroll
          for (int k = 0; k < WK; ++k) m[j][0] = fmaxf(m[j][0], x[k].x), m[j][1] = fmaxf(m[j][1], x[k].z);
          const float to[2] = {m[j][0] == -CUDART_INF_F ? 0.f : m[j][0], m[j][1] == -CUDART_INF_F ? 0.f : m[j][1]};
          l[j][0] = l[j][1] = 0.f;
#pragma unroll
          for (int k = 0; k < WK; ++k) l[j][0] += x[k].y * ex2(x[k].x - to[0]), l[j][1] += x[k].w * ex2(x[k].z - to[1]);
          unit[j][0] *= ex2(st.m[j][0] - to[0]), unit[j][1] *= ex2(st.m[j][1] - to[1]);
#pragma unroll
          for (int t = 0; t < S::MT; ++t) {
            st.o[j][t][0] *= unit[j][0], st.o[j][t][1] *= unit[j][1];
            st.o[j][t][2] *= unit[j][0], st.o[j][t][3] *= unit[j][1];
          }
          unit[j][0] = unit[j][1] = 1.f;
        }
        // half of the warps hand their outputs to the other half, twice: the second time in the place that the giver has read itself
#pragma unroll
        for (int half = WK / 2; half >= 1; half /= 2) {
          const int region = half == WK / 2 ? (wk % half) : 1;
          float4* there = reinterpret_cast<float4*>(smem + L::O + (region * WR + wr) * (L::RW * DH * 4)) + lane;
          if (wk >= half && wk < 2 * half) {
#pragma unroll
            for (int j = 0; j < NR; ++j)
#pragma unroll
              for (int t = 0; t < S::MT; ++t) there[(j * S::MT + t) * 32] = make_float4(st.o[j][t][0], st.o[j][t][1], st.o[j][t][2], st.o[j][t][3]);
          }
          meet();
          if (wk < half) {
#pragma unroll
            for (int j = 0; j < NR; ++j)
#pragma unroll
              for (int t = 0; t < S::MT; ++t) {
                const float4 x = there[(j * S::MT + t) * 32];
                st.o[j][t][0] += x.x, st.o[j][t][1] += x.y, st.o[j][t][2] += x.z, st.o[j][t][3] += x.w;
              }
          }
        }
      }
      if (wk == 0 && ok) {
        const bool direct = w.active <= 1;
        const size_t part_row = (((size_t)at[0] * gridDim.y + at[1]) * p.parts + part) * L::RB;
#pragma unroll
        for (int j = 0; j < NR; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int row = row0 + 8 * j + 2 * c + i;
            if (row > last) continue;
            const float f = direct ? (l[j][i] == 0.f ? 0.f : unit[j][i] / l[j][i]) : unit[j][i];
            const size_t to = (direct ? out_at(p, w, row) : (part_row + row) * DH) + r * (DH / 8);
#pragma unroll
            for (int t = 0; t < S::MT; t += 2) {
              const float x[4] = {st.o[j][t][i] * f, st.o[j][t][2 + i] * f, st.o[j][t + 1][i] * f, st.o[j][t + 1][2 + i] * f};
              if (direct)
                store4<F32>(p.out, to + 2 * t, x[0], x[1], x[2], x[3]);
              else
                *reinterpret_cast<float4*>(p.part_o + to + 2 * t) = make_float4(x[0], x[1], x[2], x[3]);
            }
            if (!direct && r == 0) *reinterpret_cast<float2*>(p.part_ml + (part_row + row) * 2) = make_float2(m[j][i], l[j][i]);
          }
      }
    }
    const uint32_t turn = n & 1u;
    if (!tc::mbar_wait_warp(base + L::ASK_FULL + 8 * turn, (n >> 1) & 1u, abort_flag, p.status)) break;
    const bool more = read_answer(base + L::ANSWER + 16 * turn, at);
    __syncwarp();
    if (lane == 0) arrive(base + L::ASK_EMPTY + 8 * turn);
    if (!more) break;
  }
}

// Joins the parts of an item's keys, in the order of the keys: m = max m_k, o = sum o_k 2^(m_k - m) / sum l_k 2^(m_k - m).
// grid: items, key/value heads * row blocks.
template <bool F32, int RB>
__global__ __launch_bounds__(128) void kv8_join_kernel(const AttnParams8 p) {
  pdl_begin();
  const Work w = work_of<RB>(p, blockIdx.x, blockIdx.y);
  if (w.rows <= 0 || w.active <= 1) return;
  const size_t first = (((size_t)blockIdx.x * gridDim.y + blockIdx.y) * p.parts) * RB;
  const int quads = p.head_dim / 4;
  for (int i = threadIdx.x; i < w.rows * quads; i += 128) {
    const int row = i / quads, d = i % quads * 4;
    float m = -CUDART_INF_F, l = 0.f;
    for (int k = 0; k < w.active; ++k) m = fmaxf(m, p.part_ml[(first + (size_t)k * RB + row) * 2]);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < w.active; ++k) {
      const size_t at = first + (size_t)k * RB + row;
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

template <int DH, bool F32, int NR, int WR>
int launch_attention(AttnParams8 p, int n_items, cudaStream_t stream) {
  using L = Layout<DH, F32, NR, WR>;
  const auto kernel = kv8_attention_kernel<DH, F32, NR, WR>;
  // The ring: what a block's share of an SM's shared memory (228 KB, 1 KB a block kept by the system) leaves, at most the tiles that a part
  // has.  A multiple of the warps along the keys: a place of the ring then belongs to one of them for good.  Were it to change
  // hands, a warp could ask for the second filling of a place whose first is still on its way to another warp, and the barrier's parity, which
  // tells two fillings apart and not three, would say that it is there.  (From one work to the next a place may change hands: the
  // warps have met in between, all of the first's fillings used.)
  constexpr int SHARE = (L::S::AT_ONCE == 3 ? 75 : L::S::AT_ONCE == 2 ? 113 : 200) * 1024;
  constexpr int ROOM = (SHARE - L::RING) / L::SLOT, MOST = (ROOM < L::MAX_RING ? ROOM : L::MAX_RING) / L::WK * L::WK;
  static_assert(MOST >= 2 * L::WK && MOST % L::WK == 0, "too few tiles");
  const int tiles = (p.chunk + L::S::TB * BLOCK - 1) / (L::S::TB * BLOCK), want = (tiles + L::WK - 1) / L::WK * L::WK;
  p.ring = want < 2 * L::WK ? 2 * L::WK : want < MOST ? want : MOST;
  const int bytes = L::RING + p.ring * L::SLOT;
  if (bytes > 48 * 1024) {
    const int rc = (int)note_launch(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::RING + MOST * L::SLOT));
    if (rc != 0) return take_launch_error();
  }
  const int y = p.n_kv_heads * p.row_blocks;
  const dim3 grid(n_items, y, p.parts);
  if (bytes > 48 * 1024)
    launch_pdl_all_shared(kernel, grid, dim3(160), bytes, stream, p);
  else
    launch_pdl(kernel, grid, dim3(160), bytes, stream, p);
  if (p.parts > 1) launch_pdl(kv8_join_kernel<F32, L::RB>, dim3(n_items, y), dim3(128), 0, stream, p);
  return 0;
}

// Heads of 32 to 256 in steps of 32; rows: of a block of threads, 8, 16, 32 or 64.
template <bool F32>
int dispatch_attention8(const AttnParams8& p, int n_items, int rows, cudaStream_t stream) {
  switch (p.head_dim) {
#define CASE(D)                                                                 \
  case D:                                                                       \
    return rows == 8    ? launch_attention<D, F32, 1, 1>(p, n_items, stream)    \
           : rows == 16 ? launch_attention<D, F32, 2, 1>(p, n_items, stream)    \
           : rows == 32 ? launch_attention<D, F32, 2, 2>(p, n_items, stream)    \
                        : launch_attention<D, F32, 2, 4>(p, n_items, stream);
    CASE(32) CASE(64) CASE(96) CASE(128) CASE(160) CASE(192) CASE(224) CASE(256)
#undef CASE
  }
  return -2;
}

int attention8_f32(const AttnParams8& p, int n_items, int rows, cudaStream_t stream);
int attention8_bf16(const AttnParams8& p, int n_items, int rows, cudaStream_t stream);

}  // namespace kv8
}  // namespace rl
