// Attention over the 8-bit cache on mma.sync (kv8.cuh has the format): the function of attention_kernels.cuh with keys and values
// code * scale.
//
// A block of threads takes up to 8 * NR * WR rows: the queries of one item (a decoded token, or up to 64 queries of a prompt portion) times
// the heads that share one key/value head, so that grouped heads read each key once.  Its four warps are WR along the rows times 4 / WR along the
// keys; the keys of an item may besides be cut over blocks of the grid, whose results a second kernel joins.
//
// Keys stand along the long side of the products, S^T = K Q^T and O^T = V^T P^T, so that a decoded token of up to eight heads a group wastes
// none of the 16 rows of an mma.sync and a code is turned into a half once for all rows.  No operand passes through shared memory to be
// rearranged.  The inner index of S may be ordered at will, if Q and K are ordered alike: the lane of key r and inner quarter c takes the
// pieces c, c + 4, ... of 16 bytes of its key's row as they lie, each word of which is one step of 16 (Q's fragments are laid out to match,
// once).  The rows of O^T may be ordered at will: the lane r takes the consecutive bytes r * head dim / 8 ... of four keys' rows, and
// a byte permutation of two rows gives the pairs of keys that the operand wants.  Which key is which row of S^T is free too: rows 2c
// and 2c+1 are keys c and c+4, so that neighbouring lanes read neighbouring rows of V.  P^T is S^T's fragment transposed in registers (movmatrix).
//
// Scales: the 16 keys of a block share a key scale, by which their scores are multiplied.  A block of values is one inner step of P V, so its
// probabilities are multiplied by its scale.  The outputs therefore have a maximum of their own beside the softmax's: T, the largest score +
// log2(value scale) that the row has seen; probabilities enter P V as halves of 2^(score + log2 scale - T + 15).  The key that moves the output most
// thus stands at 2^15 (exactly, where it alone matters) whatever the scales are, keys down to 2^-29 of it keep all of their 11 bits (relative error
// 2^-11, against 2^-8 of a bfloat16 output), and none is off by more than 2^-40 of it.  What a row does not see has no part in T.  (Probabilities
// against the largest scale so far, which may belong to keys of no weight or out of sight, lost bits from a ratio of 2^-18 on and everything at
// 2^-40.)  In 32 bits both maxima are rounded up: all factors that follow from them are exact then.  Q is brought to halves row by row with a power
// of two that puts its largest entry at 2^14 (a bfloat16 fits exactly, within 2^-28 of the row's largest); in 32 bits Q and P are two halves each, a
// value and what its rounding left, so that products are exact to 2^-22.  Sums, maxima and outputs are float32.
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
  int row_blocks;      // blocks of rows of an item and key/value head
  int n_entries;       // items * row_blocks
  int balanced;        // 0: a unit (an entry's rows for one key/value head) a block; else all tiles of all units in equal runs
  int cost;            // balanced: what beginning a unit counts for, in tiles
  int* plan;           // a run's length, then what the entries before each entry come to for one head [n_entries + 1]
  float* part_o;       // [blocks][2][rows][head dim], results of units that a run has not the whole of
  float* part_ml;      // [blocks][2][rows][2]
  int ring, region;    // tiles that the ring holds; bytes of one warp's outputs on their way to another
  int* status;
};

// An entry: rows of an item, for any key/value head, and the keys that any of them sees.
struct Work {
  int req, first_row, rows;           // rows: of the item and a key/value head, from first_row on; 0 or less: none
  int token0, pos0;                   // token and position of the item's first query
  int first_block, n_blocks;          // blocks of 16 keys from one at a multiple of four to the last in sight
  int first_seen;                     // the first in sight
  int slot;
  // tiles of tb blocks: one where there is no key in sight (the rows get zeros all the same), none where there are no rows
  __device__ __forceinline__ int tiles(int tb) const { return rows <= 0 ? 0 : max(1, (n_blocks + tb - 1) / tb); }
};

template <int RB>
__device__ __forceinline__ Work work_of(const AttnParams8& p, int entry) {
  Work w;
  const int item = p.row_blocks == 1 ? entry : entry / p.row_blocks;
  const int group = p.n_heads / p.n_kv_heads;
  w.req = p.is_tiles ? p.items[2 * item] : p.items[item];
  const int t0 = p.is_tiles ? p.items[2 * item + 1] : 0;
  // Blocks of 128 rows of heads that stand alone take two tiles of 64 queries at once, where the list has them next to one another: the first of them both,
  // the second nothing.
  int before[2] = {-1, 0}, next[2] = {-1, 0};
  if (RB == 2 * TILE_QUERIES && group == 1 && p.is_tiles && p.row_blocks == 1) {
    if (item > 0) before[0] = p.items[2 * item - 2], before[1] = p.items[2 * item - 1];
    if (item + 1 < p.n_entries) next[0] = p.items[2 * item + 2], next[1] = p.items[2 * item + 3];
  }
  const int qs = p.q_start[w.req], q_len = p.q_start[w.req + 1] - qs, kv_len = p.kv_len[w.req];
  const bool first_half = t0 % (2 * TILE_QUERIES) == 0;
  const bool paired = first_half ? next[0] == w.req && next[1] == t0 + TILE_QUERIES : t0 % TILE_QUERIES == 0 && before[0] == w.req && before[1] == t0 - TILE_QUERIES;
  const int n_q = paired && !first_half ? 0 : min(!p.is_tiles ? 1 : paired ? 2 * TILE_QUERIES : TILE_QUERIES, q_len - t0);
  w.first_row = (entry - item * p.row_blocks) * RB;
  w.rows = min(RB, n_q * group - w.first_row);
  w.token0 = qs + t0;
  w.pos0 = kv_len - q_len + t0;
  w.slot = p.slots[w.req];
  const int q_lo = p.is_tiles ? w.first_row / group : 0, q_hi = p.is_tiles && w.rows > 0 ? (w.first_row + w.rows - 1) / group : 0;
  if (w.token0 < 0 || w.token0 + q_hi >= p.n_tokens) w.rows = 0;  // a description that does not fit the queries
  const int lo = p.window > 0 ? max(0, w.pos0 + q_lo - p.window + 1) : 0;
  const int hi = w.slot < 0 ? 0 : w.pos0 + q_hi + 1;  // padding of a fixed-size batch sees nothing
  w.first_seen = lo / BLOCK;
  w.first_block = w.first_seen / 4 * 4;  // so that a tile lies within a page of 64 tokens or more
  w.n_blocks = hi > lo && w.rows > 0 ? (hi + BLOCK - 1) / BLOCK - w.first_block : 0;
  return w;
}

// The rows of a unit: where its queries and outputs are.
struct Rows {
  int token0, pos0, first_row, rows, head_kv;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The same with results down to 2^-149.
__device__ __forceinline__ float ex2_small(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 1 / x to 2^-23, without the branches of a rounded division.
__device__ __forceinline__ float reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// d += a (hi + lo), hi and lo the halves of a 32-bit operand.  The instruction cuts its sums off, always towards zero, which adds up over a head of 256
// or a context of thousands; so its sums are of one step of 16 alone, and those are added by rounding.  Measured (relative to 64 bits, heads of
// 256, 2000 keys): 4.4e-7, in one sum 1.6e-6, summed plainly in 32 bits 1.3e-6.
__device__ __forceinline__ void add_both(float (&d)[4], const uint32_t (&a)[4], uint32_t hi0, uint32_t hi1, uint32_t lo0, uint32_t lo1) {
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  mma16816(x, a, lo0, lo1);
  mma16816(x, a, hi0, hi1);
#pragma unroll
  for (int i = 0; i < 4; ++i) d[i] += x[i];
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

// A lane's quarter of a key's row: its pieces of CHUNK bytes, four of which make a stretch of the row.  p: the first of them.
template <int DH, int CHUNK>
__device__ __forceinline__ void load_key(const uint8_t* p, uint32_t (&w)[DH / 16]) {
#pragma unroll
  for (int i = 0; i < DH / (4 * CHUNK); ++i) {
    if constexpr (CHUNK == 16) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + 64 * i);
      w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(p + 32 * i);
      w[2 * i] = v.x, w[2 * i + 1] = v.y;
    }
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
  // Q's fragments in registers, else read from shared memory step by step: with two eights of rows a head of 128 has none left for them (measured, us, in
  // registers / not: 1024 queries of 4096, 32 heads on 8, 395 / 347, 8 x 5 queries of 20001 92 / 83, 12 heads of 64 in 32 bits, 2 x 1024, 84.8 / 80.2).
  static constexpr bool Q_IN_REGS = KSTEPS * QPARTS * NR <= (NR == 1 ? 16 : 8);
  static constexpr int Q_BYTES = NR * QPARTS * KSTEPS * 256;
  static constexpr int CHUNK = DH % 64 == 0 ? 16 : 8;  // bytes of a key's row that a lane takes at once; the four lanes of a row take neighbouring ones
  static constexpr int AT_ONCE = NR == 1 && DH <= 128 && !F32 ? 3 : NR == 1 || DH <= 160 ? 2 : 1;  // blocks of threads on an SM (registers)
};

// Up to eight rows of queries as the B fragments of K Q^T, in shared memory: frag[eight][part][step][lane] is that lane's two words.  Row r of
// the fragment is row `first + r` of the unit; rows at or beyond the unit's are left as they are (nobody looks at what comes of them).
// `factor` [8 * NR] gets what a row's scores are multiplied by.  By a whole warp, rows r0 .. r0 + N - 1: loads, then what becomes of them.
template <int DH, bool F32, int NR, int N>
struct Queries {
  using S = Shapes<DH, F32, NR>;
  float x[N][DH / 32];
  __device__ __forceinline__ void load(const AttnParams8& p, const Rows& w, int first, int r0) {
    const int lane = threadIdx.x & 31, group = p.n_heads / p.n_kv_heads;
#pragma unroll
    for (int r = 0; r < N; ++r) {
      const int row = first + r0 + r;  // of the block of rows
      const int i = w.first_row + row, q = p.is_tiles ? i / group : 0, h = w.head_kv * group + i - q * group;
      const size_t at = (size_t)(w.token0 + q) * p.q_stride + (size_t)h * DH + lane;
#pragma unroll
      for (int k = 0; k < DH / 32; ++k) {
        x[r][k] = 0.f;
        if (row < w.rows) {
          if constexpr (F32)
            x[r][k] = reinterpret_cast<const float*>(p.q)[at + 32 * k];
          else
            x[r][k] = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.q)[at + 32 * k]);
        }
      }
    }
  }
  __device__ __forceinline__ void lay(const AttnParams8& p, const Rows& w, int first, int r0, uint8_t* frag, float* factor) const {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int r = r0 + n;
      if (first + r >= w.rows) break;  // (the same in all lanes)
      float top = 0.f;
#pragma unroll
      for (int k = 0; k < DH / 32; ++k) top = fmaxf(top, fabsf(x[n][k]));
      top = warp_max(top);
      // the power of two that puts the largest entry between 2^14 and 2^15, with the sign of the scale: factors are positive, and the largest score is the
      // largest product (kept within the exponents for which both factors are normal numbers)
      const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -110), 127);
      const float up = copysignf(__uint_as_float((uint32_t)(14 - e + 127) << 23), p.scale), down = __uint_as_float((uint32_t)(e - 14 + 127) << 23);
      if (lane == 0) factor[r] = down * fabsf(p.scale) * 1.4426950408889634f;
#pragma unroll
      for (int k = 0; k < DH / 32; ++k) {
        const int d = lane + 32 * k, c = d / S::CHUNK % 4, step = d / (4 * S::CHUNK) * (S::CHUNK / 4) + d % S::CHUNK / 4;
        uint8_t* place = frag + ((r / 8 * S::QPARTS) * S::KSTEPS + step) * 256 + ((r % 8) * 4 + c) * 8 + d % 4 * 2;
        const float v = x[n][k] * up;
        const __half hi = __float2half_rn(v);
        *reinterpret_cast<__half*>(place) = hi;
        if constexpr (F32) *reinterpret_cast<__half*>(place + S::KSTEPS * 256) = __float2half_rn(v - __half2float(hi));
      }
    }
  }
};

constexpr float NOTHING = -1.7e38f;  // the maximum of no score: finite, so that differences are never of two infinities

// A warp's state over the keys it has seen: 8 * NR rows, of which a lane holds two of each eight (2c and 2c + 1, c = lane % 4).
template <int DH, int NR>
struct State {
  float o[NR][DH / 16][4];  // tile i: entries [0], [1] are dim r * DH / 8 + 2 i of the two rows (r = lane / 4), [2], [3] the dim after it
  float t[NR][2];           // the largest score + log2(value scale), in units of log 2; o is the sum of 2^(score - t + 15) * v
  float to_p[NR][2];        // 2^(15 + m - t): from a probability times its value scale to what enters the product
  float m[NR][2], l[NR][2]; // maximum (in units of log 2) and sum of 2^(score - m); the sum is over this lane's keys only until the end
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < NR; ++n) {
#pragma unroll
      for (int i = 0; i < 2; ++i) t[n][i] = m[n][i] = NOTHING, l[n][i] = to_p[n][i] = 0.f;
#pragma unroll
      for (int i = 0; i < DH / 16; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    }
  }
};

// S^T = K Q^T of TB blocks of 16 keys: kw[b][half] are the lane's words of its two keys of block b.
template <int DH, bool F32, int NR>
__device__ __forceinline__ void multiply_keys(
    float (&s)[Shapes<DH, F32, NR>::TB][NR][4], const uint32_t (&kw)[Shapes<DH, F32, NR>::TB][2][DH / 16], const uint2* q_frag,
    const uint2 (&q_regs)[Shapes<DH, F32, NR>::Q_IN_REGS ? Shapes<DH, F32, NR>::KSTEPS * Shapes<DH, F32, NR>::QPARTS * NR : 1]) {
  using S = Shapes<DH, F32, NR>;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int b = 0; b < S::TB; ++b)
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
    for (int b = 0; b < S::TB; ++b) {
      const uint32_t a[4] = {decode2((uint16_t)kw[b][0][k]), decode2((uint16_t)kw[b][1][k]), decode2((uint16_t)(kw[b][0][k] >> 16)),
                             decode2((uint16_t)(kw[b][1][k] >> 16))};
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        if constexpr (F32)
          add_both(s[b][n], a, q[n][0].x, q[n][0].y, q[n][1].x, q[n][1].y);
        else
          mma16816(s[b][n], a, q[n][0].x, q[n][0].y);
      }
    }
  }
}

// The softmax's step over the scores of a tile, and O^T += V^T P^T.  ks, vs: the blocks' scales; ks negative: a block that is not there.
// v_of(b, v): the lane's words of the values of block b, rows c, c + 4, c + 8, c + 12.  sight: every row sees every key (WHOLE), all rows see the same
// (ALIKE: decoded tokens), or not; key0 is the first key's position and pos the lane's rows'.  A tile is nearly always whole, and the checks
// are as many instructions as the rest.  (One body with branches that all lanes take alike: three bodies, one a sight, were no faster.)
enum Sight { WHOLE, ALIKE, APART };
template <int DH, bool F32, int NR, class VOf>
__device__ __forceinline__ void use_scores(const Sight sight, State<DH, NR>& st, float (&s)[Shapes<DH, F32, NR>::TB][NR][4], VOf v_of,
                                           const float (&ks)[Shapes<DH, F32, NR>::TB], const float (&vs)[Shapes<DH, F32, NR>::TB],
                                           const float (&factor)[NR][2], int key0, const int (&pos)[NR][2], int window) {
  using S = Shapes<DH, F32, NR>;
  constexpr int TB = S::TB;
  const int lane = threadIdx.x & 31, r = lane >> 2;
  const int key_row = (r >> 1) + 4 * (r & 1);  // of the block: this lane's first key, and 8 more the second
  // scores in units of log 2: s * f; keys out of a row's sight at minus infinity
  float f[TB][NR][2], top[NR][2];
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int b = 0; b < TB; ++b) f[b][n][i] = factor[n][i] * ks[b];
  if (sight != WHOLE) {
#pragma unroll
    for (int b = 0; b < TB; ++b)
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int key = key0 + b * BLOCK + key_row + 8 * h;
            const bool hidden = ks[b] < 0.f || key > pos[n][i] || (window > 0 && key <= pos[n][i] - window);
            s[b][n][2 * h + i] = hidden ? -CUDART_INF_F : s[b][n][2 * h + i] * f[b][n][i];
          }
          f[b][n][i] = 1.f;
        }
  }
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      top[n][i] = NOTHING;
#pragma unroll
      for (int b = 0; b < TB; ++b) top[n][i] = fmaxf(top[n][i], fmaxf(s[b][n][i], s[b][n][2 + i]) * f[b][n][i]);
    }
  // log2 of a value scale (its exponent as the low bits of a float); from 2^-111 on, so that 2^(15 + m - t) is a float
  auto log_of = [](float v) { return fmaxf(__uint_as_float(0x4B000000u | (__float_as_uint(v) >> 23)) - 8388735.f, -111.f); };
  float scale_top = vs[0];
#pragma unroll
  for (int b = 1; b < TB; ++b) scale_top = fmaxf(scale_top, vs[b]);
  const float log_top = log_of(scale_top);
  bool grown = false;
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int o = 4; o < 32; o *= 2) top[n][i] = fmaxf(top[n][i], __shfl_xor_sync(0xffffffffu, top[n][i], o));
      // (the largest score and the largest scale may be of different keys: whether t grows is looked at below)
      grown |= top[n][i] > st.m[n][i] || top[n][i] + log_top > st.t[n][i];
    }
  if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      float turn[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float t = NOTHING;
#pragma unroll
        for (int b = 0; b < TB; ++b) t = fmaxf(t, fmaxf(s[b][n][i], s[b][n][2 + i]) * f[b][n][i] + log_of(vs[b]));
#pragma unroll
        for (int o = 4; o < 32; o *= 2) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
        t = fmaxf(st.t[n][i], F32 ? ceilf(t) : t);
        const float m = fmaxf(st.m[n][i], F32 ? ceilf(top[n][i]) : top[n][i]);
        st.l[n][i] *= ex2(st.m[n][i] - m);
        turn[i] = ex2(st.t[n][i] - t);
        st.m[n][i] = m, st.t[n][i] = t;
        st.to_p[n][i] = ex2_small(15.f + (m - t));
      }
#pragma unroll
      for (int t = 0; t < S::MT; ++t) {
        st.o[n][t][0] *= turn[0], st.o[n][t][1] *= turn[1];
        st.o[n][t][2] *= turn[0], st.o[n][t][3] *= turn[1];
      }
    }
  }
#pragma unroll
  for (int b = 0; b < TB; ++b) {
    uint32_t hi[NR][2], lo[NR][2];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float x[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          x[i] = ex2(fmaf(s[b][n][2 * h + i], f[b][n][i], -st.m[n][i]));
          st.l[n][i] += x[i];
          x[i] = x[i] * vs[b] * st.to_p[n][i];  // (in this order: the two factors' product may be no float where the probability is 0)
        }
        hi[n][h] = pack_half(x[0], x[1]);
        if constexpr (F32) lo[n][h] = transpose8(rest_half(x[0], x[1], hi[n][h]));
        hi[n][h] = transpose8(hi[n][h]);
      }
    uint32_t v[4][DH / 32];
    v_of(b, v);
    // Where a row does not see every key, a value that is NaN (of a token it does not see, or of whatever lies behind the last key) must not
    // reach it: 0 * NaN is NaN.  Such codes are counted row by row over the keys that the row does see, and taken out of the product.
    if (sight == ALIKE) {  // (no row sees a key that its neighbour does not: the hidden keys' values are no value at all)
      const int c = lane & 3;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = key0 + b * BLOCK + c + 4 * i;
        const bool hidden = ks[b] < 0.f || key > pos[0][0] || (window > 0 && key <= pos[0][0] - window);
#pragma unroll
        for (int t = 0; t < DH / 32; ++t) v[i][t] = hidden ? 0u : v[i][t];
      }
    }
    if (sight == APART) {
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
          for (int h = 0; h < 2; ++h)
            sees[n][h] = transpose8((s[b][n][2 * h] == -CUDART_INF_F ? 0u : 0x3C00u) | (s[b][n][2 * h + 1] == -CUDART_INF_F ? 0u : 0x3C000000u));
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
          if constexpr (F32)
            add_both(st.o[n][2 * t + h], a, hi[n][0], hi[n][1], lo[n][0], lo[n][1]);
          else
            mma16816(st.o[n][2 * t + h], a, hi[n][0], hi[n][1]);
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
__device__ __forceinline__ size_t out_at(const AttnParams8& p, const Rows& w, int row) {
  const int group = p.n_heads / p.n_kv_heads, i = w.first_row + row, q = p.is_tiles ? i / group : 0;
  return (size_t)(w.token0 + q) * p.out_stride + (size_t)(w.head_kv * group + i - q * group) * p.head_dim;
}

// Shared memory: barriers, the next block asked for, segments, queries and their factors, maxima and sums, outputs on their way to another
// warp (p.region bytes each), the ring.
template <int DH, bool F32, int NR, int WR>
struct Layout {
  using S = Shapes<DH, F32, NR>;
  static constexpr int RW = 8 * NR;                            // rows of a warp
  static constexpr int RB = RW * WR, WK = 4 / WR;              // rows of a block, warps along the keys
  static constexpr int MAX_RING = 16;
  static constexpr int FULL = 0, EMPTY = 8 * MAX_RING, SEG_FULL = 16 * MAX_RING, SEG_EMPTY = SEG_FULL + 16, ASK = SEG_EMPTY + 16;
  static constexpr int ANSWER = ASK + 16, SEG = ANSWER + 16, ABORT = SEG + 64;
  static constexpr int Q = 512;
  static constexpr int AHEAD = WR == 1 ? 2 : 1;                // segments whose queries are laid out at once: by the fetching warp, ahead
  static constexpr int FACTOR = Q + AHEAD * WR * S::Q_BYTES;
  static constexpr int ML = FACTOR + AHEAD * RB * 4;           // [WK][RB][2]
  static constexpr int O = (ML + (WK > 1 ? WK * RB * 8 : 0) + 15) / 16 * 16;  // [WK / 2][WR]
  static constexpr int PLANE = S::TB * BLOCK * DH;             // codes of a tile's keys, and of its values
  static constexpr int SLOT = 2 * PLANE + (S::TB == 4 ? 32 : 16);  // and 2 * TB scales
  static_assert(ABORT + 16 <= Q, "barriers and queries overlap");
  __host__ __device__ static constexpr int ring_at(int region) { return (O + (WK > 1 ? WK / 2 * WR * region : 0) + 127) / 128 * 128; }
};

// What the fetching warp tells the others: a unit's rows and the tiles of it that are theirs.
struct Segment {
  int n_tiles;  // -1: no more
  int key0;     // the first tile's first key
  int part;     // where the result goes: -1 to the output, else to part_o
  Rows rows;
};

__device__ __forceinline__ void arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }

// The next block of the grid that has not started yet, taken over by this one: asked for by one thread, answered in shared memory.
__device__ __forceinline__ void ask_for_block(uint32_t answer, uint32_t bar) {
  tc::mbar_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer), "r"(bar) : "memory");
}
__device__ __forceinline__ bool read_answer(uint32_t answer, int& x) {
  uint32_t there, y;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 h;\n\t"
      "ld.shared.b128 h, [%3];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
      "selp.u32 %2, 1, 0, p;\n\t"
      "mov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, %1, _, _}, h;\n\t}"
      : "=r"(x), "=r"(y), "=r"(there)
      : "r"(answer)
      : "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the place is written again by the next answer
  return there != 0;
}

// Four warps that compute and one that fetches, through a ring of tiles.  Which tiles, by p.balanced:
//
// 0: grid entries x key/value heads, a unit a block; but a block that is done takes over the next one that has not started, and its
// fetching warp is by then ahead in that one's keys: a block of short contexts ends long before its loads have been worth their latency.
//
// 1: the tiles of all units in a row, and in front of each unit's the cost of beginning one, are cut into as many equal runs as blocks stand on the device
// at once (but runs of at least p.cost + 4 tiles, or of up to p.cost + 16 where there is one for each SM), whatever the lengths.  A unit that a
// run has the whole of goes to the output; of others, a run has at most two, and kv8_join_kernel joins their parts.  32 contexts of up to 16384 tokens, 8 heads of 128: 114 us in parts of 1536
// keys that blocks take over from one another, which leaves the last of them waiting for the longest; 100 so, of 85 of traffic.
// What bounds it where units are short (64 decoded tokens of 25 heads of 64 and up to 1023 keys: 40 us, 16.6 of traffic) is latency: a block takes
// 17,000 cycles for a unit of ten tiles, of which its warps compute 6,600; fifteen warps an SM issue in 29 % of the cycles.
//
// The fetching warp tells the others what comes next by a segment, two of which may be open, and lays the queries out for them (decoded tokens: the
// loads of queries, and all that hangs on the batch's description, are then as far ahead as the keys).  Codes and scales come by
// cp.async, 512 bytes of a block an instruction; pages are looked up and addresses formed for 16 blocks of keys at once, a lane a block and plane.
// With a bulk copy for every block and plane (a page may be no longer) the warp took 700 to 1000 cycles for a tile of 8 KB, about 100 a
// copy, and was what everything waited for.
template <int DH, bool F32, int NR, int WR>
__global__ __launch_bounds__(160, Shapes<DH, F32, NR>::AT_ONCE) void kv8_attention_kernel(const AttnParams8 p) {
  using S = Shapes<DH, F32, NR>;
  using L = Layout<DH, F32, NR, WR>;
  constexpr int TB = S::TB, WK = L::WK;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t base = tc::smem_u32(smem);
  const int ring_at = L::ring_at(p.region);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::ABORT);
  Segment* segments = reinterpret_cast<Segment*>(smem + L::SEG);
  static_assert(sizeof(Segment) == 32, "two segments in 64 bytes");
  const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);
  const uint32_t n_ring = (uint32_t)p.ring;
  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < n_ring; ++i) {
      tc::mbar_init(base + L::FULL + 8 * i, 33);  // each lane's copies, and one arrival for what is stored
      tc::mbar_init(base + L::EMPTY + 8 * i, WR);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(base + L::SEG_FULL + 8 * i, 1);
      tc::mbar_init(base + L::SEG_EMPTY + 8 * i, 4);
    }
    tc::mbar_init(base + L::ASK, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  pdl_begin();
  int* before = reinterpret_cast<int*>(smem + ring_at);  // balanced: what the entries before each come to for one head; the ring's place, before its first use
  if (p.balanced) {
    for (int e = threadIdx.x; e < p.n_entries; e += 160) {
      const int tiles = work_of<L::RB>(p, e).tiles(TB);
      before[e] = tiles > 0 ? p.cost + tiles : 0;
    }
    __syncthreads();
    if (warp == 0) {
      int sum = 0;
      for (int e = 0; e < p.n_entries; e += 32) {
        int x = e + lane < p.n_entries ? before[e + lane] : 0;
        const int own = x;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
          const int y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        if (e + lane < p.n_entries) before[e + lane] = sum + x - own;
        sum += __shfl_sync(0xffffffffu, x, 31);
      }
      if (lane == 0) before[p.n_entries] = sum;
    }
  }
  __syncthreads();
  uint32_t slot = 0, phase = 0;  // of the ring, for the next tile (of this warp's, where it computes)

  if (warp == 4) {
    const int page_blocks = p.page_size / BLOCK;
    const int plane = lane >> 4, of_batch = lane & 15;  // lanes 0 to 15 look after the keys of 16 blocks in a row, the others after their values
    bool ok = true;
    uint32_t told = 0;

    // tiles [i0, i1) of the entry w for head h; part as in Segment
    auto serve = [&](const Work& w, int h, int i0, int i1, int part) {
      const uint32_t turn = told & 1u;
      if (told >= 2) ok = tc::mbar_wait_warp(base + L::SEG_EMPTY + 8 * turn, ((told >> 1) & 1u) ^ 1u, abort_flag, p.status);
      if (!ok) return;
      const Rows rows{w.token0, w.pos0, w.first_row, w.rows, h};
      const int b0 = w.first_block + i0 * TB, b1 = min(w.first_block + i1 * TB, w.first_block + w.n_blocks);
      const bool has_table = w.slot < p.bt_rows;
      const int* table = p.block_table + (size_t)(has_table ? w.slot : 0) * p.bt_cols;
      auto look_up = [&](int b) {  // the page of block b, by this lane; -1: none, -2: not wanted
        if (b >= b1 || b < w.first_seen) return -2;
        const int entry = b / page_blocks;
        return has_table && entry < p.bt_cols ? table[entry] : -1;
      };
      int ahead = look_up(b0 + of_batch);  // the pages of 16 blocks are looked up while the 16 before are fetched
      Queries<DH, F32, NR, 8> queries;
      if constexpr (L::AHEAD == 2) queries.load(p, rows, 0, 0);
      const uint8_t* src = nullptr;
      const float* scale = nullptr;
      uint32_t all_there = 0;
      int i = 0, n = i1 - i0;  // tiles fetched, and all of them
      auto fetch = [&]() {     // the next tile, into its place of the ring, which is free
        const int in_batch = i % (16 / TB);
        if (in_batch == 0) {
          const int b = b0 + i * TB + of_batch;
          int page = ahead;
          ahead = look_up(b + 16);
          if (page != -2 && (page < 0 || page >= p.n_pages)) {
            atomicOr(p.status, RL_STATUS_BAD_PAGE);
            page = -1;
          }
          const int sub = b % page_blocks;
          const size_t row = ((size_t)(2 * max(page, 0) + plane)) * p.n_kv_heads + h;
          src = p.pool + (row * p.page_size + sub * BLOCK) * DH;
          scale = p.scales + row * page_blocks + sub;
          all_there = __ballot_sync(0xffffffffu, page >= 0);
        }
        const uint32_t bar = base + L::FULL + 8 * slot, to = base + ring_at + slot * L::SLOT;
        if (of_batch / TB == in_batch) {  // the lanes whose blocks the tile has
          const uint32_t at = to + 2 * L::PLANE + (uint32_t)(plane * TB + of_batch % TB) * 4;
          if ((all_there >> lane) & 1u)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(at), "l"(scale) : "memory");
          else
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(plane == 0 ? -1.f : 0.f) : "memory");
        }
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int b = 0; b < TB; ++b) {
            const int of = half * 16 + in_batch * TB + b;  // the lane that knows where
            const unsigned long long from = __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), of) + lane * 16;
            if (!((all_there >> of) & 1u)) continue;  // (the same in all lanes)
#pragma unroll
            for (int k = 0; k < DH / 32; ++k)
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + half * L::PLANE + (b * DH / 32 + k) * 512 + lane * 16), "l"(from + k * 512) : "memory");
          }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(bar) : "memory");
        __syncwarp();
        if (lane == 0) arrive(bar);  // what was stored, not copied, is seen behind this
        ++i;
        if (++slot == n_ring) slot = 0, phase ^= 1u;
      };
      // as many tiles as there is room for at once, one for each of the others, before the queries are laid out
      while (i < n && i < WK && __all_sync(0xffffffffu, tc::mbar_try_wait(base + L::EMPTY + 8 * slot, phase ^ 1u))) fetch();
      if (lane == 0) segments[turn] = Segment{n, b0 * BLOCK, part, rows};
      if constexpr (L::AHEAD == 2) {
        uint8_t* frag = smem + L::Q + turn * S::Q_BYTES;
        float* factor = reinterpret_cast<float*>(smem + L::FACTOR) + turn * L::RB;
        queries.lay(p, rows, 0, 0, frag, factor);
#pragma unroll
        for (int r0 = 8; r0 < L::RW; r0 += 8) {
          if (w.rows <= r0) break;
          queries.load(p, rows, 0, r0);
          queries.lay(p, rows, 0, r0, frag, factor);
        }
      }
      __syncwarp();
      if (lane == 0) arrive(base + L::SEG_FULL + 8 * turn);
      ++told;
      while (i < n) {
        ok = tc::mbar_wait_warp(base + L::EMPTY + 8 * slot, phase ^ 1u, abort_flag, p.status);
        if (!ok) break;
        fetch();
      }
    };

    if (p.balanced) {
      const long total = (long)before[p.n_entries] * p.n_kv_heads;  // (more than 2^31 for thousands of rows' blocks over a million tokens)
      const int blocks = (int)gridDim.x;
      const int run = (int)max((total + blocks - 1) / blocks, min(max((total + p.balanced - 1) / p.balanced, p.cost + 4L), p.cost + 16L));
      if (blockIdx.x == 0) {  // for the kernel that joins
        for (int e = lane; e <= p.n_entries; e += 32) p.plan[1 + e] = before[e];
        if (lane == 0) p.plan[0] = run;
      }
      long at = (long)blockIdx.x * run;
      const long end = min(total, at + run);
      int entry = 0;  // the last entry that begins at or before `at`
      for (int hi = p.n_entries; hi - entry > 1;) {
        const int mid = (entry + hi) >> 1;
        if ((long)before[mid] * p.n_kv_heads <= at)
          entry = mid;
        else
          hi = mid;
      }
      int rest = (int)(at - (long)before[entry] * p.n_kv_heads);  // of the entry, that earlier runs have
      __syncwarp();  // the last reading of `before`; the other warps are past it too (the ring is written from here on)
      for (; at < end && ok; ++entry) {
        const Work w = work_of<L::RB>(p, entry);
        const int tiles = w.tiles(TB);
        if (tiles == 0) continue;
        int h = rest / (p.cost + tiles), off = rest - h * (p.cost + tiles);
        rest = 0;
        for (; h < p.n_kv_heads && at < end && ok; ++h) {
          const int n = (int)min((long)(p.cost + tiles - off), end - at), i0 = max(off - p.cost, 0), i1 = max(off + n - p.cost, 0);
          if (i1 > i0) serve(w, h, i0, i1, i1 - i0 == tiles ? -1 : (int)blockIdx.x * 2 + (off >= p.cost ? 0 : 1));
          at += n;
          off = 0;
        }
      }
    } else {
      int unit = blockIdx.x;  // heads of an entry next to one another: their blocks of a page lie so too, and are read at about the same time
      for (uint32_t n = 0;; ++n) {
        __syncwarp();  // the answer before this one has been read by every lane: the next goes into the same place
        if (lane == 0) ask_for_block(base + L::ANSWER, base + L::ASK);
        __syncwarp();
        const int entry = unit / p.n_kv_heads;
        const Work w = work_of<L::RB>(p, entry);
        const int tiles = w.tiles(TB);
        if (tiles > 0 && ok) serve(w, unit - entry * p.n_kv_heads, 0, tiles, -1);
        // the answer is waited for whatever happens: it is on its way into this block's shared memory
        if (!tc::mbar_wait_warp(base + L::ASK, n & 1u, abort_flag, p.status)) {
          if (lane == 0) tc::mbar_wait_quiet(base + L::ASK, n & 1u);
          ok = false;
        }
        if (!ok || !read_answer(base + L::ANSWER, unit)) break;
      }
    }
    if (ok) {
      const uint32_t turn = told & 1u;
      if (told >= 2) ok = tc::mbar_wait_warp(base + L::SEG_EMPTY + 8 * turn, ((told >> 1) & 1u) ^ 1u, abort_flag, p.status);
      if (lane == 0 && ok) {
        segments[turn].n_tiles = -1;
        arrive(base + L::SEG_FULL + 8 * turn);
      }
    }
    if (*abort_flag) asm volatile("cp.async.wait_all;" ::: "memory");  // copies still in flight must land before the block leaves
    return;
  }

  const int wr = warp % WR, wk = warp / WR;
  const int group = p.n_heads / p.n_kv_heads, r = lane >> 2, c = lane & 3;
  auto meet = [&]() { asm volatile("bar.sync 1, 128;" ::: "memory"); };
  // A warp that gives up a wait goes on through the barriers below without its work, the others meet it there; and all four leave together, at the
  // beginning of a segment that one of them did not get.
  auto all_four = [&](bool mine) {
    uint32_t all;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbar.red.and.pred p, 1, 128, q;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(all) : "r"((uint32_t)mine) : "memory");
    return all != 0;
  };
  bool ok = true;
  uint32_t place = 0;  // of the ring, for the first tile of the segment at hand
  for (uint32_t n = 0;; ++n) {
    const uint32_t turn = n & 1u;
    const bool told = ok && tc::mbar_wait_warp(base + L::SEG_FULL + 8 * turn, (n >> 1) & 1u, abort_flag, p.status);
    if (!all_four(told)) break;
    const int4 s0 = reinterpret_cast<const int4*>(segments + turn)[0], s1 = reinterpret_cast<const int4*>(segments + turn)[1];
    const int n_tiles = s0.x, first_key = s0.y, part = s0.z;
    if (n_tiles < 0) break;
    const Rows rows{s0.w, s1.x, s1.y, s1.z, s1.w};
    const int last = rows.rows - 1, row0 = L::RW * wr;
    const uint32_t q_turn = L::AHEAD == 2 ? turn : 0u;
    uint8_t* q_at = smem + L::Q + (q_turn + wr) * S::Q_BYTES;
    float* factors = reinterpret_cast<float*>(smem + L::FACTOR) + q_turn * L::RB + wr * L::RW;
    if constexpr (L::AHEAD == 1) {
      constexpr int N = L::RW / WK < 8 ? L::RW / WK : 8;  // rows of this warp's to lay out, eight at a time
#pragma unroll
      for (int r0 = 0; r0 < L::RW / WK; r0 += N) {
        Queries<DH, F32, NR, N> queries;
        queries.load(p, rows, row0, wk * (L::RW / WK) + r0);
        queries.lay(p, rows, row0, wk * (L::RW / WK) + r0, q_at, factors);
      }
      if (WK > 1)
        meet();
      else
        __syncwarp();
    }
    const uint2* q_frag = reinterpret_cast<const uint2*>(q_at);
    uint2 q_regs[S::Q_IN_REGS ? S::KSTEPS * S::QPARTS * NR : 1];
    if constexpr (S::Q_IN_REGS) {
#pragma unroll
      for (int i = 0; i < S::KSTEPS * S::QPARTS * NR; ++i) q_regs[i] = q_frag[i * 32 + lane];
    }
    // rows behind the last one stand where it stands, so that they hide nothing
    auto position = [&](int row) { return p.is_tiles ? rows.pos0 + (rows.first_row + min(row, last)) / group : rows.pos0; };
    State<DH, NR> st;
    st.clear();
    float factor[NR][2];
    int pos[NR][2];
#pragma unroll
    for (int j = 0; j < NR; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = row0 + 8 * j + 2 * c + i;
        factor[j][i] = row <= last ? factors[8 * j + 2 * c + i] : 0.f;  // (rows behind the last one: scores that never grow)
        pos[j][i] = position(row);
      }
    const int pos_lo = position(row0), pos_hi = position(row0 + L::RW - 1);
    slot = (place + (uint32_t)wk) % n_ring, phase = ((place + (uint32_t)wk) / n_ring) & 1u;
    for (int i = wk; i < n_tiles && ok; i += WK) {
      ok = tc::mbar_wait_warp(base + L::FULL + 8 * slot, phase, abort_flag, p.status);
      if (!ok) break;
      const int key0 = first_key + i * TB * BLOCK;
      if (row0 <= last && key0 <= pos_hi && !(p.window > 0 && key0 + TB * BLOCK - 1 <= pos_lo - p.window)) {
        const uint8_t* codes = smem + ring_at + slot * L::SLOT;
        const float* scales = reinterpret_cast<const float*>(codes + 2 * L::PLANE);
        float ks[TB], vs[TB];
        bool there = true;
#pragma unroll
        for (int b = 0; b < TB; ++b) ks[b] = scales[b], vs[b] = scales[TB + b], there = there && ks[b] >= 0.f;
        const bool whole = there && key0 + TB * BLOCK - 1 <= pos_lo && (p.window <= 0 || key0 > pos_hi - p.window);
        uint32_t kw[TB][2][S::KSTEPS];
#pragma unroll
        for (int b = 0; b < TB; ++b)
#pragma unroll
          for (int h = 0; h < 2; ++h) load_key<DH, S::CHUNK>(codes + (b * BLOCK + 8 * h + (r >> 1) + 4 * (r & 1)) * DH + c * S::CHUNK, kw[b][h]);
        float s[TB][NR][4];
        multiply_keys<DH, F32, NR>(s, kw, q_frag, q_regs);
        auto v_of = [&](int b, uint32_t(&v)[4][DH / 32]) {
#pragma unroll
          for (int j = 0; j < 4; ++j) load_words<DH / 32>(codes + L::PLANE + (b * BLOCK + c + 4 * j) * DH + r * (DH / 8), v[j]);
        };
        use_scores<DH, F32, NR>(whole ? WHOLE : pos_lo == pos_hi ? ALIKE : APART, st, s, v_of, ks, vs, factor, key0, pos, p.window);
      }
      __syncwarp();
      if (lane == 0) arrive(base + L::EMPTY + 8 * slot);
      slot += WK;
      if (slot >= n_ring) slot -= n_ring, phase ^= 1u;
    }
    place += (uint32_t)n_tiles;

    // sums over the eight lanes of a row, and over the warps along the keys; outputs as means of what this block has seen (a mean is no larger than the
    // largest value, a sum may be)
    float l[NR][2], m[NR][2];
#pragma unroll
    for (int j = 0; j < NR; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        m[j][i] = st.m[j][i], l[j][i] = st.l[j][i];
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
        l[j][0] = l[j][1] = 0.f;
#pragma unroll
        for (int k = 0; k < WK; ++k) l[j][0] += x[k].y * ex2(x[k].x - m[j][0]), l[j][1] += x[k].w * ex2(x[k].z - m[j][1]);
      }
    }
#pragma unroll
    for (int j = 0; j < NR; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // (2^-15 / l and 2^(t - m) one after the other: their product may be too small)
        const float inv = l[j][i] == 0.f ? 0.f : 3.0517578125e-05f * reciprocal(l[j][i]), up = ex2(st.t[j][i] - m[j][i]);
#pragma unroll
        for (int t = 0; t < S::MT; ++t) {
          st.o[j][t][i] = st.o[j][t][i] * inv * up;
          st.o[j][t][2 + i] = st.o[j][t][2 + i] * inv * up;
        }
      }
    if constexpr (WK > 1) {
      // Half of the warps hand their outputs to the other half, twice: the second time in the place that the giver has read itself.  A lane has rows
      // 2c and 2c + 1 of each eight: where a block never has more than two (or four, six), only lanes of c = 0 (1, 2) have any.
      const int columns = WR == 1 && NR == 1 ? p.region / (S::MT * 16 * 8) : 4;
      const int mine = WR == 1 && NR == 1 ? r * columns + c : lane, lanes = 8 * columns;
#pragma unroll
      for (int half = WK / 2; half >= 1; half /= 2) {
        const int region = half == WK / 2 ? (wk % half) : 1;
        float4* there = reinterpret_cast<float4*>(smem + L::O + (region * WR + wr) * p.region) + mine;
        if (wk >= half && wk < 2 * half && c < columns) {
#pragma unroll
          for (int j = 0; j < NR; ++j)
#pragma unroll
            for (int t = 0; t < S::MT; ++t) there[(j * S::MT + t) * lanes] = make_float4(st.o[j][t][0], st.o[j][t][1], st.o[j][t][2], st.o[j][t][3]);
        }
        meet();
        if (wk < half && c < columns) {
#pragma unroll
          for (int j = 0; j < NR; ++j)
#pragma unroll
            for (int t = 0; t < S::MT; ++t) {
              const float4 x = there[(j * S::MT + t) * lanes];
              st.o[j][t][0] += x.x, st.o[j][t][1] += x.y, st.o[j][t][2] += x.z, st.o[j][t][3] += x.w;
            }
        }
      }
    }
    if (wk == 0 && ok) {
#pragma unroll
      for (int j = 0; j < NR; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = row0 + 8 * j + 2 * c + i;
          if (row > last) continue;
          const size_t part_row = (size_t)part * L::RB + row;
          const size_t to = (part < 0 ? out_at(p, rows, row) : part_row * DH) + r * (DH / 8);
#pragma unroll
          for (int t = 0; t < S::MT; t += 2) {
            const float x[4] = {st.o[j][t][i], st.o[j][t][2 + i], st.o[j][t + 1][i], st.o[j][t + 1][2 + i]};
            if (part < 0)
              store4<F32>(p.out, to + 2 * t, x[0], x[1], x[2], x[3]);
            else
              *reinterpret_cast<float4*>(p.part_o + to + 2 * t) = make_float4(x[0], x[1], x[2], x[3]);
          }
          if (part >= 0 && r == 0) *reinterpret_cast<float2*>(p.part_ml + part_row * 2) = make_float2(m[j][i], l[j][i]);
        }
    }
    __syncwarp();
    if (lane == 0) arrive(base + L::SEG_EMPTY + 8 * turn);
  }
}

// Joins the parts of the units that lie in several runs, in the order of the keys.  A part has the mean o_k of its values, its maximum m_k and its sum l_k:
// the whole is the mean of the means, weighed by l_k 2^(m_k - m), m = max m_k.  grid: entries, key/value heads, eights of rows.
template <bool F32, int RB>
__global__ __launch_bounds__(128) void kv8_join_kernel(const AttnParams8 p) {
  pdl_begin();
  const int run = p.plan[0], mine = p.plan[1 + blockIdx.x], cost = p.plan[2 + blockIdx.x] - mine;
  if (cost <= 0) return;
  const long begin = (long)mine * p.n_kv_heads + (long)blockIdx.y * cost + p.cost;
  const int first = (int)(begin / run), parts = (int)((begin + cost - p.cost - 1) / run) - first + 1;
  if (parts <= 1) return;
  const Work w = work_of<RB>(p, blockIdx.x);
  const Rows rows{w.token0, w.pos0, w.first_row, w.rows, (int)blockIdx.y};
  // a block's part lies in the first of its two places if its run begins among the unit's tiles, else in the second
  auto part_row = [&](int k, int row) { return ((size_t)(first + k) * 2 + ((long)(first + k) * run < begin ? 1 : 0)) * RB + row; };
  const int quads = p.head_dim / 4, row0 = blockIdx.z * 8, n_rows = min(8, w.rows - row0);
  for (int i = threadIdx.x; i < n_rows * quads; i += 128) {
    const int row = row0 + i / quads, d = i % quads * 4;
    float m = NOTHING, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);  // the mean so far
    for (int k = 0; k < parts; k += 4) {         // four parts' loads on their way at once
      float2 ml[4];
      float4 part[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const size_t at = part_row(k + j, row);
        const bool there = k + j < parts;
        ml[j] = there ? *reinterpret_cast<const float2*>(p.part_ml + at * 2) : make_float2(NOTHING, 0.f);
        part[j] = there ? *reinterpret_cast<const float4*>(p.part_o + at * p.head_dim + d) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      const float most = fmaxf(fmaxf(m, ml[0].x), fmaxf(ml[1].x, fmaxf(ml[2].x, ml[3].x)));
      float w[4], before = l * ex2(m - most);
      l = before;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = ml[j].y * ex2(ml[j].x - most), l += w[j];
      m = most;
      const float inv = l == 0.f ? 0.f : reciprocal(l);
      before *= inv;
      o.x *= before, o.y *= before, o.z *= before, o.w *= before;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float f = w[j] * inv;
        o.x += part[j].x * f, o.y += part[j].y * f, o.z += part[j].z * f, o.w += part[j].w * f;
      }
    }
    store4<F32>(p.out, out_at(p, rows, row) + d, o.x, o.y, o.z, o.w);
  }
}

// How a kernel is laid out on an SM: blocks at once, tiles of the ring, bytes of a handover region and of shared memory.
struct Fit {
  int blocks, ring, region, bytes;
};

template <int DH, bool F32, int NR, int WR>
Fit fit_of(int most_rows) {
  using L = Layout<DH, F32, NR, WR>;
  // lanes of the columns that have rows (use of `columns` in the kernel)
  const int columns = WR == 1 && NR == 1 ? ((most_rows < 8 ? most_rows : 8) + 1) / 2 : 4;
  Fit f;
  f.region = NR * L::S::MT * 16 * 8 * columns;
  // The ring: what a block's share of an SM's shared memory (228 KB, 1 KB a block kept by the system) leaves.  A multiple of the warps along the
  // keys: a place of the ring then belongs to one of them while a segment lasts.  Were it to change hands, a warp could ask for the second
  // filling of a place whose first is still on its way to another warp, and the barrier's parity, which tells two fillings apart and not
  // three, would say that it is there.  (From one segment to the next a place may change hands: the warps have met in between, all of the
  // first's fillings used.)
  for (f.blocks = L::S::AT_ONCE;; --f.blocks) {
    const int room = ((f.blocks == 3 ? 75 : f.blocks == 2 ? 113 : 200) * 1024 - L::ring_at(f.region)) / L::SLOT;
    f.ring = (room < L::MAX_RING ? room : L::MAX_RING) / L::WK * L::WK;
    if (f.ring >= 2 * L::WK || f.blocks == 1) break;
  }
  f.bytes = L::ring_at(f.region) + f.ring * L::SLOT;
  return f;
}

// fit != nullptr: nothing is launched, only the layout told.
template <int DH, bool F32, int NR, int WR>
int launch_attention(AttnParams8 p, int most_rows, int blocks, Fit* fit, cudaStream_t stream) {
  using L = Layout<DH, F32, NR, WR>;
  const Fit f = fit_of<DH, F32, NR, WR>(most_rows);
  if (f.ring < 2 * L::WK || f.bytes > 227 * 1024) return -9;  // (no head size that is taken comes here)
  if (fit != nullptr) {
    *fit = f;
    return 0;
  }
  p.ring = f.ring;
  p.region = f.region;
  p.cost = 8;  // about 2 us
  if (p.balanced && (p.n_entries + 1) * 4 > f.ring * L::SLOT) return -10;  // the ring's place holds the entries' tiles at first
  const auto kernel = kv8_attention_kernel<DH, F32, NR, WR>;
  const int rc = (int)note_launch(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, f.bytes));
  if (rc != 0) return take_launch_error();
  launch_pdl_all_shared(kernel, p.balanced ? dim3(blocks) : dim3((unsigned)p.n_entries * p.n_kv_heads), dim3(160), f.bytes, stream, p);
  if (p.balanced) launch_pdl(kv8_join_kernel<F32, L::RB>, dim3(p.n_entries, p.n_kv_heads, L::RB / 8), dim3(128), 0, stream, p);
  return 0;
}

// Heads of 32 to 256 in steps of 32; rows: of a block of threads, 8, 16, 32 or 64.
template <bool F32>
int dispatch_attention8(const AttnParams8& p, int rows, int blocks, Fit* fit, cudaStream_t stream) {
  const int most_rows = p.is_tiles ? rows : p.n_heads / p.n_kv_heads;  // that a unit can have
  switch (p.head_dim) {
#define CASE(D)                                                                               \
  case D:                                                                                     \
    return rows == 8    ? launch_attention<D, F32, 1, 1>(p, most_rows, blocks, fit, stream)  \
           : rows == 16 ? launch_attention<D, F32, 2, 1>(p, most_rows, blocks, fit, stream)  \
           : rows == 32 ? launch_attention<D, F32, 2, 2>(p, most_rows, blocks, fit, stream)  \
                        : launch_attention<D, F32, 2, 4>(p, most_rows, blocks, fit, stream);
    CASE(32) CASE(64) CASE(96) CASE(128) CASE(160) CASE(192) CASE(224) CASE(256)
#undef CASE
  }
  return -2;
}

int attention8_f32(const AttnParams8& p, int rows, int blocks, Fit* fit, cudaStream_t stream);
int attention8_bf16(const AttnParams8& p, int rows, int blocks, Fit* fit, cudaStream_t stream);

}  // namespace kv8
}  // namespace rl
