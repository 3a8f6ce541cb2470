// Attention over the 8-bit cache on tcgen05, for many rows (bfloat16, head sizes 64 and 128): the function of kv8_attention.cuh.
//
// A block of threads takes 128 rows, queries times the heads that share one key/value head, and walks their keys in tiles of 128.  Its warps:
//   0-7    bring codes from memory to registers, a tile ahead, turn them into halves (exact) and write those into the swizzled layouts that the
//          products read, keys and values apart, two stages of each;
//   8-15   softmax, two groups of four warps on alternate tiles, a thread a row: read the scores from tensor memory, write the
//          probabilities back over them as halves (head 64: beside them).  Each group has a maximum, a sum and an output of its own; they meet at the end of the unit;
//   16     issues S = Q K^T (M 128, N 128) and O += P V (P taken from tensor memory, V as it lies);
//   17     says which tiles of which unit come next.
// Tensor memory: two tiles of scores, 128 columns each, and two outputs of head dim columns.
//
// Scales as in kv8_attention.cuh: a block of 16 keys is 16 columns of the scores, so a key scale is a factor of 16 columns' exponents and a value
// scale one of their probabilities, which are held as halves of 2^(score + log2 scale - m - u).  m: the row's maximum, which follows when it has grown by
// more than 2^8; m + u goes with T there, the largest score + log2 scale that the row has seen: the output stays in tensor memory and is multiplied
// only when T would put a half above 2^15, and then T stands at 2^11.  So the key that moves the output most stands between 2^10 and 2^15, keys down to
// 2^-24 of it keep all of their 11 bits, and none is off by more than 2^-35 of it.
//
// What bounds it: 128 x 128 exponentials take 1024 cycles of an SM, the products of a tile 1024 (head 128) or 512; turning 32 KB of codes into
// halves takes 260 issue slots a scheduler.  Work is shared over the SMs in equal runs of tiles, as there.  Measured: a tile takes 3,350 cycles at
// head 128; 2048 queries of 32 heads (8 of keys) after 16,384 776 us, 0.39 of the measured rate of a product of that many operations; on mma.sync 2,608.
#pragma once
#include "kv8_attention.cuh"

namespace rl {
namespace kv8 {

constexpr int TC_ROWS = 128, TC_KEYS = 128, TC_BLOCKS = TC_KEYS / BLOCK, TC_THREADS = 576;

template <int DH>
struct TcLayout {
  static constexpr int SUBS = DH / 64;                 // stretches of 64 entries, 128 bytes of halves: a row of the swizzle
  static constexpr int SUB_BYTES = 128 * 128;          // 128 rows of one
  // tensor memory: scores at 0 and 128, outputs at 256 and 256 + DH, probabilities (64 columns) over the group's scores, or behind all where there is room
  static constexpr bool P_APART = DH == 64;
  __device__ __forceinline__ static uint32_t p_col(int g) { return P_APART ? 384u + 64u * (uint32_t)g : 128u * (uint32_t)g; }
  static constexpr int MAT = SUBS * SUB_BYTES;
  static constexpr int Q = 0, K = MAT, V = K + 2 * MAT;
  static constexpr int NAN_BITS = V + 2 * MAT;         // [stage][key][DH / 16] a bit for each value of a tile that not every row sees whole: NaN
  static constexpr int NAN_SOME = NAN_BITS + 2 * TC_KEYS * (DH / 8);  // [stage][8 warps]: whether there is one
  static constexpr int ML = NAN_SOME + 2 * 8 * 4;      // [group][128 rows] maximum, sum, u + 11, whether there is anything
  static constexpr int FACTOR = ML + 2 * 128 * 16;     // [128 rows]
  static constexpr int SEG = FACTOR + 512;             // two segments
  static constexpr int BARS = SEG + 2 * 64;
  static constexpr int BYTES = BARS + 8 * 24 + 16 + 1024;  // and room to align
};

enum TcBar { SEG_FULL = 0, SEG_EMPTY = 2, K_FULL = 4, K_EMPTY = 6, V_FULL = 8, V_EMPTY = 10, S_FULL = 12, P_READY = 14, PV_DONE = 16, Q_READY = 18, O_FREE = 19, WEIGHED = 20, TC_BARS = 22 };

__device__ __forceinline__ void mma_from_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// half x half -> float32, M 128; b_mn: B has its N dimension contiguous
__host__ __device__ constexpr uint32_t tc_instr_desc(int n, bool b_mn) {
  return (1u << 4) | (b_mn ? (1u << 16) : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// An MN-major tile, 128-byte swizzle: rows of 64 entries, groups of eight rows 1024 bytes apart, the next 64 columns a stretch of 128 rows on.
__device__ __forceinline__ uint64_t tc_desc_mn(uint32_t addr) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(128 * 128 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
               "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
__device__ __forceinline__ void tmem_store8(uint32_t at, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
               "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_load(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                 "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
                 "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_wait_load16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                 "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float m;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}
// Two float32 values as one register pair, for the instructions that take two at a time.
__device__ __forceinline__ uint64_t pair(float lo, float hi) { return (uint64_t)__float_as_uint(lo) | ((uint64_t)__float_as_uint(hi) << 32); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// What the planning warp tells the others.
struct TcSegment {
  int n_tiles;  // -1: no more
  int key0;     // the first tile's first key
  int part;     // as in Segment
  int token0, pos0, first_row, rows, head_kv;
  int slot, first_seen, end_block;  // the block table's row; blocks of 16 keys from first_seen to end_block - 1 are wanted
  int pos_lo, pos_hi;               // positions of the first and the last row
  int pad[3];
};

// Registers: 576 threads are launched with 96 each; eight warps that convert give 24 each to eight that do the softmax (8 * 72 + 8 * 120 + 2 * 96 =
// 18 * 96, two of each on every quarter of the SM).
template <int DH>
__global__ __launch_bounds__(TC_THREADS, 1) void kv8_attention_tc_kernel(const AttnParams8 p) {
  using L = TcLayout<DH>;
  extern __shared__ uint8_t tc_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)tc_smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t base = tc::smem_u32(smem);
  auto bar = [&](int which) { return base + L::BARS + 8 * (uint32_t)which; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::BARS + 8 * 24);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  TcSegment* segments = reinterpret_cast<TcSegment*>(smem + L::SEG);
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(bar(SEG_FULL + i), 1);
      tc::mbar_init(bar(SEG_EMPTY + i), 17);
      tc::mbar_init(bar(K_FULL + i), 8);
      tc::mbar_init(bar(K_EMPTY + i), 1);
      tc::mbar_init(bar(V_FULL + i), 8);
      tc::mbar_init(bar(V_EMPTY + i), 1);
      tc::mbar_init(bar(S_FULL + i), 1);
      tc::mbar_init(bar(P_READY + i), 4);
      tc::mbar_init(bar(PV_DONE + i), 1);
      tc::mbar_init(bar(WEIGHED + i), 4);
    }
    tc::mbar_init(bar(Q_READY), 8);
    tc::mbar_init(bar(O_FREE), 8);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 16) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    // Kernels behind are let in by this warp, when the block has its tensor memory: one that takes some before it waits for this kernel could otherwise
    // stand on the SM first, and each would wait for the other.
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // what the entries before each come to for one head, in the place of the first keys
  int* before = reinterpret_cast<int*>(smem + L::K);
  for (int e = threadIdx.x; e < p.n_entries; e += TC_THREADS) {
    const int tiles = work_of<TC_ROWS>(p, e).tiles(TC_BLOCKS);
    before[e] = tiles > 0 ? p.cost + tiles : 0;
  }
  __syncthreads();
  if (warp == 17) {
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
    __syncwarp();
    if (lane == 0) before[p.n_entries] = sum;
    __syncwarp();
  }
  // the run of this block, before the numbers' place is written over
  long at = 0, end = 0;
  int entry = 0, rest = 0;
  if (warp == 17) {
    const long total = (long)before[p.n_entries] * p.n_kv_heads;  // (more than 2^31 for thousands of rows' blocks over a million tokens)
    const int blocks = (int)gridDim.x;
    const int run = (int)max((total + blocks - 1) / blocks, p.cost + 1L);
    if (blockIdx.x == 0) {  // for the kernel that joins
      for (int e = lane; e <= p.n_entries; e += 32) p.plan[1 + e] = before[e];
      if (lane == 0) p.plan[0] = run;
    }
    at = (long)blockIdx.x * run;
    end = min(total, at + run);
    for (int hi = p.n_entries; hi - entry > 1;) {  // the last entry that begins at or before `at`
      const int mid = (entry + hi) >> 1;
      if ((long)before[mid] * p.n_kv_heads <= at)
        entry = mid;
      else
        hi = mid;
    }
    rest = (int)(at - (long)before[entry] * p.n_kv_heads);
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const int group = p.n_heads / p.n_kv_heads, page_blocks = p.page_size / BLOCK;
  // b / page_blocks for block numbers below 2^24 and pages of up to 256 blocks: the high half of b * (2^32 / page_blocks + 1)
  const uint32_t per_page = page_blocks > 1 ? 0xFFFFFFFFu / (uint32_t)page_blocks + 1u : 0u;
  auto page_index = [&](int b) { return per_page != 0u ? (int)__umulhi((uint32_t)b, per_page) : b; };
  auto wait = [&](int which, uint32_t parity) { return tc::mbar_wait_warp(bar(which), parity, abort_flag, p.status); };
  // The segment at hand, for the roles below; false when there is none.
  auto next_segment = [&](uint32_t n, TcSegment& s) {
    if (!wait(SEG_FULL + (int)(n & 1u), (n >> 1) & 1u)) return false;
    const int4* from = reinterpret_cast<const int4*>(segments + (n & 1u));
    const int4 a = from[0], b = from[1], c = from[2];
    s = TcSegment{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w, c.x, c.y, c.z, c.w, from[3].x, {}};
    return s.n_tiles >= 0;
  };
  auto done_with = [&](uint32_t n) {
    __syncwarp();
    if (lane == 0) arrive(bar(SEG_EMPTY + (int)(n & 1u)));
  };
  auto page_of = [&](const TcSegment& s, int b) {  // of block b; -1: none, -2: not wanted
    if (b < s.first_seen || b >= s.end_block) return -2;
    const int e = page_index(b);
    return s.slot < p.bt_rows && e < p.bt_cols ? p.block_table[(size_t)s.slot * p.bt_cols + e] : -1;
  };
  // whether every row of the block of threads sees every key of a tile
  auto is_whole = [&](const TcSegment& s, int key0) {
    return key0 + TC_KEYS - 1 <= s.pos_lo && (p.window <= 0 || key0 > s.pos_hi - p.window) && key0 >= s.first_seen * BLOCK;
  };

  if (warp < 8) {
    // ---- codes to halves ----
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;" ::: "memory");
    constexpr int PIECES = DH / 32;                    // of 16 codes, a thread, of the keys of a tile
    constexpr int APART = 256 / DH;                    // blocks of 16 keys between two of a thread's pieces
    // four neighbouring lanes take 64 codes of a key, the next four the same of the next key: eight lanes then write all of the banks
    const int t = threadIdx.x, key_in_block = t / 4 % 16, part = t % 4 + (DH == 128 ? t / 64 % 2 * 4 : 0), own_block = t / DH;
    const int to_values = p.n_kv_heads * page_blocks;  // blocks of 16 keys from a block of keys to that of its values
    const int in_block = key_in_block * DH + part * 16;
    const uint8_t* own_pool = p.pool + in_block;
    // where the piece's halves go: a row of 128 bytes a key, 16-byte pieces swizzled by the key (key % 8 is that of key_in_block)
    const uint32_t own_row = (uint32_t)(part / 4) * L::SUB_BYTES + (uint32_t)(own_block * BLOCK + key_in_block) * 128u;
    const uint32_t own_chunk = (uint32_t)((part % 4 * 2) ^ (key_in_block & 7)) << 4;
    uint4 keys[PIECES], values[PIECES];                // loaded, to be converted next
    uint32_t count = 0;
    TcSegment s;
    bool ok = true;
    for (uint32_t n = 0; ok && next_segment(n, s); ++n) {
      // lanes look after a tile's eight blocks (lane % 8): the table's entry, and from it which of the pool's blocks has its keys (of a block that
      // is not there, the first: what is read is hidden from every row, and its values are looked through for NaN)
      auto look_up = [&](int i) { return i < s.n_tiles ? page_of(s, s.key0 / BLOCK + i * TC_BLOCKS + (lane & 7)) : -2; };
      auto place_of = [&](int page, int i) {
        if (page != -2 && (page < 0 || page >= p.n_pages)) {
          atomicOr(p.status, RL_STATUS_BAD_PAGE);
          page = -1;
        }
        const int b = s.key0 / BLOCK + i * TC_BLOCKS + (lane & 7);
        return page < 0 ? 0 : (page * 2 * p.n_kv_heads + s.head_kv) * page_blocks + b - page_index(b) * page_blocks;
      };
      auto load = [&](uint4(&to)[PIECES], int place, int plane) {
#pragma unroll
        for (int j = 0; j < PIECES; ++j)
          to[j] = __ldcg(reinterpret_cast<const uint4*>(own_pool + (size_t)(uint32_t)(__shfl_sync(0xffffffffu, place, own_block + APART * j) + plane) * (BLOCK * DH)));
      };
      // 16 codes as two 16-byte pieces of a row of halves
      auto store = [&](uint32_t mat, int j, const uint4& codes) {
        const uint32_t to = mat + own_row + (uint32_t)j * (APART * BLOCK * 128);
        const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
        for (int h = 0; h < 2; ++h)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + (h ? own_chunk ^ 16u : own_chunk)), "r"(decode2((uint16_t)w[2 * h])),
                       "r"(decode2((uint16_t)(w[2 * h] >> 16))), "r"(decode2((uint16_t)w[2 * h + 1])), "r"(decode2((uint16_t)(w[2 * h + 1] >> 16)))
                       : "memory");
      };
      auto tell = [&](int which) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) arrive(bar(which));
      };
      auto convert_keys = [&](uint4(&from)[PIECES], int i) {
        const uint32_t of = count + (uint32_t)i, stage = of & 1u;
        ok = ok && wait(K_EMPTY + (int)stage, ((of >> 1) & 1u) ^ 1u);
        if (!ok) return;
#pragma unroll
        for (int j = 0; j < PIECES; ++j) store(base + L::K + stage * L::MAT, j, from[j]);
        tell(K_FULL + (int)stage);
      };
      auto convert_values = [&](uint4(&from)[PIECES], int i, bool there) {
        const uint32_t of = count + (uint32_t)i, stage = of & 1u;
        ok = ok && wait(V_EMPTY + (int)stage, ((of >> 1) & 1u) ^ 1u);
        if (!ok) return;
        if (!there || !is_whole(s, s.key0 + i * TC_KEYS)) {
          // Values that are NaN must not reach rows that do not see them (0 * NaN is NaN): taken out, and noted for the rows that do.
          uint16_t* bits = reinterpret_cast<uint16_t*>(smem + L::NAN_BITS) + stage * (TC_KEYS * (DH / 16));
          uint32_t some = 0;
#pragma unroll
          for (int j = 0; j < PIECES; ++j) {
            uint32_t w[4] = {from[j].x, from[j].y, from[j].z, from[j].w}, found = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t bad = __vcmpeq4(w[k] & 0x7F7F7F7Fu, 0x7F7F7F7Fu);
              w[k] &= ~bad;
              found |= (((bad & 0x08040201u) * 0x01010101u) >> 24) << (4 * k);  // a bit a byte
            }
            from[j] = make_uint4(w[0], w[1], w[2], w[3]);
            bits[((own_block + APART * j) * BLOCK + key_in_block) * (DH / 16) + part] = (uint16_t)found;
            some |= found;
          }
          const bool any = __any_sync(0xffffffffu, some != 0u);
          if (lane == 0) reinterpret_cast<int*>(smem + L::NAN_SOME)[stage * 8 + warp] = any;
        }
#pragma unroll
        for (int j = 0; j < PIECES; ++j) store(base + L::V + stage * L::MAT, j, from[j]);
        tell(V_FULL + (int)stage);
      };
      // Keys go two tiles ahead of values: scores of tile i + 2 are asked for when the product of tile i's probabilities ends, and that end is what the
      // values of tile i + 2 wait for.  What was converted makes room for the next tile's load; table entries are looked up one more ahead.
      auto all_there = [&](int page) { return __all_sync(0xffffffffu, page >= 0 && page < p.n_pages); };
      const int e0 = look_up(0), e1 = look_up(1), e2 = look_up(2);
      int entry_ahead = look_up(3);
      // places of the values of the next tiles: keys are three tiles ahead when they are loaded
      int v0 = place_of(e0, 0), v1 = place_of(e1, 1), v2 = place_of(e2, 2);
      bool t0 = all_there(e0), t1 = all_there(e1), t2 = all_there(e2);
      load(keys, v0, 0);
      load(values, v0, to_values);
      convert_keys(keys, 0);
      load(keys, v1, 0);
      if (s.n_tiles > 1) convert_keys(keys, 1);
      load(keys, v2, 0);
#pragma unroll 1
      for (int i = 0; i < s.n_tiles && ok; ++i) {
        convert_values(values, i, t0);
        load(values, v1, to_values);
        if (i + 2 < s.n_tiles) convert_keys(keys, i + 2);
        const int v3 = place_of(entry_ahead, i + 3);
        load(keys, v3, 0);
        v1 = v2, v2 = v3;
        t0 = t1, t1 = t2, t2 = all_there(entry_ahead);
        entry_ahead = look_up(i + 4);
      }
      count += (uint32_t)s.n_tiles;
      done_with(n);
    }
  } else if (warp < 16) {
    // ---- softmax ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 120;" ::: "memory");
    const int g = (warp - 8) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_at = tmem + lanes + (uint32_t)g * 128u, o_at = tmem + lanes + 256u, p_at = tmem + lanes + L::p_col(g);
    auto meet = [&]() { asm volatile("bar.sync 1, 256;" ::: "memory"); };
    auto all_of_us = [&](bool mine) {
      uint32_t all;
      asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbar.red.and.pred p, 1, 256, q;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(all) : "r"((uint32_t)mine) : "memory");
      return all != 0;
    };
    float4* ml = reinterpret_cast<float4*>(smem + L::ML);
    float* factors = reinterpret_cast<float*>(smem + L::FACTOR);
    uint32_t s_count = 0, pv_count = 0, v_count = 0, others = 0;  // of this group's tiles; of all tiles (stages go by them); of the other group's
    TcSegment s;
    bool ok = true;
    for (uint32_t n = 0;; ++n) {
      const bool have = ok && next_segment(n, s);
      if (!all_of_us(have)) break;
      const bool row_ok = row < s.rows, some_row = quarter * 32 < s.rows;
      const int i_row = s.first_row + min(row, s.rows - 1), q = i_row / group, h = s.head_kv * group + i_row - q * group;
      const int qpos = s.pos0 + q;
      float factor = 0.f;
      if (g == 0) {  // this row's queries as halves, by a power of two that puts the largest entry between 2^14 and 2^15
        const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(p.q) + (size_t)(s.token0 + q) * p.q_stride + (size_t)h * DH);
        uint4 w[DH / 8];
#pragma unroll
        for (int c = 0; c < DH / 8; ++c) w[c] = row_ok ? src[c] : make_uint4(0u, 0u, 0u, 0u);
        float top = 0.f;
#pragma unroll
        for (int c = 0; c < DH / 8; ++c) {
          const uint32_t u[4] = {w[c].x, w[c].y, w[c].z, w[c].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) top = max3(top, fabsf(__uint_as_float(u[k] << 16)), fabsf(__uint_as_float(u[k] & 0xFFFF0000u)));
        }
        const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -110), 127);
        const float up = copysignf(__uint_as_float((uint32_t)(14 - e + 127) << 23), p.scale);  // (the sign of the scale, so that factors are positive)
        factor = __uint_as_float((uint32_t)(e - 14 + 127) << 23) * fabsf(p.scale) * 1.4426950408889634f;
#pragma unroll
        for (int c = 0; c < DH / 8; ++c) {
          const uint32_t u[4] = {w[c].x, w[c].y, w[c].z, w[c].w};
          uint32_t half2[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) half2[k] = pack_half(__uint_as_float(u[k] << 16) * up, __uint_as_float(u[k] & 0xFFFF0000u) * up);
          *reinterpret_cast<uint4*>(smem + L::Q + (c / 8) * L::SUB_BYTES + row * 128 + (((c % 8) ^ (row & 7)) << 4)) = make_uint4(half2[0], half2[1], half2[2], half2[3]);
        }
        factors[row] = factor;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      meet();
      if (lane == 0) arrive(bar(Q_READY));
      if (g == 1) factor = factors[row];
      float m = NOTHING, l = 0.f, t = NOTHING;  // maximum, sum of 2^(score - m), largest score + log2(value scale)
      int u = 0;
      uint32_t bad[DH / 32] = {};  // dims that a NaN value in this row's sight has
      bool any_bad = false;
      // scales: lanes 0 to 7 of a tile's blocks of keys, 8 to 15 of values; pages a tile of this group ahead of that
      int page = lane < 16 && g < s.n_tiles ? page_of(s, s.key0 / BLOCK + g * TC_BLOCKS + (lane & 7)) : -2;
      auto scale_of = [&](int i) {
        if (lane >= 16 || page < 0 || page >= p.n_pages) return lane < 8 ? -1.f : 0.f;
        const int b = s.key0 / BLOCK + i * TC_BLOCKS + (lane & 7), sub = b - page_index(b) * page_blocks;
        return __ldcg(p.scales + ((size_t)(2 * page + (lane >> 3)) * p.n_kv_heads + s.head_kv) * page_blocks + sub);
      };
      float scale_ahead = scale_of(g);
      if (lane < 16) page = g + 2 < s.n_tiles ? page_of(s, s.key0 / BLOCK + (g + 2) * TC_BLOCKS + (lane & 7)) : -2;
      bool first = true;
      for (int i = g; i < s.n_tiles && ok; i += 2) {
        const float scale = scale_ahead;
        if (i + 2 < s.n_tiles) {
          scale_ahead = scale_of(i + 2);
          if (lane < 16) page = i + 4 < s.n_tiles ? page_of(s, s.key0 / BLOCK + (i + 4) * TC_BLOCKS + (lane & 7)) : -2;
        }
        const int key0 = s.key0 + i * TC_KEYS;
        const bool there = __all_sync(0xffffffffu, lane >= 8 || scale >= 0.f);
        const bool whole = there && is_whole(s, key0);
        // of the eight blocks: what scores are multiplied by, and the value scales' exponents
        float f[8];
        int ve[8];
#pragma unroll
        for (int b = 0; b < 8; ++b) {
          const float ks = __shfl_sync(0xffffffffu, scale, b), vs = __shfl_sync(0xffffffffu, scale, 8 + b);
          f[b] = factor * ks;
          ve[b] = (int)(__float_as_uint(vs) >> 23) - 127;
        }
        ok = wait(S_FULL + g, s_count & 1u);
        if (!ok) break;
        ++s_count;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (some_row) {
          // the tile's maxima, in units of log 2
          // (columns from lo_vis to hi_vis - 1 are of keys that the row sees)
          const int hi_vis = qpos - key0 + 1, lo_vis = p.window > 0 ? qpos - p.window + 1 - key0 : 0;
          float top = NOTHING, top_t = NOTHING;
          uint32_t ra[32], rb[32];  // two blocks' columns each, one on its way while the other is used
          auto most_of = [&](const uint32_t(&x)[32], int b) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float y[2] = {NOTHING, NOTHING};
#pragma unroll
              for (int k = 0; k < 16; k += 2) y[k / 2 & 1] = max3(y[k / 2 & 1], __uint_as_float(x[16 * h + k]), __uint_as_float(x[16 * h + k + 1]));
              const float z = fmaxf(y[0], y[1]) * f[b + h];
              top = fmaxf(top, z);
              top_t = fmaxf(top_t, z + (float)ve[b + h]);
            }
          };
          if (whole) {
            tc::tmem_load32(s_at, ra);
            tmem_wait_load(ra);
            tc::tmem_load32(s_at + 32u, rb);
            most_of(ra, 0);
            tmem_wait_load(rb);
            tc::tmem_load32(s_at + 64u, ra);
            most_of(rb, 2);
            tmem_wait_load(ra);
            tc::tmem_load32(s_at + 96u, rb);
            most_of(ra, 4);
            tmem_wait_load(rb);
            most_of(rb, 6);
          } else {
#pragma unroll 1
            for (int b = 0; b < 8; b += 2) {
              const float k0 = __shfl_sync(0xffffffffu, scale, b), k1 = __shfl_sync(0xffffffffu, scale, b + 1);
              const float v0 = __shfl_sync(0xffffffffu, scale, 8 + b), v1 = __shfl_sync(0xffffffffu, scale, 9 + b);
              tc::tmem_load32(s_at + 16u * b, ra);
              tmem_wait_load(ra);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float ks = h ? k1 : k0;
                const int lo = lo_vis - (b + h) * BLOCK, hi = ks < 0.f ? 0 : hi_vis - (b + h) * BLOCK;
                float y = NOTHING;
#pragma unroll
                for (int k = 0; k < 16; ++k) y = k >= lo && k < hi ? fmaxf(y, __uint_as_float(ra[16 * h + k])) : y;
                const float z = y == NOTHING ? NOTHING : y * (factor * ks);
                top = fmaxf(top, z);
                top_t = fmaxf(top_t, z + (float)((int)(__float_as_uint(h ? v1 : v0) >> 23) - 127));
              }
            }
          }
          t = fmaxf(t, top_t);
          const bool up = top > m + 8.f || m == NOTHING;
          const float m_new = up ? fmaxf(m, top) : m;
          const int u_new = up || t - m_new > (float)(u + 15) ? (int)ceilf(t - m_new) - 11 : u;
          if (__any_sync(0xffffffffu, m_new != m || u_new != u)) {
            const float turn = ex2(m - m_new + (float)(u - u_new));
            l *= ex2(m - m_new);
            if (!first) {
              ok = wait(PV_DONE + g, (pv_count - 1u) & 1u);
              if (ok) {
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                for (int c = 0; c < DH; c += 16) {
                  uint32_t r[16];
                  tc::tmem_load16(o_at + (uint32_t)(g * DH + c), r);
                  tmem_wait_load16(r);
#pragma unroll
                  for (int k = 0; k < 16; ++k) r[k] = __float_as_uint(__uint_as_float(r[k]) * turn);
                  tmem_store16(o_at + (uint32_t)(g * DH + c), r);
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
              }
            }
            m = m_new, u = u_new;
          }
          // The groups take turns at what follows, tile by tile: side by side they would both wait for the exponentials and then both for the products.
          if (ok && i > 0) ok = wait(WEIGHED + (1 - g), (others + (uint32_t)(i - 1) / 2u) & 1u);
          if (L::P_APART && ok && !first) {  // the group's probabilities before these have been used
            ok = wait(PV_DONE + g, (pv_count - 1u) & 1u);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          }
          // Probabilities times value scale, over the scores that have been read: the scale is a power of two and goes into the exponent (from 2^-60 on:
          // what lies below adds nothing to a half), and the sum of a block's is brought back by it.
          auto weigh = [&](const uint32_t(&x)[32], int b) {
            uint32_t packed[16];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int e = max(ve[b + h] - u, -60);
              const float from = (float)e - m;
              const uint64_t f2 = pair(f[b + h], f[b + h]), from2 = pair(from, from);
              uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll
              for (int k = 0; k < 16; k += 2) {
                const uint64_t y = fma2((uint64_t)x[16 * h + k] | ((uint64_t)x[16 * h + k + 1] << 32), f2, from2);
                const float x0 = ex2(__uint_as_float((uint32_t)y)), x1 = ex2(__uint_as_float((uint32_t)(y >> 32)));
                sum2[k / 2 & 1] = add2(sum2[k / 2 & 1], pair(x0, x1));
                packed[8 * h + k / 2] = pack_half(x0, x1);
              }
              const uint64_t both = add2(sum2[0], sum2[1]);
              l = fmaf(__uint_as_float((uint32_t)both) + __uint_as_float((uint32_t)(both >> 32)), __uint_as_float((uint32_t)max(127 - e, 0) << 23), l);
            }
            tmem_store16(p_at + 8u * b, packed);
          };
          if (whole) {
            tc::tmem_load32(s_at, ra);
            tmem_wait_load(ra);
            tc::tmem_load32(s_at + 32u, rb);
            weigh(ra, 0);
            tmem_wait_load(rb);
            tc::tmem_load32(s_at + 64u, ra);
            weigh(rb, 2);
            tmem_wait_load(ra);
            tc::tmem_load32(s_at + 96u, rb);
            weigh(ra, 4);
            tmem_wait_load(rb);
            weigh(rb, 6);
          } else {
#pragma unroll 1
            for (int b = 0; b < 8; b += 2) {
              const float k0 = __shfl_sync(0xffffffffu, scale, b), k1 = __shfl_sync(0xffffffffu, scale, b + 1);
              const float v0 = __shfl_sync(0xffffffffu, scale, 8 + b), v1 = __shfl_sync(0xffffffffu, scale, 9 + b);
              uint32_t packed[16];
              tc::tmem_load32(s_at + 16u * b, ra);
              tmem_wait_load(ra);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float ks = h ? k1 : k0, by = factor * ks;
                const int lo = lo_vis - (b + h) * BLOCK, hi = ks < 0.f ? 0 : hi_vis - (b + h) * BLOCK;
                const int e = max((int)(__float_as_uint(h ? v1 : v0) >> 23) - 127 - u, -60);
                const float from = (float)e - m;
                float sum = 0.f;
#pragma unroll
                for (int k = 0; k < 16; k += 2) {
                  float x0 = ex2(fmaf(__uint_as_float(ra[16 * h + k]), by, from)), x1 = ex2(fmaf(__uint_as_float(ra[16 * h + k + 1]), by, from));
                  x0 = k >= lo && k < hi ? x0 : 0.f;
                  x1 = k + 1 >= lo && k + 1 < hi ? x1 : 0.f;
                  sum += x0 + x1;
                  packed[8 * h + k / 2] = pack_half(x0, x1);
                }
                l = fmaf(sum, __uint_as_float((uint32_t)max(127 - e, 0) << 23), l);
              }
              tmem_store16(p_at + 8u * b, packed);
            }
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
        __syncwarp();
        if (lane == 0 && ok) arrive(bar(WEIGHED + g));
        if (!whole && ok) {  // values that are NaN, of the keys that this row sees
          const uint32_t stage = (v_count + (uint32_t)i) & 1u;
          ok = wait(V_FULL + (int)stage, ((v_count + (uint32_t)i) >> 1) & 1u);
          int some = 0;
          {
#pragma unroll
            for (int k = 0; k < 8; ++k) some |= reinterpret_cast<const int*>(smem + L::NAN_SOME)[stage * 8 + k];
          }
          if (ok && some) {
            const uint32_t* bits = reinterpret_cast<const uint32_t*>(smem + L::NAN_BITS) + stage * (TC_KEYS * (DH / 32));
            for (int k = 0; k < TC_KEYS; ++k) {
              const bool hidden = __shfl_sync(0xffffffffu, scale, k / BLOCK) < 0.f || key0 + k > qpos || (p.window > 0 && key0 + k <= qpos - p.window);
#pragma unroll
              for (int d = 0; d < DH / 32; ++d) bad[d] |= hidden ? 0u : bits[k * (DH / 32) + d];
            }
            any_bad = true;
          }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0 && ok) arrive(bar(P_READY + g));
        ++pv_count;
        first = false;
      }
      v_count += (uint32_t)s.n_tiles;
      others += (uint32_t)(s.n_tiles + g) / 2u;
      // the unit's end: both groups' outputs, each group half of the columns
      if (ok && !first) ok = wait(PV_DONE + g, (pv_count - 1u) & 1u);
      ml[g * 128 + row] = make_float4(m, l, (float)(u + 11), first ? 0.f : 1.f);
      uint32_t* bad_at = reinterpret_cast<uint32_t*>(smem + L::Q) + row * (DH / 32);  // [group][row]: the queries are used
      const bool bad_somewhere = !all_of_us(!any_bad);
      if (bad_somewhere) {
#pragma unroll
        for (int d = 0; d < DH / 32; ++d) bad_at[g * 128 * (DH / 32) + d] = bad[d];
        meet();
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (ok && some_row) {
        const float4 a = ml[row], b = ml[128 + row];
        const float top = fmaxf(a.x, b.x), fa = ex2(a.x - top), fb = ex2(b.x - top), sum = a.y * fa + b.y * fb;
        // means (which are no larger than the largest value; a sum may be); the powers of two in halves, of which neither is too small or too large
        const float by = sum == 0.f ? 0.f : 4.8828125e-4f * reciprocal(sum), ua = ex2(0.5f * (a.x - top + a.z)), ub = ex2(0.5f * (b.x - top + b.z));  // 2^-11
        const size_t part_row = (size_t)s.part * TC_ROWS + row;
        const size_t to = s.part < 0 ? (size_t)(s.token0 + q) * p.out_stride + (size_t)h * DH : part_row * DH;
#pragma unroll 1
        for (int c = g * (DH / 2); c < (g + 1) * (DH / 2); c += 32) {
          uint32_t ra[32], rb[32];
          tc::tmem_load32(o_at + (uint32_t)c, ra);
          tc::tmem_load32(o_at + (uint32_t)(DH + c), rb);
          tmem_wait_load(ra);
          tmem_wait_load(rb);
          float o[32];
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = (a.w != 0.f ? __uint_as_float(ra[k]) * by * ua * ua : 0.f) + (b.w != 0.f ? __uint_as_float(rb[k]) * by * ub * ub : 0.f);
          if (bad_somewhere) {
            const uint32_t word = bad_at[c / 32] | bad_at[128 * (DH / 32) + c / 32];
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if ((word >> k) & 1u) o[k] = CUDART_NAN_F;
          }
          if (row_ok) {
            if (s.part < 0) {
#pragma unroll
              for (int k = 0; k < 32; k += 8) {
                uint32_t u[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const __nv_bfloat162 x = __floats2bfloat162_rn(o[k + 2 * j], o[k + 2 * j + 1]);
                  u[j] = *reinterpret_cast<const uint32_t*>(&x);
                }
                *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(p.out) + to + c + k) = make_uint4(u[0], u[1], u[2], u[3]);
              }
            } else {
#pragma unroll
              for (int k = 0; k < 32; k += 4) *reinterpret_cast<float4*>(p.part_o + to + c + k) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
            }
          }
        }
        if (s.part >= 0 && row_ok && g == 0) *reinterpret_cast<float2*>(p.part_ml + part_row * 2) = make_float2(top, sum);
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) arrive(bar(O_FREE));
      done_with(n);
    }
  } else if (warp == 16) {
    // ---- products: the whole warp walks, one lane issues ----
    constexpr uint32_t idesc_s = tc_instr_desc(TC_KEYS, false), idesc_o = tc_instr_desc(DH, true);
    const uint64_t q_desc = tc::smem_desc(base + L::Q), k_desc = tc::smem_desc(base + L::K), v_desc = tc_desc_mn(base + L::V);
    uint32_t count = 0, p_count[2] = {0, 0};
    TcSegment s;
    bool ok = true;
    for (uint32_t n = 0; ok && next_segment(n, s); ++n) {
      ok = wait(Q_READY, n & 1u);
      auto issue_s = [&](int i) {  // scores of tile i, where those of the group's tile before were, or the probabilities that they became
        const int g = i & 1;
        const uint32_t stage = (count + (uint32_t)i) & 1u;
        if (!L::P_APART && p_count[g] > 0) ok = wait(PV_DONE + g, (p_count[g] - 1u) & 1u);
        if (ok) ok = wait(K_FULL + (int)stage, ((count + (uint32_t)i) >> 1) & 1u);
        if (!ok) return;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (tc::elect_one()) {
#pragma unroll
          for (int k = 0; k < DH / 16; ++k) {  // descriptors count 16-byte units: a step of 16 halves is 2
            const uint64_t off = (uint64_t)((k / 4) * (L::SUB_BYTES >> 4) + (k % 4) * 2);
            tc::mma_f16(tmem + (uint32_t)g * 128u, q_desc + off, k_desc + (uint64_t)(stage * (L::MAT >> 4)) + off, idesc_s, k != 0 ? 1u : 0u);
          }
          tc::mma_commit(bar(K_EMPTY + (int)stage));
          tc::mma_commit(bar(S_FULL + g));
        }
        __syncwarp();
      };
      if (ok) issue_s(0);
      if (ok && s.n_tiles > 1) issue_s(1);
      for (int i = 0; i < s.n_tiles && ok; ++i) {
        const int g = i & 1;
        const uint32_t stage = (count + (uint32_t)i) & 1u;
        if (i == 0 && n > 0) ok = wait(O_FREE, (n - 1u) & 1u);
        if (ok) ok = wait(P_READY + g, p_count[g] & 1u);
        if (L::P_APART && ok && i + 2 < s.n_tiles) issue_s(i + 2);
        if (ok) ok = wait(V_FULL + (int)stage, ((count + (uint32_t)i) >> 1) & 1u);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (tc::elect_one()) {
#pragma unroll
          for (int k = 0; k < TC_KEYS / 16; ++k)  // 16 keys: eight columns of packed probabilities, 16 rows of values
            mma_from_tmem(tmem + 256u + (uint32_t)(g * DH), tmem + L::p_col(g) + (uint32_t)(k * 8), v_desc + (uint64_t)(stage * (L::MAT >> 4) + k * (2048 >> 4)), idesc_o,
                          i >= 2 || k != 0 ? 1u : 0u);
          tc::mma_commit(bar(V_EMPTY + (int)stage));
          tc::mma_commit(bar(PV_DONE + g));
        }
        __syncwarp();
        ++p_count[g];
        if (!L::P_APART && i + 2 < s.n_tiles) issue_s(i + 2);
      }
      count += (uint32_t)s.n_tiles;
      done_with(n);
    }
  } else {
    // ---- which tiles come next ----
    uint32_t told = 0;
    bool ok = true;
    auto say = [&](const TcSegment& s) {
      const uint32_t turn = told & 1u;
      if (told >= 2) ok = wait(SEG_EMPTY + (int)turn, ((told >> 1) & 1u) ^ 1u);
      if (ok && lane == 0) {
        segments[turn] = s;
        arrive(bar(SEG_FULL + (int)turn));
      }
      __syncwarp();
      ++told;
    };
    for (; at < end && ok; ++entry) {
      const Work w = work_of<TC_ROWS>(p, entry);
      const int tiles = w.tiles(TC_BLOCKS);
      if (tiles == 0) continue;
      int h = rest / (p.cost + tiles), off = rest - h * (p.cost + tiles);
      rest = 0;
      for (; h < p.n_kv_heads && at < end && ok; ++h) {
        const int n = (int)min((long)(p.cost + tiles - off), end - at), i0 = max(off - p.cost, 0), i1 = max(off + n - p.cost, 0);
        if (i1 > i0)
          say(TcSegment{i1 - i0, (w.first_block + i0 * TC_BLOCKS) * BLOCK, i1 - i0 == tiles ? -1 : (int)blockIdx.x * 2 + (off >= p.cost ? 0 : 1), w.token0,
                        w.pos0, w.first_row, w.rows, h, w.slot, w.first_seen, w.first_block + w.n_blocks, w.pos0 + w.first_row / group,
                        w.pos0 + (w.first_row + w.rows - 1) / group, {}});
        at += n;
        off = 0;
      }
    }
    if (ok) say(TcSegment{-1});
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 16) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

template <int DH>
int launch_attention_tc(AttnParams8 p, int blocks, cudaStream_t stream) {
  using L = TcLayout<DH>;
  static_assert(L::BYTES <= 227 * 1024, "shared memory");
  if ((p.n_entries + 1) * 4 > 2 * L::MAT) return -10;  // the keys' place holds the entries' tiles at first
  const auto kernel = kv8_attention_tc_kernel<DH>;
  const int rc = (int)note_launch(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::BYTES));
  if (rc != 0) return take_launch_error();
  p.cost = 6;
  launch_pdl_split(false, kernel, dim3(blocks), dim3(TC_THREADS), L::BYTES, stream, p);
  launch_pdl(kv8_join_kernel<false, TC_ROWS>, dim3(p.n_entries, p.n_kv_heads, TC_ROWS / 8), dim3(128), 0, stream, p);
  return 0;
}

}  // namespace kv8
}  // namespace rl
