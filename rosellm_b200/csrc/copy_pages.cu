// Copies of whole cache pages in many pools at once: page src[i] to page dst[i] of every layer's codes, scales or rows, in one launch.
//
// A copy moves each byte twice, so its floor is the memory's copy bandwidth; what costs otherwise is one launch a pool (two a layer).
// A block of threads takes a run of 16-byte units (4-byte ones where a page's size is no multiple of 16) of one pool's
// copies, several loads of a thread on their way before its first store.
// Measured: 1024 pages of 24 layers 245 us, the copy bandwidth (a pool at a time with indexing 7,588); one page of 12 layers 3.0 us, a launch.
#include "common.cuh"

namespace rl {

constexpr int COPY_POOLS = 96;    // pools of one launch (its arguments hold them)
constexpr int COPY_THREADS = 256;
constexpr int COPY_UNITS = 8;     // units of a thread

struct CopyTable {
  char* base[COPY_POOLS];
  unsigned int units[COPY_POOLS];        // of a page
  unsigned int first_block[COPY_POOLS];  // of this pool's run of blocks
  int n_pools, wide;                     // wide: 16-byte units
};

template <typename U>
__device__ __forceinline__ void copy_run(char* base, unsigned int units, unsigned int block, const int* __restrict__ pairs, int n_pairs,
                                         int n_pages, int* status) {
  const unsigned long long total = (unsigned long long)units * n_pairs;
  const unsigned long long at = (unsigned long long)block * (COPY_THREADS * COPY_UNITS) + threadIdx.x;
  U v[COPY_UNITS];
  U* to[COPY_UNITS];
#pragma unroll
  for (int i = 0; i < COPY_UNITS; ++i) {
    const unsigned long long u = at + (unsigned long long)i * COPY_THREADS;
    to[i] = nullptr;
    if (u < total) {
      const unsigned int pair = (unsigned int)(u / units), off = (unsigned int)(u - (unsigned long long)pair * units);
      const int src = pairs[2 * pair], dst = pairs[2 * pair + 1];
      if (src >= 0 && src < n_pages && dst >= 0 && dst < n_pages) {
        v[i] = reinterpret_cast<const U*>(base)[(size_t)src * units + off];
        to[i] = reinterpret_cast<U*>(base) + (size_t)dst * units + off;
      } else {
        atomicOr(status, RL_STATUS_BAD_PAGE);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < COPY_UNITS; ++i)
    if (to[i] != nullptr) *to[i] = v[i];
}

__global__ __launch_bounds__(COPY_THREADS) void copy_pages_kernel(const __grid_constant__ CopyTable table, const int* __restrict__ pairs,
                                                                  int n_pairs, int n_pages, int* status) {
  pdl_begin();
  int lo = 0, hi = table.n_pools - 1;  // the last pool whose run begins at or before this block
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (table.first_block[mid] <= blockIdx.x)
      lo = mid;
    else
      hi = mid - 1;
  }
  if (table.wide)
    copy_run<uint4>(table.base[lo], table.units[lo], blockIdx.x - table.first_block[lo], pairs, n_pairs, n_pages, status);
  else
    copy_run<uint32_t>(table.base[lo], table.units[lo], blockIdx.x - table.first_block[lo], pairs, n_pairs, n_pages, status);
}

}  // namespace rl

// bases[n_pools]: the pools' first pages; page_bytes[n_pools]: multiples of 4 (pages lie one behind the other); pairs int32 [n_pairs][2]
// on the device.  Pools whose base and page are multiples of 16 bytes are copied in such units.
RL_EXPORT int rl_copy_pages(const void* const* bases, const long* page_bytes, int n_pools, const int* pairs, int n_pairs, int n_pages,
                            int* status, cudaStream_t stream) {
  if (n_pairs <= 0 || n_pools <= 0) return 0;
  for (int i = 0; i < n_pools; ++i)
    if (page_bytes[i] <= 0 || page_bytes[i] % 4 != 0 || (uintptr_t)bases[i] % 4 != 0 || page_bytes[i] / 4 > 0x7fffffffL) return -2;
  for (int wide = 1; wide >= 0; --wide) {
    int i = 0;
    while (i < n_pools) {
      rl::CopyTable table;
      table.n_pools = 0;
      table.wide = wide;
      unsigned long long blocks = 0;
      for (; i < n_pools && table.n_pools < rl::COPY_POOLS; ++i) {
        const int is_wide = page_bytes[i] % 16 == 0 && (uintptr_t)bases[i] % 16 == 0;
        if (is_wide != wide) continue;
        const unsigned long long units = (unsigned long long)page_bytes[i] / (wide ? 16 : 4);
        const unsigned long long per = (unsigned long long)rl::COPY_THREADS * rl::COPY_UNITS;
        const unsigned long long more = (units * n_pairs + per - 1) / per;
        if (blocks + more > 0x7fffffffULL) {
          if (blocks == 0) return -3;  // one pool's copies alone are too many for a grid
          break;
        }
        table.base[table.n_pools] = (char*)bases[i];
        table.units[table.n_pools] = (unsigned int)units;
        table.first_block[table.n_pools] = (unsigned int)blocks;
        ++table.n_pools;
        blocks += more;
      }
      if (blocks == 0) break;
      rl::launch_pdl(rl::copy_pages_kernel, dim3((unsigned int)blocks), dim3(rl::COPY_THREADS), 0, stream, table, pairs, n_pairs, n_pages, status);
    }
  }
  RL_CHECK_LAUNCH();
  return 0;
}
