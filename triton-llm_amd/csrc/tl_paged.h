// Internal header of the paged KV cache kernels (tl_paged.hip, tl_window.hip): how a
// position of a sequence is found in the page pool.  Not part of the C ABI.
//
// A pool holds n_pages pages of (n_kv_head, page_size, d_k); page_size is a power of two
// from 16 to 1024.  Position t of sequence b lies in page table[b][t >> shift], row
// t & (page_size - 1).  The kernels walk positions in aligned blocks of 16, which lie in one page
// each, so a block needs one table entry and one 64-bit base address, and rows inside
// it 32-bit offsets: pools of any size are reached.  An entry outside [0, n_pages) names no
// page: nothing is read or written through it, and its positions count as hidden.
#pragma once

#include "tl_common.h"

#include <type_traits>

namespace tlpg {

constexpr int kBlk = 16;  // positions of a block
constexpr int kBlkShift = 4;
constexpr int kMinPage = 16, kMaxPage = 1024;

struct PageMap {
  const int32_t* table;  // [batch][max_pages]
  int max_pages, n_pages, shift;
};

// log2 of a page size the kernels take, -1 for any other.
static inline int page_shift(int page_size) {
  if (page_size < kMinPage || page_size > kMaxPage || (page_size & (page_size - 1))) return -1;
  return __builtin_ctz((unsigned)page_size);
}

// Values equal on every lane, moved to scalar registers.
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uni(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)x >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

// Sums over the lanes up to and with each, by DPP moves: rows of 16 first, then row to row.
__device__ __forceinline__ int wave_scan(int x) {
  auto add = [&](auto ctrl, auto rows) {
    x += __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, decltype(rows)::value, 0xF, false);
  };
  add(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xF>{});  // row_shr:1
  add(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xF>{});
  add(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xF>{});
  add(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xF>{});
  add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});  // row_bcast:15 into rows 1 and 3
  add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});  // row_bcast:31 into rows 2 and 3
  return x;
}

__device__ __forceinline__ int last_lane(int x) { return uni(__builtin_amdgcn_readlane(x, 63)); }

}  // namespace tlpg
