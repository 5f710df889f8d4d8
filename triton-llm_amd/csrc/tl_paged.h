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

#include <initializer_list>
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

// A tensor of rows of `row` bytes at base + i0 s0 + i1 s1 + i2 s2, i_k < n[k], strides s[k] in bytes.
struct Rows3 {
  const void* base;
  int64_t n[3], s[3], row;
  Rows3 upward() const {  // the same rows from the lowest on
    Rows3 t = *this;
    for (int i = 0; i < 3; ++i)
      if (s[i] < 0) t.base = (const char*)t.base + (n[i] - 1) * s[i], t.s[i] = -s[i];
    return t;
  }
  // bytes from the first to behind the last of what the dims of strides below m span
  int64_t span(int64_t m) const {
    int64_t e = row;
    for (int i = 0; i < 3; ++i)
      if (s[i] < m) e += (n[i] - 1) * s[i];
    return e;
  }
};

// Whether two such tensors may share a byte.  Not if their spans do not meet, nor if they lie side by side in the rows of one
// buffer: all strides from some size on are multiples of m, and what the smaller ones span is apart modulo m.
static inline bool rows_overlap(const Rows3& x, const Rows3& y) {
  const Rows3 a = x.upward(), b = y.upward();
  if (!tl_overlap(a.base, (size_t)a.span(INT64_MAX), b.base, (size_t)b.span(INT64_MAX))) return false;
  for (const Rows3* t : {&a, &b})
    for (int i = 0; i < 3; ++i) {
      const int64_t least = t->s[i];
      if (t->n[i] < 2 || least < 1) continue;
      int64_t m = 0;
      for (const Rows3* u : {&a, &b})
        for (int k = 0; k < 3; ++k)
          if (u->n[k] > 1 && u->s[k] >= least)
            for (int64_t d = u->s[k]; d;) {  // m = gcd(m, d)
              const int64_t r = m % d;
              m = d;
              d = r;
            }
      const int64_t ea = a.span(least), eb = b.span(least);
      const int64_t from_a = (int64_t)(((uintptr_t)b.base % m + m - (uintptr_t)a.base % m) % m);  // a's start to b's
      if (ea <= from_a && eb <= m - from_a) return false;
    }
  return true;
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

// Of a workgroup of kScanWaves waves: the sum over its threads up to and with each, and of all.  Every thread takes part.
constexpr int kScanWaves = 16;
struct Scan {
  int64_t incl, total;
};
__device__ __forceinline__ Scan block_scan(int64_t x, int64_t (&sums)[kScanWaves]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t y = __shfl_up(x, off);
    if (lane >= off) x += y;
  }
  __syncthreads();  // the sums of the scan before have been read
  if (lane == 63) sums[wave] = x;
  __syncthreads();
  int64_t s = sums[lane & (kScanWaves - 1)];
#pragma unroll
  for (int off = 1; off < kScanWaves; off <<= 1) {
    const int64_t y = __shfl_up(s, off);
    if ((lane & (kScanWaves - 1)) >= off) s += y;
  }
  const int64_t before = __shfl(s, wave ? wave - 1 : 0);
  return Scan{x + (wave ? before : 0), __shfl(s, kScanWaves - 1)};
}

// The same of N numbers at once, whose sums fit in 32 bits, of a workgroup of W waves.  FRESH: nobody has used `sums` since a barrier.
template <bool FRESH = false, int N, int W>
__device__ __forceinline__ void block_scan(int (&x)[N], int (&total)[N], int (&sums)[N][W]) {
  const int lane = threadIdx.x & 63, wave = uni((int)threadIdx.x >> 6);
  if (!FRESH) __syncthreads();  // the sums of the scan before have been read
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] = wave_scan(x[i]);
    if (lane == 63) sums[i][wave] = x[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int s = wave_scan(lane < W ? sums[i][lane] : 0);
    total[i] = last_lane(s);
    if (wave) x[i] += __builtin_amdgcn_readlane(s, wave - 1);
  }
}

}  // namespace tlpg
