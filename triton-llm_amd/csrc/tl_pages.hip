// Page tables that the GPU keeps: which pages the sequences' new tokens go to (assign_pages) and the pages of ended
// sequences given back (release_pages), from lengths that lie on the device.  No counterpart in the reference.
//
// The pages that no sequence has are a stack: free_pages[0 .. counts[0]), the next one to be taken last.
//
// release: with h_b = ceil(lens_b / page) and the entries e of columns keep_b <= c < h_b of the ended sequences that name a
//   page, in the order (b, c), the i-th of them goes to free_pages[counts[0] + i].
// assign: sequence b needs n_b = ceil((lens_b + new_b) / page) - ceil(lens_b / page) pages; N_b = n_0 + .. + n_b.  It is
//   granted where n_b = 0 or N_b <= counts[0], and its i-th new page is free_pages[counts[0] - 1 - (N_b - n_b) - i].  Row
//   t of the packed batch is token t - starts_b of the sequence with starts_b <= t < starts_(b+1), starts the sums of new_lens.
//
// Few numbers are read and written: what counts is how many dependent loads and launches stand one behind the other.
#include "tl_paged.h"

using namespace tlpg;

namespace {

constexpr int kThreads = 64 * kScanWaves;
constexpr int kWaves = kScanWaves;
constexpr int kMostBatch = 65535;
constexpr int kOneBatch = 1024;     // sequences that one workgroup holds in LDS
constexpr int kOneTokens = 8192;    // rows that one workgroup writes
constexpr int kFillThreads = 256;
constexpr int kSearchLds = 4096;    // sequences that the rows' workgroups search in LDS

struct AssignParams {
  const int32_t* lens;
  const int32_t* new_lens;
  int32_t* table;
  const int32_t* free_pages;
  const int32_t* counts;
  int32_t* counts_out;
  int32_t* slots;
  int32_t* positions;
  int32_t* starts;
  int32_t* ends;
  int32_t* first;  // workspace, by sequence: its first new page's place from the free list's end on, -1: not granted
  int32_t* base;   // workspace: pages on the free list before the call
  int batch, max_pages, n_pages, shift, tokens;
};

__device__ __forceinline__ int64_t pages_of(int64_t n, int shift) { return (n + (1 << shift) - 1) >> shift; }

// Grants, sequence by sequence, 1024 at a time; put(b, start, first, len) is called for each of them.  Sums can pass 32 bits: they are
// of the upper and the lower halves of numbers that are cut off above what can be granted.
struct GrantLds {
  int sums[2][kWaves];
  int taken, denied;
};
template <typename Put>
__device__ __forceinline__ int grant(const AssignParams& p, GrantLds& lds, Put put) {
  const int avail = min(max(p.counts[0], 0), p.n_pages);
  const int64_t cap = (int64_t)p.max_pages << p.shift;
  if (threadIdx.x == 0) lds.taken = lds.denied = 0;
  int64_t tokens = 0, needed = 0;
  for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
    const int b = b0 + (int)threadIdx.x;
    const int64_t len = b < p.batch ? p.lens[b] : 0;
    const int add = b < p.batch ? max(p.new_lens[b], 0) : 0;
    int x[2] = {add & 0xFFFF, add >> 16}, total[2];
    block_scan(x, total, lds.sums);
    const int64_t end = tokens + ((int64_t)x[1] << 16) + x[0];
    const bool fine = len >= 0 && len + add <= cap && end <= p.tokens;
    const int need = fine ? (int)(pages_of(len + add, p.shift) - pages_of(len, p.shift)) : 0;
    tokens += ((int64_t)total[1] << 16) + total[0];
    x[0] = need & 0xFFFF, x[1] = need >> 16;
    block_scan(x, total, lds.sums);
    const int64_t upto = needed + ((int64_t)x[1] << 16) + x[0];
    const bool granted = fine && (need == 0 || upto <= avail);
    needed += ((int64_t)total[1] << 16) + total[0];
    if (b < p.batch) {
      const int64_t start = end - add;
      const int s = (int)(start < p.tokens ? start : p.tokens);
      const int f = granted ? (int)(need ? upto - need : 0) : -1;
      p.starts[b] = s;
      p.ends[b] = (int)(granted ? len + add : len);
      if (b == p.batch - 1) p.starts[p.batch] = (int)(end < p.tokens ? end : p.tokens);
      put(b, s, f, (int)len);
      // granted needs are the first ones: their sum is the largest granted N_b
      if (granted && need) atomicMax(&lds.taken, (int)upto);
      if (!granted && add) atomicAdd(&lds.denied, 1);
    }
  }
  __syncthreads();
  // every thread has read counts, which counts_out may be
  if (threadIdx.x == 0) {
    p.counts_out[0] = avail - lds.taken;
    p.counts_out[1] = lds.denied;
  }
  return avail;
}

// Row t's slot and position, and the table's entry where it is a page's first.  starts_at, first_at, len_at: by sequence.
template <typename S, typename F, typename L>
__device__ __forceinline__ void place_row(const AssignParams& p, int t, int avail, S starts_at, F first_at, L len_at) {
  int lo = 0, hi = p.batch;  // the last sequence with starts <= t, those without rows before it passed over
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts_at(mid) <= t) lo = mid;
    else hi = mid;
  }
  int slot = -1, pos = -1;
  const int first = first_at(lo);
  if (first >= 0 && t < starts_at(lo + 1)) {
    const int len = len_at(lo);
    pos = len + (t - starts_at(lo));
    const int c = pos >> p.shift, fresh = c - (int)pages_of(len, p.shift);
    int32_t* entry = p.table + (int64_t)lo * p.max_pages + c;
    int page = fresh >= 0 ? p.free_pages[avail - 1 - first - fresh] : *entry;
    if ((unsigned)page >= (unsigned)p.n_pages) page = -1;
    const int in = pos & ((1 << p.shift) - 1);
    if (fresh >= 0 && in == 0) *entry = page;
    slot = page < 0 ? -1 : (page << p.shift) + in;
  }
  p.slots[t] = slot;
  p.positions[t] = pos;
}

// Few sequences and rows: one workgroup, one launch.
__global__ __launch_bounds__(kThreads) void assign_one_kernel(AssignParams p) {
  __shared__ GrantLds lds;
  __shared__ int s_start[kOneBatch + 1], s_first[kOneBatch], s_len[kOneBatch];
  const int avail = grant(p, lds, [&](int b, int start, int first, int len) {
    s_start[b] = start;
    s_first[b] = first;
    s_len[b] = len;
    if (b == p.batch - 1) s_start[p.batch] = p.starts[p.batch];
  });
  for (int t = threadIdx.x; t < p.tokens; t += kThreads)
    place_row(p, t, avail, [&](int b) { return s_start[b]; }, [&](int b) { return s_first[b]; },
              [&](int b) { return s_len[b]; });
}

__global__ __launch_bounds__(kThreads) void assign_grant_kernel(AssignParams p) {
  __shared__ GrantLds lds;
  const int avail = grant(p, lds, [&](int b, int, int first, int) { p.first[b] = first; });
  if (threadIdx.x == 0) *p.base = avail;
}

__global__ __launch_bounds__(kFillThreads) void assign_rows_kernel(AssignParams p) {
  __shared__ int s_start[kSearchLds + 1];
  const bool lds = p.batch <= kSearchLds;
  if (lds)
    for (int b = threadIdx.x; b <= p.batch; b += kFillThreads) s_start[b] = p.starts[b];
  const int avail = *p.base;
  __syncthreads();
  const int t = (int)blockIdx.x * kFillThreads + (int)threadIdx.x;
  if (t >= p.tokens) return;
  auto first = [&](int b) { return p.first[b]; };
  auto len = [&](int b) { return p.lens[b]; };
  if (lds) place_row(p, t, avail, [&](int b) { return s_start[b]; }, first, len);
  else place_row(p, t, avail, [&](int b) { return p.starts[b]; }, first, len);
}

struct ReleaseParams {
  const int32_t* table;
  const int32_t* lens;
  const int32_t* ended;
  const int32_t* keep;  // NULL: none
  int32_t* free_pages;
  const int32_t* counts;
  int32_t* counts_out;
  int32_t* lens_out;
  int batch, max_pages, n_pages, shift;
};

// One workgroup.  The columns that are given back are cut into pieces of 64, (sequence, column), and a wave takes kPieces of them at
// a time: what names a page is counted by a ballot, the waves' counts meet in LDS, and every wave finds its places by a scan of all of
// them.  The next pieces are on their way meanwhile.
constexpr int kPieces = 4;
constexpr int kRound = kPieces * kWaves;  // pieces of a round: as many as a wave has lanes
static_assert(kRound == 64, "a wave scans a round's counts");
constexpr int kMap = 1024;  // pieces whose sequences are known at a time

__global__ __launch_bounds__(kThreads) void release_kernel(ReleaseParams p) {
  __shared__ int sums[1][kWaves];
  __shared__ int s_piece[kThreads + 1], s_lo[kThreads], s_hi[kThreads];  // by sequence: its first piece, its columns
  __shared__ int s_seq[kMap];                                            // by piece: its sequence
  __shared__ int s_count[2][kRound];
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
  int64_t at = min(max(p.counts[0], 0), p.n_pages);
  for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
    const int b = b0 + tid;
    int lo = 0, hi = 0;
    if (b < p.batch) {
      const int len = p.lens[b];
      const bool ended = p.ended[b] != 0;
      const int keep = p.keep ? p.keep[b] : 0;
      if (ended) {
        const int64_t held = pages_of(max(len, 0), p.shift);
        lo = max(keep, 0);
        hi = (int)(held < p.max_pages ? held : p.max_pages);
      }
      p.lens_out[b] = ended ? 0 : len;
    }
    const int pieces = lo < hi ? (hi - lo + 63) >> 6 : 0;
    int x[1] = {pieces}, total[1];
    block_scan(x, total, sums);
    const int first = x[0] - pieces;
    s_piece[tid] = first;
    s_lo[tid] = lo;
    s_hi[tid] = hi;
    for (int m0 = 0; m0 < total[0]; m0 += kMap) {
      __syncthreads();  // the map of the pieces before has been read
      for (int i = max(first, m0); i < min(first + pieces, m0 + kMap); ++i) s_seq[i - m0] = tid;
      __syncthreads();
      const int n = min(total[0] - m0, kMap);
      // this wave's pieces of round r
      auto load = [&](int r, int (&page)[kPieces]) {
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
          const int i = r * kRound + wave * kPieces + k;
          page[k] = -1;
          if (i < n) {
            const int s = s_seq[i];
            const int c = s_lo[s] + 64 * (m0 + i - s_piece[s]) + lane;
            if (c < s_hi[s]) page[k] = p.table[(int64_t)(b0 + s) * p.max_pages + c];
          }
        }
      };
      const int rounds = (n + kRound - 1) / kRound;
      int page[kPieces];
      load(0, page);
      for (int r = 0; r < rounds; ++r) {
        uint64_t is[kPieces];
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
          is[k] = __ballot((unsigned)page[k] < (unsigned)p.n_pages);
          if (lane == k) s_count[r & 1][wave * kPieces + k] = __popcll(is[k]);
        }
        int next[kPieces];
        if (r + 1 < rounds) load(r + 1, next);
        __syncthreads();
        const int c = s_count[r & 1][lane], upto = wave_scan(c);
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
          const int64_t to = at + __builtin_amdgcn_readlane(upto - c, wave * kPieces + k) +
                             __popcll(is[k] & (((uint64_t)1 << lane) - 1));
          if (((is[k] >> lane) & 1) && to < p.n_pages) p.free_pages[to] = page[k];
        }
        at += last_lane(upto);
#pragma unroll
        for (int k = 0; k < kPieces; ++k) page[k] = r + 1 < rounds ? next[k] : -1;
      }
    }
  }
  // every thread has read counts, which counts_out may be, before a barrier above
  if (tid == 0) {
    p.counts_out[0] = (int)(at < p.n_pages ? at : p.n_pages);
    p.counts_out[1] = (int)(at < p.n_pages ? 0 : at - p.n_pages);
  }
}

bool apart(const void* a, int64_t na, const void* b, int64_t nb) {
  return !a || !b || !tl_overlap(a, (size_t)na * 4, b, (size_t)nb * 4);
}

}  // namespace

extern "C" {

size_t tl_pages_workspace_bytes(int batch) {
  return batch < 1 || batch > kMostBatch ? 0 : (((size_t)batch + 4) * 4 + 15) & ~(size_t)15;
}

int tl_release_pages(const int32_t* page_table, int max_pages, int page_size, const int32_t* lens, const int32_t* ended,
                     const int32_t* keep, int batch, int32_t* free_pages, int n_pages, const int32_t* counts,
                     int32_t* counts_out, int32_t* lens_out, void* stream) {
  const int shift = page_shift(page_size);
  if (!page_table || !lens || !ended || !free_pages || !counts || !counts_out || !lens_out || batch < 1 || max_pages < 1 ||
      n_pages < 1 || shift < 0)
    return TL_ERR_INVALID;
  if (batch > kMostBatch || ((int64_t)max_pages << shift) > INT32_MAX) return TL_ERR_UNSUPPORTED;
  const struct {
    const void* at;
    int64_t n;
  } in[] = {{page_table, (int64_t)batch * max_pages}, {ended, batch}, {keep, batch}, {lens, batch}, {counts, 2}},
    out[] = {{free_pages, n_pages}, {lens_out, batch}, {counts_out, 2}};
  for (int o = 0; o < 3; ++o) {
    for (int i = 0; i < 5; ++i)
      if (!(o == 1 && i == 3 && lens_out == lens) && !(o == 2 && i == 4 && counts_out == counts) &&
          !apart(in[i].at, in[i].n, out[o].at, out[o].n))
        return TL_ERR_INVALID;
    for (int i = 0; i < o; ++i)
      if (!apart(out[i].at, out[i].n, out[o].at, out[o].n)) return TL_ERR_INVALID;
  }
  ReleaseParams p{page_table, lens, ended, keep, free_pages, counts, counts_out, lens_out, batch, max_pages, n_pages, shift};
  hipLaunchKernelGGL(release_kernel, dim3(1), dim3(kThreads), 0, tl_resolve_stream(stream), p);
  return tl_launch_status();
}

int tl_assign_pages(const int32_t* lens, const int32_t* new_lens, int batch, int32_t* page_table, int max_pages,
                    int page_size, const int32_t* free_pages, int n_pages, const int32_t* counts, int32_t* counts_out,
                    int max_tokens, int32_t* slots, int32_t* positions, int32_t* starts, int32_t* ends, void* workspace,
                    size_t workspace_bytes, void* stream) {
  const int shift = page_shift(page_size);
  if (!lens || !new_lens || !page_table || !free_pages || !counts || !counts_out || !starts || !ends || !workspace ||
      (max_tokens > 0 && (!slots || !positions)) || batch < 1 || max_pages < 1 || n_pages < 1 || max_tokens < 0 || shift < 0 ||
      ((uintptr_t)workspace & 15))
    return TL_ERR_INVALID;
  // a slot is a 32-bit number, and so is a position
  if (batch > kMostBatch || ((int64_t)max_pages << shift) > INT32_MAX || ((int64_t)n_pages << shift) > INT32_MAX)
    return TL_ERR_UNSUPPORTED;
  if (workspace_bytes < tl_pages_workspace_bytes(batch)) return TL_ERR_INVALID;
  const struct {
    const void* at;
    int64_t n;
  } in[] = {{lens, batch}, {new_lens, batch}, {free_pages, n_pages}, {counts, 2}},
    out[] = {{page_table, (int64_t)batch * max_pages}, {slots, max_tokens}, {positions, max_tokens}, {starts, batch + 1},
             {ends, batch}, {counts_out, 2}, {workspace, batch + 4}};
  for (int o = 0; o < 7; ++o) {
    if (out[o].n == 0) continue;
    for (int i = 0; i < 4; ++i)
      if (!(o == 5 && i == 3 && counts_out == counts) && !apart(in[i].at, in[i].n, out[o].at, out[o].n))
        return TL_ERR_INVALID;
    for (int i = 0; i < o; ++i)
      if (out[i].n && !apart(out[i].at, out[i].n, out[o].at, out[o].n)) return TL_ERR_INVALID;
  }
  AssignParams p{lens, new_lens, page_table, free_pages, counts, counts_out, slots, positions, starts, ends,
                 (int32_t*)workspace + 4, (int32_t*)workspace, batch, max_pages, n_pages, shift, max_tokens};
  hipStream_t st = tl_resolve_stream(stream);
  if (batch <= kOneBatch && max_tokens <= kOneTokens) {
    hipLaunchKernelGGL(assign_one_kernel, dim3(1), dim3(kThreads), 0, st, p);
    return tl_launch_status();
  }
  hipLaunchKernelGGL(assign_grant_kernel, dim3(1), dim3(kThreads), 0, st, p);
  const int e = tl_launch_status();
  if (e || max_tokens == 0) return e;
  hipLaunchKernelGGL(assign_rows_kernel, dim3((unsigned)(((int64_t)max_tokens + kFillThreads - 1) / kFillThreads)), dim3(kFillThreads), 0, st, p);
  return tl_launch_status();
}

}  // extern "C"
