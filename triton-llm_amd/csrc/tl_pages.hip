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
constexpr int kOneEntries = 32768;  // table entries that one workgroup looks through
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

// Grants, sequence by sequence, 1024 at a time; put(b, start, first, len) is called for each of them.
template <typename Put>
__device__ __forceinline__ int grant(const AssignParams& p, int64_t (&sums)[kWaves], Put put) {
  const int avail = min(max(p.counts[0], 0), p.n_pages);
  const int64_t cap = (int64_t)p.max_pages << p.shift;
  int64_t tokens = 0, needed = 0, taken = 0, denied = 0;
  for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
    const int b = b0 + (int)threadIdx.x;
    const int64_t len = b < p.batch ? p.lens[b] : 0;
    const int64_t add = b < p.batch ? max(p.new_lens[b], 0) : 0;
    const Scan t = block_scan(add, sums);
    const int64_t end = tokens + t.incl;
    const bool fine = len >= 0 && len + add <= cap && end <= p.tokens;
    const int64_t need = fine ? pages_of(len + add, p.shift) - pages_of(len, p.shift) : 0;
    const Scan n = block_scan(need, sums);
    const int64_t upto = needed + n.incl;
    const bool granted = fine && (need == 0 || upto <= avail);
    if (b < p.batch) {
      const int64_t start = end - add;
      const int s = (int)(start < p.tokens ? start : p.tokens);
      const int f = granted ? (int)(need ? upto - need : 0) : -1;
      p.starts[b] = s;
      p.ends[b] = (int)(granted ? len + add : len);
      if (b == p.batch - 1) p.starts[p.batch] = (int)(end < p.tokens ? end : p.tokens);
      put(b, s, f, (int)len);
    }
    // granted needs are the first ones: their sum is the largest granted N_b
    taken += block_scan(granted ? need : 0, sums).total;
    denied += block_scan(!granted && add > 0 ? 1 : 0, sums).total;
    tokens += t.total;
    needed += n.total;
  }
  // every thread has read counts, which counts_out may be, before the scans' barriers
  if (threadIdx.x == 0) {
    p.counts_out[0] = avail - (int)taken;
    p.counts_out[1] = (int)denied;
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
  __shared__ int64_t sums[kWaves];
  __shared__ int s_start[kOneBatch + 1], s_first[kOneBatch], s_len[kOneBatch];
  const int avail = grant(p, sums, [&](int b, int start, int first, int len) {
    s_start[b] = start;
    s_first[b] = first;
    s_len[b] = len;
    if (b == p.batch - 1) s_start[p.batch] = p.starts[p.batch];
  });
  __syncthreads();
  for (int t = threadIdx.x; t < p.tokens; t += kThreads)
    place_row(p, t, avail, [&](int b) { return s_start[b]; }, [&](int b) { return s_first[b]; },
              [&](int b) { return s_len[b]; });
}

__global__ __launch_bounds__(kThreads) void assign_grant_kernel(AssignParams p) {
  __shared__ int64_t sums[kWaves];
  const int avail = grant(p, sums, [&](int b, int, int first, int) { p.first[b] = first; });
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
  int32_t* found;  // workspace, by sequence: entries that name a page
  int32_t* base;
  int batch, max_pages, n_pages, shift;
};

// Columns [lo, hi) of sequence b that are given back.
struct Span {
  int lo, hi;
};
__device__ __forceinline__ Span span_of(const ReleaseParams& p, int b) {
  if (p.ended[b] == 0) return Span{0, 0};
  const int64_t held = pages_of(max(p.lens[b], 0), p.shift);
  return Span{p.keep ? max(p.keep[b], 0) : 0, (int)(held < p.max_pages ? held : p.max_pages)};
}

// Entries of a sequence that name a page, a wave at a time; see(page, how many before it) for each.
template <typename See>
__device__ __forceinline__ int walk(const ReleaseParams& p, int b, const Span& s, See see) {
  const int lane = threadIdx.x & 63;
  const int32_t* row = p.table + (int64_t)b * p.max_pages;
  int n = 0;
  for (int c0 = s.lo; c0 < s.hi; c0 += 256) {
    int page[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) page[u] = c0 + 64 * u + lane < s.hi ? row[c0 + 64 * u + lane] : -1;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool is = (unsigned)page[u] < (unsigned)p.n_pages;
      const uint64_t all = __ballot(is);
      if (is) see(page[u], n + __popcll(all & (((uint64_t)1 << lane) - 1)));
      n += __popcll(all);
    }
  }
  return n;
}

__device__ __forceinline__ void put_back(const ReleaseParams& p, int64_t at, int page) {
  if (at < p.n_pages) p.free_pages[at] = page;
}
__device__ __forceinline__ void put_counts(const ReleaseParams& p, int base, int64_t found) {
  const int64_t n = base + found;
  p.counts_out[0] = (int)(n < p.n_pages ? n : p.n_pages);
  p.counts_out[1] = (int)(n < p.n_pages ? 0 : n - p.n_pages);
}

// Few table entries: one workgroup, a wave a sequence, one launch.
__global__ __launch_bounds__(kThreads) void release_one_kernel(ReleaseParams p) {
  __shared__ int64_t sums[kWaves];
  __shared__ int s_found[kOneBatch];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int base = min(max(p.counts[0], 0), p.n_pages);
  for (int b = wave; b < p.batch; b += kWaves) {
    const int n = walk(p, b, span_of(p, b), [](int, int) {});
    if (lane == 0) s_found[b] = n;
  }
  __syncthreads();
  const int mine = (int)threadIdx.x < p.batch ? s_found[threadIdx.x] : 0;
  const Scan s = block_scan(mine, sums);
  if ((int)threadIdx.x < p.batch) s_found[threadIdx.x] = (int)(s.incl - mine);
  if (threadIdx.x == 0) put_counts(p, base, s.total);
  __syncthreads();
  for (int b = wave; b < p.batch; b += kWaves) {
    const int64_t at = (int64_t)base + s_found[b];
    walk(p, b, span_of(p, b), [&](int page, int i) { put_back(p, at + i, page); });
    const int len = p.lens[b];
    if (lane == 0) p.lens_out[b] = p.ended[b] ? 0 : len;
  }
}

__global__ __launch_bounds__(256) void release_count_kernel(ReleaseParams p) {
  const int b = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6);
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.base = min(max(p.counts[0], 0), p.n_pages);
  if (b >= p.batch) return;
  const int n = walk(p, b, span_of(p, b), [](int, int) {});
  if ((threadIdx.x & 63) == 0) p.found[b] = n;
}

__global__ __launch_bounds__(256) void release_put_kernel(ReleaseParams p) {
  const int b = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (b >= p.batch) return;
  const Span s = span_of(p, b);
  const bool last = b == p.batch - 1;
  if (s.lo < s.hi || last) {
    int64_t before = 0;
    for (int i = lane; i < b; i += 64) before += p.found[i];
#pragma unroll
    for (int off = 32; off; off >>= 1) before += __shfl_xor(before, off);
    const int base = *p.base;
    walk(p, b, s, [&](int page, int i) { put_back(p, base + before + i, page); });
    if (last && lane == 0) put_counts(p, base, before + p.found[b]);
  }
  const int len = p.lens[b];
  if (lane == 0) p.lens_out[b] = p.ended[b] ? 0 : len;
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
                     int32_t* counts_out, int32_t* lens_out, void* workspace, size_t workspace_bytes, void* stream) {
  const int shift = page_shift(page_size);
  if (!page_table || !lens || !ended || !free_pages || !counts || !counts_out || !lens_out || !workspace || batch < 1 ||
      max_pages < 1 || n_pages < 1 || shift < 0 || ((uintptr_t)workspace & 15))
    return TL_ERR_INVALID;
  if (batch > kMostBatch || ((int64_t)max_pages << shift) > INT32_MAX) return TL_ERR_UNSUPPORTED;
  if (workspace_bytes < tl_pages_workspace_bytes(batch)) return TL_ERR_INVALID;
  const struct {
    const void* at;
    int64_t n;
  } in[] = {{page_table, (int64_t)batch * max_pages}, {ended, batch}, {keep, batch}, {lens, batch}, {counts, 2}},
    out[] = {{free_pages, n_pages}, {lens_out, batch}, {counts_out, 2}, {workspace, batch + 4}};
  for (int o = 0; o < 4; ++o) {
    for (int i = 0; i < 5; ++i)
      if (!(o == 1 && i == 3 && lens_out == lens) && !(o == 2 && i == 4 && counts_out == counts) &&
          !apart(in[i].at, in[i].n, out[o].at, out[o].n))
        return TL_ERR_INVALID;
    for (int i = 0; i < o; ++i)
      if (!apart(out[i].at, out[i].n, out[o].at, out[o].n)) return TL_ERR_INVALID;
  }
  ReleaseParams p{page_table, lens, ended, keep, free_pages, counts, counts_out, lens_out,
                  (int32_t*)workspace + 4, (int32_t*)workspace, batch, max_pages, n_pages, shift};
  hipStream_t st = tl_resolve_stream(stream);
  if (batch <= kOneBatch && (int64_t)batch * max_pages <= kOneEntries) {
    hipLaunchKernelGGL(release_one_kernel, dim3(1), dim3(kThreads), 0, st, p);
    return tl_launch_status();
  }
  const dim3 grid((batch + 3) / 4);
  hipLaunchKernelGGL(release_count_kernel, grid, dim3(256), 0, st, p);
  const int e = tl_launch_status();
  if (e) return e;
  hipLaunchKernelGGL(release_put_kernel, grid, dim3(256), 0, st, p);
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
