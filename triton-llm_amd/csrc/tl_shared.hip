// Attention of one new token a sequence where groups of sequences begin with the same pages: what a group shares is read
// once for all of its sequences.  No counterpart in the reference (one sequence a cache, smollm2_triton/model.py:190-225).
//
//   o_b = softmax(scale q_b . K^T over positions 0 .. L_b - 1) V
//
// Positions 0 .. S_g - 1 lie in the same pages for every sequence b of group g.  The softmax's state over them, with m
// the maximum, l = sum 2^(s_j - m) and acc = sum 2^(s_j - m) v_j (log2 domain, fp32), comes from one product of all the group's
// queries with the shared keys; the state over a sequence's own positions S_g .. L_b - 1 from its queries alone.  States
// are joined as m = max m_i, l = sum l_i 2^(m_i - m), acc likewise, and o = acc / l.
//
// A sequence shorter than S_g, or the only one of its group, is taken as one that shares nothing.
//
// A step has one plan (plan_one_kernel, one workgroup), from the lengths, which only the device knows: which sequences share, and a
// list of items, each a tile of up to 128 query rows of one KV head and a range of keys, a group's or a sequence's own.  It holds for
// every layer.  A layer's attention: a workgroup an item (shared_kernel) and, where a row's keys are in several items, their join
// (shared_join_kernel).
#include "tl_attn_narrow.h"

#include <math.h>

using namespace tlat;
using namespace tlpg;

namespace {

constexpr int kThreads = 256;
constexpr int kBM = 128;  // query rows of an item at most
constexpr int kMostBatch = 65535;
// Key tiles of an item at least, if there are more: 2 / 4 / 8, with 4 sequences behind 496 positions, 9 / 3 heads of 64, fp32,
// plan and call 19.0 / 23.3 / 32.0 us; 2 groups of 8 behind 2000 each, 15 / 5 heads of 64, fp16, four layers, 50.7 / 53.2 / 64.2.
constexpr int kMinTiles = 2;
constexpr int kScanThreads = 64 * kScanWaves;

// Rows row0 .. of R: row r is query head hkv * group + r % group of the i0 + r / group-th sequence that shares (i0 < 0: of sequence
// b), over positions [lo, hi) of sequence b's pages.  lo is a multiple of 16 but for a sequence's first own ones.
struct Item {
  int b, hkv, lo, hi;
  int i0, row0, R, out;  // out: the first row's place in the workspace, -1: the rows go to o, as these are all their keys
};
constexpr int kFour = -2;  // i0: of sequence b, rows 0 .. R of KV heads hkv .. hkv + 3, a wave each
// Where the results of a sequence's heads are: of head hkv * group + g, the shared keys' at p_base + (hkv * p_parts + k) * R +
// r0 + g and its own ones' at s_base + (hkv * s_parts + k) * group + g.
struct Join {
  int R, p_base, p_parts, r0;
  int s_base, s_parts, done, spare;  // done: there is nothing to join
};
struct Group {
  int shared, i0, R, tiles;
  int parts, item, row, spare;
};

// The plan's layout, from sizes that host and device know.
struct PlanDims {
  int batch, n_groups, n_kv, group;
  int slots;  // workgroups that the device holds at once, about
  // A unit is a KV head and a row tile of a group, or a KV head of a sequence.  The key tiles of all are at most slots * share, and of
  // a unit's parts of `share` one is not full.
  __host__ __device__ int64_t max_items() const {
    const int64_t tiles = (int64_t)batch * group / kBM + (batch / 2 < n_groups ? batch / 2 : n_groups);
    return slots + n_kv * (batch + tiles);
  }
  __host__ __device__ int64_t max_rows() const { return (int64_t)slots * kBM + 2ll * n_kv * group * batch; }
  __host__ __device__ int64_t joins_at() const { return 64; }
  __host__ __device__ int64_t items_at() const { return joins_at() + batch * (int64_t)sizeof(Join); }
  __host__ __device__ int64_t groups_at() const { return items_at() + max_items() * (int64_t)sizeof(Item); }
  __host__ __device__ int64_t before_at() const { return groups_at() + n_groups * (int64_t)sizeof(Group); }
  __host__ __device__ int64_t order_at() const { return before_at() + 4 * ((int64_t)batch + 1); }
  __host__ __device__ int64_t named_at() const { return order_at() + 4 * (int64_t)batch; }
  __host__ __device__ int64_t bytes() const { return (named_at() + 4 * (int64_t)batch + 255) & ~(int64_t)255; }
  // A word that a plan of other sizes does not begin with.
  __host__ __device__ uint32_t check(int cap, int esize, int d_k) const {
    uint32_t h = 0x9E3779B9u;
    for (int x : {batch, n_groups, n_kv, group, slots, cap, esize, d_k}) h = (h ^ (uint32_t)x) * 0x01000193u + (h >> 15);
    return h;
  }
};
struct Head {
  uint32_t check;
  int n_items;
};

struct PlanParams {
  const int32_t* lens;
  const int32_t* members;
  const int32_t* starts;
  const int32_t* shared;
  char* plan;
  PlanDims d;
  int len_add, cap, bn;
  int fours;  // one item for four KV heads is possible
  uint32_t check;
};

// Key tiles from lo to hi, the first of them at lo's block of 16.
__device__ __forceinline__ int tiles_of(int lo, int hi, int bn) {
  return lo < hi ? (hi - (lo & ~(kBlk - 1)) + bn - 1) / bn : 0;
}
// Key tiles of an item at most: as many as `slots` workgroups have each if all end together.
__device__ __forceinline__ int share_of(int64_t work, int slots) {
  if (work < 1 << 30) return max((int)((unsigned)(work + slots - 1) / (unsigned)slots), kMinTiles);
  return (int)min(max((work + slots - 1) / slots, (int64_t)kMinTiles), (int64_t)1 << 30);
}
// Sequences of one own tile: an item for four KV heads where an item a head would be half a round of the device.  195 sequences of 11 to 16
// own positions, 24 / 8 heads of 128, bf16, 22.9 -> 20.3 us a layer; 120 of up to 60, 15 / 5 heads of 64, fp16, 15.1 -> 14.9; but 64
// of up to 500 behind 8192, of which eight have one tile, 32.2 -> 32.8.
__device__ __forceinline__ bool by_fours(const PlanParams& p, int64_t ones) { return p.fours && 2 * ones * p.d.n_kv >= p.d.slots; }
// A sequence's own positions lo .. len - 1: t tiles in `parts` parts a KV head, items `at` on, whose rows are `base` on in the
// workspace (-1: o).
struct Own {
  int b, lo, len, t;
  int parts, base, at, four;
};
// Its items of KV head h.
__device__ __forceinline__ void own_items(const PlanParams& p, Item* items, const Own& x, int h) {
  const int lo16 = x.lo & ~(kBlk - 1);
  if (x.four) {
    if (h % 4 == 0) items[x.at + h / 4] = Item{x.b, h, x.lo, x.len, kFour, 0, p.d.group, x.base < 0 ? -1 : x.base + h * p.d.group};
    return;
  }
  const int each = x.parts ? x.t / x.parts : 0, more = x.parts ? x.t - each * x.parts : 0;
  int t0 = 0;
  for (int k = 0; k < x.parts; ++k) {
    const int t1 = t0 + each + (k < more ? 1 : 0);
    items[x.at + h * x.parts + k] = Item{x.b, h, t0 ? lo16 + t0 * p.bn : x.lo, min(x.len, lo16 + t1 * p.bn), -1, 0, p.d.group,
                                         x.base < 0 ? -1 : x.base + (h * x.parts + k) * p.d.group};
    t0 = t1;
  }
}
// Item e of those of shared positions.  Workgroups are dealt to the 8 XCDs in turn: the row tiles of one range of keys stand 8
// apart.
__device__ __forceinline__ Item group_item(const PlanParams& p, const Group* groups, const int* order, int e) {
  int lo = 0, hi = p.d.n_groups;  // the last group that begins at or before e, those without items passed over
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (groups[mid].item <= e) lo = mid;
    else hi = mid;
  }
  const Group g = groups[lo];
  const int rt = (g.R + kBM - 1) / kBM, ranges = p.d.n_kv * g.parts, in = e - g.item;
  const int whole = ranges / 8 * 8 * rt;
  int tile, range;
  if (in < whole) {
    const int r = in / 8, q = r / rt;
    range = q * 8 + in % 8;
    tile = r - q * rt;
  } else {
    const int some = ranges % 8;
    tile = (in - whole) / some;
    range = ranges - some + (in - whole) - tile * some;
  }
  const int h = range / g.parts, k = range - h * g.parts;
  const int each = g.tiles / g.parts, more = g.tiles - each * g.parts;
  const int t0 = k * each + min(k, more), t1 = t0 + each + (k < more ? 1 : 0);
  return Item{order[g.i0], h, t0 * p.bn, min(g.shared, t1 * p.bn), g.i0, tile * kBM, g.R, g.row + range * g.R + tile * kBM};
}

// As many sequences and groups as threads at most, a thread each of either: what the threads need of one another is in LDS.  Few
// waves where they do: a step of the plan is a barrier more than anything (16 sequences, 6.4 us with 16 waves, 5.6
// with 4, 4.9 since three of its scans share no sums and wait for nobody's reads).  Items are many waves' work: 256 sequences of 8 KV
// heads, 4 / 8 / 16 waves 9.2 / 8.5 / 9.6 us.
template <int W>
__global__ __launch_bounds__(64 * W) void plan_one_kernel(PlanParams p) {
  constexpr int kThreads = 64 * W;
  __shared__ int s_start[kThreads + 1], s_shared[kThreads], s_before[kThreads + 1], s_order[kThreads], s_named[kThreads],
      s_len[kThreads];
  __shared__ Group s_group[kThreads];
  __shared__ Own s_own[kThreads];
  __shared__ int s_in[1][W], s_work[3][W], s_places[4][W], s_bucket[64], s_back;
  const PlanDims& d = p.d;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = tid < d.batch ? p.members[tid] : -1;
  s_named[tid] = -1;
  if (tid < 64) s_bucket[tid] = 0;
  if (tid < d.n_groups) {
    s_start[tid] = min(max(p.starts[tid], 0), d.batch);
    s_shared[tid] = min(max(p.shared[tid], 0), p.cap);
  }
  if (tid == 0) {
    s_start[d.n_groups] = min(max(p.starts[d.n_groups], 0), d.batch);
    s_back = 0;
  }
  if (tid < d.batch) {
    const int64_t n = (int64_t)p.lens[tid] + p.len_add;
    s_len[tid] = (int)(n < 0 ? 0 : n > p.cap ? p.cap : n);
  }
  __syncthreads();
  // this thread's sequence: its group, and whether it shares if the group does
  int g = 0;
  bool listed = (unsigned)b < (unsigned)d.batch && tid >= s_start[0] && tid < s_start[d.n_groups];
  if (listed) atomicMax(&s_named[b], tid);
  if (tid < d.n_groups && s_start[tid + 1] < s_start[tid]) s_back = 1;
  for (int hi = d.n_groups; hi - g > 1;) {
    const int mid = (g + hi) >> 1;
    if (s_start[mid] <= tid) g = mid;
    else hi = mid;
  }
  const int len = listed ? s_len[b] : 0;
  __syncthreads();
  const int shared = s_back ? 0 : s_shared[g];  // starts that go back: groups overlap, and nobody shares
  listed = listed && s_named[b] == tid;  // a sequence named twice is its last place's
  const bool in = listed && shared > 0 && len >= shared;
  int n_in[1] = {in ? 1 : 0}, all_in[1];
  block_scan<true>(n_in, all_in, s_in);
  if (tid < d.batch) s_before[tid] = n_in[0] - (in ? 1 : 0);
  if (tid == 0) s_before[d.batch] = all_in[0];
  if (in) {
    s_order[n_in[0] - 1] = b;
    ((int*)(p.plan + d.order_at()))[n_in[0] - 1] = b;
  }
  __syncthreads();
  auto sharing = [&](int i) { return s_before[max(s_start[i + 1], s_start[i])] - s_before[s_start[i]]; };
  Group gr{};
  if (tid < d.n_groups && sharing(tid) >= 2)
    gr = Group{s_shared[tid], s_before[s_start[tid]], sharing(tid) * d.group, tiles_of(0, s_shared[tid], p.bn), 0, 0, 0, 0};
  const int row_tiles = (gr.R + kBM - 1) / kBM;
  const int peers = sharing(g), place = s_before[tid < d.batch ? tid : 0] - s_before[s_start[g]];
  const bool shares = in && peers >= 2;
  // work in 64 bits: the tiles' upper and lower halves
  const int t = listed ? tiles_of(shares ? shared : 0, len, p.bn) : 0;
  const int64_t both = (int64_t)row_tiles * gr.tiles + t;
  int w[3] = {(int)(both & 0xFFFF), (int)(both >> 16), t == 1}, work[3];
  block_scan<true>(w, work, s_work);
  const int share = share_of((((int64_t)work[1] << 16) + work[0]) * d.n_kv, d.slots);
  gr.parts = gr.R ? (gr.tiles + share - 1) / share : 0;
  const int parts = (t + share - 1) / share;
  const bool direct = !shares && parts == 1;
  const int gi = d.n_kv * gr.parts * ((gr.R + kBM - 1) / kBM), gn = d.n_kv * gr.parts * gr.R;
  const bool four = t == 1 && by_fours(p, work[2]);
  const int oi = four ? (d.n_kv + 3) / 4 : d.n_kv * parts, on = direct ? 0 : d.n_kv * parts * d.group;
  int x[4] = {gi, gn, oi, on}, total[4];
  block_scan<true>(x, total, s_places);
  gr.item = x[0] - gi;
  gr.row = x[1] - gn;
  if (tid < d.n_groups) s_group[tid] = gr;
  // Where there are more items than workgroups the longest own ones come first, by 64ths of a share, so that the launch ends with short
  // ones (64 sequences of 1 to 500 own positions, 24 / 8 heads of 128, bf16: 27.9 -> 24.7 us).  Among equals whoever comes first.
  int own_at = x[2] - oi;
  if (total[0] + total[2] > d.slots) {
    const int bucket = parts ? 63 - min(63, (int)((int64_t)(four ? 4 : t / parts) * 64 / share)) : 0;
    if (oi) atomicAdd(&s_bucket[bucket], oi);
    __syncthreads();
    if (wave == 0) {
      const int n = s_bucket[lane];
      s_bucket[lane] = wave_scan(n) - n;
    }
    __syncthreads();
    if (oi) own_at = atomicAdd(&s_bucket[bucket], oi);
  } else {
    __syncthreads();
  }
  Item* const items = (Item*)(p.plan + d.items_at());
  Join* const joins = (Join*)(p.plan + d.joins_at());
  for (int e = tid; e < total[0]; e += kThreads) items[e] = group_item(p, s_group, s_order, e);
  if (tid < d.batch && s_named[tid] < 0) joins[tid] = Join{0, 0, 0, 0, 0, 0, 1, 0};
  if (listed) {
    const int base = total[1] + x[3] - on;
    const Group& of = s_group[g];
    joins[b] = shares ? Join{of.R, of.row, of.parts, place * d.group, base, parts, 0, 0} : Join{0, 0, 0, 0, base, parts, direct, 0};
    s_own[tid] = Own{b, shares ? shared : 0, len, t, parts, direct ? -1 : base, total[0] + own_at, four};
  } else {
    s_own[tid] = Own{0, 0, 0, 0, 0, 0, 0, 0};
  }
  __syncthreads();
  for (int i = tid; i < d.batch * d.n_kv; i += kThreads) own_items(p, items, s_own[i / d.n_kv], i % d.n_kv);
  if (tid == 0) *(Head*)p.plan = Head{p.check, total[0] + total[2]};
}

// Any number of them, 1024 at a time, with what the threads need of one another in the plan itself.
__global__ __launch_bounds__(kScanThreads) void plan_many_kernel(PlanParams p) {
  __shared__ int64_t sums[kScanWaves];
  __shared__ int s_back;
  const PlanDims& d = p.d;
  Item* const items = (Item*)(p.plan + d.items_at());
  Join* const joins = (Join*)(p.plan + d.joins_at());
  Group* const groups = (Group*)(p.plan + d.groups_at());
  int* const before = (int*)(p.plan + d.before_at());  // sequences that share before the i-th of the list
  int* const order = (int*)(p.plan + d.order_at());    // the sequences that share
  int* const named = (int*)(p.plan + d.named_at());    // the last place of the list that names a sequence, -1: none
  const int tid = threadIdx.x;
  auto start_of = [&](int g) { return min(max(p.starts[g], 0), d.batch); };
  // The i-th of the list: its sequence (-1: none) and group, tokens, positions that it shares if the group does.
  struct Member {
    int b, g, len, shared;
  };
  auto member = [&](int i) {
    Member m{-1, 0, 0, 0};
    if (i >= d.batch || i < start_of(0) || i >= start_of(d.n_groups)) return m;
    int lo = 0, hi = d.n_groups;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (start_of(mid) <= i) lo = mid;
      else hi = mid;
    }
    m.g = lo;
    const int b = p.members[i];
    if ((unsigned)b >= (unsigned)d.batch || named[b] != i) return m;
    m.b = b;
    const int64_t len = (int64_t)p.lens[b] + p.len_add;
    m.len = (int)(len < 0 ? 0 : len > p.cap ? p.cap : len);
    const int sh = s_back ? 0 : min(max(p.shared[lo], 0), p.cap);
    m.shared = m.len >= sh ? sh : 0;
    return m;
  };

  for (int b = tid; b < d.batch; b += kScanThreads) named[b] = -1;
  if (tid == 0) s_back = 0;
  __syncthreads();
  for (int g = tid; g < d.n_groups; g += kScanThreads)
    if (start_of(g + 1) < start_of(g)) s_back = 1;  // starts that go back: groups overlap, and nobody shares
  for (int i = tid; i < d.batch; i += kScanThreads) {
    const int b = p.members[i];
    if (i >= start_of(0) && i < start_of(d.n_groups) && (unsigned)b < (unsigned)d.batch) atomicMax(&named[b], i);
  }
  __syncthreads();
  for (int b = tid; b < d.batch; b += kScanThreads)
    if (named[b] < 0) joins[b] = Join{0, 0, 0, 0, 0, 0, 1, 0};
  // who shares
  int64_t n = 0;
  for (int i0 = 0; i0 < d.batch; i0 += kScanThreads) {
    const Member m = member(i0 + tid);
    const int in = m.shared > 0 ? 1 : 0;
    const Scan s = block_scan(in, sums);
    const int at = (int)(n + s.incl) - in;
    if (i0 + tid < d.batch) before[i0 + tid] = at;
    if (in) order[at] = m.b;
    n += s.total;
  }
  if (tid == 0) before[d.batch] = (int)n;
  __syncthreads();
  // the groups' key tiles, and where their items and results begin
  int64_t work = 0;
  for (int g0 = 0; g0 < d.n_groups; g0 += kScanThreads) {
    const int g = g0 + tid;
    int64_t w = 0;
    Group x{};
    if (g < d.n_groups) {
      const int s = start_of(g), e = max(start_of(g + 1), s);
      x.i0 = before[s];
      const int in = before[e] - x.i0;
      if (in >= 2) {
        x.shared = min(max(p.shared[g], 0), p.cap);
        x.R = in * d.group;
        x.tiles = tiles_of(0, x.shared, p.bn);
        w = (int64_t)((x.R + kBM - 1) / kBM) * x.tiles;
      }
      groups[g] = x;
    }
    work += block_scan(w, sums).total;
  }
  __syncthreads();
  // place of a sequence among its group's that share, -1: it shares nothing
  auto place = [&](const Member& m, int i) {
    return m.shared <= 0 || groups[m.g].R == 0 ? -1 : before[i] - groups[m.g].i0;
  };
  int64_t ones = 0;
  for (int i0 = 0; i0 < d.batch; i0 += kScanThreads) {
    const Member m = member(i0 + tid);
    const int t = m.b >= 0 ? tiles_of(place(m, i0 + tid) >= 0 ? m.shared : 0, m.len, p.bn) : 0;
    work += block_scan(t, sums).total;
    ones += block_scan(t == 1, sums).total;
  }
  const int share = share_of(work * d.n_kv, d.slots);
  int64_t item = 0, row = 0;
  for (int g0 = 0; g0 < d.n_groups; g0 += kScanThreads) {
    const int g = g0 + tid;
    int64_t ni = 0, nr = 0;
    Group x{};
    if (g < d.n_groups) {
      x = groups[g];
      x.parts = x.R ? (int)((x.tiles + share - 1) / share) : 0;
      ni = (int64_t)d.n_kv * x.parts * ((x.R + kBM - 1) / kBM);
      nr = (int64_t)d.n_kv * x.parts * x.R;
    }
    const Scan si = block_scan(ni, sums), sr = block_scan(nr, sums);
    if (g < d.n_groups) {
      x.item = (int)(item + si.incl - ni);
      x.row = (int)(row + sr.incl - nr);
      groups[g] = x;
    }
    item += si.total;
    row += sr.total;
  }
  __syncthreads();
  const int group_items = (int)item;
  for (int i0 = 0; i0 < d.batch; i0 += kScanThreads) {
    const Member m = member(i0 + tid);
    const int j = m.b >= 0 ? place(m, i0 + tid) : -1;
    const int lo = j >= 0 ? m.shared : 0, t = m.b >= 0 ? tiles_of(lo, m.len, p.bn) : 0, parts = (t + share - 1) / share;
    const bool direct = j < 0 && parts == 1;
    const bool four = t == 1 && by_fours(p, ones);
    const int oi = four ? (d.n_kv + 3) / 4 : d.n_kv * parts, on = direct ? 0 : d.n_kv * parts * d.group;
    const Scan si = block_scan(oi, sums), sn = block_scan(on, sums);
    if (m.b >= 0) {
      const int base = (int)(row + sn.incl - on);
      const Group& of = groups[m.g];
      joins[m.b] = j >= 0 ? Join{of.R, of.row, of.parts, j * d.group, base, parts, 0, 0} : Join{0, 0, 0, 0, base, parts, direct, 0};
      const Own x{m.b, lo, m.len, t, parts, direct ? -1 : base, (int)(item + si.incl) - oi, four};
      for (int h = 0; h < d.n_kv; ++h) own_items(p, items, x, h);
    }
    item += si.total;
    row += sn.total;
  }
  for (int e = tid; e < group_items; e += kScanThreads) items[e] = group_item(p, groups, order, e);
  if (tid == 0) *(Head*)p.plan = Head{p.check, (int)item};
}

struct SharedParams {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  PageMap pm;
  const char* plan;
  PlanDims d;
  uint32_t check;
  uint32_t group_magic;  // row / group = mulhi(row, group_magic) (group > 1)
  int n_head;
  float2* ml;   // by row of results: m and l
  float* acc;   // [row][D]
  int vec_out;
  int64_t q_sb, q_sh, o_sb, o_sh;
  int64_t k_sp, k_sh, k_sr, v_sp, v_sh, v_sr;
  float scale_log2;
};

// LDS of a workgroup: two key tiles of the wide form, and for the narrow one as many blocks of 16 keys a wave as keep two workgroups
// (three at d_k 64 in 16 bits) on a CU.
template <typename T, int D>
constexpr int lds_bytes() { return D * T::size == 128 ? 48 << 10 : 64 << 10; }

// Few rows, 16 NRB (tl_attn_narrow.h).
template <typename T, int D, int NRB>
__device__ __forceinline__ void narrow_item(const SharedParams& p, const Item& it, char* smem, float2 (&s_ml)[4][32]) {
  using N = Narrow<T, D>;
  using B = typename T::bits;
  constexpr int NB = lds_bytes<T, D>() / (8 * kBlk * D * T::size);  // blocks in a wave's ring
  const int lane = threadIdx.x & 63, wave = uni((int)threadIdx.x >> 6);
  const int lr = lane & 15, g = lane >> 4;
  const int b0 = it.lo >> kBlkShift;
  const int blocks = ((it.hi + kBlk - 1) >> kBlkShift) - b0;
  NarrowKeys k{p.pm, it.b, (const char*)((const B*)p.k + it.hkv * p.k_sh), (const char*)((const B*)p.v + it.hkv * p.v_sh),
               p.k_sp * T::size, p.v_sp * T::size, (uint32_t)(p.k_sr * T::size), (uint32_t)(p.v_sr * T::size), it.hi,
               (blocks - wave + 3) >> 2};
  auto pos_of = [&](int t) { return (b0 + wave + 4 * t) << kBlkShift; };
  // the first pages are on their way while the queries' rows are found
  int pages = narrow_pages(k, 0, pos_of);
  typename N::Q q[NRB];
#pragma unroll
  for (int rb = 0; rb < NRB; ++rb) {
    const int row = it.row0 + 16 * rb + lr;
    const bool there = row < it.R;
    const int seq = p.d.group == 1 ? row : (int)__umulhi((uint32_t)row, p.group_magic);
    const int hq = there ? it.hkv * p.d.group + (row - seq * p.d.group) : 0;
    const int b = !there || it.i0 < 0 ? it.b : ((const int*)(p.plan + p.d.order_at()))[it.i0 + seq];
    N::load_q(q[rb], (const char*)((const B*)p.q + b * p.q_sb + hq * p.q_sh), there && p.scale_log2 != 0.f, g,
              p.scale_log2 < 0.f ? 0x80000000u : 0u);
  }
  NarrowState<D, NRB> st;
  auto whole = [&](int pos) { return pos >= it.lo && pos + kBlk <= it.hi; };
  auto seen = [&](int key, int) { return key >= it.lo && key < it.hi; };
  const float scale = p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2);
  // a sequence's own keys are read once in the launch: they need not stay in the caches (8 groups of 32 sequences with up to 1000 own
  // positions behind 4096 shared ones, 24 / 8 heads of 128, bf16: 140 -> 130 us a layer)
  narrow_stream<T, D, NRB, NB>(st, q, k, pages, smem, wave, lane, scale, it.i0 < 0, pos_of, whole, seen);
  narrow_join<T, D, NRB>(st, smem, s_ml, wave, lane);
  constexpr int CH = D / 4;
  const int rows = min(it.R - it.row0, 16 * NRB);
  for (int i = threadIdx.x; i < rows * CH; i += kThreads) {
    const int r = i / CH, c = i - r * CH;
    float m, l;
    const f32x4 a = narrow_result<D, NRB>(smem, s_ml, r, c, m, l);
    if (it.out < 0) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      B* out = (B*)p.o + it.b * p.o_sb + (int64_t)(it.hkv * p.d.group + r) * p.o_sh + 4 * c;
      store4<T>(out, a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv, p.vec_out);
    } else {
      const int64_t at = it.out + r;
      if (c == 0) p.ml[at] = make_float2(m, l);
      *(f32x4*)(p.acc + at * D + 4 * c) = a;
    }
  }
}

// One key tile of a sequence's own, a wave a KV head: no join, and a fourth of the workgroups.
template <typename T, int D, int NRB>
__device__ __forceinline__ void four_item(const SharedParams& p, const Item& it, char* smem) {
  using N = Narrow<T, D>;
  using B = typename T::bits;
  constexpr int NB = lds_bytes<T, D>() / (8 * kBlk * D * T::size);
  const int lane = threadIdx.x & 63, wave = uni((int)threadIdx.x >> 6);
  const int lr = lane & 15, g = lane >> 4;
  const int hkv = it.hkv + wave;
  if (hkv >= p.d.n_kv) return;
  const int b0 = it.lo >> kBlkShift;
  NarrowKeys k{p.pm, it.b, (const char*)((const B*)p.k + hkv * p.k_sh), (const char*)((const B*)p.v + hkv * p.v_sh),
               p.k_sp * T::size, p.v_sp * T::size, (uint32_t)(p.k_sr * T::size), (uint32_t)(p.v_sr * T::size), it.hi,
               ((it.hi + kBlk - 1) >> kBlkShift) - b0};
  auto pos_of = [&](int t) { return (b0 + t) << kBlkShift; };
  const int pages = narrow_pages(k, 0, pos_of);
  typename N::Q q[NRB];
#pragma unroll
  for (int rb = 0; rb < NRB; ++rb) {
    const int r = 16 * rb + lr;
    const bool there = r < it.R;
    N::load_q(q[rb], (const char*)((const B*)p.q + it.b * p.q_sb + (hkv * p.d.group + (there ? r : 0)) * p.q_sh),
              there && p.scale_log2 != 0.f, g, p.scale_log2 < 0.f ? 0x80000000u : 0u);
  }
  NarrowState<D, NRB> st;
  auto whole = [&](int pos) { return pos >= it.lo && pos + kBlk <= it.hi; };
  auto seen = [&](int key, int) { return key >= it.lo && key < it.hi; };
  const float scale = p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2);
  narrow_stream<T, D, NRB, NB>(st, q, k, pages, smem, wave, lane, scale, true, pos_of, whole, seen);
#pragma unroll
  for (int rb = 0; rb < NRB; ++rb) {
    const float l = tlp::sum_xor32(sum_xor16(st.l[rb]));
    const int r = 16 * rb + lr;
    if (r >= it.R) continue;
    if (it.out < 0) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      B* out = (B*)p.o + it.b * p.o_sb + (int64_t)(hkv * p.d.group + r) * p.o_sh + 4 * g;
#pragma unroll
      for (int db = 0; db < D / 16; ++db) {
        const f32x4 a = st.o[rb][db];
        store4<T>(out + 16 * db, a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv, p.vec_out);
      }
    } else {
      const int64_t at = it.out + wave * p.d.group + r;
      if (g == 0) p.ml[at] = make_float2(st.m[rb] - Tile<T, D>::kLift, l);
#pragma unroll
      for (int db = 0; db < D / 16; ++db) *(f32x4*)(p.acc + at * D + 16 * db + 4 * g) = st.o[rb][db];
    }
  }
}

// More rows: 4 waves of 32.  Key tiles by LDS-DMA, the next one while this one is used.
template <typename T, int D>
__device__ __forceinline__ void wide_item(const SharedParams& p, const Item& it, char* smem) {
  using TL = Tile<T, D>;
  using B = typename T::bits;
  constexpr int BN = tile_keys<T>();
  constexpr int ROWB = D * T::size;
  constexpr int TILEB = BN * ROWB;
  constexpr int NSL = ROWB / 16;    // 16-byte slots of a row
  constexpr int RPR = 1024 / ROWB;  // rows of one LDS-DMA
  constexpr int WROWS = BN / 4;     // rows that a wave loads of a tile: within one block of 16
  constexpr int NDMA = WROWS / RPR;
  constexpr int NDB = TL::NDB, NMB = TL::NMB;
  constexpr int TB = BN / kBlk;  // blocks of a tile
  static_assert(WROWS <= kBlk && kBlk % WROWS == 0 && NDMA >= 1, "a wave's rows lie in one block");
  const int* order = (const int*)(p.plan + p.d.order_at());

  const int lane = threadIdx.x & 63, wave = uni((int)threadIdx.x >> 6);
  const int lq = lane & 31, h = lane >> 5;
  const int lo16 = it.lo & ~(kBlk - 1);
  const int tiles = (it.hi - lo16 + BN - 1) / BN;
  const int32_t* table = p.pm.table + (int64_t)it.b * p.pm.max_pages;

  // The pages of 64 / TB tiles from pages_t on, lane by lane: tile (pages_t + lane / TB)'s block lane % TB.
  int pages = 0, pages_t = 0;
  uint64_t gone_lanes = 0;
  auto look_up = [&](int t) __attribute__((always_inline)) {
    pages_t = t;
    const int e = (lo16 + min(t + lane / TB, tiles - 1) * BN + kBlk * (lane % TB)) >> p.pm.shift;
    pages = e < p.pm.max_pages ? table[e] : -1;
    gone_lanes = __ballot((unsigned)pages >= (unsigned)p.pm.n_pages);
  };
  look_up(0);

  // this lane's row
  const int row = it.row0 + 32 * wave + lq;
  const bool there = row < it.R;
  const bool wave_rows = it.row0 + 32 * wave < it.R;
  const int seq = p.d.group == 1 ? row : (int)__umulhi((uint32_t)row, p.group_magic);
  const int hq = it.hkv * p.d.group + (row - seq * p.d.group);
  const int b = !there || it.i0 < 0 ? it.b : order[it.i0 + seq];
  typename TL::Q q;
  TL::load_q(q, (const char*)((const B*)p.q + b * p.q_sb + (there ? hq : 0) * p.q_sh), there && p.scale_log2 != 0.f, h,
             p.scale_log2 < 0.f ? 0x80000000u : 0u);
  const float scale = p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2);

  const uint32_t k_row = (uint32_t)(p.k_sr * T::size), v_row = (uint32_t)(p.v_sr * T::size);
  uint32_t koff[NDMA], voff[NDMA];
#pragma unroll
  for (int i = 0; i < NDMA; ++i) {
    const int r = i * RPR + lane / NSL, rt = wave * WROWS + r;
    koff[i] = r * k_row + (((lane % NSL) ^ k_swz<T, D>(rt)) << 4);
    voff[i] = r * v_row + (((lane % NSL) ^ v_swz<T, D>(rt)) << 4);
  }
  const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) char*)smem;
  // Rows past the last key, and rows of pages that are not there, read as zeros.
  const char* const kbase = (const char*)((const B*)p.k + it.hkv * p.k_sh);
  const char* const vbase = (const char*)((const B*)p.v + it.hkv * p.v_sh);
  auto load_tile = [&](int t, int buf) __attribute__((always_inline)) {
    const int pos0 = lo16 + t * BN + wave * WROWS;
    int rows = min(max(it.hi - pos0, 0), WROWS);
    const int id = __builtin_amdgcn_readlane(pages, (t - pages_t) * TB + (wave * WROWS) / kBlk);
    const int in = pos0 & ((1 << p.pm.shift) - 1);
    const bool page = (unsigned)id < (unsigned)p.pm.n_pages;
    if (!page) rows = 0;
    const int64_t at = page ? id : 0;
    const i32x4 rk = uniform_rsrc(kbase + at * p.k_sp * T::size + (int64_t)in * k_row, rows ? (rows - 1) * k_row + ROWB : 0);
    const i32x4 rv = uniform_rsrc(vbase + at * p.v_sp * T::size + (int64_t)in * v_row, rows ? (rows - 1) * v_row + ROWB : 0);
    const uint32_t la = lds0 + buf * 2 * TILEB + wave * WROWS * ROWB;
#pragma unroll
    for (int i = 0; i < NDMA; ++i) lds_dma16(rk, koff[i], la + i * 1024);
#pragma unroll
    for (int i = 0; i < NDMA; ++i) lds_dma16(rv, voff[i], la + TILEB + i * 1024);
  };

  f32x16 o[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[db][r] = 0.f;
  float m = -INFINITY, l = 0.f;
  f32x16 la;  // kSumMfma: the row's sum in every register
#pragma unroll
  for (int r = 0; r < 16; ++r) la[r] = 0.f;

  // One key tile: scores, softmax, O^T.  whole: every key of it is seen.
  auto step = [&](int k0, const char* kt, uint32_t gone, bool whole) __attribute__((always_inline)) {
    f32x16 s[NMB];
    __builtin_amdgcn_s_setprio(1);
    TL::scores(s, q, kt, lq, h);
    __builtin_amdgcn_s_setprio(0);
    if (!whole) {
      asm volatile("");  // a branch: as selects the tests would run for every tile
      const int lo = it.lo - k0 - 4 * h, hi = it.hi - k0 - 4 * h;
#pragma unroll
      for (int mb = 0; mb < NMB; ++mb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int kl = 32 * mb + 8 * (r >> 2) + (r & 3);
          s[mb][r] = kl >= lo && kl < hi && !((gone >> (2 * mb + (r >> 3))) & 1) ? s[mb][r] : -INFINITY;
        }
    }
    float mx = s[0][0];
#pragma unroll
    for (int mb = 0; mb < NMB; ++mb)
#pragma unroll
      for (int r = 0; r < 16; r += 2)
        mx = __builtin_elementwise_maximum(__builtin_elementwise_maximum(mx, s[mb][r]), s[mb][r + 1]);
    mx = tlp::max_xor32(mx) * scale;
    // the maximum moves only when a score passes it by kRescale (it only bounds the exponents)
    if (__any(mx > m + TL::kRescale)) {
      const float mn = fmaxf(m, mx);
      const float a = fast_exp2(m - (mn == -INFINITY ? 0.f : mn));
      m = mn;
      l *= a;
      if constexpr (TL::kSumMfma) {
#pragma unroll
        for (int r = 0; r < 16; ++r) la[r] *= a;
      }
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] *= a;
    }
    const float shift = m == -INFINITY ? 0.f : m - TL::kLift;
#pragma unroll
    for (int mb = 0; mb < NMB; ++mb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[mb][r] = fast_exp2(fmaf(s[mb][r], scale, -shift));
        if (!TL::kSumMfma) l += s[mb][r];
      }
    __builtin_amdgcn_s_setprio(1);
    // whole weights, as paged_attention_decode has them: these items wait for memory more than for the products (64 sequences behind
    // 8192 positions 67.4 -> 70.0 us for two layers and their plan, 256 behind 8 prefixes 242.9 -> 242.5)
    TL::template values<true>(o, la, s, kt + TILEB, lane);
    __builtin_amdgcn_s_setprio(0);
  };

  load_tile(0, 0);
  for (int t = 0; t < tiles; ++t) {
    wait_vmcnt<0>();  // this wave's rows of tile t are in LDS
    lds_barrier();    // everybody's are, and tile t - 1 has been read
    const int buf = t & 1;
    const uint32_t gone = (uint32_t)(gone_lanes >> ((t - pages_t) * TB)) & ((1u << TB) - 1);
    if (t + 1 < tiles) {
      if (t + 1 - pages_t == 64 / TB) look_up(t + 1);
      load_tile(t + 1, buf ^ 1);
    }
    if (!wave_rows) continue;
    const int k0 = lo16 + t * BN;
    step(k0, smem + buf * 2 * TILEB, gone, k0 >= it.lo && k0 + BN <= it.hi && gone == 0);
  }
  if (!there) return;
  l = TL::kSumMfma ? la[0] : tlp::sum_xor32(l);
  if (it.out < 0) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    B* out = (B*)p.o + b * p.o_sb + hq * p.o_sh;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int a = 0; a < 4; ++a)
        store4<T>(out + 32 * db + 8 * a + 4 * h, o[db][4 * a] * inv, o[db][4 * a + 1] * inv, o[db][4 * a + 2] * inv,
                  o[db][4 * a + 3] * inv, p.vec_out);
    return;
  }
  const int64_t at = it.out + 32 * wave + lq;
  if (h == 0) p.ml[at] = make_float2(m - TL::kLift, l);
  float* out = p.acc + at * D;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int a = 0; a < 4; ++a)
      *(f32x4*)(out + 32 * db + 8 * a + 4 * h) = f32x4{o[db][4 * a], o[db][4 * a + 1], o[db][4 * a + 2], o[db][4 * a + 3]};
}

// A workgroup an item, by its rows.
template <typename T, int D>
__global__ __launch_bounds__(kThreads, 2) void shared_kernel(SharedParams p) {
  __shared__ __attribute__((aligned(1024))) char smem[lds_bytes<T, D>()];
  __shared__ float2 s_ml[4][32];
  const Head head = *(const Head*)p.plan;
  const Item it = ((const Item*)(p.plan + p.d.items_at()))[blockIdx.x];  // the grid is no larger than the room for them
  if (head.check != p.check || (int)blockIdx.x >= head.n_items) return;
  const int rows = it.R - it.row0;
  if (it.i0 == kFour) {
    if (rows <= 16) four_item<T, D, 1>(p, it, smem);
    else four_item<T, D, 2>(p, it, smem);
    return;
  }
  if (rows <= 16) narrow_item<T, D, 1>(p, it, smem, s_ml);
  else if (rows <= 32) narrow_item<T, D, 2>(p, it, smem, s_ml);
  else wide_item<T, D>(p, it, smem);
}

// A wave a query head of a sequence: the states of its items, shared ones first, 4 (d_k 128: 2) at a time side by side in the wave, 16
// bytes a lane (17 states of 64 features: 3.6 us, one by one 4.9).  Every load that goes by the plan alone, of up to 32 states (16), is
// on its way before the first is waited for; twice as many at d_k 128 took the registers of half the waves (256 sequences, 7.0 us for
// 5.4).  (A join by the last of a sequence's items to end, in the same launch: the shared keys' last item joins a whole tile's rows,
// one after the other; 64 sequences behind 8192 positions took 57 us for 25 + 5.8, 16 beams 14.7 for 6.4 + 4.9.)
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void shared_join_kernel(SharedParams p) {
  using B = typename T::bits;
  constexpr int LPR = D / 4, G = 64 / LPR, U = 8;  // lanes of a row, rows of a load, loads on their way
  const int lane = threadIdx.x & 63, sub = lane / LPR, c = lane % LPR;
  const int b = blockIdx.y, hq = (int)blockIdx.x * (kThreads / 64) + uni((int)threadIdx.x >> 6);
  if (hq >= p.n_head) return;
  const Head head = *(const Head*)p.plan;
  const Join x = ((const Join*)(p.plan + p.d.joins_at()))[b];
  if (head.check != p.check || x.done) return;
  const int hkv = hq / p.d.group, g = hq - hkv * p.d.group;
  const int parts = x.p_parts + x.s_parts;
  const int p_row = x.p_base + hkv * x.p_parts * x.R + x.r0 + g;
  const int s_row = x.s_base + (hkv * x.s_parts - x.p_parts) * p.d.group + g;
  auto row_of = [&](int k) { return k < x.p_parts ? p_row + k * x.R : s_row + k * p.d.group; };
  auto ml_at = [&](int k) { return k < parts ? p.ml[row_of(k)] : make_float2(-INFINITY, 0.f); };
  f32x4 r[U];
  auto load = [&](int k0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * G + sub;
      r[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (k0 + u * G < parts && k < parts) r[u] = *(const f32x4*)(p.acc + (int64_t)row_of(k) * D + 4 * c);
    }
  };
  const float2 e0 = ml_at(lane);
  load(0);
  float mx = e0.x;
  for (int k = lane + 64; k < parts; k += 64) mx = fmaxf(mx, ml_at(k).x);
#pragma unroll
  for (int off = 32; off; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off));
  const float base = mx == -INFINITY ? 0.f : mx;
  float l = 0.f, w = 0.f;
  f32x4 a = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < parts; k0 += U * G) {
    if ((k0 & 63) == 0) {
      const float2 e = k0 ? ml_at(k0 + lane) : e0;
      w = fast_exp2(e.x - base);
      l += e.y * w;
    }
    if (k0) load(k0);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k0 + u * G < parts) {
        const float wu = __shfl(w, (k0 + u * G + sub) & 63);
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = fmaf(r[u][i], wu, a[i]);
      }
  }
#pragma unroll
  for (int off = 32; off; off >>= 1) l += __shfl_xor(l, off);
#pragma unroll
  for (int off = LPR; off < 64; off <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] += __shfl_xor(a[i], off);
  if (sub) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  store4<T>((B*)p.o + b * p.o_sb + (int64_t)hq * p.o_sh + 4 * c, a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv, p.vec_out);
}

template <typename T, int D>
int launch_shared(const SharedParams& p, hipStream_t st) {
  hipLaunchKernelGGL((shared_kernel<T, D>), dim3((unsigned)p.d.max_items()), dim3(kThreads), 0, st, p);
  const int e = tl_launch_status();
  if (e) return e;
  constexpr int kHeads = kThreads / 64;
  hipLaunchKernelGGL((shared_join_kernel<T, D>), dim3((unsigned)((p.n_head + kHeads - 1) / kHeads), (unsigned)p.d.batch), dim3(kThreads), 0, st, p);
  return tl_launch_status();
}

bool known_dtype(int dtype) { return dtype == TL_DTYPE_F32 || dtype == TL_DTYPE_F16 || dtype == TL_DTYPE_BF16; }

// Sizes of a plan; false: not supported.
bool dims_of(PlanDims& d, int batch, int n_groups, int n_head, int n_kv_head, int d_k) {
  if (batch < 1 || batch > kMostBatch || n_groups < 1 || n_groups > kMostBatch || n_head < 1 || n_kv_head < 1 ||
      n_head % n_kv_head || n_head / n_kv_head > kBM || (d_k != 64 && d_k != 128))
    return false;
  // Two workgroups a CU.  (Three fit at d_k 64 in 16 bits, 15 / 5 heads: 64 sequences behind 8192 positions 20.0 us with two, 21.3
  // with three; 256 of up to 1000 own positions behind 8 prefixes 45.7 and 42.7; in fp32, where two fit, 80 behind 2 of 6624 32.3 and 36.1.)
  d = PlanDims{batch, n_groups, n_kv_head, n_head / n_kv_head, 2 * tl_device_cus()};
  // rows are divided by a multiplication (see the windowed attention's), items and rows counted in 32 bits
  const int64_t rows = (int64_t)batch * d.group + kBM;
  return rows * d.group < ((int64_t)1 << 32) && d.max_items() < (1 << 30) && d.max_rows() < (1 << 30);
}

}  // namespace

extern "C" {

size_t tl_shared_plan_bytes(int batch, int n_groups, int n_head, int n_kv_head, int d_k) {
  PlanDims d;
  return dims_of(d, batch, n_groups, n_head, n_kv_head, d_k) ? (size_t)d.bytes() : 0;
}

size_t tl_shared_workspace_bytes(int batch, int n_groups, int n_head, int n_kv_head, int d_k) {
  PlanDims d;
  return dims_of(d, batch, n_groups, n_head, n_kv_head, d_k) ? (size_t)d.max_rows() * (d_k + 2) * sizeof(float) : 0;
}

int tl_shared_plan(const int32_t* cache_lens, int len_add, const int32_t* members, const int32_t* group_starts,
                   const int32_t* shared_lens, int batch, int n_groups, int n_head, int n_kv_head, int d_k, int max_pages,
                   int page_size, int dtype, void* plan, size_t plan_bytes, void* stream) {
  const int shift = page_shift(page_size);
  if (!cache_lens || !members || !group_starts || !shared_lens || !plan || batch < 1 || n_groups < 1 || n_head < 1 ||
      n_kv_head < 1 || n_head % n_kv_head || max_pages < 1 || shift < 0 || !known_dtype(dtype) || ((uintptr_t)plan & 15))
    return TL_ERR_INVALID;
  const int64_t cap = (int64_t)max_pages << shift;
  if (cap > (1 << 30)) return TL_ERR_INVALID;
  PlanParams p{};
  if (!dims_of(p.d, batch, n_groups, n_head, n_kv_head, d_k)) return TL_ERR_UNSUPPORTED;
  if (plan_bytes < (size_t)p.d.bytes()) return TL_ERR_INVALID;
  const struct {
    const void* at;
    int64_t n;
  } in[] = {{cache_lens, batch}, {members, batch}, {group_starts, n_groups + 1}, {shared_lens, n_groups}};
  for (const auto& x : in)
    if (tl_overlap(plan, (size_t)p.d.bytes(), x.at, (size_t)x.n * 4)) return TL_ERR_INVALID;
  p.lens = cache_lens;
  p.members = members;
  p.starts = group_starts;
  p.shared = shared_lens;
  p.plan = (char*)plan;
  p.len_add = len_add;
  p.cap = (int)cap;
  const int esize = dtype == TL_DTYPE_F32 ? 4 : 2;
  p.bn = esize == 4 ? tile_keys<F32>() : tile_keys<BF16>();
  p.fours = n_kv_head > 1 && p.d.group <= 32;
  p.check = p.d.check(p.cap, esize, d_k);
  hipStream_t st = tl_resolve_stream(stream);
  const int most = batch > n_groups ? batch : n_groups;
  if (most <= 128) hipLaunchKernelGGL(plan_one_kernel<4>, dim3(1), dim3(256), 0, st, p);
  else if (most <= 512) hipLaunchKernelGGL(plan_one_kernel<8>, dim3(1), dim3(512), 0, st, p);
  else if (most <= 1024) hipLaunchKernelGGL(plan_one_kernel<16>, dim3(1), dim3(1024), 0, st, p);
  else hipLaunchKernelGGL(plan_many_kernel, dim3(1), dim3(kScanThreads), 0, st, p);
  return tl_launch_status();
}

int tl_paged_attention_shared(const void* q, const void* k_pages, const void* v_pages, const int32_t* page_table, int max_pages,
                              int n_pages, int page_size, const void* plan, size_t plan_bytes, int n_groups, void* o,
                              void* workspace, size_t workspace_bytes, int batch, int n_head, int n_kv_head, int d_k,
                              const int64_t* q_strides, const int64_t* k_page_strides, const int64_t* v_page_strides,
                              const int64_t* o_strides, float sm_scale, int dtype, void* stream) {
  if (batch == 0 || n_head == 0) return 0;
  const int shift = page_shift(page_size);
  if (!q || !k_pages || !v_pages || !page_table || !plan || !o || !workspace || batch < 0 || n_groups < 1 || n_head < 0 ||
      n_kv_head < 1 || n_head % n_kv_head || max_pages < 1 || n_pages < 1 || shift < 0 || !q_strides || !k_page_strides ||
      !v_page_strides || !o_strides || !known_dtype(dtype) || ((uintptr_t)workspace & 15) || ((uintptr_t)plan & 15))
    return TL_ERR_INVALID;
  const int64_t cap = (int64_t)max_pages << shift;
  if (cap > (1 << 30)) return TL_ERR_INVALID;
  SharedParams p{};
  if (!dims_of(p.d, batch, n_groups, n_head, n_kv_head, d_k)) return TL_ERR_UNSUPPORTED;
  if (plan_bytes < (size_t)p.d.bytes() ||
      workspace_bytes < tl_shared_workspace_bytes(batch, n_groups, n_head, n_kv_head, d_k))
    return TL_ERR_INVALID;
  // rows are moved 16 bytes at a time, a block of 16 with 32-bit offsets
  const int esize = dtype == TL_DTYPE_F32 ? 4 : 2;
  const int64_t vec = 16 / esize;
  const int64_t read[] = {q_strides[0],      q_strides[1],      k_page_strides[0], k_page_strides[1],
                          k_page_strides[2], v_page_strides[0], v_page_strides[1], v_page_strides[2]};
  for (int64_t s : read)
    if (s < 0 || s % vec) return TL_ERR_UNSUPPORTED;
  if (o_strides[0] < 0 || o_strides[1] < 0) return TL_ERR_UNSUPPORTED;
  if (k_page_strides[2] > (1 << 24) || v_page_strides[2] > (1 << 24)) return TL_ERR_UNSUPPORTED;
  if (((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages) & 15) return TL_ERR_UNSUPPORTED;
  // an item's workgroup may write o while others still read q
  auto rows = [&](const void* at, int64_t n0, int64_t n1, int64_t n2, int64_t s0, int64_t s1, int64_t s2) {
    return Rows3{at, {n0, n1, n2}, {s0 * esize, s1 * esize, s2 * esize}, (int64_t)d_k * esize};
  };
  const Rows3 out = rows(o, batch, n_head, 1, o_strides[0], o_strides[1], 0);
  auto pool = [&](const void* at, const int64_t* s) { return rows(at, n_pages, n_kv_head, page_size, s[0], s[1], s[2]); };
  if (rows_overlap(out, rows(q, batch, n_head, 1, q_strides[0], q_strides[1], 0)) ||
      rows_overlap(out, pool(k_pages, k_page_strides)) || rows_overlap(out, pool(v_pages, v_page_strides)))
    return TL_ERR_INVALID;
  p.q = q;
  p.k = k_pages;
  p.v = v_pages;
  p.o = o;
  p.pm = PageMap{page_table, max_pages, n_pages, shift};
  p.plan = (const char*)plan;
  p.check = p.d.check((int)cap, esize, d_k);
  p.group_magic = (uint32_t)((((uint64_t)1 << 32) + p.d.group - 1) / p.d.group);
  p.n_head = n_head;
  p.ml = (float2*)workspace;
  p.acc = (float*)workspace + 2 * p.d.max_rows();
  p.vec_out = ((uintptr_t)o % (4 * esize)) == 0 && o_strides[0] % 4 == 0 && o_strides[1] % 4 == 0;
  p.q_sb = q_strides[0], p.q_sh = q_strides[1];
  p.o_sb = o_strides[0], p.o_sh = o_strides[1];
  p.k_sp = k_page_strides[0], p.k_sh = k_page_strides[1], p.k_sr = k_page_strides[2];
  p.v_sp = v_page_strides[0], p.v_sh = v_page_strides[1], p.v_sr = v_page_strides[2];
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  hipStream_t st = tl_resolve_stream(stream);
  switch (dtype) {
    case TL_DTYPE_F32: return d_k == 64 ? launch_shared<F32, 64>(p, st) : launch_shared<F32, 128>(p, st);
    case TL_DTYPE_F16: return d_k == 64 ? launch_shared<F16, 64>(p, st) : launch_shared<F16, 128>(p, st);
    default: return d_k == 64 ? launch_shared<BF16, 64>(p, st) : launch_shared<BF16, 128>(p, st);
  }
}

}  // extern "C"
