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
// Two steps.  The plan (plan_kernel, one workgroup), from the lengths, which only the device knows: which sequences share,
// and the list of items, each a tile of up to 128 query rows of one KV head and a range of keys, all of about the same length.
// It holds for every layer of a model's step.  Then each layer's attention: a workgroup an item (shared_kernel) and, where a
// row's keys are in several items, their join (shared_join_kernel).
#include "tl_attn_tile.h"
#include "tl_paged.h"

#include <math.h>

using namespace tlat;
using namespace tlpg;

namespace {

constexpr int kThreads = 256;
constexpr int kBM = 128;  // query rows of an item at most
constexpr int kMostBatch = 65535;
constexpr int kMinTiles = 4;  // key tiles of an item at least
constexpr int kScanThreads = 64 * kScanWaves;

// Rows row0 .. of a block of R: row r is query head hkv * group + r % group of the i0 + r / group-th sequence that shares (i0
// < 0: of sequence b), over positions [lo, hi) of sequence b's pages.  lo is a multiple of 16 but for the first own ones.
struct Item {
  int b, hkv, lo, hi;
  int i0, row0, R, out;  // out: where the rows' results go in the workspace, -1: to o, as they are all there is
};
// Where the results of a sequence's heads are: of head hkv * group + g, the shared keys' at p_base + (hkv * p_parts + k) * R +
// r0 + g and its own ones' at s_base + (hkv * s_parts + k) * group + g.
struct Join {
  int b, R, p_base, p_parts;
  int r0, s_base, s_parts, done;  // done: an item has written o itself, or there is nothing to write
};
struct Group {
  int shared, i0, R, tiles;
  int parts, item, row, spare;
};

// The plan's layout, from sizes that host and device know.
struct PlanDims {
  int batch, n_groups, n_kv, group, slots;
  __host__ __device__ int64_t max_items() const {
    const int64_t tiles = (int64_t)batch * group / kBM + (batch / 2 < n_groups ? batch / 2 : n_groups);
    return slots + n_kv * (batch + tiles);
  }
  // rows of partial results: parts are at most 1 + tiles / share, and sum tiles / share at most slots
  __host__ __device__ int64_t max_rows() const { return (int64_t)slots * (kBM + group) + 2ll * n_kv * group * batch; }
  __host__ __device__ int64_t items_at() const { return 64; }
  __host__ __device__ int64_t joins_at() const { return items_at() + max_items() * (int64_t)sizeof(Item); }
  __host__ __device__ int64_t groups_at() const { return joins_at() + batch * (int64_t)sizeof(Join); }
  __host__ __device__ int64_t before_at() const { return groups_at() + n_groups * (int64_t)sizeof(Group); }
  __host__ __device__ int64_t order_at() const { return before_at() + 4 * ((int64_t)batch + 1); }
  __host__ __device__ int64_t bytes() const { return (order_at() + 4 * (int64_t)batch + 255) & ~(int64_t)255; }
  // A word that a plan of other sizes does not begin with.
  __host__ __device__ uint32_t check(int cap, int esize, int d_k) const {
    uint32_t h = 0x9E3779B9u;
    for (int x : {batch, n_groups, n_kv, group, slots, cap, esize, d_k}) h = (h ^ (uint32_t)x) * 0x01000193u + (h >> 15);
    return h;
  }
};
struct Head {
  uint32_t check;
  int n_items, n_joins;
};

struct PlanParams {
  const int32_t* lens;
  const int32_t* members;
  const int32_t* starts;
  const int32_t* shared;
  char* plan;
  PlanDims d;
  int len_add, cap, bn;
  uint32_t check;
};

__global__ __launch_bounds__(kScanThreads) void plan_kernel(PlanParams p) {
  __shared__ int64_t sums[kScanWaves];
  const PlanDims& d = p.d;
  Item* const items = (Item*)(p.plan + d.items_at());
  Join* const joins = (Join*)(p.plan + d.joins_at());
  Group* const groups = (Group*)(p.plan + d.groups_at());
  int* const before = (int*)(p.plan + d.before_at());  // sequences that share before the i-th of the list
  int* const order = (int*)(p.plan + d.order_at());    // the sequences that share
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
    if ((unsigned)b >= (unsigned)d.batch) return m;
    m.b = b;
    const int64_t len = (int64_t)p.lens[b] + p.len_add;
    m.len = (int)(len < 0 ? 0 : len > p.cap ? p.cap : len);
    const int sh = min(max(p.shared[lo], 0), p.cap);
    m.shared = m.len >= sh ? sh : 0;
    return m;
  };
  auto tiles_of = [&](int lo, int hi) { return lo < hi ? (hi - (lo & ~(kBlk - 1)) + p.bn - 1) / p.bn : 0; };

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
  // the groups' and the sequences' units: one for each KV head and row tile
  int64_t work = 0, units = 0, rows = 0;
  for (int g0 = 0; g0 < d.n_groups; g0 += kScanThreads) {
    const int g = g0 + tid;
    int64_t w = 0, u = 0;
    Group x{};
    if (g < d.n_groups) {
      const int s = start_of(g), e = max(start_of(g + 1), s);
      x.i0 = before[s];
      const int in = before[e] - x.i0;
      if (in >= 2) {
        x.shared = min(max(p.shared[g], 0), p.cap);
        x.R = in * d.group;
        x.tiles = tiles_of(0, x.shared);
        u = (x.R + kBM - 1) / kBM;
        w = u * x.tiles;
      }
      groups[g] = x;
    }
    work += block_scan(w, sums).total;
    units += block_scan(u, sums).total;
    rows += block_scan(x.R, sums).total;
  }
  if (rows > (int64_t)d.batch * d.group) {  // starts that go back: groups overlap, and nobody shares
    for (int g = tid; g < d.n_groups; g += kScanThreads) groups[g].R = groups[g].tiles = 0;
    work = units = 0;
  }
  __syncthreads();
  // place of a sequence among its group's that share, -1: it shares nothing
  auto place = [&](const Member& m, int i) {
    if (m.shared <= 0 || groups[m.g].R == 0) return -1;
    const int j = before[i] - groups[m.g].i0;
    return j >= 0 && j < groups[m.g].R / d.group ? j : -1;
  };
  for (int i0 = 0; i0 < d.batch; i0 += kScanThreads) {
    const Member m = member(i0 + tid);
    int t = 0;
    if (m.b >= 0) t = tiles_of(place(m, i0 + tid) >= 0 ? m.shared : 0, m.len);
    work += block_scan(t, sums).total;
    units += block_scan(t > 0 ? 1 : 0, sums).total;
  }
  work *= d.n_kv;
  units *= d.n_kv;
  // Key tiles of an item: items are about `slots`, and each unit's last one is short.
  const int64_t aim = max((int64_t)d.slots - units, (int64_t)d.slots / 2);
  const int64_t share = max((work + aim - 1) / aim, (int64_t)kMinTiles);
  // where the groups' items and results begin
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
  const int p_items = (int)item;
  // the sequences' own items, and where their results are
  for (int i0 = 0; i0 < d.batch; i0 += kScanThreads) {
    const int i = i0 + tid;
    const Member m = member(i);
    const int j = m.b >= 0 ? place(m, i) : -1;
    const int lo = j >= 0 ? m.shared : 0;
    const int t = m.b >= 0 ? tiles_of(lo, m.len) : 0;
    const int parts = (int)((t + share - 1) / share);
    const bool direct = j < 0 && parts == 1;
    const Scan si = block_scan((int64_t)d.n_kv * parts, sums);
    const int64_t nr = direct ? 0 : (int64_t)d.n_kv * parts * d.group;
    const Scan sr = block_scan(nr, sums);
    const int base = (int)(row + sr.incl - nr);
    if (i < d.batch) {
      Join x{m.b, 0, 0, 0, 0, base, parts, direct || m.b < 0 ? 1 : 0};
      if (j >= 0) {
        const Group& g = groups[m.g];
        x.R = g.R, x.p_base = g.row, x.p_parts = g.parts, x.r0 = j * d.group;
      }
      joins[i] = x;
      Item* at = items + item + si.incl - (int64_t)d.n_kv * parts;
      const int lo16 = lo & ~(kBlk - 1);
      for (int h = 0; h < d.n_kv; ++h) {
        int t0 = 0;
        for (int k = 0; k < parts; ++k) {
          const int t1 = t0 + t / parts + (k < t % parts ? 1 : 0);
          *at++ = Item{m.b, h, t0 ? lo16 + t0 * p.bn : lo, min(m.len, lo16 + t1 * p.bn), -1, 0, d.group,
                       direct ? -1 : base + (h * parts + k) * d.group};
          t0 = t1;
        }
      }
    }
    item += si.total;
    row += sr.total;
  }
  // The groups' items.  Workgroups are dealt to the 8 XCDs in turn: the row tiles of one range of keys stand 8 apart.
  for (int e = tid; e < p_items; e += kScanThreads) {
    int lo = 0, hi = d.n_groups;  // the last group that begins at or before e, those without items passed over
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (groups[mid].item <= e) lo = mid;
      else hi = mid;
    }
    const Group g = groups[lo];
    const int rt = (g.R + kBM - 1) / kBM, ranges = d.n_kv * g.parts, in = e - g.item;
    const int whole = ranges / 8 * 8 * rt;
    int tile, range;
    if (in < whole) {
      range = in / (8 * rt) * 8 + in % 8;
      tile = in / 8 % rt;
    } else {
      const int some = ranges % 8;
      range = ranges - some + (in - whole) % some;
      tile = (in - whole) / some;
    }
    const int h = range / g.parts, k = range - h * g.parts;
    const int each = g.tiles / g.parts, more = g.tiles % g.parts;
    const int t0 = k * each + min(k, more), t1 = t0 + each + (k < more ? 1 : 0);
    items[e] = Item{order[g.i0], h, t0 * p.bn, min(g.shared, t1 * p.bn), g.i0, tile * kBM, g.R,
                    g.row + range * g.R + tile * kBM};
  }
  if (tid == 0) *(Head*)p.plan = Head{p.check, (int)item, d.batch};
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

// 4 waves of 32 rows; key tiles by LDS-DMA, the next one while this one is used.  Every row sees every key of the item.
template <typename T, int D>
__global__ __launch_bounds__(kThreads, 2) void shared_kernel(SharedParams p) {
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
  __shared__ __attribute__((aligned(1024))) char smem[4 * TILEB];  // (K, V) twice

  const Head head = *(const Head*)p.plan;
  if (head.check != p.check || (int)blockIdx.x >= head.n_items) return;
  const Item it = ((const Item*)(p.plan + p.d.items_at()))[blockIdx.x];
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
    TL::values(o, la, s, kt + TILEB, lane);
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
  if (h == 0) p.ml[at] = make_float2(m, l);
  float* out = p.acc + at * D;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int a = 0; a < 4; ++a)
      *(f32x4*)(out + 32 * db + 8 * a + 4 * h) = f32x4{o[db][4 * a], o[db][4 * a + 1], o[db][4 * a + 2], o[db][4 * a + 3]};
}

// A wave a query head of a sequence: the states of its items, shared ones first.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void shared_join_kernel(SharedParams p) {
  using B = typename T::bits;
  constexpr int NJ = D / 64, U = 8;
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * (kThreads / 64) + uni((int)threadIdx.x >> 6);
  const int i = (int)(unit / p.n_head), hq = (int)(unit - (int64_t)i * p.n_head);
  const Head head = *(const Head*)p.plan;
  if (head.check != p.check || i >= head.n_joins) return;
  const Join x = ((const Join*)(p.plan + p.d.joins_at()))[i];
  if (x.done) return;
  const int hkv = hq / p.d.group, g = hq - hkv * p.d.group;
  const int parts = x.p_parts + x.s_parts;
  auto row_of = [&](int k) {
    return k < x.p_parts ? (int64_t)x.p_base + (int64_t)(hkv * x.p_parts + k) * x.R + x.r0 + g
                         : (int64_t)x.s_base + (hkv * x.s_parts + k - x.p_parts) * p.d.group + g;
  };
  auto ml_at = [&](int k) { return k < parts ? p.ml[row_of(k)] : make_float2(-INFINITY, 0.f); };
  const float2 e0 = ml_at(lane);
  float mx = e0.x;
  for (int k = lane + 64; k < parts; k += 64) mx = fmaxf(mx, ml_at(k).x);
#pragma unroll
  for (int off = 32; off; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off));
  const float base = mx == -INFINITY ? 0.f : mx;
  float l = 0.f, a[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) a[j] = 0.f;
  for (int k0 = 0; k0 < parts; k0 += 64) {
    const float2 e = k0 ? ml_at(k0 + lane) : e0;
    const float w = fast_exp2(e.x - base);
    l += e.y * w;
    const int n = min(64, parts - k0);
    for (int k1 = 0; k1 < n; k1 += U) {
      float r[U][NJ];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < NJ; ++j) r[u][j] = k1 + u < n ? p.acc[row_of(k0 + k1 + u) * D + NJ * lane + j] : 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float wu = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), (k1 + u) & 63));
#pragma unroll
        for (int j = 0; j < NJ; ++j) a[j] = fmaf(r[u][j], wu, a[j]);
      }
    }
  }
#pragma unroll
  for (int off = 32; off; off >>= 1) l += __shfl_xor(l, off);
  B* o = (B*)p.o + x.b * p.o_sb + (int64_t)hq * p.o_sh;
#pragma unroll
  for (int j = 0; j < NJ; ++j) o[NJ * lane + j] = from_f32<T>(l == 0.f ? 0.f : a[j] / l);
}

template <typename T, int D>
int launch_shared(const SharedParams& p, hipStream_t st) {
  hipLaunchKernelGGL((shared_kernel<T, D>), dim3((unsigned)p.d.max_items()), dim3(kThreads), 0, st, p);
  const int e = tl_launch_status();
  if (e) return e;
  const int64_t waves = (int64_t)p.d.batch * p.n_head;
  hipLaunchKernelGGL((shared_join_kernel<T, D>), dim3((unsigned)((waves + 3) / 4)), dim3(kThreads), 0, st, p);
  return tl_launch_status();
}

bool known_dtype(int dtype) { return dtype == TL_DTYPE_F32 || dtype == TL_DTYPE_F16 || dtype == TL_DTYPE_BF16; }

// Sizes of a plan; false: not supported.
bool dims_of(PlanDims& d, int batch, int n_groups, int n_head, int n_kv_head, int d_k) {
  if (batch < 1 || batch > kMostBatch || n_groups < 1 || n_groups > kMostBatch || n_head < 1 || n_kv_head < 1 ||
      n_head % n_kv_head || n_head / n_kv_head > kBM || (d_k != 64 && d_k != 128))
    return false;
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
  p.check = p.d.check(p.cap, esize, d_k);
  hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(kScanThreads), 0, tl_resolve_stream(stream), p);
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
