// Attention of many query rows through a sliding window with sinks, over K and V given by
// strides or in pages.
//
// Query row i of sequence b stands at position base + i and sees key j when
//   j <= base + i,  and with a window w > 0 only  j > base + i - w  or  j < sinks.
// base is seq_k - seq_q for K / V given by strides (bottom-right, as the causal prefill) and
// cache_lens[b] for pages.  O = softmax(scale q . K^T over the keys seen) V, by one pass over the keys
// with the running maximum m and sum l of the softmax in fp32 (log2 domain).  A row that
// sees no key gives zeros.  The reference has no windows and no pages; its causal attention
// (attention_gqa.py:21-146) is window = 0.
//
// A workgroup is 4 waves of 32 query rows of one KV head, its query heads side by side (row r is token r /
// group).  It walks only the key tiles that any of its 128 rows sees: the sinks' tiles, then those from the
// first row's window on to the last row's position.  As in the causal prefill the products are transposed, S^T =
// K . Q^T and O^T = V^T . P^T, on 32 x 32 MFMA blocks: lane l of the accumulator holds query row l % 32, so
// maximum and rescale are a lane's own (one exchange between l and l ^ 32), and P^T goes from the accumulator's
// registers straight into the second product.  K / V tiles come by LDS-DMA, the next one while this one is used;
// V is read by transposing LDS reads.
//
// Bound by the matrix products and, at d_k 64, as much by exp and the conversions: 8192 tokens, window 1024, 24 / 8 heads
// of 128, bf16: 126 to 137 us; 4 x 500 rows on prefixes of 2875 to 3835, 15 / 5 heads of 64, fp16: 40.7 to 43 us, by device.
#include "tl_attn_narrow.h"

#include <math.h>

using namespace tlat;
using namespace tlpg;

namespace {

constexpr int kThreads = 256;
constexpr int kBM = 128;  // query rows of a workgroup
constexpr int kMinShare = 4;  // key tiles of a part at least
constexpr int kWaveParts = 4;  // parts of a row tile that the waves join themselves
constexpr int kMostRows = 1 << 28;     // query rows of a sequence
constexpr int kWholeWindow = 3 << 29;  // positions lie in [-2^28, 2^30 + 2^28): a window this long hides nothing, and
                                       // below it position - window fits in 32 bits

struct WinParams {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  PageMap pm;  // pages: k / v strides are {page, head, row}; else {batch, head, row}
  const int32_t* lens;
  const int32_t* new_lens;
  const int32_t* starts;  // packed rows: sequence b's are q's rows starts[b] .. starts[b + 1] - 1 (q_sb = o_sb = 0), else NULL
  int packed_rows;        // rows of q
  int batch, n_head, n_kv, group, seq_q, seq_k, n_qt;
  uint32_t group_magic;  // row / group = mulhi(row, group_magic) for the rows there are (group > 1)
  int window, sinks;
  int slots;           // workgroups that the keys are shared by; 0: a row tile's keys are not divided
  int room;            // parts that there may be (slots > 0): the workspace holds as many, the grid has as many workgroups
  int key_cap;         // key tiles of a row tile count as this many at most, so that their sum fits in 32 bits
  int q_shift, n_lvl, xcd_groups;  // how workgroups are dealt (window_fwd_kernel)
  int vec_out;         // o's rows take 4 elements at once
  uint64_t tag;        // this call's, where the waves join the parts; 0: window_join_kernel does
  uint64_t* words;     // [part][wave]: the tag where the part's results are there
  float* ws;           // partial results by part (slots > 0)
  int64_t q_sb, q_sh, q_ss;
  int64_t k_sb, k_sh, k_ss;
  int64_t v_sb, v_sh, v_ss;
  int64_t o_sb, o_sh, o_ss;
  float scale_log2;
};

// The token of a row.  Integer divisions are long dependent chains, and what runs before a short call's first
// load counts: this one is a multiplication.
__device__ __forceinline__ int token_of(const WinParams& p, int row) {
  return p.group == 1 ? row : (int)__umulhi((uint32_t)row, p.group_magic);
}

// Where a sequence's query rows stand: token i at position base + i and in row first + i of q, nq tokens, no key from `end` on.
struct Rows {
  int base, nq, end, first;
};
template <bool PAGED>
__device__ __forceinline__ Rows rows_of(const WinParams& p, int b) {
  Rows r;
  r.first = 0;
  if constexpr (PAGED) {
    // rows before position -seq_q see nothing, as those there; lengths past 2^30 count as 2^30
    r.base = min(max(p.lens[b], -p.seq_q), 1 << 30);
    if (p.starts) {
      r.first = min(max(p.starts[b], 0), p.packed_rows);
      r.nq = min(max(min(max(p.starts[b + 1], 0), p.packed_rows) - r.first, 0), p.seq_q);
    } else {
      r.nq = p.new_lens ? min(max(p.new_lens[b], 0), p.seq_q) : p.seq_q;
    }
    r.end = min(r.base + r.nq, p.pm.max_pages << p.pm.shift);
  } else {
    r.base = p.seq_k - p.seq_q;
    r.nq = p.seq_q;
    r.end = p.seq_k;
  }
  return r;
}

// The key tiles of row tile qt: ns of the sinks', then those from t0 on.
struct Keys {
  int ns, t0, tiles, end;
  __device__ __forceinline__ int key0(int t) const { return t < ns ? t : t - ns + t0; }  // in tiles
};
template <int BN>
__device__ __forceinline__ Keys keys_of(const WinParams& p, const Rows& r, int qt) {
  Keys k{0, 0, 0, r.end};
  const int p0 = r.base + token_of(p, qt * kBM);
  const int p1 = min(r.base + min(token_of(p, qt * kBM + kBM - 1) + 1, r.nq), r.end) - 1;  // last key any row sees
  if (p1 < 0) return k;
  if (p.window > 0) {
    k.t0 = min(max(p0 - p.window + 1, 0) / BN, p1 / BN + 1);  // rows past the pages may see none of the window's
    k.ns = (min(p.sinks, p1 + 1) + BN - 1) / BN;
    if (k.t0 <= k.ns) k.ns = k.t0 = 0;
  }
  k.tiles = k.ns + p1 / BN - k.t0 + 1;
  return k;
}

// How divided keys are dealt.  Every sequence's row tiles have the same number of parts, as its last one needs for
// `share` key tiles a part, and its parts, by (KV head, part, row tile), stand behind those of the sequences before it.  Only
// the device knows the lengths, so only it can make the parts about `slots`, equally long, without gaps between
// them: with a grid by the longest lengths that there could be, workgroups without work stood among the
// others, and 4 x 500 rows on prefixes of 2875 to 3835 (of at most 4608) took 47.8 us.  Lengths are walked 64 at a time by every
// workgroup; 2 rows of each of 8, 64 and 150 sequences, 131072 keys in all, 15 / 5 heads of 64, bf16, take 42, 33 and 35 us.
struct Seq {
  Rows r;
  int tiles, keys;  // row tiles, key tiles of the last of them
  int parts, all;   // parts of a row tile, of all of them and every KV head
  __device__ __forceinline__ void cut(const WinParams& p, int share) {
    parts = max(1, (int)((unsigned)(keys + share - 1) / (unsigned)share));
    all = tiles * parts * p.n_kv;
  }
};
template <int BN, bool PAGED>
__device__ __forceinline__ Seq seq_at(const WinParams& p, int b) {
  Seq s{{0, 0, 0, 0}, 0, 0, 0, 0};
  if (b < p.batch) {
    s.r = rows_of<PAGED>(p, b);
    s.tiles = (s.r.nq * p.group + kBM - 1) / kBM;
    if (s.tiles) s.keys = min(keys_of<BN>(p, s.r, s.tiles - 1).tiles, p.key_cap);
  }
  return s;
}
struct Deal {
  int share, total;
  Seq s;     // lane's sequence, of the first 64
  int incl;  // parts of all up to it
};
template <int BN, bool PAGED>
__device__ __forceinline__ Deal deal_of(const WinParams& p, int lane) {
  Deal d;
  d.s = seq_at<BN, PAGED>(p, lane);
  int work = last_lane(wave_scan(d.s.tiles * d.s.keys)), tiles = last_lane(wave_scan(d.s.tiles));
  for (int b0 = 64; b0 < p.batch; b0 += 64) {
    const Seq t = seq_at<BN, PAGED>(p, b0 + lane);
    work += last_lane(wave_scan(t.tiles * t.keys));
    tiles += last_lane(wave_scan(t.tiles));
  }
  // a sequence's last part is short: as many parts more than shares as there are row tiles.  Packed rows: single tokens and prompts
  // differ by more than that, and parts of an equal share, in more than one round, end closer together (30 tokens and 2 prompts of up to
  // 500 rows on 100 to 3500 positions, 24 / 8 heads of 128, bf16: 90 -> 82 us).
  const int aim = p.starts ? p.slots : max(p.slots - tiles * p.n_kv, p.slots / 2);
  // rounded up past the 32-bit quotient's error
  d.share = max((int)((float)work * (float)p.n_kv * __builtin_amdgcn_rcpf((float)aim) * 1.00001f) + 1, kMinShare);
  constexpr int kWhole = 1 << 30;
  while (true) {
    int longest = d.s.keys;
    d.s.cut(p, d.share);
    d.incl = wave_scan(d.s.all);
    d.total = last_lane(d.incl);
    for (int b0 = 64; b0 < p.batch; b0 += 64) {
      Seq t = seq_at<BN, PAGED>(p, b0 + lane);
      longest = max(longest, t.keys);
      t.cut(p, d.share);
      d.total += last_lane(wave_scan(t.all));
    }
    // Row tiles stay whole where their parts would take two rounds of the workgroups and two parts be as long as
    // the longest (sequences of 2 x share - 1 tiles and fewer beside short ones: 31 tokens on 4000 keys beside a prompt of 100,
    // 24 / 8 heads of 128, 99 us, cut in two 126), and where there is no room for the parts: more rows than the host said.
    if (d.share == kWhole || ((p.starts || d.total <= p.slots) && d.total <= p.room)) break;
    if (d.total <= p.room && __any(longest > 2 * d.share)) break;
    d.share = kWhole;
  }
  return d;
}
// The 64 sequences from b0 on, lane by lane: s, and the parts of all up to it.
template <int BN, bool PAGED>
__device__ __forceinline__ int parts_upto(const WinParams& p, const Deal& d, int b0, int lane, Seq& s) {
  s = d.s;
  int incl = d.incl;
  for (int b = 64; b <= b0; b += 64) {
    const int base = last_lane(incl);
    s = seq_at<BN, PAGED>(p, b + lane);
    s.cut(p, d.share);
    incl = base + wave_scan(s.all);
  }
  return incl;
}
// Lane li's sequence, on every lane.
__device__ __forceinline__ Seq seq_of_lane(const Seq& s, int li) {
  auto of = [&](int x) { return uni(__builtin_amdgcn_readlane(x, li)); };
  return Seq{{of(s.r.base), of(s.r.nq), of(s.r.end), of(s.r.first)}, of(s.tiles), of(s.keys), of(s.parts), of(s.all)};
}

// A part's results: 32 rows a wave, each wave's m and l (by row) and then its O^T, the registers as
// they lie in the lanes.
template <int D>
constexpr size_t part_floats() { return (size_t)4 * (64 + 64 * (D / 2)); }

// The only row tile of a sequence of at most 16 NRB rows: the first wave's lanes get what they would hold after the tiles t_lo .. t_hi - 1.
template <typename T, int D, int NRB>
__device__ __forceinline__ void narrow_tile(const WinParams& p, int b, int hkv, const Rows& rw, const Keys& ks, int t_lo, int t_hi,
                                            char* smem, float2 (&s_ml)[4][32], f32x16 (&o)[D / 32], float& m, float& l) {
  using N = Narrow<T, D>;
  using B = typename T::bits;
  constexpr int BN = tile_keys<T>(), TB = BN / kBlk;
  constexpr int NB = 4 * BN / (8 * kBlk) < 1 ? 1 : 4 * BN / (8 * kBlk);  // blocks in a wave's ring: 4 tiles of LDS
  const int lane = threadIdx.x & 63, wave = uni((int)threadIdx.x >> 6);
  const int lr = lane & 15, g = lane >> 4;
  const int rows = rw.nq * p.group;
  NarrowKeys k{p.pm, b, (const char*)((const B*)p.k + hkv * p.k_sh), (const char*)((const B*)p.v + hkv * p.v_sh),
               p.k_sb * T::size, p.v_sb * T::size, (uint32_t)(p.k_ss * T::size), (uint32_t)(p.v_ss * T::size), ks.end,
               ((t_hi - t_lo) * TB - wave + 3) >> 2};
  auto pos_of = [&](int t) {
    const int i = wave + 4 * t, tile = t_lo + i / TB;
    return ks.key0(tile) * BN + kBlk * (i % TB);
  };
  int pages = narrow_pages(k, 0, pos_of);
  typename N::Q q[NRB];
  int pos[NRB];
#pragma unroll
  for (int rb = 0; rb < NRB; ++rb) {
    const int row = 16 * rb + lr, tok = token_of(p, row);
    const bool there = row < rows;
    pos[rb] = rw.base + tok;
    N::load_q(q[rb], (const char*)((const B*)p.q + (there ? hkv * p.group + (row - tok * p.group) : 0) * p.q_sh +
                                   (int64_t)(rw.first + (there ? tok : 0)) * p.q_ss),
              there && p.scale_log2 != 0.f, g, p.scale_log2 < 0.f ? 0x80000000u : 0u);
  }
  NarrowState<D, NRB> st;
  auto whole = [&](int at) {
    return at + kBlk - 1 <= rw.base && at + kBlk <= ks.end &&
           (p.window <= 0 || at > rw.base + rw.nq - 1 - p.window || at + kBlk <= p.sinks);
  };
  auto seen = [&](int key, int rb) {
    return key <= pos[rb] && key < ks.end && (p.window <= 0 || key > pos[rb] - p.window || key < p.sinks);
  };
  const float scale = p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2);
  narrow_stream<T, D, NRB, NB>(st, q, k, pages, smem, wave, lane, scale, true, pos_of, whole, seen);
  narrow_join<T, D, NRB>(st, smem, s_ml, wave, lane);
  const int lq = lane & 31, h = lane >> 5;
  if (wave == 0 && lq < rows) {
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const f32x4 x = narrow_result<D, NRB>(smem, s_ml, lq, 8 * db + 2 * a + h, m, l);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[db][4 * a + e] = x[e];
      }
  }
}

// PACKED (and PAGED): the rows are packed (p.starts), and a row tile of few rows goes by 16 x 16 products: a packed batch is mostly
// single tokens, whose 128-row tiles would be empty but for a few rows.
template <typename T, int D, bool PAGED, bool PACKED>
__global__ __launch_bounds__(kThreads, 2) void window_fwd_kernel(WinParams p) {
  using TL = Tile<T, D>;
  using B = typename T::bits;
  constexpr int BN = tile_keys<T>();
  constexpr int ROWB = D * T::size;
  constexpr int TILEB = BN * ROWB;
  constexpr int NSL = ROWB / 16;              // 16-byte slots of a row
  constexpr int RPR = 1024 / ROWB;            // rows of one LDS-DMA
  constexpr int WROWS = BN / 4;               // rows that a wave loads of a tile: within one block of 16
  constexpr int NDMA = WROWS / RPR;
  constexpr int NDB = TL::NDB, NMB = TL::NMB;
  static_assert(WROWS <= kBlk && kBlk % WROWS == 0 && NDMA >= 1, "a wave's rows lie in one block");

  __shared__ __attribute__((aligned(1024))) char smem[4 * TILEB];  // (K, V) twice

  const int lane = threadIdx.x & 63;
  // Workgroups are dealt to the 8 XCDs in turn, and an XCD's L2 should hold the keys of few (sequence, KV head)s.
  // Undivided: these are cut into every 2^q_shift-th row tile, so that a multiple of 8 groups is dealt to the XCDs;
  // within an XCD the longest rows come first.  Divided: an XCD takes a contiguous range of the parts; packed rows' parts, which are
  // not equal work, are dealt in turn, the KV head first, so that with 8 of them an XCD reads one head's keys (30 tokens and 2 prompts
  // of up to 500 rows, 24 / 8 heads of 128, bf16: 82.5 -> 77 us).
  const int xcd = blockIdx.x % 8, at = blockIdx.x / 8;
  int b, hkv, qt, part = 0, parts = 1, place = 0, stride = 0;  // stride: places from part to part
  Rows rw;
  if (p.slots > 0) {
    const Deal d = deal_of<BN, PAGED>(p, lane);
    const int per = (d.total + 7) / 8;
    place = PACKED ? (int)blockIdx.x : xcd * per + at;
    if ((!PACKED && at >= per) || place >= d.total) return;
    Seq s;
    int b0 = 0, incl = parts_upto<BN, PAGED>(p, d, 0, lane, s);
    while (last_lane(incl) <= place) {
      b0 += 64;
      incl = parts_upto<BN, PAGED>(p, d, b0, lane, s);
    }
    const int li = uni(__ffsll((unsigned long long)__ballot(incl > place)) - 1);
    b = b0 + li;
    const int before = uni(__builtin_amdgcn_readlane(incl - s.all, li));
    s = seq_of_lane(s, li);
    rw = s.r;
    const int in = place - before;
    parts = s.parts;
    stride = s.tiles;
    int r;
    if constexpr (PACKED) {
      r = (int)((unsigned)in / (unsigned)p.n_kv);
      hkv = in - r * p.n_kv;
      place = before + hkv * parts * s.tiles + r;
    } else {
      hkv = (int)((unsigned)in / (unsigned)(parts * s.tiles));
      r = in - hkv * parts * s.tiles;
    }
    part = (int)((unsigned)r / (unsigned)s.tiles);
    qt = s.tiles - 1 - (r - part * s.tiles);
  } else {
    const int lvl = (int)((unsigned)at / (unsigned)p.xcd_groups);
    const int grp = (at - lvl * p.xcd_groups) * 8 + xcd;
    const int kvh = grp >> p.q_shift;
    qt = ((p.n_lvl - 1 - lvl) << p.q_shift) + (grp - (kvh << p.q_shift));
    if (qt >= p.n_qt || kvh >= p.batch * p.n_kv) return;
    b = (int)((unsigned)kvh / (unsigned)p.n_kv);
    hkv = kvh - b * p.n_kv;
    rw = rows_of<PAGED>(p, b);
  }
  const Keys ks = keys_of<BN>(p, rw, qt);
  if (qt * kBM >= rw.nq * p.group) return;

  const int wave = uni((int)threadIdx.x >> 6);
  const int lq = lane & 31, h = lane >> 5;

  // this lane's row: query head hkv * group + row % group of token row / group
  const int row = qt * kBM + 32 * wave + lq;
  const int tok = token_of(p, row);
  const int hq = hkv * p.group + (row - tok * p.group);
  const bool there = tok < rw.nq;
  const int pos = rw.base + tok;
  typename TL::Q q;
  TL::load_q(q, (const char*)((const B*)p.q + b * p.q_sb + hq * p.q_sh + (int64_t)(rw.first + tok) * p.q_ss),
             there && p.scale_log2 != 0.f,
             h, p.scale_log2 < 0.f ? 0x80000000u : 0u);
  const float scale = p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2);

  // ---- tile loads --------------------------------------------------------------
  const uint32_t k_row = (uint32_t)(p.k_ss * T::size), v_row = (uint32_t)(p.v_ss * T::size);
  uint32_t koff[NDMA], voff[NDMA];
#pragma unroll
  for (int i = 0; i < NDMA; ++i) {
    const int r = i * RPR + lane / NSL, rt = wave * WROWS + r;
    koff[i] = r * k_row + (((lane % NSL) ^ k_swz<T, D>(rt)) << 4);
    voff[i] = r * v_row + (((lane % NSL) ^ v_swz<T, D>(rt)) << 4);
  }
  const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) char*)smem;
  // The pages of 64 / TB tiles from pages_t on, lane by lane: tile (pages_t + lane / TB)'s block lane % TB; gone: which of
  // these there are not.  A load for each tile would be waited for with every LDS-DMA before it, which the compiler does
  // not know of, and scalar loads with every LDS read: 4 x 500 rows on prefixes took 48.5 and 53.1 us, 45.4 so.
  constexpr int TB = BN / kBlk;
  int pages = 0, pages_t = 0;
  uint64_t gone_lanes = 0;
  int t_lo = 0, t_hi = ks.tiles;
  if (parts > 1) {
    const int each = (int)((unsigned)ks.tiles / (unsigned)parts), more = ks.tiles - each * parts;
    t_lo = part * each + min(part, more);
    t_hi = t_lo + each + (part < more ? 1 : 0);
  }
  auto look_up = [&](int t) __attribute__((always_inline)) {
    if constexpr (PAGED) {
      pages_t = t;
      const int e = (ks.key0(min(t + lane / TB, t_hi - 1)) * BN + kBlk * (lane % TB)) >> p.pm.shift;
      pages = e < p.pm.max_pages ? p.pm.table[(int64_t)b * p.pm.max_pages + e] : -1;
      gone_lanes = __ballot((unsigned)pages >= (unsigned)p.pm.n_pages);
    }
  };
  // Rows past the last key, and rows of pages that are not there, read as zeros.
  const char* const kbase = (const char*)((const B*)p.k + (PAGED ? 0 : b * p.k_sb) + hkv * p.k_sh);
  const char* const vbase = (const char*)((const B*)p.v + (PAGED ? 0 : b * p.v_sb) + hkv * p.v_sh);
  auto load_tile = [&](int t, int buf) __attribute__((always_inline)) {
    const int pos0 = ks.key0(t) * BN + wave * WROWS;
    int rows = min(max(ks.end - pos0, 0), WROWS);
    int64_t ka, va;
    if constexpr (PAGED) {
      const int id = __builtin_amdgcn_readlane(pages, (t - pages_t) * TB + (wave * WROWS) / kBlk);
      const int in = pos0 & ((1 << p.pm.shift) - 1);
      const bool page = (unsigned)id < (unsigned)p.pm.n_pages;
      if (!page) rows = 0;
      const int64_t at = page ? id : 0;
      ka = at * p.k_sb * T::size + (int64_t)in * k_row;
      va = at * p.v_sb * T::size + (int64_t)in * v_row;
    } else {
      ka = (int64_t)pos0 * k_row;
      va = (int64_t)pos0 * v_row;
    }
    const i32x4 rk = uniform_rsrc(kbase + ka, rows ? (rows - 1) * k_row + ROWB : 0);
    const i32x4 rv = uniform_rsrc(vbase + va, rows ? (rows - 1) * v_row + ROWB : 0);
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

  // this wave's first and last position
  const int row0 = qt * kBM + 32 * wave;
  const int wp0 = uni(rw.base + token_of(p, row0));
  const int wp1 = uni(rw.base + min(token_of(p, row0 + 31), rw.nq - 1));
  const bool wave_rows = row0 < rw.nq * p.group;

  // One key tile: scores, softmax, O^T.  all: every row sees every key.
  auto step = [&](int k0, const char* kt, uint32_t gone, bool all) __attribute__((always_inline)) {
    f32x16 s[NMB];
    // matrix phases win over the other workgroup's softmax: 133 -> 130.4 us at 8192 tokens
    __builtin_amdgcn_s_setprio(1);
    TL::scores(s, q, kt, lq, h);
    __builtin_amdgcn_s_setprio(0);
    if (!all) {
      asm volatile("");  // a branch: as selects the tests would run for every tile
      // key k0 + kl + 4 h of this lane is seen if kl <= hi and (kl > lo or kl < sk)
      const int off = k0 + 4 * h;
      const int hi = min(pos, ks.end - 1) - off;
      const int lo = p.window > 0 ? pos - off - p.window : -BN - 1;
      const int sk = p.sinks - off;
#pragma unroll
      for (int mb = 0; mb < NMB; ++mb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int kl = 32 * mb + 8 * (r >> 2) + (r & 3);
          s[mb][r] = kl <= hi && (kl > lo || kl < sk) ? s[mb][r] : -INFINITY;
        }
      if (gone) {
        asm volatile("");
#pragma unroll
        for (int mb = 0; mb < NMB; ++mb)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if ((gone >> (2 * mb + (r >> 3))) & 1) s[mb][r] = -INFINITY;
      }
    }
    // IEEE maximum: one v_maximum3_f32 for two scores, where fmaxf first quiets its operands
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

  bool narrow = false;
  if constexpr (PACKED) {
    narrow = rw.nq * p.group <= 32;
    if (narrow) {
      __shared__ float2 s_ml[4][32];
      if (rw.nq * p.group <= 16) narrow_tile<T, D, 1>(p, b, hkv, rw, ks, t_lo, t_hi, smem, s_ml, o, m, l);
      else narrow_tile<T, D, 2>(p, b, hkv, rw, ks, t_lo, t_hi, smem, s_ml, o, m, l);
    }
  }
  if (!narrow) {
    if (t_lo < t_hi) {
      look_up(t_lo);
      load_tile(t_lo, 0);
    }
    for (int t = t_lo; t < t_hi; ++t) {
      wait_vmcnt<0>();  // this wave's rows of tile t are in LDS
      lds_barrier();    // everybody's are, and tile t - 1 has been read
      const int buf = (t - t_lo) & 1;
      const uint32_t gone = PAGED ? (uint32_t)(gone_lanes >> ((t - pages_t) * TB)) & ((1u << TB) - 1) : 0;
      if (t + 1 < t_hi) {
        if (PAGED && t + 1 - pages_t == 64 / TB) look_up(t + 1);
        load_tile(t + 1, buf ^ 1);
      }
      const int k0 = ks.key0(t) * BN;
      // does any row of this wave see a key of the tile, and does every row see all of them
      const bool any = wave_rows && k0 <= wp1 && (p.window <= 0 || k0 + BN - 1 > wp0 - p.window || k0 < p.sinks);
      if (!any) continue;
      const bool all = k0 + BN - 1 <= wp0 && k0 + BN <= ks.end && gone == 0 &&
                       (p.window <= 0 || k0 > wp1 - p.window || k0 + BN <= p.sinks);
      const char* kt = smem + buf * 2 * TILEB;
      step(k0, kt, gone, all);
    }
    l = TL::kSumMfma ? la[0] : tlp::sum_xor32(l);
  }
  // Divided keys: a wave leaves its part's results.  Where a row tile has few parts (p.tag: see window_entry) it waits for
  // its stores and then leaves the call's tag.  A wave that
  // finds the tags of all parts there (the last one does; several may, and write the same) adds them up in the
  // parts' order and takes the tags away, for a graph's next replay.  Nothing waits for another workgroup.  Stores,
  // tags and loads are device-coherent (sc1), which orders them across XCDs without write-backs of a cache.
  if (parts > 1) {
    if (!wave_rows) return;
    constexpr int kSc1 = 16;
    constexpr uint32_t kWaveBytes = (64 + 64 * (D / 2)) * 4;
    auto part_rsrc = [&](int k) {
      return __builtin_amdgcn_make_buffer_rsrc((char*)(p.ws + (size_t)k * part_floats<D>()) + wave * kWaveBytes, (short)0,
                                               (int)kWaveBytes, kBufRsrcWord3);
    };
    const auto mine = part_rsrc(place);
    const int o_at = 256 + 16 * lane, ml_at = 8 * lq;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const f32x4 x = {o[db][4 * a], o[db][4 * a + 1], o[db][4 * a + 2], o[db][4 * a + 3]};
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), mine, o_at, (4 * db + a) * 1024, kSc1);
      }
    if (h == 0) __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(m), __float_as_uint(l)}, mine, ml_at, 0, kSc1);
    if (!p.tag) return;
    wait_vmcnt<0>();
    const int first = place - part * stride;
    auto word = [&](int k) { return p.words + 4 * (size_t)(first + k * stride) + wave; };
    if (lane == 0) __hip_atomic_store(word(part), p.tag, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    wait_vmcnt<0>();
    bool all = true;
    for (int k0 = 0; k0 < parts; k0 += 64) {
      uint64_t x = p.tag;
      if (k0 + lane < parts) x = __hip_atomic_load(word(k0 + lane), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      all = all && __all(x == p.tag);
    }
    if (!all) return;
    asm volatile("" ::: "memory");
    float top = -INFINITY;
    for (int k = 0; k < parts; ++k)
      top = fmaxf(top, __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(part_rsrc(first + k * stride), ml_at, 0, kSc1)));
    const float shift = top == -INFINITY ? 0.f : top;
    l = 0.f;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[db][r] = 0.f;
    for (int k = 0; k < parts; ++k) {
      const auto rs = part_rsrc(first + k * stride);
      const u32x2 ml = __builtin_amdgcn_raw_buffer_load_b64(rs, ml_at, 0, kSc1);
      u32x4 x[NDB][4];
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int a = 0; a < 4; ++a) x[db][a] = __builtin_amdgcn_raw_buffer_load_b128(rs, o_at, (4 * db + a) * 1024, kSc1);
      const float f = fast_exp2(__uint_as_float(ml.x) - shift);
      l = fmaf(__uint_as_float(ml.y), f, l);
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[db][4 * a + e] = fmaf(__uint_as_float(x[db][a][e]), f, o[db][4 * a + e]);
    }
    for (int k = lane; k < parts; k += 64) __hip_atomic_store(word(k), (uint64_t)0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (!there) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  B* out = (B*)p.o + b * p.o_sb + hq * p.o_sh + (int64_t)(rw.first + tok) * p.o_ss;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int a = 0; a < 4; ++a)
      store4<T>(out + 32 * db + 8 * a + 4 * h, o[db][4 * a] * inv, o[db][4 * a + 1] * inv, o[db][4 * a + 2] * inv,
                o[db][4 * a + 3] * inv, p.vec_out);
}

// Joins the parts of a row tile where the waves do not: the same lanes that wrote them.
template <typename T, int D, bool PAGED>
__global__ __launch_bounds__(kThreads) void window_join_kernel(WinParams p) {
  using B = typename T::bits;
  constexpr int BN = tile_keys<T>();
  const int tile = blockIdx.x, db = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lq = lane & 31, h = lane >> 5;
  const int kvh = tile / p.n_qt;
  const int qt = tile - kvh * p.n_qt;
  const int b = kvh / p.n_kv;
  const int hkv = kvh - b * p.n_kv;
  if (qt * kBM >= rows_of<PAGED>(p, b).nq * p.group) return;
  const Deal d = deal_of<BN, PAGED>(p, lane);
  Seq s;
  const int incl = parts_upto<BN, PAGED>(p, d, b & ~63, lane, s);
  const int before = uni(__builtin_amdgcn_readlane(incl - s.all, b & 63));
  s = seq_of_lane(s, b & 63);
  const int parts = s.parts;
  if (qt >= s.tiles || parts <= 1) return;
  const int row = qt * kBM + 32 * wave + lq;
  const int tok = token_of(p, row);
  if (tok >= s.r.nq) return;
  const int hq = hkv * p.group + (row - tok * p.group);
  const float* w = p.ws + ((size_t)before + hkv * parts * s.tiles + (s.tiles - 1 - qt)) * part_floats<D>() +
                   (size_t)wave * (64 + 64 * (D / 2));
  const size_t step = (size_t)s.tiles * part_floats<D>();  // from part to part
  float m = -INFINITY;
  for (int i = 0; i < parts; ++i) m = fmaxf(m, w[i * step + 2 * lq]);
  const float shift = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  f32x4 o[4];
#pragma unroll
  for (int a = 0; a < 4; ++a) o[a] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < parts; ++i) {
    const float* wi = w + i * step;
    const float2 ml = *(const float2*)(wi + 2 * lq);
    const float f = fast_exp2(ml.x - shift);
    l = fmaf(ml.y, f, l);
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const f32x4 x = *(const f32x4*)(wi + 64 + (4 * db + a) * 256 + 4 * lane);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[a][e] = fmaf(x[e], f, o[a][e]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  B* out = (B*)p.o + b * p.o_sb + hq * p.o_sh + (int64_t)(s.r.first + tok) * p.o_ss;
#pragma unroll
  for (int a = 0; a < 4; ++a)
    store4<T>(out + 32 * db + 8 * a + 4 * h, o[a][0] * inv, o[a][1] * inv, o[a][2] * inv, o[a][3] * inv, p.vec_out);
}

// Key tiles that one row tile can have at most.
int64_t most_tiles(int64_t keys, int window, int sinks, int group, int bn) {
  int64_t n = (keys + bn - 1) / bn;
  if (window > 0) {
    const int64_t w = ((int64_t)window + kBM / group + 1) / bn + 2 + ((int64_t)sinks + bn - 1) / bn;
    n = n < w ? n : w;
  }
  return n < 1 ? 1 : n;
}

// Whether the keys of the row tiles are divided, and by how many workgroups: where the row tiles alone would not fill
// the device and a row tile can have several parts (1 x 100 rows on 4000 keys, 15 / 5 heads, d_k 64, fp16: 22.0 us,
// undivided 58; 1000 causal rows, 9 / 3 heads: 14.4 and 18.5).  The 16-bit kernels and fp32 at d_k 128 take as many
// workgroups as fit (1 x 500 rows on 4000 keys, 24 / 8 heads, d_k 128: fp16 39.6 us, one a CU 47; fp32 at 300 rows on
// 2000 keys 86 and 98); fp32 at d_k 64 is bound by its matrix products, which one workgroup a CU keeps busy (1023
// rows, window 256: 25.0 us, with two 30.1).  Returns the most parts there can be (0: undivided).
int64_t plan_slots(WinParams& p, int64_t tiles, int64_t keys, int d_k, int esize) {
  const int bn = esize == 2 ? 64 : 32;
  const int64_t most = most_tiles(keys, p.window, p.sinks, p.group, bn);
  const int64_t slots = (int64_t)tl_device_cus() * (d_k == 128 ? 2 : esize == 4 ? 1 : 3);
  p.slots = tiles < 1 || tiles >= slots || most < 2 * kMinShare ? 0 : (int)slots;
  const int64_t parts = tiles * ((most + kMinShare - 1) / kMinShare);
  return !p.slots ? 0 : parts < 2 * slots + tiles ? parts : 2 * slots + tiles;
}

// The call's row tiles: by the rows that the sequences have where the host knows them (counts), else as if all had seq_q.  A
// padded batch planned by seq_q is taken for one with many row tiles, and its keys stay whole: one sequence of 500 rows on 4000
// keys among 8 slots, 24 / 8 heads of 128, 41.1 us by its rows, 108 by seq_q (alone 39.5); beside seven tokens on 16000 keys
// 94 and 320.
// Packed rows are so many in all, whatever the lengths.
int64_t row_tiles(const WinParams& p, const int32_t* counts) {
  if (!counts) {
    const int64_t all = (int64_t)p.batch * p.n_qt, packed = p.batch + (int64_t)p.packed_rows * p.group / kBM;
    return (p.packed_rows && packed < all ? packed : all) * p.n_kv;
  }
  int64_t n = 0;
  for (int b = 0; b < p.batch; ++b) {
    const int64_t rows = counts[b] < 0 ? 0 : counts[b] < p.seq_q ? counts[b] : p.seq_q;
    n += (rows * p.group + kBM - 1) / kBM;
  }
  return n * p.n_kv;
}

// Rows that token_of() divides exactly: the magic's excess, below group, times a row stays below 2^32.  (Rows of the
// last tile count.)
bool rows_ok(int64_t seq_q, int64_t group) { return (seq_q * group + kBM) * group < ((int64_t)1 << 32); }

// Workspace of so many parts: their tags, then their results.
size_t words_bytes(int64_t parts) { return ((size_t)parts * 4 * sizeof(uint64_t) + 255) & ~(size_t)255; }
size_t part_bytes(int d_k) { return (d_k == 64 ? part_floats<64>() : part_floats<128>()) * sizeof(float); }

template <typename T, int D>
int launch_window(WinParams& p, bool paged, hipStream_t st) {
  const int64_t tiles = (int64_t)p.batch * p.n_kv * p.n_qt;
  if (tiles > (1 << 27)) return TL_ERR_UNSUPPORTED;
  const int64_t units = (int64_t)p.batch * p.n_kv;
  p.q_shift = 3;  // units << q_shift is a multiple of 8
  while (p.q_shift > 0 && units % (16 >> p.q_shift) == 0) --p.q_shift;
  p.n_lvl = (p.n_qt + (1 << p.q_shift) - 1) >> p.q_shift;
  p.xcd_groups = (int)((units << p.q_shift) / 8);
  const dim3 grid(p.slots > 0 ? (unsigned)((p.room + 7) / 8 * 8) : (unsigned)(8 * p.xcd_groups * p.n_lvl));
  if (p.starts) hipLaunchKernelGGL((window_fwd_kernel<T, D, true, true>), grid, dim3(kThreads), 0, st, p);
  else if (paged) hipLaunchKernelGGL((window_fwd_kernel<T, D, true, false>), grid, dim3(kThreads), 0, st, p);
  else hipLaunchKernelGGL((window_fwd_kernel<T, D, false, false>), grid, dim3(kThreads), 0, st, p);
  const int e = tl_launch_status();
  if (e || p.slots == 0 || p.tag) return e;
  const dim3 join((unsigned)tiles, D / 32);
  if (paged) hipLaunchKernelGGL((window_join_kernel<T, D, true>), join, dim3(kThreads), 0, st, p);
  else hipLaunchKernelGGL((window_join_kernel<T, D, false>), join, dim3(kThreads), 0, st, p);
  return tl_launch_status();
}

template <typename T>
int launch_window_d(WinParams& p, bool paged, int d_k, hipStream_t st) {
  return d_k == 64 ? launch_window<T, 64>(p, paged, st) : launch_window<T, 128>(p, paged, st);
}

int window_entry(WinParams& p, bool paged, int64_t keys, const int32_t* counts, void* workspace, size_t workspace_bytes, int d_k,
                 const int64_t* qs, const int64_t* ks, const int64_t* vs, const int64_t* os, float sm_scale, int dtype, void* stream) {
  if (!p.q || !p.k || !p.v || !p.o || !qs || !ks || !vs || !os || p.batch < 0 || p.n_head < 0 || p.n_kv < 1 ||
      p.n_head % p.n_kv || p.seq_q < 0 || p.window < 0 || p.sinks < 0)
    return TL_ERR_INVALID;
  if (dtype != TL_DTYPE_F32 && dtype != TL_DTYPE_F16 && dtype != TL_DTYPE_BF16) return TL_ERR_INVALID;
  if (d_k != 64 && d_k != 128) return TL_ERR_UNSUPPORTED;
  if (p.seq_q > kMostRows || p.seq_k > (1 << 29)) return TL_ERR_UNSUPPORTED;
  if (p.window >= kWholeWindow) p.window = 0;
  // rows are moved 16 bytes at a time, a block of 16 with 32-bit offsets
  const int esize = dtype == TL_DTYPE_F32 ? 4 : 2;
  const int64_t vec = 16 / esize;
  for (int i = 0; i < 3; ++i) {
    if (qs[i] < 0 || ks[i] < 0 || vs[i] < 0 || os[i] < 0) return TL_ERR_UNSUPPORTED;
    if (qs[i] % vec || ks[i] % vec || vs[i] % vec) return TL_ERR_UNSUPPORTED;
  }
  if (ks[2] > (1 << 24) || vs[2] > (1 << 24)) return TL_ERR_UNSUPPORTED;
  if (((uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.v) & 15) return TL_ERR_UNSUPPORTED;
  p.q_sb = qs[0], p.q_sh = qs[1], p.q_ss = qs[2];
  p.k_sb = ks[0], p.k_sh = ks[1], p.k_ss = ks[2];
  p.v_sb = vs[0], p.v_sh = vs[1], p.v_ss = vs[2];
  p.o_sb = os[0], p.o_sh = os[1], p.o_ss = os[2];
  // a workgroup writes o while others still read q, k and v
  const int64_t row = (int64_t)d_k * esize;
  auto rows = [&](const void* at, int64_t n0, int64_t n1, int64_t n2, const int64_t* s) {
    return Rows3{at, {n0, n1, n2}, {s[0] * esize, s[1] * esize, s[2] * esize}, row};
  };
  const int64_t n0 = paged ? p.pm.n_pages : p.batch, n2 = paged ? (int64_t)1 << p.pm.shift : p.seq_k;
  const int64_t q0 = p.starts ? 1 : p.batch, q2 = p.starts ? p.packed_rows : p.seq_q;
  const Rows3 out = rows(p.o, q0, p.n_head, q2, os);
  if (rows_overlap(out, rows(p.q, q0, p.n_head, q2, qs)) || rows_overlap(out, rows(p.k, n0, p.n_kv, n2, ks)) ||
      rows_overlap(out, rows(p.v, n0, p.n_kv, n2, vs)))
    return TL_ERR_INVALID;
  p.group = p.n_head / p.n_kv;
  if (!rows_ok(p.seq_q, p.group)) return TL_ERR_UNSUPPORTED;
  p.group_magic = (uint32_t)((((uint64_t)1 << 32) + p.group - 1) / p.group);
  p.n_qt = (p.seq_q * p.group + kBM - 1) / kBM;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.vec_out = ((uintptr_t)p.o % (4 * esize)) == 0 && os[0] % 4 == 0 && os[1] % 4 == 0 && os[2] % 4 == 0;
  hipStream_t st = tl_resolve_stream(stream);
  if (counts) {  // a graph's replays may come with other counts
    hipStreamCaptureStatus c;
    if (hipStreamIsCapturing(st, &c) != hipSuccess || c != hipStreamCaptureStatusNone) counts = nullptr;
  }
  const int64_t tiles = row_tiles(p, counts);
  const int64_t most_parts = plan_slots(p, tiles, keys, d_k, esize);
  if (p.slots > 0) {
    p.room = (int)most_parts;
    const int64_t cap = INT32_MAX / ((int64_t)p.batch * p.n_qt);
    p.key_cap = (int)(cap < (1 << 20) ? cap : 1 << 20);
    // without room for the parts the keys stay undivided
    if (!workspace || workspace_bytes < words_bytes(most_parts) + (size_t)most_parts * part_bytes(d_k) || ((uintptr_t)workspace & 15)) p.slots = 0;
    // Few parts are joined by the wave that ends last, without a second launch; many would be added up one after the
    // other by one wave.  us joined by the waves / by a second launch: 1023 rows, window 256, fp32 (2 parts) 25.0 / 26.2,
    // 4 x 500 rows on prefixes (3 parts) 43.5 / 44.8; 500 rows on 4000 keys, d_k 128 (5 parts) 43.7 / 39.6, 100 rows (21
    // parts) 40.7 / 27.6.
    p.tag = p.slots <= kWaveParts * tiles ? tl_arrival_tag() : 0;
    p.words = (uint64_t*)workspace;
    p.ws = (float*)((char*)workspace + words_bytes(most_parts));
  }
  switch (dtype) {
    case TL_DTYPE_F32: return launch_window_d<F32>(p, paged, d_k, st);
    case TL_DTYPE_F16: return launch_window_d<F16>(p, paged, d_k, st);
    default: return launch_window_d<BF16>(p, paged, d_k, st);
  }
}

}  // namespace

extern "C" {

size_t tl_window_workspace_bytes(int batch, int n_head, int n_kv_head, int seq_q, int most_keys, int d_k, int window,
                                 int sinks, int dtype) {
  return tl_paged_prefill_workspace_bytes(nullptr, batch, n_head, n_kv_head, seq_q, most_keys, d_k, window, sinks, dtype);
}

size_t tl_paged_prefill_workspace_bytes(const int32_t* host_new_lens, int batch, int n_head, int n_kv_head, int seq_q,
                                        int most_keys, int d_k, int window, int sinks, int dtype) {
  return tl_paged_packed_workspace_bytes(host_new_lens, 0, batch, n_head, n_kv_head, seq_q, most_keys, d_k, window, sinks,
                                         dtype);
}

size_t tl_paged_packed_workspace_bytes(const int32_t* host_new_lens, int n_rows, int batch, int n_head, int n_kv_head,
                                       int seq_q, int most_keys, int d_k, int window, int sinks, int dtype) {
  if (n_rows < 0) return 0;
  if (n_rows > 0 && seq_q > n_rows) seq_q = n_rows;
  if (batch < 1 || n_head < 1 || n_kv_head < 1 || n_head % n_kv_head || seq_q < 1 || seq_q > kMostRows || most_keys < 1 ||
      window < 0 || sinks < 0 || (d_k != 64 && d_k != 128) || !rows_ok(seq_q, n_head / n_kv_head) ||
      (dtype != TL_DTYPE_F32 && dtype != TL_DTYPE_F16 && dtype != TL_DTYPE_BF16))
    return 0;
  WinParams p{};
  p.batch = batch;
  p.n_kv = n_kv_head;
  p.group = n_head / n_kv_head;
  p.packed_rows = n_rows;
  p.seq_q = seq_q;
  p.n_qt = (seq_q * p.group + kBM - 1) / kBM;
  p.window = window;
  p.sinks = sinks;
  const int64_t parts = plan_slots(p, row_tiles(p, host_new_lens), most_keys, d_k, dtype == TL_DTYPE_F32 ? 4 : 2);
  return parts ? words_bytes(parts) + (size_t)parts * part_bytes(d_k) : 0;
}

int tl_window_attention(const void* q, const void* k, const void* v, void* o, void* workspace, size_t workspace_bytes,
                        int batch, int n_head, int n_kv_head, int seq_q, int seq_k, int d_k, const int64_t* q_strides, const int64_t* k_strides,
                        const int64_t* v_strides, const int64_t* o_strides, float sm_scale, int window, int sinks,
                        int dtype, void* stream) {
  if (batch == 0 || n_head == 0 || seq_q == 0) return 0;
  if (seq_k < 1) return TL_ERR_INVALID;
  WinParams p{};
  p.q = q;
  p.k = k;
  p.v = v;
  p.o = o;
  p.batch = batch;
  p.n_head = n_head;
  p.n_kv = n_kv_head;
  p.seq_q = seq_q;
  p.seq_k = seq_k;
  p.window = window;
  p.sinks = sinks;
  return window_entry(p, false, seq_k, nullptr, workspace, workspace_bytes, d_k, q_strides, k_strides, v_strides, o_strides,
                      sm_scale, dtype, stream);
}

int tl_paged_attention_prefill(const void* q, const void* k_pages, const void* v_pages, const int32_t* page_table,
                               int max_pages, int n_pages, int page_size, const int32_t* cache_lens,
                               const int32_t* new_lens, void* o, void* workspace, size_t workspace_bytes, int batch,
                               int n_new, int n_head, int n_kv_head, int d_k, const int64_t* q_strides, const int64_t* k_page_strides,
                               const int64_t* v_page_strides, const int64_t* o_strides, float sm_scale, int window,
                               int sinks, int dtype, void* stream) {
  return tl_paged_attention_prefill_counted(q, k_pages, v_pages, page_table, max_pages, n_pages, page_size, cache_lens,
                                            new_lens, nullptr, o, workspace, workspace_bytes, batch, n_new, n_head, n_kv_head,
                                            d_k, q_strides, k_page_strides, v_page_strides, o_strides, sm_scale, window,
                                            sinks, dtype, stream);
}

int tl_paged_attention_prefill_counted(const void* q, const void* k_pages, const void* v_pages, const int32_t* page_table,
                                       int max_pages, int n_pages, int page_size, const int32_t* cache_lens,
                                       const int32_t* new_lens, const int32_t* host_new_lens, void* o, void* workspace,
                                       size_t workspace_bytes, int batch, int n_new, int n_head, int n_kv_head, int d_k,
                                       const int64_t* q_strides, const int64_t* k_page_strides,
                                       const int64_t* v_page_strides, const int64_t* o_strides, float sm_scale, int window,
                                       int sinks, int dtype, void* stream) {
  if (batch == 0 || n_head == 0 || n_new == 0) return 0;
  if (host_new_lens && !new_lens) return TL_ERR_INVALID;
  const int shift = page_shift(page_size);
  if (!page_table || !cache_lens || max_pages < 1 || n_pages < 1 || shift < 0 ||
      ((int64_t)max_pages << shift) > (1 << 30))
    return TL_ERR_INVALID;
  WinParams p{};
  p.q = q;
  p.k = k_pages;
  p.v = v_pages;
  p.o = o;
  p.pm = PageMap{page_table, max_pages, n_pages, shift};
  p.lens = cache_lens;
  p.new_lens = new_lens;
  p.batch = batch;
  p.n_head = n_head;
  p.n_kv = n_kv_head;
  p.seq_q = n_new;
  p.window = window;
  p.sinks = sinks;
  return window_entry(p, true, (int64_t)max_pages << shift, host_new_lens, workspace, workspace_bytes, d_k, q_strides, k_page_strides,
                      v_page_strides, o_strides, sm_scale, dtype, stream);
}

int tl_paged_attention_packed(const void* q, const void* k_pages, const void* v_pages, const int32_t* page_table, int max_pages,
                              int n_pages, int page_size, const int32_t* cache_lens, const int32_t* starts,
                              const int32_t* host_new_lens, void* o, void* workspace, size_t workspace_bytes, int batch,
                              int n_rows, int max_new, int n_head, int n_kv_head, int d_k, const int64_t* q_strides,
                              const int64_t* k_page_strides, const int64_t* v_page_strides, const int64_t* o_strides,
                              float sm_scale, int window, int sinks, int dtype, void* stream) {
  if (batch == 0 || n_head == 0 || n_rows == 0 || max_new == 0) return 0;
  const int shift = page_shift(page_size);
  if (!page_table || !cache_lens || !starts || n_rows < 0 || max_pages < 1 || n_pages < 1 || shift < 0 ||
      ((int64_t)max_pages << shift) > (1 << 30) || !q_strides || !o_strides)
    return TL_ERR_INVALID;
  WinParams p{};
  p.q = q;
  p.k = k_pages;
  p.v = v_pages;
  p.o = o;
  p.pm = PageMap{page_table, max_pages, n_pages, shift};
  p.lens = cache_lens;
  p.starts = starts;
  p.packed_rows = n_rows;
  p.batch = batch;
  p.n_head = n_head;
  p.n_kv = n_kv_head;
  p.seq_q = max_new < n_rows ? max_new : n_rows;
  p.window = window;
  p.sinks = sinks;
  const int64_t qs[] = {0, q_strides[1], q_strides[0]}, os[] = {0, o_strides[1], o_strides[0]};
  return window_entry(p, true, (int64_t)max_pages << shift, host_new_lens, workspace, workspace_bytes, d_k, qs,
                      k_page_strides, v_page_strides, os, sm_scale, dtype, stream);
}

}  // extern "C"
