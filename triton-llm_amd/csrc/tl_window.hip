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
// A workgroup is 4 waves of 32 query rows of one head.  It walks only the key tiles that any of
// its 128 rows sees: the sinks' tiles, then those from the first row's window on to the last row's
// position.  As in the causal prefill the products are transposed, S^T = K . Q^T and
// O^T = V^T . P^T, on 32 x 32 MFMA blocks: lane l of the accumulator holds query row l % 32, so maximum and
// rescale are a lane's own (one exchange between l and l ^ 32), and P^T goes from the accumulator's
// registers straight into the second product.  K / V tiles come by LDS-DMA, the next one while this
// one is used; V is read by transposing LDS reads.
#include "tl_paged.h"
#include "tl_prefill.h"

#include <math.h>

using namespace tlpg;

namespace {

constexpr int kThreads = 256;
constexpr int kBM = 128;  // query rows of a workgroup
constexpr float kRescaleLog2 = 8.f;

struct WinParams {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  PageMap pm;  // pages: k / v strides are {page, head, row}; else {batch, head, row}
  const int32_t* lens;
  const int32_t* new_lens;
  int batch, n_head, n_kv, group, seq_q, seq_k, n_qt;
  int window, sinks;
  int64_t q_sb, q_sh, q_ss;
  int64_t k_sb, k_sh, k_ss;
  int64_t v_sb, v_sh, v_ss;
  int64_t o_sb, o_sh, o_ss;
  float scale_log2;
};

// Keys of a tile.  fp32 rows are twice as long: half as many keys in the same LDS.
template <typename T>
constexpr int tile_keys() { return T::size == 2 ? 64 : 32; }

// Slot of 16-byte chunk c of LDS row r is c ^ swz(r).  K: the 32 rows of an operand read take the same
// chunk.  V: a transposing read takes 4 consecutive rows (see tl_prefill.hip); fp32 V
// is read 32 consecutive words at a time and needs none.
template <typename T, int D>
__device__ __forceinline__ int k_swz(int r) {
  if constexpr (T::size == 2) return tlp::lds_swz<D>(r);
  else return r & 15;
}
template <typename T, int D>
__device__ __forceinline__ int v_swz(int r) {
  if constexpr (T::size == 4) return 0;
  else return D == 64 ? 2 * ((r >> 1) & 1) : 4 * (r & 3);
}

// The matrix products of one 32-row block, by storage type.
template <typename T, int D>
struct Tile;

template <typename T, int D>
struct Tile16 {
  using M = Mfma<T>;
  using frag = typename M::frag;
  static constexpr int ROWB = D * 2, NKS = D / 16, NDB = D / 32, NMB = 2;
  struct Q {
    frag f[NKS];
  };
  static __device__ __forceinline__ void load_q(Q& q, const char* row, bool there, int h) {
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      u32x4 x = u32x4{0u, 0u, 0u, 0u};
      if (there) x = *(const u32x4*)(row + 32 * ks + 16 * h);
      q.f[ks] = __builtin_bit_cast(frag, x);
    }
  }
  static __device__ __forceinline__ void scores(f32x16 (&s)[NMB], const Q& q, const char* kt, int lq, int h) {
#pragma unroll
    for (int mb = 0; mb < NMB; ++mb) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[mb][r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
        const u32x4 a = *(const u32x4*)(kt + (32 * mb + lq) * ROWB + (((2 * ks + h) ^ k_swz<T, D>(lq)) << 4));
        s[mb] = M::mma(__builtin_bit_cast(frag, a), q.f[ks], s[mb]);
      }
    }
  }
  // s holds the probabilities; they are rounded to the storage type here (at most half a step
  // each, as the causal prefill does), the sum l is of the unrounded ones.
  static __device__ __forceinline__ void values(f32x16 (&o)[NDB], const f32x16 (&s)[NMB], const char* vt, int lane) {
    typedef short v4s __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) v4s lds_v4s;
    const auto* lds = (const __attribute__((address_space(3))) char*)vt;
    const int g = lane >> 4, e = (lane >> 2) & 3, c = lane & 3;
#pragma unroll
    for (int tt = 0; tt < 2 * NMB; ++tt) {
      u32x4 pw;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x[2] = {s[tt >> 1][8 * (tt & 1) + 2 * j], s[tt >> 1][8 * (tt & 1) + 2 * j + 1]};
        pw[j] = pack2<T>(x);
      }
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        const int chunk = 4 * db + 2 * (g & 1) + (c >> 1);
        const int off = (16 * tt + 4 * (g >> 1) + e) * ROWB + ((chunk ^ v_swz<T, D>(e)) << 4) + 8 * (c & 1);
        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(lds + off));
        const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(lds + off + 8 * ROWB));
        const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
        o[db] = M::mma(__builtin_bit_cast(frag, u32x4{a.x, a.y, b.x, b.y}), __builtin_bit_cast(frag, pw), o[db]);
      }
    }
  }
};

template <int D>
struct Tile32 {
  static constexpr int ROWB = D * 4, NDB = D / 32, NMB = 1;
  struct Q {
    float f[D / 2];  // features h D / 2 .. of the row
  };
  static __device__ __forceinline__ void load_q(Q& q, const char* row, bool there, int h) {
#pragma unroll
    for (int c = 0; c < D / 8; ++c) {
      f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
      if (there) x = *(const f32x4*)(row + h * (D * 2) + 16 * c);
#pragma unroll
      for (int i = 0; i < 4; ++i) q.f[4 * c + i] = x[i];
    }
  }
  static __device__ __forceinline__ void scores(f32x16 (&s)[NMB], const Q& q, const char* kt, int lq, int h) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[0][r] = 0.f;
#pragma unroll
    for (int c = 0; c < D / 8; ++c) {
      const f32x4 a = *(const f32x4*)(kt + lq * ROWB + (((h * (D / 8) + c) ^ k_swz<F32, D>(lq)) << 4));
#pragma unroll
      for (int i = 0; i < 4; ++i) s[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], q.f[4 * c + i], s[0], 0, 0, 0);
    }
  }
  static __device__ __forceinline__ void values(f32x16 (&o)[NDB], const f32x16 (&s)[NMB], const char* vt, int lane) {
    const int lq = lane & 31, h = lane >> 5;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int key = 8 * (r >> 2) + 4 * h + (r & 3);
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        const float a = *(const float*)(vt + key * ROWB + (32 * db + lq) * 4);
        o[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, s[0][r], o[db], 0, 0, 0);
      }
    }
  }
};

template <int D>
struct Tile<BF16, D> : Tile16<BF16, D> {};
template <int D>
struct Tile<F16, D> : Tile16<F16, D> {};
template <int D>
struct Tile<F32, D> : Tile32<D> {};

template <typename T, int D, bool PAGED>
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

  // Workgroups are dealt to the 8 XCDs in turn; XCD x takes a contiguous range of (sequence, KV head,
  // query head, tile), so that few KV heads share its L2.
  const int n_items = p.batch * p.n_head * p.n_qt;
  const int per = (n_items + 7) / 8;
  const int item = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
  if ((int)(blockIdx.x / 8) >= per || item >= n_items) return;
  const int head = item / p.n_qt;
  const int qt = p.n_qt - 1 - (item - head * p.n_qt);  // the longest rows first
  const int b = head / p.n_head;
  const int hq = head - b * p.n_head;
  const int hkv = hq / p.group;

  const int lane = threadIdx.x & 63;
  const int wave = uni((int)threadIdx.x >> 6);
  const int lq = lane & 31, h = lane >> 5;

  int base, nq, key_end;  // position of row 0, rows, keys behind which nothing is read
  if constexpr (PAGED) {
    constexpr int kFar = 1 << 30;
    base = min(max(p.lens[b], -kFar), kFar);
    nq = p.new_lens ? min(max(p.new_lens[b], 0), p.seq_q) : p.seq_q;
    key_end = min(base + nq, p.pm.max_pages << p.pm.shift);
  } else {
    base = p.seq_k - p.seq_q;
    nq = p.seq_q;
    key_end = p.seq_k;
  }
  if (qt * kBM >= nq) return;

  // the key tiles: ns of the sinks, then from t0 on
  const int p0 = base + qt * kBM;
  const int p1 = min(base + min(qt * kBM + kBM, nq), key_end) - 1;  // last key any row sees
  int ns = 0, t0 = 0, nt = 0;
  if (p1 >= 0) {
    const int te = p1 / BN;
    if (p.window > 0) {
      t0 = max(p0 - p.window + 1, 0) / BN;
      ns = (min(p.sinks, p1 + 1) + BN - 1) / BN;
      if (t0 <= ns) ns = t0 = 0;
    }
    nt = ns + te - t0 + 1;
  }
  auto tile_key0 = [&](int t) { return (t < ns ? t : t - ns + t0) * BN; };

  const int row = qt * kBM + 32 * wave + lq;  // this lane's query row
  const int pos = base + row;
  const bool there = row < nq;
  typename TL::Q q;
  TL::load_q(q, (const char*)((const B*)p.q + b * p.q_sb + hq * p.q_sh + (int64_t)min(row, nq - 1) * p.q_ss), there, h);

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
  const int32_t* table = PAGED ? p.pm.table + (int64_t)b * p.pm.max_pages : nullptr;
  // lane i < BN / 16: the page of the tile's block i, -1 where there is none
  auto tile_pages = [&](int t) {
    int id = -1;
    if constexpr (PAGED) {
      const int e = (tile_key0(t) + kBlk * lane) >> p.pm.shift;
      if (lane < BN / kBlk && e < p.pm.max_pages) id = table[e];
      if ((unsigned)id >= (unsigned)p.pm.n_pages) id = -1;
    }
    return id;
  };
  // Rows past key_end, and rows of pages that are not there, read as zeros.
  auto load_tile = [&](int t, int buf, int pages) {
    const int pos0 = tile_key0(t) + wave * WROWS;
    int rows = min(max(key_end - pos0, 0), WROWS);
    const char *kb, *vb;
    if constexpr (PAGED) {
      const int id = __builtin_amdgcn_readlane(pages, (wave * WROWS) / kBlk);
      const int in = pos0 & ((1 << p.pm.shift) - 1);
      if (id < 0) rows = 0;
      const int64_t at = id < 0 ? 0 : id;
      kb = (const char*)((const B*)p.k + at * p.k_sb + hkv * p.k_sh + in * p.k_ss);
      vb = (const char*)((const B*)p.v + at * p.v_sb + hkv * p.v_sh + in * p.v_ss);
    } else {
      kb = (const char*)((const B*)p.k + b * p.k_sb + hkv * p.k_sh + pos0 * p.k_ss);
      vb = (const char*)((const B*)p.v + b * p.v_sb + hkv * p.v_sh + pos0 * p.v_ss);
    }
    const i32x4 rk = uniform_rsrc(kb, rows ? (rows - 1) * k_row + ROWB : 0);
    const i32x4 rv = uniform_rsrc(vb, rows ? (rows - 1) * v_row + ROWB : 0);
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

  const int wp0 = uni(base + qt * kBM + 32 * wave);  // this wave's first position
  const int wp1 = min(wp0 + 31, base + nq - 1);
  const bool wave_rows = qt * kBM + 32 * wave < nq;

  int pages = nt > 0 ? tile_pages(0) : -1;
  if (nt > 0) load_tile(0, 0, pages);
  int next_pages = nt > 1 ? tile_pages(1) : -1;
  for (int t = 0; t < nt; ++t) {
    wait_vmcnt<0>();  // this wave's rows of tile t are in LDS
    lds_barrier();    // everybody's are, and tile t - 1 has been read
    const int there_now = pages;
    if (t + 1 < nt) {
      load_tile(t + 1, (t + 1) & 1, next_pages);
      pages = next_pages;
      if (t + 2 < nt) next_pages = tile_pages(t + 2);
    }
    const int k0 = tile_key0(t);
    // does any row of this wave see a key of the tile, and does every row see all of them
    const bool any = wave_rows && k0 <= wp1 && (p.window <= 0 || k0 + BN - 1 > wp0 - p.window || k0 < p.sinks);
    if (!any) continue;
    uint32_t gone = 0;  // blocks that have no page
    if constexpr (PAGED) gone = (uint32_t)__ballot(there_now < 0) & ((1u << (BN / kBlk)) - 1);
    const bool all = k0 + BN - 1 <= wp0 && k0 + BN <= key_end && gone == 0 &&
                     (p.window <= 0 || k0 > wp1 - p.window || k0 + BN <= p.sinks);
    const char* kt = smem + (t & 1) * 2 * TILEB;
    const char* vt = kt + TILEB;
    f32x16 s[NMB];
    TL::scores(s, q, kt, lq, h);
    if (!all) {
#pragma unroll
      for (int mb = 0; mb < NMB; ++mb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = k0 + 32 * mb + 8 * (r >> 2) + 4 * h + (r & 3);
          const bool seen = key_seen(key, pos, p.window, p.sinks) && key < key_end && !((gone >> (2 * mb + (r >> 3))) & 1);
          s[mb][r] = seen ? s[mb][r] : -INFINITY;
        }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int mb = 0; mb < NMB; ++mb)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[mb][r]);
    mx = tlp::max_xor32(mx) * p.scale_log2;
    // a negative scale turns the order round: the maximum is then the smallest score's
    if (p.scale_log2 < 0.f) {
      float mn = INFINITY;
#pragma unroll
      for (int mb = 0; mb < NMB; ++mb)
#pragma unroll
        for (int r = 0; r < 16; ++r) mn = fminf(mn, s[mb][r] == -INFINITY ? INFINITY : s[mb][r]);
      mx = -tlp::max_xor32(-mn);
      mx = mx == INFINITY ? -INFINITY : mx * p.scale_log2;
    }
    if (__any(mx > m + kRescaleLog2)) {
      const float mn = fmaxf(m, mx);
      const float a = fast_exp2(m - (mn == -INFINITY ? 0.f : mn));
      m = mn;
      l *= a;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] *= a;
    }
    const float shift = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int mb = 0; mb < NMB; ++mb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float x = s[mb][r];
        const float e = fast_exp2(fmaf(x, p.scale_log2, -shift));
        s[mb][r] = all || x != -INFINITY ? e : 0.f;
        l += s[mb][r];
      }
    TL::values(o, s, vt, lane);
  }

  l = tlp::sum_xor32(l);
  if (!there) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  B* out = (B*)p.o + b * p.o_sb + hq * p.o_sh + (int64_t)row * p.o_ss;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int d = 32 * db + 8 * a + 4 * h;
#pragma unroll
      for (int i = 0; i < 4; ++i) out[d + i] = from_f32<T>(o[db][4 * a + i] * inv);
    }
}

template <typename T, int D>
int launch_window(const WinParams& p, bool paged, hipStream_t st) {
  const int64_t items = (int64_t)p.batch * p.n_head * p.n_qt;
  if (items > (1 << 30)) return TL_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)((items + 7) / 8 * 8));
  if (paged) hipLaunchKernelGGL((window_fwd_kernel<T, D, true>), grid, dim3(kThreads), 0, st, p);
  else hipLaunchKernelGGL((window_fwd_kernel<T, D, false>), grid, dim3(kThreads), 0, st, p);
  return tl_launch_status();
}

int window_entry(WinParams& p, bool paged, int d_k, const int64_t* qs, const int64_t* ks, const int64_t* vs,
                 const int64_t* os, float sm_scale, int dtype, void* stream) {
  if (!p.q || !p.k || !p.v || !p.o || !qs || !ks || !vs || !os || p.batch < 0 || p.n_head < 0 || p.n_kv < 1 ||
      p.n_head % p.n_kv || p.seq_q < 0 || p.window < 0 || p.sinks < 0)
    return TL_ERR_INVALID;
  if (dtype != TL_DTYPE_F32 && dtype != TL_DTYPE_F16 && dtype != TL_DTYPE_BF16) return TL_ERR_INVALID;
  if (d_k != 64 && d_k != 128) return TL_ERR_UNSUPPORTED;
  if (p.seq_q > (1 << 29) || p.seq_k > (1 << 29)) return TL_ERR_UNSUPPORTED;
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
  p.group = p.n_head / p.n_kv;
  p.n_qt = (p.seq_q + kBM - 1) / kBM;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  hipStream_t st = tl_resolve_stream(stream);
  switch (dtype) {
    case TL_DTYPE_F32: return d_k == 64 ? launch_window<F32, 64>(p, paged, st) : launch_window<F32, 128>(p, paged, st);
    case TL_DTYPE_F16: return d_k == 64 ? launch_window<F16, 64>(p, paged, st) : launch_window<F16, 128>(p, paged, st);
    default: return d_k == 64 ? launch_window<BF16, 64>(p, paged, st) : launch_window<BF16, 128>(p, paged, st);
  }
}

}  // namespace

extern "C" {

int tl_window_attention(const void* q, const void* k, const void* v, void* o, int batch, int n_head, int n_kv_head,
                        int seq_q, int seq_k, int d_k, const int64_t* q_strides, const int64_t* k_strides,
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
  return window_entry(p, false, d_k, q_strides, k_strides, v_strides, o_strides, sm_scale, dtype, stream);
}

int tl_paged_attention_prefill(const void* q, const void* k_pages, const void* v_pages, const int32_t* page_table,
                               int max_pages, int n_pages, int page_size, const int32_t* cache_lens,
                               const int32_t* new_lens, void* o, int batch, int n_new, int n_head, int n_kv_head,
                               int d_k, const int64_t* q_strides, const int64_t* k_page_strides,
                               const int64_t* v_page_strides, const int64_t* o_strides, float sm_scale, int window,
                               int sinks, int dtype, void* stream) {
  if (batch == 0 || n_head == 0 || n_new == 0) return 0;
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
  return window_entry(p, true, d_k, q_strides, k_page_strides, v_page_strides, o_strides, sm_scale, dtype, stream);
}

}  // extern "C"
