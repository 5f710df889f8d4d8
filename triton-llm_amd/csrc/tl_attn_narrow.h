// Internal header: attention of few query rows, at most 32, over keys in pages, on 16 x 16 matrix products (tl_shared.hip,
// tl_window.hip).  Not part of the C ABI.
//
// A workgroup is 4 waves.  Every wave by itself takes blocks of 16 keys, its own ring of them coming by LDS-DMA without a barrier, and
// keeps the running maximum and sum of the softmax over its keys (fp32, log2 domain); the waves' states are joined through LDS at the
// end.  Against 32 x 32 blocks on one wave, the tile shared by all four: a short call waits for a quarter of the products (4
// sequences, fp32: 13.1 -> 5.1 us), and a wave that computes is not always the same SIMD's.
//
// With 16-bit types a weight goes into the product with V in two words, its rounding and what that left out (2^-16 of it in bf16,
// less in fp16), so that no weight's rounding shows: the products are not what these calls wait for (256 sequences behind 8
// prefixes, 243.5 us either way; 64 behind one of 8192, 68.5 and 69.4).
#pragma once

#include "tl_attn_tile.h"
#include "tl_paged.h"

#include <math.h>

namespace tlat {

using namespace tlpg;

__device__ __forceinline__ float max_xor16(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_xor16(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The 16 x 16 matrix products of 16 keys with 16 query rows: scores S^T = K . Q^T, a lane then holding query row lane % 16 and
// keys 4 (lane / 16) .. + 3, which is how O^T = V^T . P^T takes the weights.
template <typename T, int D>
struct Narrow;

template <typename T, int D>
struct Narrow16 {
  static constexpr int ROWB = D * 2;
  struct Q {
    u32x4 f[D / 32];
  };
  static __device__ __forceinline__ int kswz(int r) { return k_swz<T, D>(r); }
  static __device__ __forceinline__ int vswz(int r) { return v_swz<T, D>(r & 3); }
  static __device__ __forceinline__ void load_q(Q& q, const char* row, bool there, int g, uint32_t sign) {
    sign |= sign >> 16;
#pragma unroll
    for (int ks = 0; ks < D / 32; ++ks) {
      u32x4 x = u32x4{0u, 0u, 0u, 0u};
      if (there) x = *(const u32x4*)(row + 64 * ks + 16 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] ^= sign;
      q.f[ks] = x;
    }
  }
  template <int NRB>
  static __device__ __forceinline__ void scores(f32x4 (&s)[NRB], const Q (&q)[NRB], const char* kt, int lr, int g) {
#pragma unroll
    for (int rb = 0; rb < NRB; ++rb) s[rb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < D / 32; ++ks) {
      const u32x4 a = *(const u32x4*)(kt + lr * ROWB + (((4 * ks + g) ^ kswz(lr)) << 4));
#pragma unroll
      for (int rb = 0; rb < NRB; ++rb) {
        if constexpr (T::code == TL_DTYPE_BF16)
          s[rb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, q[rb].f[ks]), s[rb], 0, 0, 0);
        else
          s[rb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, q[rb].f[ks]), s[rb], 0, 0, 0);
      }
    }
  }
  typedef short v4s __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ f32x4 product(v4s a, v4s b, f32x4 c) {
    if constexpr (T::code == TL_DTYPE_BF16) return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
  }
  template <int NRB>
  static __device__ __forceinline__ void values(f32x4 (&o)[NRB][D / 16], const f32x4 (&w)[NRB], const char* vt, int lane) {
    typedef __attribute__((address_space(3))) v4s lds_v4s;
    const int g = lane >> 4, e = (lane >> 2) & 3, c = lane & 3;
    u32x2 pw[NRB], rest[NRB];
#pragma unroll
    for (int rb = 0; rb < NRB; ++rb) {
      float x[2] = {w[rb][0], w[rb][1]}, y[2] = {w[rb][2], w[rb][3]}, r[4];
      pw[rb] = u32x2{pack2<T>(x), pack2<T>(y)};
      unpack2<T>(pw[rb].x, r[0], r[1]);
      unpack2<T>(pw[rb].y, r[2], r[3]);
      x[0] -= r[0], x[1] -= r[1], y[0] -= r[2], y[1] -= r[3];
      rest[rb] = u32x2{pack2<T>(x), pack2<T>(y)};
    }
    const auto* row = (const __attribute__((address_space(3))) char*)vt + (4 * g + e) * ROWB + 8 * (c & 1);
#pragma unroll
    for (int db = 0; db < D / 16; ++db) {
      const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(row + (((2 * db + (c >> 1)) ^ vswz(e)) << 4)));
#pragma unroll
      for (int rb = 0; rb < NRB; ++rb) {
        o[rb][db] = product(a, __builtin_bit_cast(v4s, pw[rb]), o[rb][db]);
        o[rb][db] = product(a, __builtin_bit_cast(v4s, rest[rb]), o[rb][db]);
      }
    }
  }
};

template <int D>
struct Narrow32 {
  static constexpr int ROWB = D * 4;
  struct Q {
    float f[D / 4];  // features g D / 4 .. of the row
  };
  static __device__ __forceinline__ int kswz(int r) { return r & 15; }
  static __device__ __forceinline__ int vswz(int r) { return 4 * ((r >> 2) & 3); }
  static __device__ __forceinline__ void load_q(Q& q, const char* row, bool there, int g, uint32_t sign) {
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      u32x4 x = u32x4{0u, 0u, 0u, 0u};
      if (there) x = *(const u32x4*)(row + g * D + 16 * c);
#pragma unroll
      for (int i = 0; i < 4; ++i) q.f[4 * c + i] = __uint_as_float(x[i] ^ sign);
    }
  }
  template <int NRB>
  static __device__ __forceinline__ void scores(f32x4 (&s)[NRB], const Q (&q)[NRB], const char* kt, int lr, int g) {
#pragma unroll
    for (int rb = 0; rb < NRB; ++rb) s[rb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      const f32x4 a = *(const f32x4*)(kt + lr * ROWB + (((g * (D / 16) + c) ^ kswz(lr)) << 4));
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int rb = 0; rb < NRB; ++rb) s[rb] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], q[rb].f[4 * c + i], s[rb], 0, 0, 0);
    }
  }
  template <int NRB>
  static __device__ __forceinline__ void values(f32x4 (&o)[NRB][D / 16], const f32x4 (&w)[NRB], const char* vt, int lane) {
    const int g = lane >> 4, lr = lane & 15;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int db = 0; db < D / 16; ++db) {
        const float a = *(const float*)(vt + (4 * g + i) * ROWB + (((4 * db + (lr >> 2)) ^ vswz(4 * g)) << 4) + 4 * (lr & 3));
#pragma unroll
        for (int rb = 0; rb < NRB; ++rb) o[rb][db] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, w[rb][i], o[rb][db], 0, 0, 0);
      }
  }
};

template <int D>
struct Narrow<BF16, D> : Narrow16<BF16, D> {};
template <int D>
struct Narrow<F16, D> : Narrow16<F16, D> {};
template <int D>
struct Narrow<F32, D> : Narrow32<D> {};

// Where a workgroup's keys are: sequence b's pages, one KV head.  Strides in bytes.
struct NarrowKeys {
  PageMap pm;
  int b;
  const char* k;
  const char* v;
  int64_t k_sp, v_sp;
  uint32_t k_row, v_row;
  int end;   // no key from here on
  int mine;  // blocks of this wave
};

template <int D, int NRB>
struct NarrowState {
  f32x4 o[NRB][D / 16];
  float m[NRB], l[NRB];
};

// Lane i: the page of this wave's block t + i, which begins at position pos_of(t + i).
template <typename Pos>
__device__ __forceinline__ int narrow_pages(const NarrowKeys& k, int t, Pos pos_of) {
  const int lane = threadIdx.x & 63;
  const int e = pos_of(min(t + lane, max(k.mine - 1, 0))) >> k.pm.shift;
  return e < k.pm.max_pages ? k.pm.table[(int64_t)k.b * k.pm.max_pages + e] : -1;
}

// This wave's blocks 0 .. k.mine - 1.  pages: narrow_pages(k, 0, pos_of).  NB: blocks of a wave's ring, of 2 * 16 rows each, in smem.
// whole(pos): whether every row sees the whole block at pos; seen(key, rb): whether this lane's row of row block rb sees a key.
template <typename T, int D, int NRB, int NB, typename Q, typename Pos, typename Whole, typename Seen>
__device__ __forceinline__ void narrow_stream(NarrowState<D, NRB>& st, const Q (&q)[NRB], const NarrowKeys& k, int pages, char* smem,
                                              int wave, int lane, float scale, bool nontemporal, Pos pos_of, Whole whole,
                                              Seen seen) {
  using N = Narrow<T, D>;
  constexpr int ROWB = D * T::size, BLKB = kBlk * ROWB;
  constexpr int NSL = ROWB / 16, RPR = 1024 / ROWB, NDMA = BLKB / 1024;
  static_assert(NB >= 1 && NB <= 3 && RPR >= 1, "the waits below");
  const int lr = lane & 15, g = lane >> 4;
  uint32_t koff[NDMA], voff[NDMA];
#pragma unroll
  for (int i = 0; i < NDMA; ++i) {
    const int r = i * RPR + lane / NSL;
    koff[i] = r * k.k_row + (((lane % NSL) ^ N::kswz(r)) << 4);
    voff[i] = r * k.v_row + (((lane % NSL) ^ N::vswz(r)) << 4);
  }
  char* const ring = smem + wave * NB * 2 * BLKB;
  const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) char*)ring;
  uint32_t gone = 0;  // places of the ring whose page is not there
  // Rows past the last key, and rows of pages that are not there, read as zeros.
  auto load = [&](int t) __attribute__((always_inline)) {
    const int pos = uni(pos_of(t));
    const int id = __builtin_amdgcn_readlane(pages, t & 63);
    const bool page = (unsigned)id < (unsigned)k.pm.n_pages;
    const int rows = page ? min(max(k.end - pos, 0), kBlk) : 0;
    const int64_t at = page ? id : 0;
    const int in = pos & ((1 << k.pm.shift) - 1);
    const i32x4 rk = uniform_rsrc(k.k + at * k.k_sp + (int64_t)in * k.k_row, rows ? (rows - 1) * k.k_row + ROWB : 0);
    const i32x4 rv = uniform_rsrc(k.v + at * k.v_sp + (int64_t)in * k.v_row, rows ? (rows - 1) * k.v_row + ROWB : 0);
    const int place = t % NB;
    gone = (gone & ~(1u << place)) | ((page ? 0u : 1u) << place);
    const uint32_t la = lds0 + place * 2 * BLKB;
    if (nontemporal) {
#pragma unroll
      for (int i = 0; i < NDMA; ++i) lds_dma16_nt(rk, koff[i], la + i * 1024);
#pragma unroll
      for (int i = 0; i < NDMA; ++i) lds_dma16_nt(rv, voff[i], la + BLKB + i * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < NDMA; ++i) lds_dma16(rk, koff[i], la + i * 1024);
#pragma unroll
      for (int i = 0; i < NDMA; ++i) lds_dma16(rv, voff[i], la + BLKB + i * 1024);
    }
  };

#pragma unroll
  for (int rb = 0; rb < NRB; ++rb) {
    st.m[rb] = -INFINITY;
    st.l[rb] = 0.f;
#pragma unroll
    for (int db = 0; db < D / 16; ++db) st.o[rb][db] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll
  for (int t = 0; t < NB; ++t)
    if (t < k.mine) load(t);
  for (int t = 0; t < k.mine; ++t) {
    // blocks t + 1 .. are on their way
    const int later = min(NB - 1, k.mine - 1 - t);
    if (later >= 2) wait_vmcnt<NB >= 3 ? 4 * NDMA : 0>();
    else if (later == 1) wait_vmcnt<NB >= 2 ? 2 * NDMA : 0>();
    else wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    const char* kt = ring + (t % NB) * 2 * BLKB;
    f32x4 s[NRB];
    N::template scores<NRB>(s, q, kt, lr, g);
    const int pos = uni(pos_of(t));
    const bool hidden = (gone >> (t % NB)) & 1;
    if (hidden || !whole(pos)) {
      asm volatile("");  // a branch: as selects the tests would run for every block
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int rb = 0; rb < NRB; ++rb) s[rb][i] = !hidden && seen(pos + 4 * g + i, rb) ? s[rb][i] : -INFINITY;
    }
    float mx[NRB];
    bool grow = false;
#pragma unroll
    for (int rb = 0; rb < NRB; ++rb) {
      mx[rb] = __builtin_elementwise_maximum(__builtin_elementwise_maximum(s[rb][0], s[rb][1]),
                                             __builtin_elementwise_maximum(s[rb][2], s[rb][3]));
      mx[rb] = tlp::max_xor32(max_xor16(mx[rb])) * scale;
      grow |= mx[rb] > st.m[rb] + Tile<T, D>::kRescale;
    }
    // the maximum moves only when a score passes it by kRescale (it only bounds the exponents)
    if (__any(grow)) {
#pragma unroll
      for (int rb = 0; rb < NRB; ++rb) {
        const float mn = fmaxf(st.m[rb], mx[rb]);
        const float a = fast_exp2(st.m[rb] - (mn == -INFINITY ? 0.f : mn));
        st.m[rb] = mn;
        st.l[rb] *= a;
#pragma unroll
        for (int db = 0; db < D / 16; ++db) st.o[rb][db] *= a;
      }
    }
#pragma unroll
    for (int rb = 0; rb < NRB; ++rb) {
      const float sh = st.m[rb] == -INFINITY ? 0.f : st.m[rb] - Tile<T, D>::kLift;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[rb][i] = fast_exp2(fmaf(s[rb][i], scale, -sh));
        st.l[rb] += s[rb][i];
      }
    }
    N::template values<NRB>(st.o, s, kt + BLKB, lane);
    if (t + NB < k.mine) {
      if (((t + NB) & 63) == 0) pages = narrow_pages(k, t + NB, pos_of);
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the block's place has been read
      load(t + NB);
    }
  }
}

// The waves' states go to LDS: chunk c of row r's accumulators lies in place c ^ (r & 15).  Weights are 2^kLift times 2^(s - m): m is
// told without the lift.
template <typename T, int D, int NRB>
__device__ __forceinline__ void narrow_join(NarrowState<D, NRB>& st, char* smem, float2 (&s_ml)[4][32], int wave, int lane) {
  constexpr int ROWS = 16 * NRB, CH = D / 4;
  const int lr = lane & 15, g = lane >> 4;
#pragma unroll
  for (int rb = 0; rb < NRB; ++rb) st.l[rb] = tlp::sum_xor32(sum_xor16(st.l[rb]));
  __syncthreads();  // every wave is done with its ring
  f32x4* const acc = (f32x4*)smem;
#pragma unroll
  for (int rb = 0; rb < NRB; ++rb) {
    const int r = 16 * rb + lr;
    if (g == 0) s_ml[wave][r] = make_float2(st.m[rb] - Tile<T, D>::kLift, st.l[rb]);
#pragma unroll
    for (int db = 0; db < D / 16; ++db) acc[(wave * ROWS + r) * CH + ((4 * db + g) ^ (r & 15))] = st.o[rb][db];
  }
  __syncthreads();
}

// Chunk c of row r's joined accumulators, its m and l.
template <int D, int NRB>
__device__ __forceinline__ f32x4 narrow_result(const char* smem, const float2 (&s_ml)[4][32], int r, int c, float& m, float& l) {
  constexpr int ROWS = 16 * NRB, CH = D / 4;
  m = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; ++w) m = fmaxf(m, s_ml[w][r].x);
  const float base = m == -INFINITY ? 0.f : m;
  f32x4 a = {0.f, 0.f, 0.f, 0.f};
  l = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float2 e = s_ml[w][r];
    const float f = fast_exp2(e.x - base);
    l = fmaf(e.y, f, l);
    const f32x4 x = ((const f32x4*)smem)[(w * ROWS + r) * CH + (c ^ (r & 15))];
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = fmaf(x[i], f, a[i]);
  }
  return a;
}

}  // namespace tlat
