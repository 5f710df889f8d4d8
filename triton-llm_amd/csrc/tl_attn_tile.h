// Internal header: the matrix products of one 32-row block of queries with a tile of keys in LDS, as the windowed and the shared
// attention use them (tl_window.hip, tl_shared.hip).  Not part of the C ABI.
//
// The products are transposed, S^T = K . Q^T and O^T = V^T . P^T, on 32 x 32 MFMA blocks: lane l of the accumulator holds
// query row l % 32, and P^T goes from the accumulator's registers straight into the second product.
#pragma once

#include "tl_prefill.h"

namespace tlat {

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
  // sign: flips of the values' sign bits
  static __device__ __forceinline__ void load_q(Q& q, const char* row, bool there, int h, uint32_t sign) {
    sign |= sign >> 16;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      u32x4 x = u32x4{0u, 0u, 0u, 0u};
      if (there) x = *(const u32x4*)(row + 32 * ks + 16 * h);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] ^= sign;
      q.f[ks] = __builtin_bit_cast(frag, x);
    }
  }
  // Operands are read kAhead MFMAs ahead; the barriers keep the compiler from reading them all at
  // once, which their registers do not allow at d_k 128.
  static constexpr int kAhead = 4;
  // The sum of a row's weights.  At d_k 64 the vector unit is the limit and the matrix unit half idle: there it is one
  // more MFMA per 16 keys, ones . P^T, of the rounded weights (4 x 500 rows on prefixes, fp16: 51.4 -> 47.8 us).
  static constexpr bool kSumMfma = D == 64;
  // Weights are rounded to the storage type for the second product: an error of the size of the output's own rounding (a second
  // word a weight takes it away, and 169 us for 134 at 8192 bf16 rows, 53 for 41 at 4 x 500 fp16 ones).  A weight is 2^kLift times exp2 of its score's
  // distance to the running maximum, and that lags behind the largest score by kRescale at most.  bf16 has fp32's exponents:
  // half a step each.  fp16 ends at 2^16 and is subnormal below 2^-14: lifted by 2^9 a weight is at most 2^15, has half a
  // step down to 2^-23 of the row's largest, and below that an error of 2^-34 of it at most.  (A lift of 2^11 leaves 2^4 for
  // the lag: 6000 rows, window 1024, 15 / 5 heads of 64, scores of deviation 6, 47.5 us for 45.5; of deviation 1 43 with either.)
  static constexpr float kLift = T::code == TL_DTYPE_F16 ? 9.f : 0.f;
  static constexpr float kRescale = T::code == TL_DTYPE_F16 ? 6.f : 8.f;
  static __device__ __forceinline__ void scores(f32x16 (&s)[NMB], const Q& q, const char* kt, int lq, int h) {
    constexpr int NG = NMB * NKS;
    const char* row = kt + lq * ROWB;
    const int sw = (h ^ k_swz<T, D>(lq)) << 4;
    u32x4 f[NG];
    auto fetch = [&](int g) __attribute__((always_inline)) {
      f[g] = *(const u32x4*)(row + 32 * (g % NMB) * ROWB + (sw ^ ((g / NMB) << 5)));
    };
#pragma unroll
    for (int g = 0; g < kAhead; ++g) fetch(g);
#pragma unroll
    for (int mb = 0; mb < NMB; ++mb)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[mb][r] = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      if (g + kAhead < NG) fetch(g + kAhead);
      s[g % NMB] = M::mma(__builtin_bit_cast(frag, f[g]), q.f[g / NMB], s[g % NMB]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  // s holds the weights; they are rounded to the storage type here (see kLift).  The sum of a row's weights is
  // of the rounded ones in la (kSumMfma) and of the unrounded ones in l otherwise, in fp32 either way: a weight's rounding
  // then counts in numerator and denominator, or in the numerator alone, half a step of the output at most in both.
  // WHOLE: a weight goes into the products in two words, its rounding and what that left out (2^-16 of it in bf16, less in fp16), so
  // that no weight's rounding shows.  Packed rows go without, as padded ones do: 30 tokens beside two prompts, bf16, would take 78.2 us for
  // 73.5, 12 prompts of up to 1400, fp16, 66.3 for 49.6.
  template <bool WHOLE = false>
  static __device__ __forceinline__ void values(f32x16 (&o)[NDB], f32x16& la, const f32x16 (&s)[NMB], const char* vt,
                                                int lane) {
    typedef short v4s __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) v4s lds_v4s;
    constexpr int NG = 2 * NMB * NDB;
    const int g16 = lane >> 4, e = (lane >> 2) & 3, c = lane & 3;
    const auto* lds = (const __attribute__((address_space(3))) char*)vt + (4 * (g16 >> 1) + e) * ROWB + 8 * (c & 1);
    const int sw = ((2 * (g16 & 1) + (c >> 1)) ^ v_swz<T, D>(e)) << 4;
    u32x4 f[NG];
    u32x4 pw[2 * NMB], rest;
    auto fetch = [&](int g) __attribute__((always_inline)) {
      const auto* at = lds + 16 * (g / NDB) * ROWB + (sw ^ ((g % NDB) << 6));
      const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)at));
      const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + 8 * ROWB)));
      f[g] = u32x4{a.x, a.y, b.x, b.y};
    };
#pragma unroll
    for (int g = 0; g < kAhead; ++g) fetch(g);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const int tt = g / NDB, db = g % NDB;
      if (db == 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x[2] = {s[tt >> 1][8 * (tt & 1) + 2 * j], s[tt >> 1][8 * (tt & 1) + 2 * j + 1]};
          pw[tt][j] = pack2<T>(x);
          if constexpr (WHOLE) {
            float r[2];
            unpack2<T>(pw[tt][j], r[0], r[1]);
            r[0] = x[0] - r[0], r[1] = x[1] - r[1];
            rest[j] = pack2<T>(r);
          }
        }
      }
      if (g + kAhead < NG) fetch(g + kAhead);
      o[db] = M::mma(__builtin_bit_cast(frag, f[g]), __builtin_bit_cast(frag, pw[tt]), o[db]);
      if constexpr (WHOLE) o[db] = M::mma(__builtin_bit_cast(frag, f[g]), __builtin_bit_cast(frag, rest), o[db]);
      if (kSumMfma && db == 0) {
        const frag ones = __builtin_bit_cast(frag, u32x4{T::one_pair, T::one_pair, T::one_pair, T::one_pair});
        la = M::mma(ones, __builtin_bit_cast(frag, pw[tt]), la);
        if constexpr (WHOLE) la = M::mma(ones, __builtin_bit_cast(frag, rest), la);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

template <int D>
struct Tile32 {
  static constexpr int ROWB = D * 4, NDB = D / 32, NMB = 1;
  static constexpr bool kSumMfma = false;
  static constexpr float kLift = 0.f, kRescale = 8.f;
  struct Q {
    float f[D / 2];  // features h D / 2 .. of the row
  };
  static __device__ __forceinline__ void load_q(Q& q, const char* row, bool there, int h, uint32_t sign) {
#pragma unroll
    for (int c = 0; c < D / 8; ++c) {
      u32x4 x = u32x4{0u, 0u, 0u, 0u};
      if (there) x = *(const u32x4*)(row + h * (D * 2) + 16 * c);
#pragma unroll
      for (int i = 0; i < 4; ++i) q.f[4 * c + i] = __uint_as_float(x[i] ^ sign);
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
  template <bool WHOLE = false>  // nothing is rounded here
  static __device__ __forceinline__ void values(f32x16 (&o)[NDB], f32x16& la, const f32x16 (&s)[NMB], const char* vt,
                                                int lane) {
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

// Four neighbouring outputs, rounded to nearest even.
template <typename T>
__device__ __forceinline__ void store4(typename T::bits* d, float a, float b, float c, float e, int vec) {
  if constexpr (T::size == 4) {
    if (vec) {
      *(f32x4*)d = f32x4{a, b, c, e};
    } else {
      d[0] = __float_as_uint(a), d[1] = __float_as_uint(b), d[2] = __float_as_uint(c), d[3] = __float_as_uint(e);
    }
  } else {
    const float x[2] = {a, b}, y[2] = {c, e};
    const uint32_t lo = pack2<T>(x), hi = pack2<T>(y);
    if (vec) {
      *(u32x2*)d = u32x2{lo, hi};
    } else {
      d[0] = (uint16_t)lo, d[1] = (uint16_t)(lo >> 16), d[2] = (uint16_t)hi, d[3] = (uint16_t)(hi >> 16);
    }
  }
}

}  // namespace tlat
