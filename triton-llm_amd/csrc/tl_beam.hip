// Beam search's selection: of the J V continuations of every batch item's J beams the n best,
//   score(j, v) = s_j + x_jv - log sum_u exp x_ju,
// best first, ties to the lowest j V + v.  The reference has no beam search; it stands beside
// the sampler that replaces its _sample (smollm2_triton/model.py:566-584).
//
// Scores are ordered in 64 bits: neighbours of different beams may differ by less than a 32-bit step of
// their size.  exp, its sums and the logarithm are 64-bit too (see exp_below).
//
// Every logit is read once, by beam_scan, a wave a segment of 1024 entries of a row, bound by the 64-bit operations of exp
// (16 x 8 x 128256 bf16, 33 MB: 14.6 us, 2.3 TB/s; with a 32-bit exp 10.4; with segments of 2048 entries a call takes 2 us
// more, with 512 up to 3 more where the places are many), which leaves
//   * the segment's maximum and its sum of exp against it;
//   * the maximum of every group of 64 entries.
// beam_finish, a workgroup a batch item, has everything else from those.  The best score in a unit (a segment, or
// a group where the segments are few) is base_j + its maximum, base_j = s_j - log-sum-exp.  The units are
// dealt to 64 or 256 classes; the n-th largest of the classes' best (its upper word) is a bound that n continuations
// reach, so only units that reach it are read again, and their entries that reach it are the candidates: about n for
// scattered scores.  A candidate's rank is the number of better ones.  Where the
// candidates are many (ties, rows in order) every wave walks its units in order instead and keeps its 64 best in
// its lanes; those are the candidates then.  beam_finish is latency alone, dependent steps on one CU: 6.1 us for
// 4 x 50257, 10 us for each of 16 x 8 x 128256.
#include "tl_common.h"

#include <limits.h>
#include <math.h>

namespace {

constexpr int kST = 256;                 // threads of beam_scan
constexpr int kVec = 8;                  // neighbouring entries of a lane
constexpr int kVecs = 2;                 // of those a lane has in a segment
constexpr int kSeg = 64 * kVec * kVecs;  // entries of a segment, a wave's
constexpr int kGrp = 64;                 // entries of a group: 8 lanes
constexpr int kFT = 1024;                // threads of beam_finish
constexpr int kFW = kFT / 64;
// Up to kFewPlaces places 64 classes, ranked by one wave (4 x 50257 for 8: 9.5 us, with 256 classes 10.1); beyond them
// 256, ranked by all waves, as of 64 classes too many units reach the bound (4 of 4 x 50257 for 64: 18.7 us, with 64
// classes 57; 16 of 2 x 32000 for 32: 13.0 and 14.6).
constexpr int kFewPlaces = 16;
constexpr int kClasses = 256;
constexpr int kMaxVocab = 262144;
constexpr int kMaxBeams = 64;
constexpr int kMaxSelect = 64;
constexpr int kMaxCand = 1024;           // candidates that are ranked
constexpr int kAtOnce = 4;               // units of a thread that are read together
constexpr int kMaxList = 1024;           // units that are read again
constexpr int kUnitsAPlace = 4;          // segments a place in the selection, below which groups are the units

struct BeamParams {
  const void* logits;
  int64_t row_stride;
  const float* scores;
  int batch, beams, vocab, select;
  int n_seg, n_grp;
  int unit, n_units;  // entries of a unit, units of a row
  uint32_t unit_magic;  // u / n_units = mulhi(u, unit_magic) for every unit u (n_units > 1)
  float* gmax;    // [rows][n_grp]
  float* smax;    // [rows][n_seg]
  double* ssum;   // [rows][n_seg]
  float* out_scores;
  int32_t* out_parents;
  int32_t* out_tokens;
};

// Rows of odd length start anywhere: these loads ask for an element's alignment only.
typedef uint32_t words16 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t words32 __attribute__((ext_vector_type(4), aligned(4)));

size_t align256(size_t b) { return (b + 255) & ~size_t(255); }

// exp(x - m) for x <= m, to 2^-45 of it (any finite number for NaN).  In 64 bits throughout: continuations of different
// beams are ordered by their rows' log-sum-exp, and an error that all entries of a flat floor share does not average
// out (in 32 bits it reached 5e-7).  d log2 e = n + f with whole n and |f| <= 1/2; 2^f by its interpolation of degree 9 at the
// Chebyshev points; n goes into the exponent.  Below e^-700 it is e^-700, which no sum with a 1 in it notices.
// 64-bit products take no longer than 32-bit ones here; their number is what counts (degree 11 and a clamp that keeps
// NaN: 16 x 8 x 128256 27.3 us a call, so 24.1).
__device__ __forceinline__ double exp_below(float x, double m) {
  constexpr double kL = 1.4426950408889634;
  constexpr double kRound = 6755399441055744.0;  // 1.5 2^52: added, a number's whole part stands in its low bits
  constexpr double c[] = {1.0000000000000135,     6.9314718055994617e-01, 2.4022650695640341e-01, 5.5504108664651670e-02,
                          9.6181291939343126e-03, 1.3333558200794592e-03, 1.5403433751251010e-04, 1.5252672924850737e-05,
                          1.3259645244887111e-06, 1.0205905413765595e-07};
  const double d = fmax((double)x - m, -700.);
  const double t = fma(d, kL, kRound);
  const double f = fma(d, kL, kRound - t);
  double e = c[9];
#pragma unroll
  for (int k = 8; k >= 0; --k) e = fma(e, f, c[k]);
  return __builtin_ldexp(e, (int)__builtin_bit_cast(uint64_t, t));
}

// The IEEE maximum: NaN where either is.
__device__ __forceinline__ float max_or_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// kVec neighbouring entries of a row from i on, -inf behind its end.
template <typename T>
__device__ __forceinline__ void load_vec(float (&v)[kVec], const typename T::bits* x, int i, int vocab) {
  if (i + kVec <= vocab) {
    if constexpr (T::size == 2) {
      const words16 w = *(const words16*)(x + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) unpack2<T>(w[e], v[2 * e], v[2 * e + 1]);
    } else {
      const words32 a = *(const words32*)(x + i), b = *(const words32*)(x + i + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = __uint_as_float(a[e]);
        v[4 + e] = __uint_as_float(b[e]);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < kVec; ++e) v[e] = i + e < vocab ? to_f32<T>(x[i + e]) : -INFINITY;
  }
}

__device__ __forceinline__ double shfl_xor_d(double x, int off) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t a = __shfl_xor((uint32_t)u, off), b = __shfl_xor((uint32_t)(u >> 32), off);
  return __builtin_bit_cast(double, (uint64_t)a | ((uint64_t)b << 32));
}
__device__ __forceinline__ double shfl_d(double x, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t a = __shfl((uint32_t)u, lane), b = __shfl((uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)a | ((uint64_t)b << 32));
}

// Reductions by DPP moves, a few cycles each where a move through LDS takes about a hundred, over 8 lanes or a wave (16 x 8 x
// 128256 24.9 -> 24.1 us, 4 x 50257 9.6 -> 9.5 for beam_scan's; 9.8 -> 9.4 before for beam_finish's).
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  const int i = __float_as_int(x);
  return __int_as_float(__builtin_amdgcn_update_dpp(i, i, CTRL, 0xF, 0xF, false));
}
template <int CTRL>
__device__ __forceinline__ double dpp(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const int a = (int)u, b = (int)(u >> 32);
  const uint32_t c = __builtin_amdgcn_update_dpp(a, a, CTRL, 0xF, 0xF, false);
  const uint32_t d = __builtin_amdgcn_update_dpp(b, b, CTRL, 0xF, 0xF, false);
  return __builtin_bit_cast(double, (uint64_t)c | ((uint64_t)d << 32));
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kMirror8 = 0x141, kMirror16 = 0x140;  // quad_perm, row_half_mirror, row_mirror
__device__ __forceinline__ float max8(float x) {
  x = max_or_nan(x, dpp<kXor1>(x));
  x = max_or_nan(x, dpp<kXor2>(x));
  return max_or_nan(x, dpp<kMirror8>(x));
}
__device__ __forceinline__ float lane_f(float x, int i) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), i));
}
__device__ __forceinline__ float wave_max_of8(float x) {  // of max8's results
  x = max_or_nan(x, dpp<kMirror16>(x));
  return max_or_nan(max_or_nan(lane_f(x, 0), lane_f(x, 16)), max_or_nan(lane_f(x, 32), lane_f(x, 48)));
}

// Lane i's value, i the same on every lane.
__device__ __forceinline__ double lane_d(double x, int i) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t a = __builtin_amdgcn_readlane((uint32_t)u, i), b = __builtin_amdgcn_readlane((uint32_t)(u >> 32), i);
  return __builtin_bit_cast(double, (uint64_t)a | ((uint64_t)b << 32));
}

__device__ __forceinline__ double wave_sum(double x) {
  x += dpp<kXor1>(x);
  x += dpp<kXor2>(x);
  x += dpp<kMirror8>(x);
  x += dpp<kMirror16>(x);
  return (lane_d(x, 0) + lane_d(x, 16)) + (lane_d(x, 32) + lane_d(x, 48));
}

template <typename T>
__global__ __launch_bounds__(kST) void beam_scan_kernel(BeamParams p) {
  using B = typename T::bits;
  const int row = blockIdx.y, lane = threadIdx.x & 63;
  const int seg = blockIdx.x * (kST / 64) + (threadIdx.x >> 6);
  if (seg >= p.n_seg) return;
  const B* x = (const B*)p.logits + (int64_t)row * p.row_stride;
  float v[kVecs][kVec];
  const int i0 = seg * kSeg + lane * kVec;
#pragma unroll
  for (int k = 0; k < kVecs; ++k) load_vec<T>(v[k], x, i0 + k * 64 * kVec, p.vocab);
  // NaN anywhere makes the segment's maximum NaN, by which the row's log-sum-exp is one too
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    float g = v[k][0];
#pragma unroll
    for (int e = 1; e < kVec; ++e) g = max_or_nan(g, v[k][e]);
    g = max8(g);
    const int i = i0 + k * 64 * kVec;
    if ((lane & 7) == 0 && i < p.vocab) p.gmax[(int64_t)row * p.n_grp + i / kGrp] = g;
    m = max_or_nan(m, g);
  }
  m = wave_max_of8(m);
  const double base = m == -INFINITY ? 0. : (double)m;  // a segment of -inf alone has no mass
  double s = 0.;
#pragma unroll
  for (int k = 0; k < kVecs; ++k)
#pragma unroll
    for (int i = 0; i < kVec; ++i) s += exp_below(v[k][i], base);
  s = wave_sum(s);
  if (lane == 0) {
    p.smax[(int64_t)row * p.n_seg + seg] = m;
    p.ssum[(int64_t)row * p.n_seg + seg] = s;
  }
}

struct Cand {
  double v;
  int i;  // j V + v
};
__device__ __forceinline__ bool better(double va, int ia, double vb, int ib) {
  return va > vb || (va == vb && ia < ib);
}

// One step of a bitonic network: lanes a distance `off` apart, the better of the two to the lower
// lane where `down`.
__device__ __forceinline__ void exchange(Cand& c, int lane, int off, bool down) {
  const double v = shfl_xor_d(c.v, off);
  const int i = __shfl_xor(c.i, off);
  const bool lower = (lane & off) == 0;
  const bool mine = better(c.v, c.i, v, i);
  if (mine != (lower == down)) c.v = v, c.i = i;
}
__device__ __forceinline__ void sort64(Cand& c, int lane) {  // best in lane 0
  for (int size = 2; size <= 64; size <<= 1)
    for (int off = size >> 1; off > 0; off >>= 1) exchange(c, lane, off, (lane & size) == 0);
}

template <typename T>
__global__ __launch_bounds__(kFT) void beam_finish_kernel(BeamParams p) {
  using B = typename T::bits;
  const int item = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int J = p.beams, n = p.select;
  __shared__ double s_base[kMaxBeams];
  __shared__ double s_best[kFT];
  __shared__ uint32_t s_bound;
  __shared__ __attribute__((aligned(16))) uint32_t s_key[kClasses];
  __shared__ int s_above[kClasses];
  __shared__ int s_n_list, s_n_cand;
  __shared__ int s_list[kMaxList];
  __shared__ double s_cv[kMaxCand];
  __shared__ int s_ci[kMaxCand];

  const int U = p.n_units;
  const float* umax = (p.unit == kGrp ? p.gmax : p.smax) + (int64_t)item * J * U;
  float um[kAtOnce];  // the first of this thread's units, on their way during the sums
#pragma unroll
  for (int k = 0; k < kAtOnce; ++k) um[k] = tid + k * kFT < J * U ? umax[tid + k * kFT] : -INFINITY;
  if (tid == 0) s_n_list = s_n_cand = 0, s_bound = ~0u;
  auto beam_of = [&](int u) { return U == 1 ? u : (int)__umulhi((uint32_t)u, p.unit_magic); };
  // base_j = s_j - log-sum-exp of the row; -inf where either has no value, and such a beam has no
  // continuations
  for (int j = wave; j < J; j += kFW) {
    const int64_t row = (int64_t)item * J + j;
    const float* sm = p.smax + row * p.n_seg;
    const double* ss = p.ssum + row * p.n_seg;
    constexpr int K = kMaxVocab / kSeg / 64;
    float sx[K], m = -INFINITY;
    double part[K], s = 0.;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = lane + 64 * k;
      sx[k] = i < p.n_seg ? sm[i] : -INFINITY;
      part[k] = i < p.n_seg ? ss[i] : 0.;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) m = max_or_nan(m, sx[k]);
    m = wave_max_of8(max8(m));
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (64 * k >= p.n_seg) break;
      s += sx[k] == -INFINITY ? part[k] : part[k] * exp((double)sx[k] - (double)m);  // NaN for NaN and +inf
    }
    s = wave_sum(s);
    if (lane == 0) {
      const double base = (double)p.scores[row] - ((double)m + log(s));
      s_base[j] = base > -INFINITY && base < INFINITY ? base : -INFINITY;
    }
  }
  __syncthreads();

  // the bound: n-th best of the classes' best
  double best = -INFINITY;
#pragma unroll
  for (int k = 0; k < kAtOnce; ++k)
    if (tid + k * kFT < J * U) best = fmax(best, s_base[beam_of(tid + k * kFT)] + (double)um[k]);
  for (int u = tid + kAtOnce * kFT; u < J * U; u += kFT) best = fmax(best, s_base[beam_of(u)] + (double)umax[u]);
  s_best[tid] = best;
  // by the values' upper words, in an order of unsigned numbers: the bound may be lower than the n-th best
  auto key_of = [](double c) {
    const uint32_t hi = (uint32_t)(__builtin_bit_cast(uint64_t, c) >> 32);
    return (int32_t)hi < 0 ? ~hi : hi | 0x80000000u;
  };
  if (n <= kFewPlaces) {
    __syncthreads();
    if (wave == 0) {
      double c = -INFINITY;
#pragma unroll
      for (int w = 0; w < kFW; ++w) c = fmax(c, s_best[w * 64 + lane]);
      const uint32_t key = key_of(c);
      int above = 0;
#pragma unroll
      for (int i = 0; i < 64; ++i) above += (uint32_t)__builtin_amdgcn_readlane(key, i) > key ? 1 : 0;
      if (above < n) atomicMin(&s_bound, key);
    }
  } else {
    if (tid < kClasses) s_above[tid] = 0;
    __syncthreads();
    if (tid < kClasses) {
      double c = s_best[tid];
#pragma unroll
      for (int k = kClasses; k < kFT; k += kClasses) c = fmax(c, s_best[tid + k]);
      s_key[tid] = key_of(c);
    }
    __syncthreads();
    // every thread a class against a part of the others
    constexpr int kPart = kClasses * kClasses / kFT;
    const uint32_t* others = s_key + tid / kClasses * kPart;
    int above = 0;
#pragma unroll
    for (int i = 0; i < kPart; ++i) above += others[i] > s_key[tid % kClasses] ? 1 : 0;
    atomicAdd(&s_above[tid % kClasses], above);
    __syncthreads();
    if (tid < kClasses && s_above[tid] < n) atomicMin(&s_bound, s_key[tid]);
  }
  __syncthreads();
  // the lowest value of this upper word; -inf's has no lower one
  const uint32_t key = s_bound, bhi = key & 0x80000000u ? key & 0x7FFFFFFFu : ~key;
  const uint64_t blo = (int32_t)bhi < 0 && bhi != 0xFFF00000u ? 0xFFFFFFFFu : 0u;
  const double bound = __builtin_bit_cast(double, (uint64_t)bhi << 32 | blo);
  auto reaches = [&](double v) { return v >= bound && v > -INFINITY; };

  if (reaches(best)) {
    auto list = [&](int u, float x) {
      if (reaches(s_base[beam_of(u)] + (double)x)) {
        const int at = atomicAdd(&s_n_list, 1);
        if (at < kMaxList) s_list[at] = u;
      }
    };
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k)
      if (tid + k * kFT < J * U) list(tid + k * kFT, um[k]);
    for (int u = tid + kAtOnce * kFT; u < J * U; u += kFT) list(u, umax[u]);
  }
  __syncthreads();
  const int n_list = s_n_list;
  // this lane's entry 64 c + lane of unit u (of beam u / U)
  auto entry = [&](int u, int c, double& v, int& i) __attribute__((always_inline)) {
    const int j = beam_of(u), at = (u - j * U) * p.unit + c * 64 + lane;
    v = -INFINITY;
    i = INT_MAX;
    if (at < p.vocab) {
      v = s_base[j] + (double)to_f32<T>(((const B*)p.logits)[((int64_t)item * J + j) * p.row_stride + at]);
      i = j * p.vocab + at;
    }
  };
  auto push = [&](double v, int i) {
    const int at = atomicAdd(&s_n_cand, 1);
    if (at < kMaxCand) s_cv[at] = v, s_ci[at] = i;
  };
  if (n_list <= kMaxList && p.unit == kSeg) {
    // a wave two segments, read as beam_scan does
    for (int w = wave; w < n_list; w += 2 * kFW) {
      float x[2][kVecs][kVec];
      int j[2], at[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int wq = w + q * kFW;
        if (wq >= n_list) break;
        const int u = s_list[wq];
        j[q] = beam_of(u);
        at[q] = (u - j[q] * U) * kSeg + lane * kVec;
#pragma unroll
        for (int k = 0; k < kVecs; ++k)
          load_vec<T>(x[q][k], (const B*)p.logits + ((int64_t)item * J + j[q]) * p.row_stride, at[q] + k * 64 * kVec,
                      p.vocab);
      }
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (w + q * kFW >= n_list) break;
        const double base = s_base[j[q]];
#pragma unroll
        for (int k = 0; k < kVecs; ++k) {
          float m = x[q][k][0];
#pragma unroll
          for (int e = 1; e < kVec; ++e) m = fmaxf(m, x[q][k][e]);
          if (!reaches(base + (double)m)) continue;
#pragma unroll
          for (int e = 0; e < kVec; ++e) {
            const double v = base + (double)x[q][k][e];
            if (reaches(v)) push(v, j[q] * p.vocab + at[q] + k * 64 * kVec + e);
          }
        }
      }
    }
  } else if (n_list <= kMaxList) {
    for (int w = wave; w < n_list; w += kAtOnce * kFW) {  // a wave kAtOnce groups
      double v[kAtOnce];
      int i[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        v[k] = -INFINITY;
        if (w + k * kFW < n_list) entry(s_list[w + k * kFW], 0, v[k], i[k]);
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k)
        if (reaches(v[k])) push(v[k], i[k]);
    }
  }
  __syncthreads();
  int n_cand = s_n_cand;
  if (n_list > kMaxList || n_cand > kMaxCand) {
    __syncthreads();
    if (tid == 0) s_n_cand = 0;
    __syncthreads();
    Cand kept{-INFINITY, INT_MAX};  // this wave's 64 best so far, best in lane 0
    for (int u = wave; u < J * U; u += kFW) {
      const double uv = s_base[beam_of(u)] + (double)umax[u];
      if (!(reaches(uv) && uv >= lane_d(kept.v, 63))) continue;
      for (int c = 0; c < p.unit / 64; ++c) {
        Cand x;
        entry(u, c, x.v, x.i);
        if (!(x.v > -INFINITY)) x.v = -INFINITY, x.i = INT_MAX;
        if (!__any(better(x.v, x.i, lane_d(kept.v, 63), __builtin_amdgcn_readlane(kept.i, 63)))) continue;
        sort64(x, lane);
        // the better of i-th best and (63 - i)-th best are the 64 best of both, in a bitonic order
        const double rv = shfl_d(x.v, 63 - lane);
        const int ri = __shfl(x.i, 63 - lane);
        if (better(rv, ri, kept.v, kept.i)) kept.v = rv, kept.i = ri;
        for (int off = 32; off > 0; off >>= 1) exchange(kept, lane, off, true);
      }
    }
    if (kept.v > -INFINITY) {
      const int at = atomicAdd(&s_n_cand, 1);
      s_cv[at] = kept.v, s_ci[at] = kept.i;  // at most 16 waves of 64
    }
    __syncthreads();
    n_cand = s_n_cand;
  }
  static_assert(kMaxCand >= kFW * 64, "every wave's best fit");

  const int64_t o = (int64_t)item * n;
  for (int c = tid; c < n_cand; c += kFT) {
    const double v = s_cv[c];
    const int i = s_ci[c];
    int rank = 0;
#pragma unroll 8
    for (int k = 0; k < n_cand; ++k) rank += better(s_cv[k], s_ci[k], v, i) ? 1 : 0;
    if (rank < n) {
      p.out_scores[o + rank] = (float)v;
      p.out_parents[o + rank] = i / p.vocab;
      p.out_tokens[o + rank] = i - i / p.vocab * p.vocab;
    }
  }
  // fewer continuations than asked for
  for (int r = n_cand + tid; r < n; r += kFT) {
    p.out_scores[o + r] = -INFINITY;
    p.out_parents[o + r] = -1;
    p.out_tokens[o + r] = -1;
  }
}

int n_segments(int vocab) { return (vocab + kSeg - 1) / kSeg; }
int n_groups(int vocab) { return (vocab + kGrp - 1) / kGrp; }

size_t ws_layout(int64_t rows, int vocab, char* base, BeamParams* p) {
  const size_t R = (size_t)rows, S = (size_t)n_segments(vocab), G = (size_t)n_groups(vocab);
  const size_t gb = align256(R * G * 4), mb = align256(R * S * 4), sb = align256(R * S * 8);
  if (p) {
    p->gmax = (float*)base;
    p->smax = (float*)(base + gb);
    p->ssum = (double*)(base + gb + mb);
  }
  return gb + mb + sb;
}

template <typename T>
int launch_beam(const BeamParams& p, hipStream_t st) {
  hipLaunchKernelGGL(beam_scan_kernel<T>, dim3((p.n_seg + kST / 64 - 1) / (kST / 64), p.batch * p.beams), dim3(kST), 0,
                     st, p);
  const int e = tl_launch_status();
  if (e) return e;
  hipLaunchKernelGGL(beam_finish_kernel<T>, dim3(p.batch), dim3(kFT), 0, st, p);
  return tl_launch_status();
}

bool beam_sizes_ok(int batch, int beams, int vocab, int select) {
  return batch > 0 && beams > 0 && beams <= kMaxBeams && (int64_t)batch * beams <= 65535 && vocab > 0 &&
         vocab <= kMaxVocab && select > 0 && select <= kMaxSelect;
}

}  // namespace

extern "C" {

int tl_beam_max_select(void) { return kMaxSelect; }

size_t tl_beam_select_workspace_bytes(int batch, int beams, int vocab) {
  if (!beam_sizes_ok(batch, beams, vocab, 1)) return 0;
  return ws_layout((int64_t)batch * beams, vocab, nullptr, nullptr);
}

int tl_beam_select(const void* logits, const float* scores, int batch, int beams, int vocab, int64_t row_stride,
                   int select, float* out_scores, int32_t* out_parents, int32_t* out_tokens, void* workspace,
                   size_t workspace_bytes, int dtype, void* stream) {
  if (batch == 0 || select == 0) return 0;
  if (!logits || !scores || !out_scores || !out_parents || !out_tokens || !workspace || batch < 0 || beams < 1 ||
      vocab < 1 || select < 0 || row_stride < vocab || ((uintptr_t)workspace & 15))
    return TL_ERR_INVALID;
  if (dtype != TL_DTYPE_F32 && dtype != TL_DTYPE_F16 && dtype != TL_DTYPE_BF16) return TL_ERR_INVALID;
  if (!beam_sizes_ok(batch, beams, vocab, select)) return TL_ERR_UNSUPPORTED;
  if (workspace_bytes < tl_beam_select_workspace_bytes(batch, beams, vocab)) return TL_ERR_INVALID;
  BeamParams p{};
  p.logits = logits;
  p.row_stride = row_stride;
  p.scores = scores;
  p.batch = batch;
  p.beams = beams;
  p.vocab = vocab;
  p.select = select;
  p.n_seg = n_segments(vocab);
  p.n_grp = n_groups(vocab);
  // Segments where they are several for each place, so that few of them reach the bound, and no class is empty.  us a
  // call with segments / with groups: 16 x 8 x 128256 for 16 24.1 / 30.3, 4 x 50257 for 8 9.5 / 9.8; 1 x 50257 for 4
  // 8.5 / 8.3, 16 of 2 x 32000 for 32 34.0 / 13.0.
  const bool segments = (int64_t)beams * p.n_seg >= kUnitsAPlace * select && (int64_t)beams * p.n_seg >= 64;
  p.unit = segments ? kSeg : kGrp;
  p.n_units = segments ? p.n_seg : p.n_grp;
  // exact: at most 2^18 units in all, and n_units <= 2^12, so that the magic's excess times a unit stays below 2^32
  p.unit_magic = (uint32_t)((((uint64_t)1 << 32) + p.n_units - 1) / p.n_units);
  ws_layout((int64_t)batch * beams, vocab, (char*)workspace, &p);
  p.out_scores = out_scores;
  p.out_parents = out_parents;
  p.out_tokens = out_tokens;
  hipStream_t st = tl_resolve_stream(stream);
  switch (dtype) {
    case TL_DTYPE_F32: return launch_beam<F32>(p, st);
    case TL_DTYPE_F16: return launch_beam<F16>(p, st);
    default: return launch_beam<BF16>(p, st);
  }
}

}  // extern "C"
