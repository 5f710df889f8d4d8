// The paged KV cache: what writes it (paged_append), reads it for one new token a
// sequence (paged_decode) and copies its pages (copy_pages).
//
// The reference keeps one contiguous cache per sequence on the host
// (smollm2_triton/model.py:190-225) and has no pages; positions, RoPE and attention
// semantics are those of rope_kv_append and attention_decode here.
#include "tl_paged.h"

#include <math.h>

#include <type_traits>

using namespace tlpg;

namespace {

// ---------------------------------------------------------------------------------
// Append: rotary positions on q and k, k and v into the pages.  A padded batch's token s of sequence b has position lens[b] + s
// and finds its page in the table; a packed one's (SLOTS) comes with its position and its slot, page * page_size + row.
//
//   half         (x_i, x_{i + r/2}) -> (x_i c - x_{i + r/2} s, x_{i + r/2} c + x_i s)
//   interleaved  (x_{2i}, x_{2i+1}) likewise;   i < r / 2, r rotated features of d_k
//
// with c, s the tables' entry i of row `position`.  Products and sums are rounded one by
// one in fp32 and once to the storage type (as rope_kv_append's are, whose bits this gives).
// Bytes only: every row is read and written once.
// ---------------------------------------------------------------------------------
enum { kNoRope = 0, kHalf = 1, kInterleaved = 2 };

struct AppendParams {
  const void* q;
  void* qo;
  const void* kn;
  const void* vn;
  void* kp;
  void* vp;
  PageMap pm;
  const int32_t* lens;
  const int32_t* new_lens;  // NULL: n_new for every sequence
  const int32_t* slots;      // SLOTS: by token (batch 1), and positions (NULL without rotary positions)
  const int32_t* positions;
  int past_caches;  // SLOTS: rows are read without keeping them in the caches
  const float* cos_t;
  const float* sin_t;
  int rope_rows, rot_half;
  int batch, n_new, n_head, n_kv, d_k;
  int64_t q_sb, q_ss, q_sh;
  int64_t qo_sb, qo_ss, qo_sh;
  int64_t kn_sb, kn_ss, kn_sh;
  int64_t vn_sb, vn_ss, vn_sh;
  int64_t kp_sp, kp_sh, kp_sr;
  int64_t vp_sp, vp_sh, vp_sr;
};

// Where token s of sequence b goes (row: in its page); false: it is not written (see the header).
template <bool SLOTS>
__device__ __forceinline__ bool token_place(const AppendParams& p, int b, int s, bool rope, int& pos, int& page, int& row) {
  if constexpr (SLOTS) {
    const int slot = p.slots[s];
    pos = rope ? p.positions[s] : 0;
    page = slot >> p.pm.shift;
    row = slot & ((1 << p.pm.shift) - 1);
    if (rope && (unsigned)pos >= (unsigned)p.rope_rows) return false;
  } else {
    if (p.new_lens && s >= p.new_lens[b]) return false;
    const int64_t at = (int64_t)p.lens[b] + s;
    if (at < 0 || (at >> p.pm.shift) >= p.pm.max_pages || (rope && at >= p.rope_rows)) return false;
    pos = (int)at;
    page = p.pm.table[(int64_t)b * p.pm.max_pages + (pos >> p.pm.shift)];
    row = pos & ((1 << p.pm.shift) - 1);
  }
  return (unsigned)page < (unsigned)p.pm.n_pages;
}

// Row r of token (b, s) -- its n_head q rows, then n_kv k rows, then n_kv v rows -- as
// source and destination addresses.
template <typename B>
__device__ __forceinline__ void token_row(const AppendParams& p, int b, int s, int row, int page, int r, const B*& src,
                                          B*& dst) {
  if (r < p.n_head) {
    src = (const B*)p.q + b * p.q_sb + s * p.q_ss + r * p.q_sh;
    dst = (B*)p.qo + b * p.qo_sb + s * p.qo_ss + r * p.qo_sh;
  } else if (r < p.n_head + p.n_kv) {
    const int h = r - p.n_head;
    src = (const B*)p.kn + b * p.kn_sb + s * p.kn_ss + h * p.kn_sh;
    dst = (B*)p.kp + page * p.kp_sp + h * p.kp_sh + row * p.kp_sr;
  } else {
    const int h = r - p.n_head - p.n_kv;
    src = (const B*)p.vn + b * p.vn_sb + s * p.vn_ss + h * p.vn_sh;
    dst = (B*)p.vp + page * p.vp_sp + h * p.vp_sh + row * p.vp_sr;
  }
}

// One element pair a thread: any even d_k, any strides.
template <typename T, int MODE, bool SLOTS>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendParams p) {
  using B = typename T::bits;
  const int pairs = p.d_k / 2, rows = p.n_head + 2 * p.n_kv;
  const int64_t tid = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (tid >= (int64_t)p.batch * p.n_new * rows * pairs) return;
  const int i = (int)(tid % pairs);
  const int64_t t = tid / pairs;
  const int r = (int)(t % rows);
  const int64_t tok = t / rows;
  const int b = (int)(tok / p.n_new), s = (int)(tok % p.n_new);
  int pos, page, row;
  if (!token_place<SLOTS>(p, b, s, MODE != kNoRope, pos, page, row)) return;
  const B* src;
  B* dst;
  token_row(p, b, s, row, page, r, src, dst);
  int x = 2 * i, y = 2 * i + 1;
  if (MODE == kHalf && i < p.rot_half) x = i, y = i + p.rot_half;
  const B sx = src[x], sy = src[y];
  if (MODE != kNoRope && i < p.rot_half && r < p.n_head + p.n_kv) {
    const int64_t at = (int64_t)pos * p.rot_half + i;
    float ox, oy;
    rope_rotate_pair(to_f32<T>(sx), to_f32<T>(sy), p.cos_t[at], p.sin_t[at], ox, oy);
    dst[x] = from_f32<T>(ox);
    dst[y] = from_f32<T>(oy);
  } else {
    dst[x] = sx;
    dst[y] = sy;
  }
}

// 16 bytes of a row at once.  A row is cut into pairs of 16-byte chunks, thread j of a row's d_k / 2 / VEC
// taking one pair: in the half layout the two chunks that are turned into each other, behind the turned features
// and in the other layouts two neighbours (an interleaved chunk is turned in itself).  A thread takes
// rows g, g + R, ... of its token and loads its angles once for all of them.  8 prompts of up to 1999 tokens, 15 / 5 heads
// of 64, fp16, 72 MB: 18.4 us, 3.9 TB/s; by pairs of elements (paged_append_kernel) 51 us.
// PAST: rows are read without keeping them in the caches.
template <typename T, int MODE, bool SLOTS, bool PAST>
__global__ __launch_bounds__(256) void paged_append_vec_kernel(AppendParams p, int R) {
  using B = typename T::bits;
  constexpr int VEC = 16 / T::size;
  constexpr int UNROLL = 4;
  const int per_row = p.d_k / (2 * VEC);
  const int64_t tid = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per_tok = per_row * R;
  if (tid >= (int64_t)p.batch * p.n_new * per_tok) return;
  const int64_t tok = tid / per_tok;
  const int rest = (int)(tid - tok * per_tok);
  const int g = rest / per_row, j = rest - g * per_row;
  const int b = (int)(tok / p.n_new), s = (int)(tok - (int64_t)b * p.n_new);
  int pos, page, row;
  if (!token_place<SLOTS>(p, b, s, MODE != kNoRope, pos, page, row)) return;

  const int turned = MODE == kHalf ? p.rot_half / VEC : 0;  // pairs of chunks that turn into each other
  const bool across = MODE == kHalf && j < turned;
  const int ca = across ? j : MODE == kHalf ? 2 * turned + 2 * (j - turned) : 2 * j;
  const int cb = across ? j + turned : ca + 1;
  const bool in_a = MODE == kInterleaved && ca * VEC < 2 * p.rot_half;
  const bool in_b = MODE == kInterleaved && cb * VEC < 2 * p.rot_half;
  // angles: across, VEC of them at j VEC; inside, VEC / 2 a chunk at ca VEC / 2
  float c[VEC], sn[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) c[i] = 1.f, sn[i] = 0.f;
  if (MODE != kNoRope && (across || in_a)) {
    const int64_t at = (int64_t)pos * p.rot_half + j * VEC;
    const int n = across || in_b ? VEC : VEC / 2;
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i < n) c[i] = p.cos_t[at + i], sn[i] = p.sin_t[at + i];
  }
  auto unpack = [](const u32x4& w, float (&f)[VEC]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (T::size == 4) f[i] = __uint_as_float(w[i]);
      else unpack2<T>(w[i], f[2 * i], f[2 * i + 1]);
    }
  };
  auto pack = [](const float (&f)[VEC]) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (T::size == 4) w[i] = __float_as_uint(f[i]);
      else w[i] = (uint32_t)from_f32<T>(f[2 * i]) | ((uint32_t)from_f32<T>(f[2 * i + 1]) << 16);
    }
    return w;
  };
  const int rows = p.n_head + 2 * p.n_kv, rot_rows = p.n_head + p.n_kv;
  for (int r = g; r < rows; r += UNROLL * R) {
    u32x4 wa[UNROLL], wb[UNROLL];
    B* out[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      if (r + u * R < rows) {
        const B* src;
        token_row(p, b, s, row, page, r + u * R, src, out[u]);
        if constexpr (PAST) {
          wa[u] = __builtin_nontemporal_load((const u32x4*)(src + ca * VEC));
          wb[u] = __builtin_nontemporal_load((const u32x4*)(src + cb * VEC));
        } else {
          wa[u] = *(const u32x4*)(src + ca * VEC);
          wb[u] = *(const u32x4*)(src + cb * VEC);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      if (r + u * R < rows) {
        u32x4 oa = wa[u], ob = wb[u];
        if (MODE != kNoRope && r + u * R < rot_rows && (across || in_a)) {
          float x[VEC], y[VEC];
          unpack(wa[u], x);
          unpack(wb[u], y);
          if (MODE == kHalf) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) rope_rotate_pair(x[i], y[i], c[i], sn[i], x[i], y[i]);
          } else {
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) {
              rope_rotate_pair(x[2 * i], x[2 * i + 1], c[i], sn[i], x[2 * i], x[2 * i + 1]);
              if (in_b) rope_rotate_pair(y[2 * i], y[2 * i + 1], c[VEC / 2 + i], sn[VEC / 2 + i], y[2 * i], y[2 * i + 1]);
            }
          }
          oa = pack(x);
          if (MODE == kHalf || in_b) ob = pack(y);
        }
        *(u32x4*)(out[u] + ca * VEC) = oa;
        *(u32x4*)(out[u] + cb * VEC) = ob;
      }
    }
  }
}

// Whether every row can be moved in whole 16-byte chunks, turned features ending at a chunk's end.
template <typename T>
bool append_vec_ok(const AppendParams& p, int mode) {
  constexpr int VEC = 16 / T::size;
  if (p.d_k % (2 * VEC)) return false;
  if (mode == kHalf && p.rot_half % VEC) return false;
  if (mode == kInterleaved && (2 * p.rot_half) % VEC) return false;
  const int64_t st[] = {p.kn_sb, p.kn_ss, p.kn_sh, p.vn_sb, p.vn_ss, p.vn_sh, p.kp_sp, p.kp_sh, p.kp_sr,
                        p.vp_sp, p.vp_sh, p.vp_sr, p.q_sb,  p.q_ss,  p.q_sh,  p.qo_sb, p.qo_ss, p.qo_sh};
  for (int64_t x : st)
    if (x % VEC) return false;
  return !(((uintptr_t)p.q | (uintptr_t)p.qo | (uintptr_t)p.kn | (uintptr_t)p.vn | (uintptr_t)p.kp | (uintptr_t)p.vp) & 15);
}

template <typename T, int MODE, bool SLOTS>
int launch_append_mode(const AppendParams& p, hipStream_t st) {
  const int rows = p.n_head + 2 * p.n_kv;
  if (append_vec_ok<T>(p, MODE)) {
    // A decoded token: a thread a chunk pair.  Prompts: about 2^18 threads, each with several rows
    // for one load of its angles.
    const int64_t lanes = (int64_t)p.batch * p.n_new * (p.d_k / (2 * (16 / T::size)));
    int64_t groups = ((int64_t)1 << 18) / lanes;
    groups = groups < 1 ? 1 : groups > rows ? rows : groups;
    const int64_t blocks = (lanes * groups + 255) / 256;
    if (blocks > INT32_MAX) return TL_ERR_UNSUPPORTED;
    if (SLOTS && p.past_caches)
      hipLaunchKernelGGL((paged_append_vec_kernel<T, MODE, SLOTS, SLOTS>), dim3((unsigned)blocks), dim3(256), 0, st, p, (int)groups);
    else
      hipLaunchKernelGGL((paged_append_vec_kernel<T, MODE, SLOTS, false>), dim3((unsigned)blocks), dim3(256), 0, st, p, (int)groups);
    return tl_launch_status();
  }
  const int64_t blocks = ((int64_t)p.batch * p.n_new * rows * (p.d_k / 2) + 255) / 256;
  if (blocks > INT32_MAX) return TL_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((paged_append_kernel<T, MODE, SLOTS>), dim3((unsigned)blocks), dim3(256), 0, st, p);
  return tl_launch_status();
}

template <typename T, bool SLOTS>
int launch_append(const AppendParams& p, int mode, hipStream_t st) {
  return mode == kHalf          ? launch_append_mode<T, kHalf, SLOTS>(p, st)
         : mode == kInterleaved ? launch_append_mode<T, kInterleaved, SLOTS>(p, st)
                                : launch_append_mode<T, kNoRope, SLOTS>(p, st);
}

// ---------------------------------------------------------------------------------
// One new token a sequence over its pages: o = softmax(scale q . K^T over the keys it
// sees) V, the softmax's running maximum m and sum l kept in fp32 (log2 domain):
//   m' = max(m, s),  l' = l 2^(m - m') + 2^(s - m'),  acc' = acc 2^(m - m') + 2^(s - m') v
// and two states joined as (max m, sum l_i 2^(m_i - m), sum acc_i 2^(m_i - m)).
//
// Work.  The blocks of 16 positions that a sequence's query sees (all of them, or a
// window's and the sinks') are laid end to end, (sequence, pair, block), a pair being one KV head with up to
// 8 of its query heads, and cut into equal shares, a workgroup each, whatever the lengths.
// A share may end inside a pair and go on in the next; each piece is a segment.  A pair inside one
// share is finished there; else each segment leaves (m, l, acc) in the workspace, and
// the last of them joins them.  A share has at most one segment of a pair that began before it
// (slot 0) and one of a pair that goes on after it (slot 1), so the workspace is two
// slots a workgroup, whatever batch and length are.
//
// Bound by the reading of K and V: 64 sequences of 4096 to 16383 positions, 24 / 8 heads of 128, bf16, 2.9 GB: 444 us,
// 6.5 TB/s; shorter calls by the latency of a few dependent loads.
// ---------------------------------------------------------------------------------
constexpr int kDecThreads = 256;
constexpr int kDecWaves = kDecThreads / 64;
constexpr int kMaxShares = 2048;  // workgroups at most: bounds the workspace
constexpr int kMinShare = 4;      // blocks of a share at least: one for each wave
constexpr int64_t kPairMaxBytes = 384ll << 10;
constexpr int64_t kPairMaxAll = 64ll << 20;
constexpr int64_t kPairFewBytes = 128ll << 10;
constexpr int kPairMany = 64;
constexpr float kRescaleLog2 = 8.f;
constexpr int kAuxNontemporal = 2;  // buffer-load cache policy: nt
constexpr uint32_t kPastEnd = 0x7FFFFF00u;  // an offset that every resource here ends before

struct DecodeParams {
  const void* q;
  const void* k;
  const void* v;
  const int32_t* lens;
  PageMap pm;
  uint64_t tag;     // this call's
  uint64_t* words;  // [share][2]: the tag where that segment's results are there
  float* ws_ml;   // [share][2][heads_per_pair][2]
  float* ws_acc;  // [share][2][heads_per_pair][D]
  void* o;
  int len_add, window, sinks;
  int batch, n_head, n_kv, group;
  int heads_per_pair, n_pairs, n_shares;
  int64_t q_sb, q_sh, o_sb, o_sh;
  int64_t k_sp, k_sh, v_sp, v_sh;     // page and head strides in elements
  uint32_t k_row_bytes, v_row_bytes;  // row strides in bytes
  float scale_log2;
};

// What sequence b's query sees: len positions, `lo` the window's first; n blocks, the
// first ns of them from the sequence's start on, the others from block wb on.
struct Seen {
  int len, lo, n, ns, wb;
};
__device__ __forceinline__ Seen seen_of(const DecodeParams& p, int b) {
  Seen s;
  int64_t len = (int64_t)p.lens[b] + p.len_add;
  const int64_t cap = (int64_t)p.pm.max_pages << p.pm.shift;
  len = len < 0 ? 0 : len > cap ? cap : len;
  s.len = (int)len;
  const int nb = (int)((len + kBlk - 1) >> kBlkShift);
  s.lo = p.window > 0 && s.len > p.window ? s.len - p.window : 0;
  s.ns = s.n = nb;
  s.wb = 0;
  if (s.lo > 0) {
    const int sb = min(nb, (int)(((int64_t)p.sinks + kBlk - 1) >> kBlkShift));
    const int wb = s.lo >> kBlkShift;
    if (wb > sb) {
      s.ns = sb;
      s.wb = wb;
      s.n = sb + nb - wb;
    }
  }
  return s;
}

__device__ __forceinline__ bool row_seen(const Seen& s, int sinks, int pos) {
  return pos < s.len && (pos >= s.lo || pos < sinks);
}

// How the blocks are dealt.  Even shares of the flattened blocks, whole rounds of the waves, where the pairs are many;
// a share may then hold the end of one pair and the beginning of the next.  Where that costs a share at most two
// rounds of the waves, every pair is cut by itself into parts of `share` blocks instead, so that no workgroup runs one
// short segment after another: 8 pairs of 100 positions (d_k 128, bf16) 13.6 -> 10.0 us, 64 of 500 17.2 -> 14.2; 512 pairs
// of 10000, where the parts would be twice the shares, 441 as shares and 486 as parts.
// Batches beyond 64 are walked 64 sequences at a time, by every workgroup: 512 of 1024 positions, 24 / 8 heads of 128, bf16, take 335
// us, 64 of 8192 330.
// unit(n): what a pair of n blocks counts, blocks or parts; incl: those of sequences 0 .. lane, for all pairs.
struct Layout {
  bool padded;
  int share, total;
  int n, incl;  // lane's sequence (of the first 64)
  __device__ __forceinline__ int unit(int blocks) const { return padded ? (blocks + share - 1) / share : blocks; }
};
__device__ __forceinline__ int blocks_at(const DecodeParams& p, int b) { return b < p.batch ? seen_of(p, b).n : 0; }

__device__ __forceinline__ Layout layout_of(const DecodeParams& p, int lane) {
  Layout y;
  y.n = blocks_at(p, lane);
  y.incl = wave_scan(y.n * p.n_pairs);
  y.total = last_lane(y.incl);
  for (int b0 = 64; b0 < p.batch; b0 += 64) y.total += last_lane(wave_scan(blocks_at(p, b0 + lane) * p.n_pairs));
  const int pairs = p.batch * p.n_pairs;
  auto share_of = [&](int shares) {
    const int r = max((int)(((unsigned)y.total + shares - 1) / shares), kMinShare);
    return (r + kDecWaves - 1) / kDecWaves * kDecWaves;
  };
  y.share = share_of(p.n_shares);
  y.padded = 2 * pairs <= p.n_shares && share_of(p.n_shares - pairs) <= y.share + 2 * kDecWaves;
  if (y.padded) y.share = share_of(p.n_shares - pairs);
  if (y.padded) {
    y.incl = wave_scan(y.unit(y.n) * p.n_pairs);
    y.total = last_lane(y.incl);
    for (int b0 = 64; b0 < p.batch; b0 += 64)
      y.total += last_lane(wave_scan(y.unit(blocks_at(p, b0 + lane)) * p.n_pairs));
  }
  return y;
}

// The sequence that unit r < total belongs to, and its first unit.
struct Owner {
  int b, first;
};
__device__ __forceinline__ Owner owner_of(const DecodeParams& p, const Layout& y, int r, int lane) {
  int b0 = 0, n = y.unit(y.n) * p.n_pairs, incl = y.incl;
  while (b0 + 64 < p.batch && last_lane(incl) <= r) {
    const int base = last_lane(incl);
    b0 += 64;
    n = y.unit(blocks_at(p, b0 + lane)) * p.n_pairs;
    incl = base + wave_scan(n);
  }
  const int li = uni(__ffsll((unsigned long long)__ballot(incl > r)) - 1);
  return Owner{b0 + li, uni(__builtin_amdgcn_readlane(incl - n, li))};
}
// The first unit of sequence b.
__device__ __forceinline__ int first_of(const DecodeParams& p, const Layout& y, int b, int lane) {
  int base = 0, n = y.unit(y.n) * p.n_pairs, incl = y.incl;
  for (int b0 = 64; b0 <= b; b0 += 64) {
    base = last_lane(incl);
    n = y.unit(blocks_at(p, b0 + lane)) * p.n_pairs;
    incl = base + wave_scan(n);
  }
  return uni(__builtin_amdgcn_readlane(incl - n, b & 63));
}

template <int W>
struct Slice {
  uint32_t w[W];
};

// A row's slice at byte offset voff + soff of a block (soff the same on every lane).
template <int W>
__device__ __forceinline__ void load_slice(Slice<W>& s, __amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff) {
  if constexpr (W == 2) {
    const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, voff, soff, kAuxNontemporal));
    s.w[0] = a.x;
    s.w[1] = a.y;
  } else {
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
      const u32x4 a =
          __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, voff + 16 * i, soff, kAuxNontemporal));
      s.w[4 * i + 0] = a.x;
      s.w[4 * i + 1] = a.y;
      s.w[4 * i + 2] = a.z;
      s.w[4 * i + 3] = a.w;
    }
  }
}

template <typename T, int W>
__device__ __forceinline__ float dot_slice(const Slice<W>& q, const Slice<W>& k) {
  float d = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    if constexpr (T::code == TL_DTYPE_BF16)
      d = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, q.w[i]), __builtin_bit_cast(bf16x2, k.w[i]), d,
                                          false);
    else if constexpr (T::code == TL_DTYPE_F16)
      d = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, q.w[i]), __builtin_bit_cast(f16x2, k.w[i]), d, false);
    else
      d = fmaf(__uint_as_float(q.w[i]), __uint_as_float(k.w[i]), d);
  }
  return d;
}

// Blocks of a wave at a time in a pair's workgroup, whose waves are few: a block's K and V take D * size / 8
// registers.
template <typename T, int D>
constexpr int kPairBlocks = D * T::size == 512 ? 1 : 2;
constexpr int kPairWaves = 8;

// Wave priority by what is done of the share: without it a CU's oldest workgroup runs ahead of its youngest, and
// equal shares end far apart.
__device__ __forceinline__ void set_progress_priority(int done, int share) {
  const int q = 4 * done / share;
  if (q <= 0) __builtin_amdgcn_s_setprio(3);
  else if (q == 1) __builtin_amdgcn_s_setprio(2);
  else if (q == 2) __builtin_amdgcn_s_setprio(1);
  else __builtin_amdgcn_s_setprio(0);
}

// Buffer resource of one block of 16 rows, from wave-uniform values.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t block_rsrc(const char* base, uint32_t bytes) {
  const int64_t a = uni((int64_t)(uintptr_t)base);
  return __builtin_amdgcn_make_buffer_rsrc((void*)(uintptr_t)a, (short)0, (int)bytes, kBufRsrcWord3);
}

// Stores and loads past an XCD's L2 (sc1), which order partial results across XCDs without a write-back of a cache.
__device__ __forceinline__ void put(float* at, float x) {
  __hip_atomic_store(at, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float get(const float* at) {
  return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// After a segment of a pair that several shares have: once its stores are done the workgroup leaves the call's tag, and
// where it finds those of all segments (the last one does; several may, and write the same) it joins them, a wave a head,
// and takes the tags away, for a graph's next replay.  Nothing waits for another workgroup.  (With a
// second launch for the joins, 3.6 us, one sequence of 100 positions, 9 / 3 heads, fp32, took 9.0 us for 8.15, and 64 long
// ones 442.5 for 445.)  Lane s holds segment s's (m, l);
// accumulators are read eight segments at a time.
template <typename T, int D, int G, int NW>
__device__ __forceinline__ void join_segments(const DecodeParams& p, int b, int hq0, int n_g, int first,
                                              int parts, int wave, int lane, int& s_all) {
  constexpr int NJ = D / 64, R = 8;
  using B = typename T::bits;
  auto at_slot = [&](int s) { return (first + s) * 2 + (s == 0 ? 1 : 0); };
  wait_vmcnt<0>();
  __syncthreads();
  if (wave == 0) {
    if (lane == 0)
      __hip_atomic_store(p.words + at_slot((int)blockIdx.x - first), p.tag, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    wait_vmcnt<0>();
    bool all = true;
    for (int s0 = 0; s0 < parts; s0 += 64) {
      uint64_t x = p.tag;
      if (s0 + lane < parts) x = __hip_atomic_load(p.words + at_slot(s0 + lane), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      all = all && __all(x == p.tag);
    }
    if (lane == 0) s_all = all ? 1 : 0;
  }
  __syncthreads();
  if (!s_all) return;
  asm volatile("" ::: "memory");
  for (int g = wave; g < n_g; g += NW) {
    auto at = [&](int s) { return at_slot(s) * G + g; };
    auto load = [&](int s0, float (&r)[R][NJ]) {
#pragma unroll
      for (int k = 0; k < R; ++k)
#pragma unroll
        for (int j = 0; j < NJ; ++j) r[k][j] = s0 + k < parts ? get(p.ws_acc + (int64_t)at(s0 + k) * D + lane + 64 * j) : 0.f;
    };
    float r[R][NJ];
    load(0, r);
    auto ml = [&](int s) { return make_float2(get(p.ws_ml + 2 * at(s)), get(p.ws_ml + 2 * at(s) + 1)); };
    const float2 e0 = lane < parts ? ml(lane) : make_float2(-INFINITY, 0.f);
    float mx = e0.x;
    for (int s = lane + 64; s < parts; s += 64) mx = fmaxf(mx, get(p.ws_ml + 2 * at(s)));
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off));
    const float base = mx == -INFINITY ? 0.f : mx;
    float ls = 0.f, wl = 0.f, a[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) a[j] = 0.f;
    for (int s0 = 0; s0 < parts; s0 += R) {
      if ((s0 & 63) == 0) {
        const int s = s0 + lane;
        const float2 e = s0 == 0 ? e0 : s < parts ? ml(s) : make_float2(-INFINITY, 0.f);
        wl = s < parts ? fast_exp2(e.x - base) : 0.f;
        ls += e.y * wl;
      }
      if (s0 > 0) load(s0, r);
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wl), (s0 + k) & 63));
#pragma unroll
        for (int j = 0; j < NJ; ++j) a[j] = fmaf(r[k][j], w, a[j]);
      }
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) ls += __shfl_xor(ls, off);
    B* o = (B*)p.o + b * p.o_sb + (int64_t)(hq0 + g) * p.o_sh;
#pragma unroll
    for (int j = 0; j < NJ; ++j) o[lane + 64 * j] = from_f32<T>(ls == 0.f ? 0.f : a[j] / ls);
  }
  if (wave == 0)
    for (int s = lane; s < parts; s += 64)
      __hip_atomic_store(p.words + at_slot(s), (uint64_t)0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// 16 lanes read a row, a wave 4 rows a load and a block in 4 loads of K and 4 of V; wave w takes blocks
// w, w + NW, ... of the segment, NB of them at a time.  PAIR: a workgroup takes a whole pair (see pair_mode).
// (8 lanes with 16-byte loads for rows of 128 bytes were slower: 32 sequences, 15 / 5 heads, d_k 64, 1000 positions
// 15.2 -> 17.0 us as pairs, 17.7 -> 18.9 as shares.)
template <typename T, int D, int G, int NW, int NB, bool PAIR>
__global__ __launch_bounds__(64 * NW) void paged_decode_kernel(DecodeParams p) {
  constexpr int LPR = 16, RPL = 4;      // lanes of a row, rows of a load
  constexpr int EPL = D / LPR;          // elements of a lane's slice of a row
  constexpr int W = EPL * T::size / 4;  // its 32-bit words
  constexpr int U = kBlk / RPL;         // rows of a block that a lane reads
  using B = typename T::bits;
  const int lane = threadIdx.x & 63;
  const int wave = uni((int)threadIdx.x >> 6);
  const int sub = lane & (LPR - 1), rowg = lane / LPR;
  const int n_chunks = p.n_pairs / p.n_kv;
  __shared__ float s_m[NW][G], s_l[NW][G];
  __shared__ float s_acc[NW][G][D];
  __shared__ int s_all;
  const uint32_t k_lane = rowg * p.k_row_bytes + sub * (EPL * T::size);
  const uint32_t v_lane = rowg * p.v_row_bytes + sub * (EPL * T::size);

  // Blocks [v0, v1) of the Seen blocks of pair `pair` of sequence b; r0 of share blocks of the workgroup's
  // share are done before.
  auto segment = [&](const int b, const Seen& sn, const int pair, const int v0, const int v1, const int first,
                     const int parts, const int done, const int share) {
    const bool whole = parts == 1;
    const int slot = v0 == 0 ? 1 : 0;
    const int hkv = pair / n_chunks;
    const int hq0 = hkv * p.group + (pair - hkv * n_chunks) * G;
    const int n_g = min(G, hkv * p.group + p.group - hq0);
    Slice<W> qs[G];
    float m[G], l[G], acc[G][EPL];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const uint32_t* src =
          (const uint32_t*)((const B*)p.q + b * p.q_sb + (int64_t)min(hq0 + g, hq0 + n_g - 1) * p.q_sh + sub * EPL);
#pragma unroll
      for (int i = 0; i < W; ++i) qs[g].w[i] = g < n_g ? src[i] : 0u;
      m[g] = -INFINITY;
      l[g] = 0.f;
#pragma unroll
      for (int e = 0; e < EPL; ++e) acc[g][e] = 0.f;
    }
    const int32_t* row = p.pm.table + (int64_t)b * p.pm.max_pages;
    const int shift = p.pm.shift;
    auto block_at = [&](int v) { return v < sn.ns ? v : v - sn.ns + sn.wb; };
    const char* const kh = (const char*)p.k + hkv * p.k_sh * T::size;
    const char* const vh = (const char*)p.v + hkv * p.v_sh * T::size;

    int pages = 0;  // lane i: the page of this wave's block (it & ~63) + i
    // The wave's blocks it .. it + N - 1, from v on NW apart.
    auto blocks = [&](const int v, const int it, auto count) __attribute__((always_inline)) {
      constexpr int N = decltype(count)::value;
      Slice<W> kr[N][U], vr[N][U];
      bool full[N];
      int pos0[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int vi = v + i * NW;
        const int page = __builtin_amdgcn_readlane(pages, (it + i) & 63);
        const bool there = (unsigned)page < (unsigned)p.pm.n_pages;
        pos0[i] = block_at(vi) << kBlkShift;
        const int in_page = pos0[i] & ((1 << shift) - 1);
        const int64_t id = there ? page : 0;
        const auto krs = block_rsrc(kh + id * p.k_sp * T::size + (int64_t)in_page * p.k_row_bytes,
                                    there ? 15 * p.k_row_bytes + D * T::size : 0);
        const auto vrs = block_rsrc(vh + id * p.v_sp * T::size + (int64_t)in_page * p.v_row_bytes,
                                    there ? 15 * p.v_row_bytes + D * T::size : 0);
        full[i] = there && pos0[i] + kBlk <= sn.len && (pos0[i] >= sn.lo || pos0[i] + kBlk <= p.sinks);
        if (!there) pos0[i] = sn.len;  // hidden throughout
        if (full[i]) {
#pragma unroll
          for (int u = 0; u < U; ++u) load_slice(kr[i][u], krs, k_lane, RPL * u * p.k_row_bytes);
#pragma unroll
          for (int u = 0; u < U; ++u) load_slice(vr[i][u], vrs, v_lane, RPL * u * p.v_row_bytes);
        } else {
          // hidden rows may hold anything (NaN among it): they are not read, and count as zeros
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const bool seen = row_seen(sn, p.sinks, pos0[i] + RPL * u + rowg);
            load_slice(kr[i][u], krs, seen ? k_lane + RPL * u * p.k_row_bytes : kPastEnd, 0);
            load_slice(vr[i][u], vrs, seen ? v_lane + RPL * u * p.v_row_bytes : kPastEnd, 0);
          }
        }
      }
      float s[G][N * U];
#pragma unroll
      for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int g = 0; g < G; ++g) s[g][i * U + u] = row16_sum(dot_slice<T>(qs[g], kr[i][u])) * p.scale_log2;
        if (!full[i]) {
          asm volatile("");
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const bool seen = row_seen(sn, p.sinks, pos0[i] + RPL * u + rowg);
#pragma unroll
            for (int g = 0; g < G; ++g) s[g][i * U + u] = seen ? s[g][i * U + u] : -INFINITY;
          }
        }
      }
      // the maximum moves only when a score passes it by 2^8 (it only bounds the exponents)
      bool grow = false;
      float mb[G];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        mb[g] = s[g][0];
#pragma unroll
        for (int u = 1; u < N * U; ++u) mb[g] = fmaxf(mb[g], s[g][u]);
        grow |= mb[g] > m[g] + kRescaleLog2;
      }
      if (__any(grow)) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const float mn = fmaxf(m[g], mb[g]);
          const float a = fast_exp2(m[g] - (mn == -INFINITY ? 0.f : mn));
          m[g] = mn;
          l[g] *= a;
#pragma unroll
          for (int e = 0; e < EPL; ++e) acc[g][e] *= a;
        }
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float base = m[g] == -INFINITY ? 0.f : m[g];
#pragma unroll
        for (int u = 0; u < N * U; ++u) {
          s[g][u] = fast_exp2(s[g][u] - base);
          l[g] += s[g][u];
        }
      }
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float vf[EPL];
          if constexpr (T::size == 4) {
#pragma unroll
            for (int e = 0; e < EPL; ++e) vf[e] = __uint_as_float(vr[i][u].w[e]);
          } else {
#pragma unroll
            for (int e = 0; e < W; ++e) unpack2<T>(vr[i][u].w[e], vf[2 * e], vf[2 * e + 1]);
          }
#pragma unroll
          for (int g = 0; g < G; ++g)
#pragma unroll
            for (int e = 0; e < EPL; ++e) acc[g][e] = fmaf(s[g][i * U + u], vf[e], acc[g][e]);
        }
    };
    int v = v0 + wave, it = 0;
    auto look_up = [&]() __attribute__((always_inline)) {
      if ((it & 63) == 0) {
        const int mine = v + NW * lane;
        pages = mine < v1 ? row[block_at(mine) >> (shift - kBlkShift)] : -1;
      }
    };
    if constexpr (NB > 1) {
      for (; v + NW * (NB - 1) < v1; v += NW * NB, it += NB) {
        look_up();
        blocks(v, it, std::integral_constant<int, NB>{});
      }
    }
    for (; v < v1; v += NW, ++it) {
      look_up();
      if constexpr (!PAIR) {
        if ((it & 3) == 0) set_progress_priority(done + it * NW, share);
      }
      blocks(v, it, std::integral_constant<int, 1>{});
    }

    // join the rows of a load, then the waves
#pragma unroll
    for (int off = LPR; off <= 32; off <<= 1) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float m2 = __shfl_xor(m[g], off), l2 = __shfl_xor(l[g], off);
        const float mn = fmaxf(m[g], m2);
        const float base = mn == -INFINITY ? 0.f : mn;
        const float w1 = fast_exp2(m[g] - base), w2 = fast_exp2(m2 - base);
        m[g] = mn;
        l[g] = l[g] * w1 + l2 * w2;
#pragma unroll
        for (int e = 0; e < EPL; ++e) acc[g][e] = acc[g][e] * w1 + __shfl_xor(acc[g][e], off) * w2;
      }
    }
    __syncthreads();  // the last segment's sums have been read
    if (lane < LPR) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if (lane == 0) {
          s_m[wave][g] = m[g];
          s_l[wave][g] = l[g];
        }
#pragma unroll
        for (int e = 0; e < EPL; ++e) s_acc[wave][g][sub * EPL + e] = acc[g][e];
      }
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < n_g * D; idx += 64 * NW) {
      const int g = idx / D, d = idx - g * D;
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < NW; ++w) mx = fmaxf(mx, s_m[w][g]);
      const float base = mx == -INFINITY ? 0.f : mx;
      float a = 0.f, ls = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float wt = fast_exp2(s_m[w][g] - base);
        a += s_acc[w][g][d] * wt;
        ls += s_l[w][g] * wt;
      }
      if (whole) {
        ((B*)p.o)[b * p.o_sb + (int64_t)(hq0 + g) * p.o_sh + d] = from_f32<T>(ls == 0.f ? 0.f : a / ls);
      } else {
        const int64_t at = ((int64_t)blockIdx.x * 2 + slot) * G + g;
        put(p.ws_acc + at * D + d, a);
        if (d == 0) {
          put(p.ws_ml + at * 2, mx);
          put(p.ws_ml + at * 2 + 1, ls);
        }
      }
    }
    if constexpr (!PAIR) {
      if (!whole) join_segments<T, D, G, NW>(p, b, hq0, n_g, first, parts, wave, lane, s_all);
    }
  };

  if constexpr (PAIR) {
    const int b = (int)blockIdx.x / p.n_pairs;
    const Seen sn = seen_of(p, b);
    segment(b, sn, (int)blockIdx.x - b * p.n_pairs, 0, sn.n, 0, 1, 0, 0);
  } else {
    const Layout lay = layout_of(p, lane);
    const int64_t begin = (int64_t)blockIdx.x * lay.share;
    if (lay.padded) {
      // one segment a workgroup: part blockIdx.x - first of its pair
      const int w = (int)blockIdx.x;
      if (w < lay.total) {
        const Owner own = owner_of(p, lay, w, lane);
        const Seen sn = seen_of(p, own.b);
        const int parts = (sn.n + lay.share - 1) / lay.share;
        const int pair = (w - own.first) / parts;
        const int first = own.first + pair * parts, v0 = (w - first) * lay.share, v1 = min(v0 + lay.share, sn.n);
        segment(own.b, sn, pair, v0, v1, first, parts, 0, v1 - v0);
      }
    } else if (begin < lay.total) {
      const int r0 = (int)begin, r1 = (int)min((int64_t)lay.total, begin + lay.share);
      for (int r = r0; r < r1;) {
        const Owner own = owner_of(p, lay, r, lane);
        const Seen sn = seen_of(p, own.b);
        const int pair = (r - own.first) / sn.n;
        const int pair0 = own.first + pair * sn.n;
        const int v0 = r - pair0, v1 = min(r1 - pair0, sn.n);
        const int first = pair0 / lay.share, parts = (pair0 + sn.n - 1) / lay.share - first + 1;
        segment(own.b, sn, pair, v0, v1, first, parts, r - r0, r1 - r0);
        r = pair0 + v1;
      }
    }
    // sequences that see nothing
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
      if (seen_of(p, b).n > 0) continue;
      for (int i = threadIdx.x; i < p.n_head * D; i += 64 * NW) ((B*)p.o)[b * p.o_sb + (int64_t)(i / D) * p.o_sh + i % D] = 0;
    }
  }
}

// Blocks that one sequence's query can see at most.
int64_t most_blocks(int64_t cap, int window, int sinks) {
  int64_t n = (cap + kBlk - 1) / kBlk;
  if (window > 0) {
    const int64_t w = (int64_t)window / kBlk + 2 + ((int64_t)sinks + kBlk - 1) / kBlk;
    n = n < w ? n : w;
  }
  return n;
}

int heads_per_pair(int n_head, int n_kv) { return n_head / n_kv < 8 ? n_head / n_kv : 8; }

constexpr size_t kWordsBytes = (size_t)kMaxShares * 2 * sizeof(uint64_t);
size_t ws_ml_bytes(int hpp) { return (size_t)kMaxShares * 2 * hpp * 2 * sizeof(float); }

// A workgroup for each pair, which finishes it: no partial results, one launch.  Taken where the longest pair
// there can be (pair_bytes of K and V) is short: one CU streams it.  us a call as pairs / as shares, 250 KB a pair,
// 16 bits: 5 pairs 13.2 / 9.0, 40 pairs 13.5 / 12.0, 64 (d_k 128) 12.3 / 13.5, 96 (MHA) 10.8 / 13.4, 160 14.3 / 17.6;
// 350 KB: 32 15.1 / 12.3, 128 16.1 / 17.0, 24 (fp32) 12.5 / 10.7; 126 KB: 320 13.8 / 16.2; 50 KB: 8 7.1 / 9.2, 128 7.8 / 9.7.
bool pair_mode(const DecodeParams& p, int64_t pair_bytes) {
  const int64_t pairs = (int64_t)p.batch * p.n_pairs;
  return !tl_overrides.decode_shares && pair_bytes <= kPairMaxBytes && pair_bytes * pairs <= kPairMaxAll &&
         (pair_bytes <= kPairFewBytes || pairs >= kPairMany);
}

template <typename T, int D, int G>
int launch_decode_g(DecodeParams& p, int64_t most, hipStream_t st) {
  const int64_t pair_bytes = most / ((int64_t)p.batch * p.n_pairs) * kBlk * 2 * D * T::size;
  if (pair_mode(p, pair_bytes)) {
    hipLaunchKernelGGL((paged_decode_kernel<T, D, G, kPairWaves, kPairBlocks<T, D>, true>), dim3(p.batch * p.n_pairs),
                       dim3(64 * kPairWaves), 0, st, p);
    return tl_launch_status();
  }
  static int per_cu = 0;
  if (per_cu == 0) {
    int n = 0;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, paged_decode_kernel<T, D, G, kDecWaves, 1, false>,
                                                     kDecThreads, 0) != hipSuccess ||
        n <= 0)
      n = 1;
    per_cu = n;
  }
  int64_t shares = (int64_t)per_cu * tl_device_cus();
  shares = shares < kMaxShares ? shares : kMaxShares;
  // never more than the parts there can be; twice the pairs at least, where the device holds as many, so that the
  // pairs are cut one by one
  const int64_t pairs = (int64_t)p.batch * p.n_pairs;
  const int64_t full = (most + kMinShare - 1) / kMinShare + pairs;
  p.n_shares = (int)(shares < full ? shares : full);
  p.tag = tl_arrival_tag();
  hipLaunchKernelGGL((paged_decode_kernel<T, D, G, kDecWaves, 1, false>), dim3(p.n_shares), dim3(kDecThreads), 0, st, p);
  return tl_launch_status();
}

template <typename T, int D>
int launch_decode_d(DecodeParams& p, int64_t most, hipStream_t st) {
  switch (p.heads_per_pair) {
    case 1: return launch_decode_g<T, D, 1>(p, most, st);
    case 2: return launch_decode_g<T, D, 2>(p, most, st);
    case 3: return launch_decode_g<T, D, 3>(p, most, st);
    case 4: return launch_decode_g<T, D, 4>(p, most, st);
    case 5: return launch_decode_g<T, D, 5>(p, most, st);
    case 6: return launch_decode_g<T, D, 6>(p, most, st);
    case 7: return launch_decode_g<T, D, 7>(p, most, st);
    default: return launch_decode_g<T, D, 8>(p, most, st);
  }
}

template <typename T>
int launch_decode(DecodeParams& p, int d_k, int64_t most, hipStream_t st) {
  return d_k == 64 ? launch_decode_d<T, 64>(p, most, st) : launch_decode_d<T, 128>(p, most, st);
}

// ---------------------------------------------------------------------------------
// Page copies.  Bases and pairs ride in the kernel's argument: no upload, and a captured
// graph keeps them.  They are read from the argument segment with scalar loads (an index into
// the by-value argument would copy the arrays into registers).  120 pages of 128 KB in 32 pools, 1.0 GB
// moved: 189 us, 5.3 TB/s; 3 pages in 60 pools: 3.0 us on the device.
// ---------------------------------------------------------------------------------
constexpr int kCopyBases = 64, kCopyPairs = 256;
constexpr int kCopyBytes = 16384;  // of a page, a workgroup

struct CopyParams {
  uint64_t base[kCopyBases];
  int2 pair[kCopyPairs];  // (source, destination)
  int64_t page_stride;    // bytes
  int page_bytes, n_pairs, pieces;
};

__global__ __launch_bounds__(256) void copy_pages_kernel(CopyParams p) {
  typedef const __attribute__((address_space(4))) char* kchar;
  typedef const __attribute__((address_space(4))) uint64_t* ku64;
  const kchar args = (kchar)__builtin_amdgcn_kernarg_segment_ptr();
  const int piece = blockIdx.x, pair = blockIdx.y, cache = blockIdx.z;
  const uint64_t base = *(ku64)(args + offsetof(CopyParams, base) + 8 * cache);
  const uint64_t sd = *(ku64)(args + offsetof(CopyParams, pair) + 8 * pair);
  const int src = (int)(uint32_t)sd, dst = (int)(uint32_t)(sd >> 32);
  const int lo = piece * kCopyBytes, hi = min(p.page_bytes, lo + kCopyBytes);
  const char* s = (const char*)base + src * p.page_stride;
  char* d = (char*)base + dst * p.page_stride;
  for (int i = lo + threadIdx.x * 16; i < hi; i += 256 * 16) *(u32x4*)(d + i) = *(const u32x4*)(s + i);
}

// Entries of an int32 array on the device, by value.
struct WriteParams {
  int2 at[kCopyPairs];  // (index, value)
  int32_t* dst;
  int n;
};

__global__ __launch_bounds__(256) void write_i32_kernel(WriteParams p) {
  typedef const __attribute__((address_space(4))) char* kchar;
  typedef const __attribute__((address_space(4))) int* kint;
  const kchar args = (kchar)__builtin_amdgcn_kernarg_segment_ptr();
  if ((int)threadIdx.x >= p.n) return;
  const kint at = (kint)(args + offsetof(WriteParams, at) + 8 * threadIdx.x);
  p.dst[at[0]] = at[1];
}

bool known_dtype(int dtype) { return dtype == TL_DTYPE_F32 || dtype == TL_DTYPE_F16 || dtype == TL_DTYPE_BF16; }

// Bytes from a tensor's first element to behind its last, outer dims (n, stride) in elements.
size_t span_bytes(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t n2, int64_t s2, int64_t inner, int esize) {
  return (size_t)((n0 - 1) * s0 + (n1 - 1) * s1 + (n2 - 1) * s2 + inner) * esize;
}

}  // namespace

extern "C" {

int tl_paged_kv_append(const void* q, void* q_out, const void* k_new, const void* v_new, void* k_pages, void* v_pages,
                       const int32_t* page_table, int max_pages, int n_pages, int page_size,
                       const int32_t* cache_lens, const int32_t* new_lens, const float* cos_table,
                       const float* sin_table, int rope_rows, int rotary, int interleaved, int batch, int n_new,
                       int n_head, int n_kv_head, int d_k, const int64_t* q_strides, const int64_t* q_out_strides,
                       const int64_t* k_new_strides, const int64_t* v_new_strides, const int64_t* k_page_strides,
                       const int64_t* v_page_strides, int dtype, void* stream) {
  if (batch == 0 || n_new == 0) return 0;
  if (!k_new || !v_new || !k_pages || !v_pages || !page_table || !cache_lens || batch < 0 || n_new < 0 || n_head < 0 ||
      n_kv_head < 1 || d_k < 2 || (d_k & 1) || max_pages < 1 || n_pages < 1 || !k_new_strides || !v_new_strides ||
      !k_page_strides || !v_page_strides || !known_dtype(dtype))
    return TL_ERR_INVALID;
  const int shift = page_shift(page_size);
  if (shift < 0 || ((int64_t)max_pages << shift) > INT32_MAX) return TL_ERR_INVALID;
  if ((cos_table == nullptr) != (sin_table == nullptr)) return TL_ERR_INVALID;
  if (cos_table && (rope_rows < 0 || rotary < 2 || (rotary & 1) || rotary > d_k)) return TL_ERR_INVALID;
  const int esize = dtype == TL_DTYPE_F32 ? 4 : 2;
  AppendParams p{};
  if (q && n_head > 0) {
    if (!q_out || !q_strides || !q_out_strides) return TL_ERR_INVALID;
    if (q == q_out) {
      for (int i = 0; i < 3; ++i)
        if (q_strides[i] != q_out_strides[i]) return TL_ERR_INVALID;
    } else if (tl_overlap(q, span_bytes(batch, q_strides[0], n_new, q_strides[1], n_head, q_strides[2], d_k, esize),
                          q_out, span_bytes(batch, q_out_strides[0], n_new, q_out_strides[1], n_head, q_out_strides[2],
                                            d_k, esize))) {
      return TL_ERR_INVALID;
    }
    p.n_head = cos_table || q != q_out ? n_head : 0;  // nothing to do in place without positions
    p.q = q;
    p.qo = q_out;
    p.q_sb = q_strides[0], p.q_ss = q_strides[1], p.q_sh = q_strides[2];
    p.qo_sb = q_out_strides[0], p.qo_ss = q_out_strides[1], p.qo_sh = q_out_strides[2];
  }
  p.kn = k_new;
  p.vn = v_new;
  p.kp = k_pages;
  p.vp = v_pages;
  p.pm = PageMap{page_table, max_pages, n_pages, shift};
  p.lens = cache_lens;
  p.new_lens = new_lens;
  p.cos_t = cos_table;
  p.sin_t = sin_table;
  p.rope_rows = rope_rows;
  p.rot_half = cos_table ? rotary / 2 : 0;
  p.batch = batch;
  p.n_new = n_new;
  p.n_kv = n_kv_head;
  p.d_k = d_k;
  p.kn_sb = k_new_strides[0], p.kn_ss = k_new_strides[1], p.kn_sh = k_new_strides[2];
  p.vn_sb = v_new_strides[0], p.vn_ss = v_new_strides[1], p.vn_sh = v_new_strides[2];
  p.kp_sp = k_page_strides[0], p.kp_sh = k_page_strides[1], p.kp_sr = k_page_strides[2];
  p.vp_sp = v_page_strides[0], p.vp_sh = v_page_strides[1], p.vp_sr = v_page_strides[2];
  const int mode = !cos_table ? kNoRope : interleaved ? kInterleaved : kHalf;
  hipStream_t st = tl_resolve_stream(stream);
  switch (dtype) {
    case TL_DTYPE_F32: return launch_append<F32, false>(p, mode, st);
    case TL_DTYPE_F16: return launch_append<F16, false>(p, mode, st);
    default: return launch_append<BF16, false>(p, mode, st);
  }
}

int tl_paged_kv_append_slots(const void* q, void* q_out, const void* k_new, const void* v_new, void* k_pages, void* v_pages,
                             int n_pages, int page_size, const int32_t* slots, const int32_t* positions,
                             const float* cos_table, const float* sin_table, int rope_rows, int rotary, int interleaved,
                             int n_tokens, int n_head, int n_kv_head, int d_k, const int64_t* q_strides,
                             const int64_t* q_out_strides, const int64_t* k_new_strides, const int64_t* v_new_strides,
                             const int64_t* k_page_strides, const int64_t* v_page_strides, int dtype, void* stream) {
  if (n_tokens == 0) return 0;
  if (!k_new || !v_new || !k_pages || !v_pages || !slots || n_tokens < 0 || n_head < 0 || n_kv_head < 1 || d_k < 2 ||
      (d_k & 1) || n_pages < 1 || !k_new_strides || !v_new_strides || !k_page_strides || !v_page_strides ||
      !known_dtype(dtype))
    return TL_ERR_INVALID;
  const int shift = page_shift(page_size);
  if (shift < 0 || ((int64_t)n_pages << shift) > INT32_MAX) return TL_ERR_INVALID;
  if ((cos_table == nullptr) != (sin_table == nullptr)) return TL_ERR_INVALID;
  if (cos_table && (!positions || rope_rows < 0 || rotary < 2 || (rotary & 1) || rotary > d_k)) return TL_ERR_INVALID;
  const int esize = dtype == TL_DTYPE_F32 ? 4 : 2;
  auto rows = [&](const void* at, int64_t heads, const int64_t* s) {
    return Rows3{at, {n_tokens, heads, 1}, {s[0] * esize, s[1] * esize, 0}, (int64_t)d_k * esize};
  };
  auto pool = [&](const void* at, const int64_t* s) {
    return Rows3{at, {n_pages, n_kv_head, page_size}, {s[0] * esize, s[1] * esize, s[2] * esize}, (int64_t)d_k * esize};
  };
  const Rows3 kp = pool(k_pages, k_page_strides), vp = pool(v_pages, v_page_strides);
  const Rows3 kn = rows(k_new, n_kv_head, k_new_strides), vn = rows(v_new, n_kv_head, v_new_strides);
  if (rows_overlap(kp, kn) || rows_overlap(kp, vn) || rows_overlap(vp, kn) || rows_overlap(vp, vn)) return TL_ERR_INVALID;
  AppendParams p{};
  if (q && n_head > 0) {
    if (!q_out || !q_strides || !q_out_strides) return TL_ERR_INVALID;
    const Rows3 from = rows(q, n_head, q_strides), to = rows(q_out, n_head, q_out_strides);
    const bool same = q == q_out && q_strides[0] == q_out_strides[0] && q_strides[1] == q_out_strides[1];
    if ((!same && rows_overlap(from, to)) || rows_overlap(to, kn) || rows_overlap(to, vn) || rows_overlap(to, kp) ||
        rows_overlap(to, vp) || rows_overlap(from, kp) || rows_overlap(from, vp))
      return TL_ERR_INVALID;
    p.n_head = cos_table || q != q_out ? n_head : 0;  // nothing to do in place without positions
    p.q = q;
    p.qo = q_out;
    p.q_ss = q_strides[0], p.q_sh = q_strides[1];
    p.qo_ss = q_out_strides[0], p.qo_sh = q_out_strides[1];
  }
  p.kn = k_new;
  p.vn = v_new;
  p.kp = k_pages;
  p.vp = v_pages;
  p.pm = PageMap{nullptr, 0, n_pages, shift};
  p.slots = slots;
  p.positions = positions;
  // Rows are read once, and what is written is what attention reads next: more rows than the L2s hold are read past them.  us alone, and
  // with the attention after it, kept in the caches / past them: 17000 tokens, 9 / 3 heads of 64, fp32 (65 MB) 34.0 / 29.8, 479 / 479;
  // 8000 tokens, 24 / 8 heads of 128, bf16 (82 MB) with attention 173 / 166; 6000 tokens, 15 / 5 heads of 64, fp16 (19 MB) 10.6 / 12.2.
  // (Writing past them too: 24.6 alone in the first case, and attention loses it again: 482; 177.)
  constexpr int64_t kL2s = 32ll << 20;
  p.past_caches = (int64_t)n_tokens * (p.n_head + 2 * n_kv_head) * d_k * esize > kL2s;
  p.cos_t = cos_table;
  p.sin_t = sin_table;
  p.rope_rows = rope_rows;
  p.rot_half = cos_table ? rotary / 2 : 0;
  p.batch = 1;
  p.n_new = n_tokens;
  p.n_kv = n_kv_head;
  p.d_k = d_k;
  p.kn_ss = k_new_strides[0], p.kn_sh = k_new_strides[1];
  p.vn_ss = v_new_strides[0], p.vn_sh = v_new_strides[1];
  p.kp_sp = k_page_strides[0], p.kp_sh = k_page_strides[1], p.kp_sr = k_page_strides[2];
  p.vp_sp = v_page_strides[0], p.vp_sh = v_page_strides[1], p.vp_sr = v_page_strides[2];
  const int mode = !cos_table ? kNoRope : interleaved ? kInterleaved : kHalf;
  hipStream_t st = tl_resolve_stream(stream);
  switch (dtype) {
    case TL_DTYPE_F32: return launch_append<F32, true>(p, mode, st);
    case TL_DTYPE_F16: return launch_append<F16, true>(p, mode, st);
    default: return launch_append<BF16, true>(p, mode, st);
  }
}

size_t tl_paged_decode_workspace_bytes(int n_head, int n_kv_head, int d_k) {
  if (n_head <= 0 || n_kv_head <= 0 || n_head % n_kv_head || d_k <= 0) return 0;
  const int hpp = heads_per_pair(n_head, n_kv_head);
  return kWordsBytes + ws_ml_bytes(hpp) + (size_t)kMaxShares * 2 * hpp * d_k * sizeof(float);
}

int tl_paged_attention_decode(const void* q, const void* k_pages, const void* v_pages, const int32_t* page_table,
                              int max_pages, int n_pages, int page_size, const int32_t* cache_lens, int len_add,
                              int window, int sinks, void* o, void* workspace, size_t workspace_bytes, int batch,
                              int n_head, int n_kv_head, int d_k, const int64_t* q_strides,
                              const int64_t* k_page_strides, const int64_t* v_page_strides, const int64_t* o_strides,
                              float sm_scale, int dtype, void* stream) {
  if (batch == 0 || n_head == 0) return 0;
  if (!q || !k_pages || !v_pages || !page_table || !cache_lens || !o || !workspace || batch < 0 || n_head < 0 ||
      n_kv_head < 1 || n_head % n_kv_head || max_pages < 1 || n_pages < 1 || window < 0 || sinks < 0 || !q_strides ||
      !k_page_strides || !v_page_strides || !o_strides || !known_dtype(dtype) || ((uintptr_t)workspace & 15))
    return TL_ERR_INVALID;
  const int shift = page_shift(page_size);
  const int64_t cap = (int64_t)max_pages << (shift < 0 ? 0 : shift);
  if (shift < 0 || cap > INT32_MAX) return TL_ERR_INVALID;
  if (d_k != 64 && d_k != 128) return TL_ERR_UNSUPPORTED;
  if (batch > 65535) return TL_ERR_UNSUPPORTED;
  if (workspace_bytes < tl_paged_decode_workspace_bytes(n_head, n_kv_head, d_k)) return TL_ERR_INVALID;
  // a lane reads d_k / 16 elements of a row in 8- or 16-byte words, a block of 16 rows with 32-bit offsets
  const int esize = dtype == TL_DTYPE_F32 ? 4 : 2;
  const int64_t slice = d_k / 16;
  const int64_t strides[] = {q_strides[0], q_strides[1], k_page_strides[0], k_page_strides[1], k_page_strides[2],
                             v_page_strides[0], v_page_strides[1], v_page_strides[2]};
  for (int64_t s : strides)
    if (s < 0 || s % slice) return TL_ERR_UNSUPPORTED;
  if (((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages) % (uintptr_t)(slice * esize)) return TL_ERR_UNSUPPORTED;
  if (k_page_strides[2] > (1 << 24) || v_page_strides[2] > (1 << 24)) return TL_ERR_UNSUPPORTED;
  // o may be q, as every head's q is read before its o is written
  auto rows = [&](const void* at, int64_t n0, int64_t n1, int64_t n2, int64_t s0, int64_t s1, int64_t s2) {
    return Rows3{at, {n0, n1, n2}, {s0 * esize, s1 * esize, s2 * esize}, (int64_t)d_k * esize};
  };
  const Rows3 out = rows(o, batch, n_head, 1, o_strides[0], o_strides[1], 0);
  const bool is_q = o == q && o_strides[0] == q_strides[0] && o_strides[1] == q_strides[1];
  auto pool = [&](const void* at, const int64_t* s) { return rows(at, n_pages, n_kv_head, page_size, s[0], s[1], s[2]); };
  if ((!is_q && rows_overlap(out, rows(q, batch, n_head, 1, q_strides[0], q_strides[1], 0))) ||
      rows_overlap(out, pool(k_pages, k_page_strides)) || rows_overlap(out, pool(v_pages, v_page_strides)))
    return TL_ERR_INVALID;
  DecodeParams p{};
  p.q = q;
  p.k = k_pages;
  p.v = v_pages;
  p.lens = cache_lens;
  p.pm = PageMap{page_table, max_pages, n_pages, shift};
  p.o = o;
  p.len_add = len_add;
  p.window = window;
  p.sinks = sinks;
  p.batch = batch;
  p.n_head = n_head;
  p.n_kv = n_kv_head;
  p.group = n_head / n_kv_head;
  p.heads_per_pair = heads_per_pair(n_head, n_kv_head);
  p.n_pairs = n_kv_head * ((p.group + p.heads_per_pair - 1) / p.heads_per_pair);
  p.words = (uint64_t*)workspace;
  p.ws_ml = (float*)((char*)workspace + kWordsBytes);
  p.ws_acc = (float*)((char*)workspace + kWordsBytes + ws_ml_bytes(p.heads_per_pair));
  p.q_sb = q_strides[0], p.q_sh = q_strides[1];
  p.o_sb = o_strides[0], p.o_sh = o_strides[1];
  p.k_sp = k_page_strides[0], p.k_sh = k_page_strides[1];
  p.v_sp = v_page_strides[0], p.v_sh = v_page_strides[1];
  p.k_row_bytes = (uint32_t)(k_page_strides[2] * esize);
  p.v_row_bytes = (uint32_t)(v_page_strides[2] * esize);
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  const int64_t most = most_blocks(cap, window, sinks) * batch * p.n_pairs;
  if (most > INT32_MAX) return TL_ERR_UNSUPPORTED;  // blocks are counted in 32 bits
  hipStream_t st = tl_resolve_stream(stream);
  switch (dtype) {
    case TL_DTYPE_F32: return launch_decode<F32>(p, d_k, most, st);
    case TL_DTYPE_F16: return launch_decode<F16>(p, d_k, most, st);
    default: return launch_decode<BF16>(p, d_k, most, st);
  }
}

int tl_copy_pages(void* const* caches, int n_caches, int64_t page_bytes, int64_t page_stride_bytes, int n_pages,
                  const int32_t* host_src, const int32_t* host_dst, int count, void* stream) {
  if (n_caches == 0 || count == 0) return 0;
  if (!caches || !host_src || !host_dst || n_caches < 0 || count < 0 || n_pages < 1 || page_bytes < 16 ||
      page_bytes % 16 || page_stride_bytes < page_bytes || page_stride_bytes % 16)
    return TL_ERR_INVALID;
  for (int c = 0; c < n_caches; ++c)
    if (!caches[c] || ((uintptr_t)caches[c] & 15)) return TL_ERR_INVALID;
  for (int i = 0; i < count; ++i)
    if (host_src[i] < 0 || host_src[i] >= n_pages || host_dst[i] < 0 || host_dst[i] >= n_pages) return TL_ERR_INVALID;
  if (page_bytes > (1 << 30)) return TL_ERR_UNSUPPORTED;  // offsets in a page are 32-bit
  hipStream_t st = tl_resolve_stream(stream);
  CopyParams p;
  p.page_stride = page_stride_bytes;
  p.page_bytes = (int)page_bytes;
  p.pieces = (int)((page_bytes + kCopyBytes - 1) / kCopyBytes);
  for (int c0 = 0; c0 < n_caches; c0 += kCopyBases) {
    const int nc = n_caches - c0 < kCopyBases ? n_caches - c0 : kCopyBases;
    for (int c = 0; c < kCopyBases; ++c) p.base[c] = (uint64_t)(uintptr_t)caches[c0 + (c < nc ? c : 0)];
    for (int i0 = 0; i0 < count; i0 += kCopyPairs) {
      p.n_pairs = count - i0 < kCopyPairs ? count - i0 : kCopyPairs;
      for (int i = 0; i < kCopyPairs; ++i) {
        const int j = i0 + (i < p.n_pairs ? i : 0);
        p.pair[i] = make_int2(host_src[j], host_dst[j]);
      }
      hipLaunchKernelGGL(copy_pages_kernel, dim3(p.pieces, p.n_pairs, nc), dim3(256), 0, st, p);
      const int e = tl_launch_status();
      if (e) return e;
    }
  }
  return 0;
}

int tl_write_i32(int32_t* dst, int64_t dst_count, const int32_t* host_index, const int32_t* host_value, int count,
                 void* stream) {
  if (count == 0) return 0;
  if (!dst || !host_index || !host_value || count < 0) return TL_ERR_INVALID;
  for (int i = 0; i < count; ++i)
    if (host_index[i] < 0 || host_index[i] >= dst_count) return TL_ERR_INVALID;
  hipStream_t st = tl_resolve_stream(stream);
  WriteParams p;
  p.dst = dst;
  for (int i0 = 0; i0 < count; i0 += kCopyPairs) {
    p.n = count - i0 < kCopyPairs ? count - i0 : kCopyPairs;
    for (int i = 0; i < kCopyPairs; ++i) {
      const int j = i0 + (i < p.n ? i : 0);
      p.at[i] = make_int2(host_index[j], host_value[j]);
    }
    hipLaunchKernelGGL(write_i32_kernel, dim3(1), dim3(256), 0, st, p);
    const int e = tl_launch_status();
    if (e) return e;
  }
  return 0;
}

}  // extern "C"
