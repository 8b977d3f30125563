// Softmax attention over packed sequences of different lengths, with its gradients (gfx950): head dim 64,
// bf16 in and out, fp32 scores, statistics and sums; grouped heads, an optional causal mask, keys in a pack
// or in the slabs of a cache.
//
//   S = scale Q K^T (masked), P = softmax(S), O = P V, lse = log(sum exp S)
//   D = rowsum(dO O), dS = P (dO V^T - D), dV = P^T dO, dK = scale dS^T Q, dQ = scale dS K
//
// A packed row: the G = heads / kv_heads query heads that share a key head are G rows of one query position,
// r = i G + g.  A tile of rows then reads its keys once for all of them, a causal tile's diagonal is G times
// shorter, and one new token of 8 grouped heads is 8 rows, not 8 tiles of one.
//
// Lengths are read on the device: the grid is an upper bound that follows from the totals alone, and tile t
// belongs to the last sequence b with floor(cu[b] G / tile) + b <= t (find_tile) -- a sequence then owns
// at least ceil(its rows / tile) of these indexes, so no plan, copy or synchronisation precedes the launch.
// Everything read through cu is held to the totals, so a bad cu gives wrong rows but no access out of range.
#include "attn_tile.h"
#include "common.h"

#include <algorithm>
#include <cfloat>
#include <type_traits>

namespace i2pc {
namespace attnp {

using attn::bf16_t;
using attn::bf16x8;
using attn::f32x16;
using attn::kKV;
using attn::kTileBytes;
using attn::lds_addr;
using attn::pack_bf16;
using attn::v4s;

constexpr int kRows = 128;       // packed rows of a workgroup: 4 waves x 32

struct Args {
  const bf16_t *q, *k, *v;
  int64_t q_t, q_h, k_t, k_h, v_t, v_h;
  bf16_t* out;
  int64_t o_t, o_h;
  float* lse;
  const int32_t *cu_q, *cu_k, *k_lens;
  int B, Tq, Tk, H, Hk, G, zero_tail, nsplit;
  float c;                       // scale * log2(e)
  float* part_o;                 // [nsplit][Hk][Tq * G][64], rows normalised
  float2* part_l;                // [nsplit][Hk][Tq * G], a row's reference and its sum
  // backward
  const bf16_t* dout;
  int64_t d_t, d_h;
  bf16_t *dq, *dk, *dv;
  int64_t dq_t, dq_h, dk_t, dk_h, dv_t, dv_h;
  float scale;
  float *nlse, *ndelta;          // [H][Tq]: -lse / scale (NaN: the next two instead) and -D
  float *far_m, *far_l;          // [H][Tq]: a row's largest raw score, log2 of its sum relative to it
};

// The kernel's arguments, read again where they are used: for code that is hardly ever reached, so that its
// pointers and strides do not occupy scalar registers throughout.
typedef const __attribute__((address_space(4))) Args ConstArgs;
__device__ __forceinline__ ConstArgs* again() {
  ConstArgs* p = (ConstArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

// ------------------------------------------------------------------ lookup of a tile
__device__ __forceinline__ int cu_at(const int32_t* cu, int b, int total) {
  return b == 0 ? 0 : min(max(cu[b], 0), total);
}
// The last sequence b < entries with floor(cu[b] * mult / tile) + b <= t, 64 candidates a step; `local` becomes
// t's index within it.  (cu[b] * mult < 2^31: the host checks.)
__device__ __forceinline__ int find_tile(const int32_t* cu, int total, int mult, int tile, int entries, int t, int lane,
                                         int& local) {
  int lo = 0, n = entries, first = 0;
  while (n > 1) {
    const int step = (n + 63) >> 6;
    const int at = lane * step;
    int f = INT_MAX;
    if (at < n) f = cu_at(cu, lo + at, total) * mult / tile + lo + at;
    const int cnt = __popcll(__ballot(f <= t));
    if (cnt == 0) return -1;                     // not reached: f(0) = 0
    first = __builtin_amdgcn_readlane(f, cnt - 1);
    lo += (cnt - 1) * step;
    n = min(step, n - (cnt - 1) * step);
  }
  local = t - first;
  return __builtin_amdgcn_readfirstlane(lo);
}

struct Seq {
  int q0, lq, k0, lk;
};
// The sequence b and the tile within it that index t of a grid over `cu` (cu_q, or cu_k with BY_KEY) stands for; b = B: the
// rows behind the last sequence (zero_tail); tile < 0: nothing.  Up to 64 sequences everything is read at once, a sequence
// to a lane.  LONGEST: of up to 16 sequences those with the most keys come first, so that what ends last is short (ten
// images of 1 to 2305 tokens, twelve heads: 60 -> 56 us; the pass over the lengths costs more than that for 32 or 64).
template <bool BY_KEY, bool LONGEST>
__device__ __forceinline__ int locate(const Args& a, int mult, int rows, int t, int lane, int& tile, Seq& s) {
  const int32_t* cu = BY_KEY ? a.cu_k : a.cu_q;
  const int total = BY_KEY ? a.Tk : a.Tq;
  if (a.B <= 64) {
    const int i = min(lane, a.B - 1);
    const int q0 = i ? min(max(a.cu_q[i], 0), a.Tq) : 0, q1 = min(max(a.cu_q[i + 1], 0), a.Tq);
    const int k0 = i ? min(max(a.cu_k[i], 0), a.Tk) : 0, k1 = min(max(a.cu_k[i + 1], 0), a.Tk);
    const int most = a.k_lens ? max(0, a.k_lens[i]) : INT_MAX;
    const int lq = max(0, q1 - q0), lk = min(max(0, k1 - k0), most);
    int b;
    if (LONGEST && a.B <= 16) {
      const int n = lane < a.B ? ((BY_KEY ? lk : lq) * mult + rows - 1) / rows : 0;    // the lane's tiles
      int first = 0, all = 0;
      for (int j = 0; j < a.B; ++j) {
        const int nj = __builtin_amdgcn_readlane(n, j), cj = __builtin_amdgcn_readlane(lk, j);
        first += cj > lk || (cj == lk && j < lane) ? nj : 0;
        all += nj;
      }
      if (t >= all) {
        tile = a.zero_tail ? t - all : -1;
        return a.zero_tail ? a.B : 0;
      }
      b = max((int)__ffsll((unsigned long long)__ballot(t >= first && t < first + n)) - 1, 0);
      tile = t - __builtin_amdgcn_readlane(first, b);
    } else {
      const int f = (BY_KEY ? k0 : q0) * mult / rows + i;
      if (a.zero_tail) {
        const int end = __builtin_amdgcn_readlane(BY_KEY ? k1 : q1, a.B - 1) * mult / rows + a.B;
        if (t >= end) {
          tile = t - end;
          return a.B;
        }
      }
      b = max(__popcll(__ballot(lane < a.B && f <= t)) - 1, 0);
      tile = t - __builtin_amdgcn_readlane(f, b);
    }
    s.q0 = __builtin_amdgcn_readlane(q0, b);
    s.lq = __builtin_amdgcn_readlane(lq, b);
    s.k0 = __builtin_amdgcn_readlane(k0, b);
    s.lk = __builtin_amdgcn_readlane(lk, b);
    return b;
  }
  const int b = find_tile(cu, total, mult, rows, a.B + a.zero_tail, t, lane, tile);
  if (b == a.B) return b;
  s.q0 = __builtin_amdgcn_readfirstlane(cu_at(a.cu_q, b, a.Tq));
  s.lq = max(0, __builtin_amdgcn_readfirstlane(cu_at(a.cu_q, b + 1, a.Tq)) - s.q0);
  s.k0 = __builtin_amdgcn_readfirstlane(cu_at(a.cu_k, b, a.Tk));
  s.lk = max(0, __builtin_amdgcn_readfirstlane(cu_at(a.cu_k, b + 1, a.Tk)) - s.k0);
  if (a.k_lens) s.lk = min(s.lk, max(0, __builtin_amdgcn_readfirstlane(a.k_lens[b])));
  return b;
}

// ------------------------------------------------------------------ tiles in LDS
// 16-B chunk c of row r at c ^ swz(r), for tiles that are read both by rows (ds_read_b128, the A operand of
// S and dP) and transposed (ds_read_b64_tr_b16): a bijection of (r >> 1) & 7 whose lowest bit moves chunk
// sets {0-3} / {4-7} onto each other, so that neither read has a bank conflict.
__device__ __forceinline__ int swz(int row) {
  const int x = (row >> 1) & 7;
  return ((x & 1) << 2) | (x >> 1);
}

// 16 B (4 B) per lane global -> LDS.  Inline asm for the reason given at attn::dma16; the s_nop covers the wait
// states of M0 (1) and of scalars that come from a lane read (5), which the compiler does not see in here.
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rs, uint32_t lds_base, uint32_t voff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(lds_base), "v"(voff), "s"(rs)
               : "memory", "m0");
}
__device__ __forceinline__ void dma4(__amdgpu_buffer_rsrc_t rs, uint32_t lds_base, uint32_t voff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :
               : "s"(lds_base), "v"(voff), "s"(rs)
               : "memory", "m0");
}

// Where a tile of rows is read from.  The base is 64 bits and moves with the tile, so a sequence may span more than
// 4 GiB; moving it is a scalar addition, and so is the next tile's range: `rows` rows are left, and reads behind the
// 64 values of the last of them give zero.
template <int TILE>
struct Src {
  const uint8_t* p;
  uint32_t pitch;                // bytes from row to row
  __device__ __forceinline__ Src(const bf16_t* row, int64_t row_stride)
      : p(reinterpret_cast<const uint8_t*>(row)), pitch((uint32_t)row_stride * 2) {}
  __device__ __forceinline__ void move() { p += (uint64_t)pitch * TILE; }
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(int rows) const {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, (min(rows, TILE) - 1) * pitch + 128, 0x00020000);
  }
};

// one wave's quarter of a 64-row tile: 2 instructions of 8 rows x 128 B, to `lds` and 1 KiB behind it
struct Stage {
  uint32_t off[2];
  __device__ __forceinline__ Stage(int wid, int lane, int64_t pitch) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = (wid * 2 + j) * 8 + (lane >> 3);
      off[j] = (uint32_t)((row * pitch + ((lane & 7) ^ swz(row)) * 8) * 2);
    }
  }
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rs, uint32_t lds) const {
    dma16(rs, lds, off[0]);
    dma16(rs, lds + 1024, off[1]);
  }
};

// Where a lane reads its operands from a tile of 128-byte rows at LDS address `tile`: the A operand of a product over d
// (row lane & 31 of a 32-row block, chunk t of four) and of a product over the block's rows (columns 32 dt .. + 31 of rows
// {0-3, 8-11} + 4 (lane >> 5), by two transposing reads).  The swizzle repeats every 16 rows, so that other blocks,
// tiles and buffers are these addresses plus constants -- the offsets of the read instructions where the loops are
// unrolled over the two buffers, and no vector additions.
struct Lanes {
  uint32_t row[4], lo[2], hi[2];
  __device__ __forceinline__ Lanes(uint32_t tile, int lane) {
    const int lr = lane & 31, hh = lane >> 5;
#pragma unroll
    for (int t = 0; t < 4; ++t) row[t] = tile + lr * 128 + (((2 * t + hh) ^ swz(lr)) << 4);
    const int tg = lane >> 4, tq = (lane >> 2) & 3, tp = lane & 3, r0 = 4 * (tg >> 1) + tq, r1 = r0 + 8;
#pragma unroll
    for (int dt = 0; dt < 2; ++dt) {
      const int d0 = 32 * dt + 16 * (tg & 1) + 4 * tp, ch = d0 >> 3, within = (d0 & 7) * 2;
      lo[dt] = tile + r0 * 128 + ((ch ^ swz(r0)) << 4) + within;
      hi[dt] = tile + r1 * 128 + ((ch ^ swz(r1)) << 4) + within;
    }
  }
  __device__ __forceinline__ Lanes behind(uint32_t bytes) const {      // the addresses of another buffer
    Lanes x = *this;
#pragma unroll
    for (int t = 0; t < 4; ++t) x.row[t] += bytes;
#pragma unroll
    for (int dt = 0; dt < 2; ++dt) x.lo[dt] += bytes, x.hi[dt] += bytes;
    return x;
  }
  // `at`: bytes from `tile` to the block's first row (rows: 16 of them for a column read)
  __device__ __forceinline__ bf16x8 rows(int t, uint32_t at) const {
    return *(const __attribute__((address_space(3))) bf16x8*)(row[t] + at);
  }
  __device__ __forceinline__ bf16x8 columns(int dt, uint32_t at) const {
    const v4s l = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(lo[dt] + at));
    const v4s h = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(hi[dt] + at));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(l, h, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};
__device__ __forceinline__ bf16x8 p_frag(const uint32_t (&pk)[8], int s) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(bf16x8, u32x4{pk[4 * s], pk[4 * s + 1], pk[4 * s + 2], pk[4 * s + 3]});
}
__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ bool nonfinite(bf16x8 f) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const u32x4 u = __builtin_bit_cast(u32x4, f);
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= (u[i] & 0x7f80u) == 0x7f80u || (u[i] & 0x7f800000u) == 0x7f800000u;
  return bad;
}

// A matrix product multiplies a masked row by zero, which is NaN where that row holds an infinity or NaN.  Blocks
// that are partly masked look for such values (`bad`); a wave that met one does its sums again at the end, a row of
// K, V, Q or dO at a time and only with the rows that the mask leaves -- slow, and for such inputs only.
__device__ __forceinline__ float dot_row(const bf16_t* row, const bf16x8 (&f)[4], int hh) {
  float s = 0.f;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const bf16x8 x = *reinterpret_cast<const bf16x8*>(row + 16 * t + 8 * hh);
    bf16x8 y = f[t];
    asm volatile("" : "+v"(y));                      // its conversion is not kept in registers from row to row
#pragma unroll
    for (int j = 0; j < 8; ++j) s = fmaf((float)x[j], (float)y[j], s);
  }
  return s + __shfl_xor(s, 32);
}
__device__ __forceinline__ void add_row(f32x16 (&acc)[2], float w, const bf16_t* row, int hh) {
#pragma unroll
  for (int dt = 0; dt < 2; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const uint2 x = *reinterpret_cast<const uint2*>(row + 32 * dt + 8 * g + 4 * hh);
      const float e[4] = {__uint_as_float(x.x << 16), __uint_as_float(x.x & 0xffff0000u), __uint_as_float(x.y << 16),
                          __uint_as_float(x.y & 0xffff0000u)};
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[dt][4 * g + i] = fmaf(w, e[i], acc[dt][4 * g + i]);
    }
}

// whether this lane's part of the 32 rows at `at` has an infinity or NaN
__device__ __forceinline__ int has_nonfinite(const Lanes& ad, uint32_t at) {
  int bad = 0;
#pragma unroll
  for (int t = 0; t < 4; ++t) bad |= nonfinite(ad.rows(t, at));
  return bad;
}

// a bound that the compiler does not take apart: it would keep sixteen of its sums with constants in registers instead
__device__ __forceinline__ int whole(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// 4 consecutive values a lane and register group of an accumulator, times f, as bf16: row[32 dt + 8 g + 4 hh ...]
__device__ __forceinline__ void store_acc(bf16_t* row, const f32x16 (&o)[2], float f, int hh) {
#pragma unroll
  for (int dt = 0; dt < 2; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      uint2 w;
      w.x = pack_bf16(o[dt][4 * g + 0] * f, o[dt][4 * g + 1] * f);
      w.y = pack_bf16(o[dt][4 * g + 2] * f, o[dt][4 * g + 3] * f);
      *reinterpret_cast<uint2*>(row + 32 * dt + 8 * g + 4 * hh) = w;
    }
}

// keys that packed row r's query sees
__device__ __forceinline__ int seen(bool causal, int i, const Seq& s) {
  return causal ? min(max(i + 1 + s.lk - s.lq, 0), s.lk) : s.lk;
}

// rows [from, from + 128) of the rows behind the last sequence, as zero
__device__ __forceinline__ void zero_rows(bf16_t* out, int64_t o_t, int64_t o_h, int t0, int from, int count, int hk, int G,
                                          float* lse, int H) {
  for (int e = threadIdx.x; e < kRows * 8; e += 256) {
    const int r = from + (e >> 3);
    if (r >= count) break;
    const int i = r / G, h = hk * G + r - i * G;
    *reinterpret_cast<uint4*>(out + (t0 + i) * o_t + h * o_h + (e & 7) * 8) = make_uint4(0, 0, 0, 0);
    if (lse && (e & 7) == 0) lse[(int64_t)(t0 + i) * H + h] = -INFINITY;
  }
}

// ------------------------------------------------------------------ forward
// A row's running state, a row to a lane (its two lane halves hold different keys' probabilities and different d of O).
struct Rows {
  f32x16 o[2];                   // O^T, not normalised
  float m;                       // the reference, a raw score
  float l;                       // this half's sum of 2^(c (s - m))
  int bad;                       // met an infinity or NaN in a partly masked block
  bool far;                      // (uniform) c m of some row is too large for a product that is not rounded beside one that is
  __device__ __forceinline__ void clear() {
    for (int i = 0; i < 16; ++i) o[0][i] = o[1][i] = 0.f;
    m = l = 0.f;
    bad = 0;
    far = false;
  }
};

// 32 keys (at bytes atK, atV behind the addresses' tile) for 32 rows: p = 2^(c s - c m), one FMA and one exponential a
// score.  m moves only when a probability could pass 2^8 (harmless for the bf16 operand and the fp32 sums), so the usual
// block has no maximum and no rescale.  first: the rows' first block, which sets m (a bool, or its constant).  left: how many of
// the block's keys the lane's row sees; partial (uniform): not all of them for some row of the wave.
// c m is rounded and c s within the FMA is not: the exponent of s = m is off by up to 2^-25 |c m|, the same for a row's every
// score, which the sum takes out again -- until it leaves the exponential's range.  Rows whose |c m| is above 2^12 (`far`) take
// 2^(c (s - m)) instead, with their maximum anew in each block.
template <bool CAUSAL, class First>
__device__ __forceinline__ void attend(Rows& w, const bf16x8 (&qf)[4], const Lanes& ad, uint32_t atK, uint32_t atV, First first,
                                       bool partial, int left, float c, int hh) {
  constexpr float kThresh = 256.f, kFar = 4096.f;
  bf16x8 kf[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) kf[t] = ad.rows(t, atK);
  f32x16 st;
#pragma unroll
  for (int t = 0; t < 4; ++t) st = mfma(kf[t], qf[t], t == 0 ? f32x16{} : st);
  // V's columns are on their way while the exponentials are taken
  bf16x8 vf[2][2];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int dt = 0; dt < 2; ++dt) vf[t][dt] = ad.columns(dt, atV + 2048 * t);
  if (partial) {
    const int lim = whole(left - 4 * hh);
#pragma unroll
    for (int i = 0; i < 16; ++i) st[i] = (i & 3) + 8 * (i >> 2) < lim ? st[i] : -INFINITY;
  }
  float ls = 0.f;
  uint32_t pk[8];
  auto probs = [&](float mc) {
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const float p0 = __builtin_amdgcn_exp2f(fmaf(st[i], c, -mc));
      const float p1 = __builtin_amdgcn_exp2f(fmaf(st[i + 1], c, -mc));
      ls = i ? ls + (p0 + p1) : p0 + p1;
      pk[i >> 1] = pack_bf16(p0, p1);
    }
  };
  bool full = first || w.far;
  if (!full) {
    probs(w.m * c);
    full = __ballot(ls >= kThresh) != 0;
  }
  if (full) {
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, st[i]);
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
    mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
    // a row that sees nothing here keeps its reference; one that has met no score but -inf has the lowest finite one (and is far)
    const float m_new = fmaxf(mx, first ? -FLT_MAX : w.m);
    if (!first) {
      const float alpha = __builtin_amdgcn_exp2f((w.m - m_new) * c);
      w.l *= alpha;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        w.o[0][i] *= alpha;
        w.o[1][i] *= alpha;
      }
    }
    w.m = m_new;
    float mc = m_new * c;
    w.far = __ballot(fabsf(mc) > kFar) != 0;
    if (__builtin_expect(w.far, 0)) {
#pragma unroll
      for (int i = 0; i < 16; ++i) st[i] -= m_new;
      mc = 0.f;
    }
    probs(mc);
  }
  w.l += ls;
  if (CAUSAL && partial) w.bad |= has_nonfinite(ad, atV);
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int dt = 0; dt < 2; ++dt) w.o[dt] = mfma(vf[t][dt], p_frag(pk, t), w.o[dt]);
}

// log(sum exp(scale s)) of a row from its reference and sum: -inf for a row that saw no key (or only scores of -inf), and for
// no other
__device__ __forceinline__ float lse_of(float m, float l, float scale) {
  const float x = fmaf(m, scale, log2f(l) * 0.69314718055994531f);
  return l != 0.f && x == -INFINITY ? -FLT_MAX : x;
}

// The state of the keys [from, to) again, key by key: rows that `bad` says need it.
__device__ __forceinline__ void attend_again(Rows& w, const bf16x8 (&qf)[4], const bf16_t* K, int64_t k_t, const bf16_t* V,
                                             int64_t v_t, int from, int to, int step, int nk, float c, int hh) {
  float m = -INFINITY, l = 0.f;
  w.clear();
#pragma clang loop unroll(disable)
  for (int j = from; j < to; j += (j & 31) == 31 ? step : 1) {
    const float x = dot_row(K + j * k_t, qf, hh);
    if (j < nk) {
      const float m_new = fmaxf(m, x), alpha = m == m_new ? 1.f : __builtin_amdgcn_exp2f((m - m_new) * c);
      const float p = x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((x - m_new) * c);
      m = m_new;
      l = fmaf(l, alpha, p);
      for (int i = 0; i < 16; ++i) {
        w.o[0][i] *= alpha;
        w.o[1][i] *= alpha;
      }
      add_row(w.o, p, V + j * v_t, hh);
    }
  }
  w.m = m == -INFINITY ? 0.f : m;
  w.l = hh ? 0.f : l;                                // the whole sum; the halves' are added
}

// One workgroup: 128 / KW packed rows of one key head, over all of their keys or (SPLIT) over one of nsplit shares of
// them.  Each wave owns 32 rows, a row to a lane: S^T = K Q^T leaves a query's scores in one lane's
// registers, which then are the B operand of O^T += V^T P^T.  K and V tiles of 64 keys go through LDS by
// LDS-DMA, double-buffered.  KW 2: waves 2, 3 hold the rows of waves 0, 1 again and take the second 32 keys of each tile,
// and the two states are joined at the end: twice the workgroups, of half the length.
// Bound by the exponentials and the products together: 8 x 4096 tokens of 16 heads take 585 us in the kernel trace (940 TF; calls
// one after the other 561, 980 TF), the vector unit 77 % busy and the matrix unit 58 %, at the 1.6 to 1.7 GHz that the power limit
// leaves.  Four waves a SIMD: eight-wave workgroups of 256 rows were slower (causal prompts 118 against 107 us), as were raised
// wave priorities.  The first tile is outside the loop: with its test for a row's first block inside, the loop had no registers
// for the addresses of both buffers (2 % slower).
template <bool CAUSAL, bool SPLIT, int KW>
__global__ __launch_bounds__(256, 4) void k_attnp_fwd(const Args a) {
  constexpr int kWgRows = kRows / KW;
  __shared__ __attribute__((aligned(16))) uint8_t smem[4 * kTileBytes];
  __shared__ float ml[2][KW == 2 ? 2 : 1][KW == 2 ? 64 : 1];
  const int lane = threadIdx.x & 63, hh = lane >> 5, lr = lane & 31;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rw = KW == 2 ? wid & 1 : wid, kw = KW == 2 ? wid >> 1 : 0;
  // key heads fastest: workgroups b and b + 8 share an XCD, so with 8 heads (4, 2) each XCD (pair, four) keeps to
  // one head's keys; with a causal mask later tiles, which have the most keys, come first
  const int hk = blockIdx.x % a.Hk;
  int rest = blockIdx.x / a.Hk;
  const int split = SPLIT ? rest % a.nsplit : 0;
  if (SPLIT) rest /= a.nsplit;
  const int tiles = gridDim.x / (a.Hk * (SPLIT ? a.nsplit : 1));
  int tile;
  Seq s;
  const int b = locate<false, !CAUSAL>(a, a.G, kWgRows, CAUSAL ? tiles - 1 - rest : rest, lane, tile, s);
  if (b == a.B) {                                    // the rows behind the last sequence
    const int t0 = cu_at(a.cu_q, a.B, a.Tq);
    if (!SPLIT) zero_rows(a.out, a.o_t, a.o_h, t0, tile * kWgRows, min((tile + 1) * kWgRows, (a.Tq - t0) * a.G), hk, a.G, a.lse, a.H);
    return;
  }
  const int R = s.lq * a.G, r0 = tile * kWgRows;
  if (tile < 0 || r0 >= R) return;
  const int r = r0 + rw * 32 + lr, rc = min(r, R - 1), qi = rc / a.G, h = hk * a.G + rc - qi * a.G;
  const int nk = seen(CAUSAL, qi, s);
  // first and last row of the wave, last row of the tile (uniform)
  const int w0 = min(r0 + rw * 32, R - 1);
  const bool wave_on = r0 + rw * 32 < R;
  const int nk_first = seen(CAUSAL, w0 / a.G, s), nk_last = seen(CAUSAL, min(w0 + 31, R - 1) / a.G, s);
  int ks = 0, ke = seen(CAUSAL, (min(r0 + kWgRows, R) - 1) / a.G, s);
  if (SPLIT) {
    const int chunk = ((s.lk + a.nsplit - 1) / a.nsplit + kKV - 1) / kKV * kKV;
    ks = (int)min((int64_t)split * chunk, (int64_t)ke);
    ke = min(ke, ks + chunk);
  }

  const bf16_t* Kg = a.k + (s.k0 * a.k_t + hk * a.k_h);
  const bf16_t* Vg = a.v + (s.k0 * a.v_t + hk * a.v_h);
  const Stage stk(wid, lane, a.k_t), stv(wid, lane, a.v_t);
  Src<kKV> srck(Kg + ks * a.k_t, a.k_t), srcv(Vg + ks * a.v_t, a.v_t);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(smem)) + wid * 2048;
  auto stage = [&](int buf, int key) {               // the next tile, which starts at key
    stk.load(srck.rsrc(s.lk - key), lds0 + buf * 2 * kTileBytes);
    stv.load(srcv.rsrc(s.lk - key), lds0 + (buf * 2 + 1) * kTileBytes);
    srck.move();
    srcv.move();
  };
  if (ks < ke) stage(0, ks);
  bf16x8 qf[4];
  {
    const bf16_t* qr = a.q + (s.q0 + qi) * a.q_t + h * a.q_h;
#pragma unroll
    for (int t = 0; t < 4; ++t) qf[t] = *reinterpret_cast<const bf16x8*>(qr + 16 * t + 8 * hh);
  }
  __builtin_amdgcn_s_waitcnt(0xF70);                 // vmcnt(0), known to the compiler: Q and the first tile
  __syncthreads();

  const float c = a.c;
  Rows w;
  w.clear();
  const Lanes ad(lds_addr(smem) + kw * 4096, lane);
  auto step = [&](int key0, auto buffer, auto first) {
    constexpr int cur = decltype(buffer)::value;
    if (key0 + kKV < ke) stage(cur ^ 1, key0 + kKV);
    if (wave_on) {
      const int key = key0 + 32 * kw;
      constexpr uint32_t atK = cur * 2 * kTileBytes, atV = atK + kTileBytes;
      if (key < nk_last) {                           // some row of the wave sees these keys
        attend<CAUSAL>(w, qf, ad, atK, atV, first, key + 32 > nk_first, nk - key, c, hh);
        if (KW == 1 && key + 32 < nk_last)
          attend<CAUSAL>(w, qf, ad, atK + 4096, atV + 4096, std::false_type{}, key + 64 > nk_first, nk - key - 32, c, hh);
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the next tile landed (this wave's part)
    __syncthreads();                                     // ... and every wave's
  };
  if (ks < ke) step(ks, std::integral_constant<int, 0>{}, std::true_type{});
  for (int key0 = ks + kKV; key0 < ke; key0 += 2 * kKV) {
    step(key0, std::integral_constant<int, 1>{}, std::false_type{});
    if (key0 + kKV < ke) step(key0 + kKV, std::integral_constant<int, 0>{}, std::false_type{});
  }
  if (CAUSAL && __ballot(w.bad) != 0)
    attend_again(w, qf, Kg, a.k_t, Vg, a.v_t, ks + 32 * kw, min(ke, nk_last), KW == 2 ? 33 : 1, nk, c, hh);
  float l = w.l + __shfl_xor(w.l, 32), m = w.m;
  if constexpr (KW == 2) {
    float* x = reinterpret_cast<float*>(smem) + rw * 32 * 64 + lane;
    if (kw == 1) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[i * 64] = w.o[0][i];
        x[(16 + i) * 64] = w.o[1][i];
      }
      ml[0][rw][lane] = m;
      ml[1][rw][lane] = l;
    }
    __syncthreads();
    if (kw == 1) return;
    const float m1 = ml[0][rw][lane], l1 = ml[1][rw][lane];
    if (l1 != 0.f) {                                 // (NaN: joined too)
      // a half without a probability has no say: its reference may lie anywhere
      const bool empty = l == 0.f;
      const float mm = empty ? m1 : fmaxf(m, m1);
      const float f0 = empty ? 0.f : m == mm ? 1.f : __builtin_amdgcn_exp2f((m - mm) * c);
      const float f1 = m1 == mm ? 1.f : __builtin_amdgcn_exp2f((m1 - mm) * c);
      l = fmaf(l, f0, l1 * f1);
      m = mm;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        w.o[0][i] = fmaf(w.o[0][i], f0, x[i * 64] * f1);
        w.o[1][i] = fmaf(w.o[1][i], f0, x[(16 + i) * 64] * f1);
      }
    }
  }
  if (r >= R) return;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  if (SPLIT) {
    const int64_t row = ((int64_t)split * a.Hk + hk) * a.Tq * a.G + (int64_t)s.q0 * a.G + r;
    if (hh == 0) a.part_l[row] = make_float2(m, l);
    if (l != 0.f) {
#pragma unroll
      for (int dt = 0; dt < 2; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<float4*>(a.part_o + row * 64 + 32 * dt + 8 * g + 4 * hh) =
              make_float4(w.o[dt][4 * g] * inv, w.o[dt][4 * g + 1] * inv, w.o[dt][4 * g + 2] * inv, w.o[dt][4 * g + 3] * inv);
    }
  } else {
    store_acc(a.out + (s.q0 + qi) * a.o_t + h * a.o_h, w.o, inv, hh);
    if (hh == 0) a.lse[(int64_t)(s.q0 + qi) * a.H + h] = lse_of(m, l, a.scale);
  }
}

// Few rows (new tokens over a cache): 32 packed rows of one key head a workgroup, whose four waves take every fourth
// block of 32 keys of a share, each with its own two LDS buffers and no barrier until the end -- what counts is how many
// bytes of K and V are on their way, 8 KiB a wave.  A share is lk / nsplit keys, 256 at least.
// Bound by HBM: one token of 64 sequences over 97 to 8096 keys, 16 heads over 4: 58 us and 5 us for the join (4.4 TB/s; a copy
// reaches 4.9); one token over 131071 keys, 16 heads over 2: 15 and 4 us.
constexpr int kFew = 32;
constexpr int kFewBlock = 32 * 128;                  // bytes of 32 keys' K (or V)
template <bool CAUSAL>
__global__ __launch_bounds__(256, 2) void k_attnp_few(const Args a) {
  // per wave two buffers of K block, V block; at the end the waves' sums, rows of 68 floats
  __shared__ __attribute__((aligned(16))) uint8_t smem[4 * 4 * kFewBlock];
  __shared__ float ml[2][4][32];
  const int lane = threadIdx.x & 63, hh = lane >> 5, lr = lane & 31;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hk = blockIdx.x % a.Hk;
  int rest = blockIdx.x / a.Hk;
  const int split = rest % a.nsplit;
  int tile;
  Seq s;
  const int b = locate<false, false>(a, a.G, kFew, rest / a.nsplit, lane, tile, s);
  if (b == a.B) {
    const int t0 = cu_at(a.cu_q, a.B, a.Tq);
    if (split == 0 && a.nsplit == 1) zero_rows(a.out, a.o_t, a.o_h, t0, tile * kFew, min((tile + 1) * kFew, (a.Tq - t0) * a.G), hk, a.G, a.lse, a.H);
    return;
  }
  const int R = s.lq * a.G, r0 = tile * kFew;
  if (tile < 0 || r0 >= R) return;
  const int rc = min(r0 + lr, R - 1), qi = rc / a.G, h = hk * a.G + rc - qi * a.G;
  const int nk = seen(CAUSAL, qi, s), nk_first = seen(CAUSAL, r0 / a.G, s);
  int ke = seen(CAUSAL, (min(r0 + kFew, R) - 1) / a.G, s);
  const int chunk = max(256, ((s.lk + a.nsplit - 1) / a.nsplit + 127) / 128 * 128);
  const int ks = (int)min((int64_t)split * chunk, (int64_t)ke);
  ke = min(ke, ks + chunk);

  const bf16_t* Kg = a.k + (s.k0 * a.k_t + hk * a.k_h);
  const bf16_t* Vg = a.v + (s.k0 * a.v_t + hk * a.v_h);
  uint32_t offk[4], offv[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int row = j * 8 + (lane >> 3), ch = ((lane & 7) ^ swz(row)) * 8;
    offk[j] = (uint32_t)((row * a.k_t + ch) * 2);
    offv[j] = (uint32_t)((row * a.v_t + ch) * 2);
  }
  uint8_t* mine = smem + wid * 4 * kFewBlock;
  const int first = ks + 32 * wid;
  Src<128> srck(Kg + first * a.k_t, a.k_t), srcv(Vg + first * a.v_t, a.v_t);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(mine));
  auto stage = [&](int buf, int key) {               // the wave's next block, which starts at key
    const auto rk = srck.rsrc(s.lk - key), rv = srcv.rsrc(s.lk - key);
    const uint32_t base = lds0 + buf * 2 * kFewBlock;
#pragma unroll
    for (int j = 0; j < 4; ++j) dma16(rk, base + j * 1024, offk[j]);
#pragma unroll
    for (int j = 0; j < 4; ++j) dma16(rv, base + kFewBlock + j * 1024, offv[j]);
    srck.move();
    srcv.move();
  };
  bf16x8 qf[4];
  {
    const bf16_t* qr = a.q + (s.q0 + qi) * a.q_t + h * a.q_h;
#pragma unroll
    for (int t = 0; t < 4; ++t) qf[t] = *reinterpret_cast<const bf16x8*>(qr + 16 * t + 8 * hh);
  }
  if (first < ke) stage(0, first);
  const float c = a.c;
  Rows w;
  w.clear();
  const Lanes ad(lds_addr(mine), lane);
  auto step = [&](int key, auto buffer) {
    constexpr int cur = decltype(buffer)::value;
    if (key + 128 < ke) {
      // the other buffer's reads have returned before it is written again
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      stage(cur ^ 1, key + 128);
      asm volatile("s_waitcnt vmcnt(8)" ::: "memory");  // this block landed, the next one's 8 loads may be on their way
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    attend<CAUSAL>(w, qf, ad, cur * 2 * kFewBlock, (cur * 2 + 1) * kFewBlock, key == first, key + 32 > nk_first, nk - key, c, hh);
  };
  for (int key = first; key < ke; key += 256) {
    step(key, std::integral_constant<int, 0>{});
    if (key + 128 < ke) step(key + 128, std::integral_constant<int, 1>{});
  }
  if (CAUSAL && __ballot(w.bad) != 0) attend_again(w, qf, Kg, a.k_t, Vg, a.v_t, first, ke, 97, nk, c, hh);
  const float l = w.l + __shfl_xor(w.l, 32);

  // the four waves' sums: sum_w f_w O_w, f_w = 2^(c (m_w - m))
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  float* ow = reinterpret_cast<float*>(mine);
#pragma unroll
  for (int dt = 0; dt < 2; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<float4*>(ow + lr * 68 + 32 * dt + 8 * g + 4 * hh) =
          make_float4(w.o[dt][4 * g], w.o[dt][4 * g + 1], w.o[dt][4 * g + 2], w.o[dt][4 * g + 3]);
  if (hh == 0) {
    ml[0][wid][lr] = l == 0.f ? -INFINITY : w.m;
    ml[1][wid][lr] = l;
  }
  __syncthreads();
  const int row = threadIdx.x >> 3, d = (threadIdx.x & 7) * 8, r = r0 + row;
  if (r >= R) return;
  float m = -INFINITY, total = 0.f, acc[8] = {};
#pragma unroll
  for (int v = 0; v < 4; ++v) m = fmaxf(m, ml[0][v][row]);
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const float lv = ml[1][v][row];
    if (lv == 0.f) continue;                         // saw nothing (a NaN sum is not skipped)
    const float mv = ml[0][v][row], f = mv == m ? 1.f : __builtin_amdgcn_exp2f((mv - m) * c);
    total = fmaf(f, lv, total);
    const float* x = reinterpret_cast<const float*>(smem + v * 4 * kFewBlock) + row * 68 + d;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = fmaf(f, x[i], acc[i]);
  }
  const float inv = total == 0.f ? 0.f : 1.0f / total;
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] *= inv;
  const int i = r / a.G, hq = hk * a.G + r - i * a.G;
  if (a.nsplit == 1) {
    *reinterpret_cast<uint4*>(a.out + (s.q0 + i) * a.o_t + hq * a.o_h + d) =
        make_uint4(pack_bf16(acc[0], acc[1]), pack_bf16(acc[2], acc[3]), pack_bf16(acc[4], acc[5]), pack_bf16(acc[6], acc[7]));
    if (d == 0) a.lse[(int64_t)(s.q0 + i) * a.H + hq] = lse_of(m, total, a.scale);
  } else {
    const int64_t at = ((int64_t)split * a.Hk + hk) * a.Tq * a.G + (int64_t)s.q0 * a.G + r;
    if (d == 0) a.part_l[at] = make_float2(m, total);
    if (total != 0.f) {
      *reinterpret_cast<float4*>(a.part_o + at * 64 + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      *reinterpret_cast<float4*>(a.part_o + at * 64 + d + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
    }
  }
}

// The shares of a split call joined, W waves to a row: out = sum_s w_s O_s / sum_s w_s, w_s = l_s 2^(c (m_s - m)).  Wave v takes the
// shares 8 v .. 8 v + 7, then 8 W further, eight loads in flight; a lane is a d.  Bound by the latency of two dependent
// reads: 4 to 5 us.
template <int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void k_attnp_join(const Args a) {
  __shared__ float red[W == 1 ? 1 : W][W == 1 ? 1 : 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, v = W == 1 ? 0 : wave;
  const int64_t rows = (int64_t)a.Tq * a.G, n = W == 1 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
  if (n >= rows * a.Hk) return;
  const int hk = (int)(n / rows), row = (int)(n - hk * rows), t = row / a.G, h = hk * a.G + row - t * a.G;
  const bool tail = t >= cu_at(a.cu_q, a.B, a.Tq);
  if (tail && !a.zero_tail) return;
  const int64_t step = rows * a.Hk;                  // from share to share
  const float2* pl = a.part_l + hk * rows + row;
  const float* po = a.part_o + (hk * rows + row) * 64 + lane;
  float acc = 0.f, m = -INFINITY, total = 0.f;
  if (!tail) {
    for (int s = lane; s < a.nsplit; s += 64) {
      const float2 x = pl[s * step];
      m = fmaxf(m, x.y == 0.f ? -INFINITY : x.x);
    }
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
    for (int s0 = 8 * v; s0 < a.nsplit; s0 += 8 * W) {
      float2 l[8];
      float o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) l[j] = pl[min(s0 + j, a.nsplit - 1) * step];
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = po[min(s0 + j, a.nsplit - 1) * step * 64];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        // an empty share wrote no O; NaN shares (a NaN or infinite score) stay NaN
        const bool on = s0 + j < a.nsplit && l[j].y != 0.f;
        const float w = on ? l[j].y * __builtin_amdgcn_exp2f((l[j].x - m) * a.c) : 0.f;
        total += w;
        acc = on ? fmaf(w, o[j], acc) : acc;
      }
    }
  }
  if constexpr (W > 1) {
    red[v][lane] = acc;
    __shared__ float tot[W];
    if (lane == 0) tot[v] = total;
    __syncthreads();
    if (v) return;
    acc = total = 0.f;
#pragma unroll
    for (int u = 0; u < W; ++u) {
      acc += red[u][lane];
      total += tot[u];
    }
  }
  const __bf16 o = (__bf16)(total == 0.f ? 0.f : acc / total);
  a.out[t * a.o_t + h * a.o_h + lane] = __builtin_bit_cast(bf16_t, o);
  if (lane == 0) a.lse[(int64_t)t * a.H + h] = lse_of(m, total, a.scale);
}

// ------------------------------------------------------------------ backward
constexpr float kFarLse = 16384.f;
constexpr uint32_t kFarMark = 0x7fc0fa11u;           // a NaN of its own, for the nlse of such rows
__device__ __forceinline__ bool is_far(float lse) { return fabsf(lse) > kFarLse && lse != -INFINITY; }

// dQ: the forward's rows and tiles; per 32 keys S^T = K Q^T and dP^T = V dO^T (which starts at -D), then
// dQ^T += K^T dS^T.  KW 2 as in the forward pass.  D = rowsum(dO O) is taken on the way from the rows that the kernel holds
// anyway, and left for the dK / dV kernel: ndelta = -D, nlse = -lse / scale (-inf for a row that saw nothing, so that its
// probabilities are 0), both [H][Tq].  The rounding of O to bf16 is off in D by |dO| |O| 2^-9, which counts where a row has
// few keys (the share falls with the root of their number): there D = sum P dP is taken from the tile itself.
// lse is rounded to fp32, and a probability is off by as much: 2^-20 |lse| with the roundings on the way of lse / scale.  Rows of
// |lse| above 2^14, where that would pass bf16's own rounding, are done again at the end from their largest score and their sum,
// which are left for the dK / dV kernel too; their nlse is a NaN of its own, so that a key which such a row sees becomes NaN there
// and is done again.
// Bound as the forward pass: 8 x 4096 tokens of 16 heads 795 us, 1038 TF over the three products.  Three waves a SIMD; two
// with the blocks interleaved as in the dK / dV kernel were slower (six images' step 91 against 84 us).
template <bool CAUSAL, int KW>
__global__ __launch_bounds__(256, 3) void k_attnp_dq(const Args a) {
  constexpr int kWgRows = kRows / KW;
  __shared__ __attribute__((aligned(16))) uint8_t smem[4 * kTileBytes];
  const int lane = threadIdx.x & 63, hh = lane >> 5, lr = lane & 31;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rw = KW == 2 ? wid & 1 : wid, kw = KW == 2 ? wid >> 1 : 0;
  const int hk = blockIdx.x % a.Hk, rest = blockIdx.x / a.Hk, tiles = gridDim.x / a.Hk;
  int tile;
  Seq s;
  const int b = locate<false, !CAUSAL>(a, a.G, kWgRows, CAUSAL ? tiles - 1 - rest : rest, lane, tile, s);
  if (b == a.B) {
    const int t0 = cu_at(a.cu_q, a.B, a.Tq);
    zero_rows(a.dq, a.dq_t, a.dq_h, t0, tile * kWgRows, min((tile + 1) * kWgRows, (a.Tq - t0) * a.G), hk, a.G, nullptr, 0);
    return;
  }
  const int R = s.lq * a.G, r0 = tile * kWgRows;
  if (tile < 0 || r0 >= R) return;
  const int r = r0 + rw * 32 + lr, rc = min(r, R - 1), qi = rc / a.G, h = hk * a.G + rc - qi * a.G;
  const int nk = seen(CAUSAL, qi, s);
  const int w0 = min(r0 + rw * 32, R - 1);
  const bool wave_on = r0 + rw * 32 < R;
  const int nk_first = seen(CAUSAL, w0 / a.G, s), nk_last = seen(CAUSAL, min(w0 + 31, R - 1) / a.G, s);
  const int ke = seen(CAUSAL, (min(r0 + kWgRows, R) - 1) / a.G, s);

  const bf16_t* Kg = a.k + (s.k0 * a.k_t + hk * a.k_h);
  const bf16_t* Vg = a.v + (s.k0 * a.v_t + hk * a.v_h);
  const Stage stk(wid, lane, a.k_t), stv(wid, lane, a.v_t);
  Src<kKV> srck(Kg, a.k_t), srcv(Vg, a.v_t);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(smem)) + wid * 2048;
  auto stage = [&](int buf, int key) {
    stk.load(srck.rsrc(s.lk - key), lds0 + buf * 2 * kTileBytes);
    stv.load(srcv.rsrc(s.lk - key), lds0 + (buf * 2 + 1) * kTileBytes);
    srck.move();
    srcv.move();
  };
  if (ke > 0) stage(0, 0);
  bf16x8 qf[4], df[4];
  const bf16_t* qr = a.q + (s.q0 + qi) * a.q_t + h * a.q_h;
  const bf16_t* dr = a.dout + (s.q0 + qi) * a.d_t + h * a.d_h;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    qf[t] = *reinterpret_cast<const bf16x8*>(qr + 16 * t + 8 * hh);
    df[t] = *reinterpret_cast<const bf16x8*>(dr + 16 * t + 8 * hh);
  }
  const float c = a.c;
  const float lse = a.lse[(int64_t)(s.q0 + qi) * a.H + h];
  const float neg = lse == -INFINITY ? -INFINITY : is_far(lse) ? __uint_as_float(kFarMark) : lse != lse ? NAN : -lse / a.scale;
  const float nl = neg * c;
  float d = dot_row(a.out + (s.q0 + qi) * a.o_t + h * a.o_h, df, hh);
  __builtin_amdgcn_s_waitcnt(0xF70);
  __syncthreads();

  const Lanes ad(lds_addr(smem) + kw * 4096, lane);
  if (wave_on && nk_last <= kKV) {                   // D of rows with one tile of keys: sum P dP
    const float rounded = d;
    d = 0.f;
#pragma clang loop unroll(disable)
    for (int k2 = 0; 32 * k2 < nk_last; ++k2) {
      const Lanes at = ad.behind((uint32_t)(k2 - kw) * 4096);
      const int lim = whole(nk - 32 * k2 - 4 * hh);
      f32x16 st, dp;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        st = mfma(at.rows(t, 0), qf[t], t == 0 ? f32x16{} : st);
        dp = mfma(at.rows(t, kTileBytes), df[t], t == 0 ? f32x16{} : dp);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) d += (i & 3) + 8 * (i >> 2) < lim ? __builtin_amdgcn_exp2f(fmaf(st[i], c, nl)) * dp[i] : 0.f;
    }
    d += __shfl_xor(d, 32);
    if (nl != nl) d = rounded;
  }
  f32x16 nd, dq[2];
  for (int i = 0; i < 16; ++i) {
    nd[i] = lse == -INFINITY ? 0.f : -d;
    dq[0][i] = dq[1][i] = 0.f;
  }
  if (r < R && kw == 0 && hh == 0) {
    const int64_t at = (int64_t)h * a.Tq + s.q0 + qi;
    a.nlse[at] = neg;
    a.ndelta[at] = nd[0];
  }

  int bad = 0;
  auto step = [&](int key0, auto buffer) {
    constexpr int cur = decltype(buffer)::value;
    if (key0 + kKV < ke) stage(cur ^ 1, key0 + kKV);
    if (wave_on) {
#pragma unroll
      for (int k2 = 0; k2 < 2 / KW; ++k2) {
        const int key = key0 + 32 * (k2 + kw);
        const uint32_t atK = cur * 2 * kTileBytes + k2 * 4096, atV = atK + kTileBytes;
        if (key >= nk_last) break;
        f32x16 st, dp;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          st = mfma(ad.rows(t, atK), qf[t], t == 0 ? f32x16{} : st);
          dp = mfma(ad.rows(t, atV), df[t], t == 0 ? nd : dp);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) dp[i] *= __builtin_amdgcn_exp2f(fmaf(st[i], c, nl));
        if (key + 32 > nk_first) {                   // some row of the wave does not see all of the block
          const int lim = whole(nk - key - 4 * hh);
#pragma unroll
          for (int i = 0; i < 16; ++i) dp[i] = (i & 3) + 8 * (i >> 2) < lim ? dp[i] : 0.f;
          if (CAUSAL) bad |= has_nonfinite(ad, atK);
        }
        uint32_t pk[8];
#pragma unroll
        for (int i = 0; i < 16; i += 2) pk[i >> 1] = pack_bf16(dp[i], dp[i + 1]);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int dt = 0; dt < 2; ++dt) dq[dt] = mfma(ad.columns(dt, atK + 2048 * t), p_frag(pk, t), dq[dt]);
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };
  for (int key0 = 0; key0 < ke; key0 += 2 * kKV) {
    step(key0, std::integral_constant<int, 0>{});
    if (key0 + kKV < ke) step(key0 + kKV, std::integral_constant<int, 1>{});
  }
  ConstArgs* w = again();
  const bool far = wave_on && __ballot(nl != nl) != 0 && is_far(w->lse[(int64_t)(s.q0 + qi) * w->H + h]);
  if (wave_on && __ballot(bad != 0 || far) != 0) {
    for (int i = 0; i < 16; ++i) dq[0][i] = dq[1][i] = 0.f;
    float m = -INFINITY, l = 0.f;
    const bf16_t* K = w->k + (s.k0 * w->k_t + hk * w->k_h);
    const bf16_t* V = w->v + (s.k0 * w->v_t + hk * w->v_h);
    if (__ballot(far) != 0) {
#pragma clang loop unroll(disable)
      for (int j = 0; j < nk_last; ++j) {
        const float x = dot_row(K + j * w->k_t, qf, hh);
        if (j < nk) {
          const float m_new = fmaxf(m, x), alpha = m == m_new ? 1.f : __builtin_amdgcn_exp2f((m - m_new) * c);
          l = fmaf(l, alpha, x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((x - m_new) * c));
          m = m_new;
        }
      }
      l = log2f(l);
      if (far && r < R && kw == 0 && hh == 0) {
        const int64_t at = (int64_t)h * w->Tq + s.q0 + qi;
        w->far_m[at] = m;
        w->far_l[at] = l;
      }
    }
#pragma clang loop unroll(disable)
    for (int j = 32 * kw; j < nk_last; j += KW == 2 && (j & 31) == 31 ? 33 : 1) {
      const float x = dot_row(K + j * w->k_t, qf, hh), y = dot_row(V + j * w->v_t, df, hh);
      const float p = __builtin_amdgcn_exp2f(far ? fmaf(x - m, c, -l) : fmaf(x, c, nl));
      if (j < nk) add_row(dq, p * (y + nd[0]), K + j * w->k_t, hh);
    }
  }
  if constexpr (KW == 2) {
    float* x = reinterpret_cast<float*>(smem) + rw * 32 * 64 + lane;
    if (kw == 1) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[i * 64] = dq[0][i];
        x[(16 + i) * 64] = dq[1][i];
      }
    }
    __syncthreads();
    if (kw == 1) return;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      dq[0][i] += x[i * 64];
      dq[1][i] += x[(16 + i) * 64];
    }
  }
  if (r < R) store_acc(a.dq + (s.q0 + qi) * a.dq_t + h * a.dq_h, dq, a.scale, hh);
}

// dK, dV: 32 KW keys of one key head a workgroup, over the rows of its query heads one after the other (of one of them
// with a.nsplit = G: partial sums, joined by k_attnp_sum).  A key to a lane: S = Q K^T (which starts at -lse / scale) and
// dP = dO V^T (at -D) leave a key's column in one lane's registers, which then are the B operand of dV^T += dO^T P and
// dK^T += Q^T dS.  Tiles are of RT = 256 / KW rows: with KW 4 every wave has 32 keys and takes both 32-row blocks of a tile;
// with KW 2 waves 2, 3 hold the keys of waves 0, 1 again, a wave takes two of the four blocks and the sums are added at the
// end.  A wave's two blocks are independent: while one's exponentials are on the vector unit the other's products are on
// the matrix unit.  8 x 4096 tokens of 16 heads: 1090 us, 1009 TF over the four products (847 cycles a block, 512 of them
// on the matrix unit; the blocks interleaved and the addresses out of the loops took the whole backward pass from 1777 to
// 1693 us on one card; 1709 to 1755 on others).
template <bool CAUSAL, int KW>
__global__ __launch_bounds__(256, 2) void k_attnp_dkdv(const Args a) {
  constexpr int RT = 256 / KW, kRowBytes = RT * 128;
  // two buffers of Q tile, dO tile, RT nlse, RT ndelta
  constexpr int kBuf = 2 * kRowBytes + 8 * RT;
  __shared__ __attribute__((aligned(16))) uint8_t smem[2 * kBuf];
  const int lane = threadIdx.x & 63, hh = lane >> 5, lr = lane & 31;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kh = KW == 4 ? wid : wid & 1, qh = KW == 4 ? 0 : wid >> 1;
  const int hk = blockIdx.x % a.Hk;
  int rest = blockIdx.x / a.Hk;
  const int split = rest % a.nsplit;
  rest /= a.nsplit;
  int tile;
  Seq s;
  const int b = locate<true, false>(a, 1, 32 * KW, rest, lane, tile, s);
  if (b == a.B) {
    const int t0 = cu_at(a.cu_k, a.B, a.Tk);
    for (int e = threadIdx.x; a.nsplit == 1 && e < 32 * KW * 8; e += 256) {
      const int64_t t = t0 + tile * 32 * KW + (e >> 3);
      if (t >= a.Tk) break;
      *reinterpret_cast<uint4*>(a.dk + t * a.dk_t + hk * a.dk_h + (e & 7) * 8) = make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(a.dv + t * a.dv_t + hk * a.dv_h + (e & 7) * 8) = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  const int key0 = tile * 32 * KW;
  if (tile < 0 || key0 >= s.lk) return;
  const int kw = key0 + 32 * kh;                       // the wave's first key
  const int key = kw + lr, kc = min(key, s.lk - 1);
  // causal: key j is seen by the queries from j - (lk - lq) on
  const int off = s.lk - s.lq;
  const int i_first = CAUSAL ? max(0, key0 - off) : 0;
  const int g0 = a.nsplit == 1 ? 0 : split, g1 = a.nsplit == 1 ? a.G : split + 1;
  const bool any = i_first < s.lq;

  // a wave loads RT / 4 rows of Q and of dO, 8 an instruction
  constexpr int kOps = RT / 32;
  uint32_t offq[kOps], offd[kOps];
#pragma unroll
  for (int j = 0; j < kOps; ++j) {
    const int row = (wid * kOps + j) * 8 + (lane >> 3), ch = ((lane & 7) ^ swz(row)) * 8;
    offq[j] = (uint32_t)((row * a.q_t + ch) * 2);
    offd[j] = (uint32_t)((row * a.d_t + ch) * 2);
  }
  // and 64 of the tile's 2 RT statistics (waves 0, 1 of four with 64-row tiles)
  const bool stat_on = wid < RT / 32;
  const int stat_at = KW == 4 ? 0 : (wid & 1) * 64;
  auto q_of = [&](auto* w, int g) { return w->q + ((s.q0 + i_first) * w->q_t + (hk * w->G + g) * w->q_h); };
  auto d_of = [&](auto* w, int g) { return w->dout + ((s.q0 + i_first) * w->d_t + (hk * w->G + g) * w->d_h); };
  auto s_of = [&](auto* w, int g) {
    return ((KW == 4 ? wid : wid >> 1) ? w->ndelta : w->nlse) + (int64_t)(hk * w->G + g) * w->Tq + s.q0 + i_first + stat_at;
  };
  Src<RT> srcq(q_of(&a, g0), a.q_t), srcd(d_of(&a, g0), a.d_t);
  const float* stats = s_of(&a, g0);
  const uint32_t ldsb = __builtin_amdgcn_readfirstlane(lds_addr(smem));
  const uint32_t lds0 = ldsb + wid * kOps * 1024, ldss = ldsb + 2 * kRowBytes + wid * 256;
  int next_i = i_first, next_g = g0;                   // the tile that is loaded next
  auto stage = [&](int buf) {
    const auto rq = srcq.rsrc(s.lq - next_i), rd = srcd.rsrc(s.lq - next_i);
#pragma unroll
    for (int j = 0; j < kOps; ++j) dma16(rq, lds0 + buf * kBuf + j * 1024, offq[j]);
#pragma unroll
    for (int j = 0; j < kOps; ++j) dma16(rd, lds0 + buf * kBuf + kRowBytes + j * 1024, offd[j]);
    if (stat_on) {
      const int n = __builtin_amdgcn_readfirstlane(max(0, min(s.lq - next_i - stat_at, 64)));
      dma4(__builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(stats), 0, n * 4, 0x00020000), ldss + buf * kBuf, lane * 4);
    }
    next_i += RT;
    if (next_i < s.lq) {
      srcq.move();
      srcd.move();
      stats += RT;
    } else {                                           // the next query head
      next_i = i_first;
      ++next_g;
      ConstArgs* w = again();
      srcq.p = reinterpret_cast<const uint8_t*>(q_of(w, next_g));
      srcd.p = reinterpret_cast<const uint8_t*>(d_of(w, next_g));
      stats = s_of(w, next_g);
    }
  };
  if (any) stage(0);
  bf16x8 kf[4], vf[4];
  {
    const bf16_t* kr = a.k + (s.k0 + kc) * a.k_t + hk * a.k_h;
    const bf16_t* vr = a.v + (s.k0 + kc) * a.v_t + hk * a.v_h;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      kf[t] = *reinterpret_cast<const bf16x8*>(kr + 16 * t + 8 * hh);
      vf[t] = *reinterpret_cast<const bf16x8*>(vr + 16 * t + 8 * hh);
    }
  }
  __builtin_amdgcn_s_waitcnt(0xF70);
  __syncthreads();

  const float c = a.c;
  f32x16 dk[2], dv[2];
  for (int i = 0; i < 16; ++i) dk[0][i] = dk[1][i] = dv[0][i] = dv[1][i] = 0.f;

  int bad = 0, cur = 0;
  // the wave's blocks: rows ra and ra + kApart of a tile
  constexpr int kApart = KW == 2 ? 64 : 32;
  const int ra = 32 * qh;
  const Lanes ad0(ldsb + ra * 128, lane);
  const uint32_t stat0 = ldsb + 2 * kRowBytes + (ra + 4 * hh) * 4;
  // One tile, whose first query is i1.  EDGE: some of its queries may not see some of the workgroup's keys.  (Rows behind
  // the sequence are zero, with statistics of zero: they add nothing.)
  auto tile_step = [&](int i1, auto edge) {
    constexpr bool EDGE = decltype(edge)::value;
    constexpr uint32_t atQ = 0, atD = kRowBytes;
    if (next_g < g1) stage(cur ^ 1);
    const Lanes ad = ad0.behind(cur * kBuf);
    const uint32_t stat = stat0 + cur * kBuf;
    // What a block's products need is read a phase ahead of them: the rows of Q and dO, with -lse / scale and -D as the
    // accumulators' start values, then their transposes.
    struct Block {
      bf16x8 q[4], d[4];
      f32x16 st, dp;
    };
    auto read_rows = [&](int r, Block& x) {            // r: rows behind ra
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        x.q[t] = ad.rows(t, atQ + r * 128);
        x.d[t] = ad.rows(t, atD + r * 128);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        typedef float f32x4 __attribute__((ext_vector_type(4)));
        const f32x4 u = *(const __attribute__((address_space(3))) f32x4*)(stat + (r + 8 * q) * 4);
        const f32x4 v = *(const __attribute__((address_space(3))) f32x4*)(stat + (RT + r + 8 * q) * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) x.st[4 * q + i] = u[i], x.dp[4 * q + i] = v[i];
      }
    };
    auto read_columns = [&](int r, Block& x) {         // in place of the rows
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int dt = 0; dt < 2; ++dt) {
          x.d[2 * t + dt] = ad.columns(dt, atD + r * 128 + 2048 * t);
          x.q[2 * t + dt] = ad.columns(dt, atQ + r * 128 + 2048 * t);
        }
    };
    auto scores = [&](int r, Block& x) {               // S - lse / scale and dP - D
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        x.st = mfma(x.q[t], kf[t], x.st);
        x.dp = mfma(x.d[t], vf[t], x.dp);
      }
      if (EDGE) {
        const int lim = whole(key - off - i1 - ra - r - 4 * hh);  // the rows below this do not see the lane's key
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const bool on = (i & 3) + 8 * (i >> 2) >= lim;
          x.st[i] = on ? x.st[i] : -INFINITY;
          x.dp[i] = on ? x.dp[i] : 0.f;
        }
      }
    };
    auto probs = [&](Block& x) {                       // P and dS in place of them
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x.st[i] = __builtin_amdgcn_exp2f(x.st[i] * c);
        x.dp[i] *= x.st[i];
      }
    };
    auto sums = [&](const Block& x) {
      uint32_t pk[8], dsk[8];
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        pk[i >> 1] = pack_bf16(x.st[i], x.st[i + 1]);
        dsk[i >> 1] = pack_bf16(x.dp[i], x.dp[i + 1]);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int dt = 0; dt < 2; ++dt) {
          dv[dt] = mfma(x.d[2 * t + dt], p_frag(pk, t), dv[dt]);
          dk[dt] = mfma(x.q[2 * t + dt], p_frag(dsk, t), dk[dt]);
        }
    };
    // a phase: `reads` LDS reads, then eight products between the other block's exponentials
    auto mix = [](auto reads) {
      __builtin_amdgcn_sched_group_barrier(0x100, decltype(reads)::value, 0);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x400, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
      }
    };
    if constexpr (EDGE) {
      // one block after the other, where some query sees some key of the wave
#pragma unroll
      for (int r = 0; r <= kApart; r += kApart) {
        if (i1 + ra + r + 31 < kw - off) continue;
        Block x;
        read_rows(r, x);
        scores(r, x);
        __builtin_amdgcn_sched_barrier(0);
        bad |= has_nonfinite(ad, atQ + r * 128) | has_nonfinite(ad, atD + r * 128);
        __builtin_amdgcn_sched_barrier(0);
        read_columns(r, x);
        probs(x);
        sums(x);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      Block x, y;
      read_rows(0, x);
      __builtin_amdgcn_sched_barrier(0);
      read_rows(kApart, y);
      scores(0, x);
      __builtin_amdgcn_sched_barrier(0);
      read_columns(0, x);
      scores(kApart, y);
      probs(x);
      mix(std::integral_constant<int, 16>{});
      __builtin_amdgcn_sched_barrier(0);
      read_columns(kApart, y);
      sums(x);
      probs(y);
      mix(std::integral_constant<int, 16>{});
      __builtin_amdgcn_sched_barrier(0);
      sums(y);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    cur ^= 1;
  };
  const int i_edge = CAUSAL ? min(s.lq, key0 + 32 * KW - 1 - off) : i_first;   // from here on all keys are seen
  for (int g = g0; any && g < g1; ++g) {
    int i1 = i_first;
    if (CAUSAL)
      for (; i1 < i_edge; i1 += RT) tile_step(i1, std::true_type{});
    for (; i1 < s.lq; i1 += RT) tile_step(i1, std::false_type{});
  }
  const bool nan = dv[0][0] != dv[0][0];
  if (__ballot(nan) != 0) {
    // Done again: keys that a far row has made NaN, and those of an infinity, which the rows of zeros behind the last query have
    // (not those that a NaN has spoilt: it would again)
    bool inf = false, real = true;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = (float)kf[t][j];
        inf |= fabsf(x) == INFINITY;
        real &= x == x;
      }
    inf |= __shfl_xor((int)inf, 32) != 0;
    real &= __shfl_xor((int)real, 32) != 0;
    bad |= nan && inf && real;
    ConstArgs* w = again();
    for (int g = g0; g < g1; ++g) {
      const uint32_t* nl = reinterpret_cast<const uint32_t*>(w->nlse + (int64_t)(hk * w->G + g) * w->Tq + s.q0);
      for (int i = i_first + lane; i < s.lq; i += 64) bad |= nl[i] == kFarMark;
    }
  }
  if (__ballot(bad != 0) != 0) {
    for (int i = 0; i < 16; ++i) dk[0][i] = dk[1][i] = dv[0][i] = dv[1][i] = 0.f;
    ConstArgs* w = again();
    for (int g = g0; g < g1; ++g) {
      const int h = hk * w->G + g;
#pragma clang loop unroll(disable)
      for (int i = i_first; i < s.lq; ++i) {
        if (KW == 2 && ((i - i_first) >> 5 & 1) != qh) continue;      // the other waves' rows
        const bf16_t* qr = w->q + (s.q0 + i) * w->q_t + h * w->q_h;
        const bf16_t* dr = w->dout + (s.q0 + i) * w->d_t + h * w->d_h;
        const float x = dot_row(qr, kf, hh), y = dot_row(dr, vf, hh);
        if (!CAUSAL || i >= key - off) {
          const int64_t st = (int64_t)h * w->Tq + s.q0 + i;
          const float nl = w->nlse[st];
          const float p = __builtin_amdgcn_exp2f(__float_as_uint(nl) == kFarMark ? fmaf(x - w->far_m[st], c, -w->far_l[st]) : (x + nl) * c);
          add_row(dv, p, dr, hh);
          add_row(dk, p * (y + w->ndelta[st]), qr, hh);
        }
      }
    }
  }
  if constexpr (KW == 2) {
    // the two row halves' sums: 64 floats x 64 lanes of waves 2, 3 through LDS (32 KiB, the buffers' own)
    float* x = reinterpret_cast<float*>(smem) + kh * 64 * 64 + lane;
    if (qh == 1) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[i * 64] = dk[0][i];
        x[(16 + i) * 64] = dk[1][i];
        x[(32 + i) * 64] = dv[0][i];
        x[(48 + i) * 64] = dv[1][i];
      }
    }
    __syncthreads();
    if (qh == 1) return;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      dk[0][i] += x[i * 64];
      dk[1][i] += x[(16 + i) * 64];
      dv[0][i] += x[(32 + i) * 64];
      dv[1][i] += x[(48 + i) * 64];
    }
  }
  if (key >= s.lk) return;
  if (a.nsplit == 1) {
    store_acc(a.dk + (s.k0 + key) * a.dk_t + hk * a.dk_h, dk, a.scale, hh);
    store_acc(a.dv + (s.k0 + key) * a.dv_t + hk * a.dv_h, dv, 1.0f, hh);
    return;
  }
  float* pk = a.part_o + (((int64_t)split * a.Tk + s.k0 + key) * a.Hk + hk) * 128;       // 64 of dK, 64 of dV
#pragma unroll
  for (int dt = 0; dt < 2; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * dt + 8 * g + 4 * hh;
      *reinterpret_cast<float4*>(pk + d) = make_float4(dk[dt][4 * g], dk[dt][4 * g + 1], dk[dt][4 * g + 2], dk[dt][4 * g + 3]);
      *reinterpret_cast<float4*>(pk + 64 + d) = make_float4(dv[dt][4 * g], dv[dt][4 * g + 1], dv[dt][4 * g + 2], dv[dt][4 * g + 3]);
    }
}

// The query heads' partial sums of dK and dV added, in their order: 32 lanes a key row, four values each.  Bound by reading
// them: 60 MB (7300 tokens, 16 heads) 12 us.
__global__ __launch_bounds__(256) void k_attnp_sum(const Args a) {
  const int64_t n = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), rows = (int64_t)a.Tk * a.Hk;
  if (n >= rows) return;
  const int64_t t = n / a.Hk;
  const int hk = (int)(n - t * a.Hk), e = threadIdx.x & 31;
  const bool tail = t >= cu_at(a.cu_k, a.B, a.Tk);
  if (tail && !a.zero_tail) return;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int g = 0; !tail && g < a.nsplit; ++g) {
    const float4 x = *reinterpret_cast<const float4*>(a.part_o + (g * rows + n) * 128 + 4 * e);
    v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
  }
  const float f = e < 16 ? a.scale : 1.0f;
  bf16_t* out = e < 16 ? a.dk + t * a.dk_t + hk * a.dk_h + 4 * e : a.dv + t * a.dv_t + hk * a.dv_h + 4 * (e - 16);
  *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16(v.x * f, v.y * f), pack_bf16(v.z * f, v.w * f));
}

// ------------------------------------------------------------------ host side
inline int64_t row_tiles(const i2pc_attn_packed_desc& d, int rows) {
  return (int64_t)d.total_q * (d.heads / d.kv_heads) / rows + d.batch + (d.zero_tail ? 1 : 0);
}
// Waves over the keys of a tile (the kernels' KW): two while there are few 128-row workgroups for the chip's 1024 places,
// or not many of the different lengths that a causal mask gives them.  Measured forward, KW 1 / 2: 7200 tokens of six
// heads (380 workgroups) 38 / 31 us, 9400 of twelve heads (1010) 62 / 65 us; causal, 16 heads over 4, 7300 tokens (940)
// 76 / 65 us, 8700 tokens (1110) 112 / 108 us.
inline int key_waves(const i2pc_attn_packed_desc& d) {
  return row_tiles(d, kRows) * d.kv_heads < (d.causal ? 1200 : 700) ? 2 : 1;
}

// Sequences of 32 packed rows or fewer on average take the kernel for few rows.  (Right for any lengths: the rule only
// decides the speed.)
inline bool few_rows(const i2pc_attn_packed_desc& d) {
  return (int64_t)d.total_q * (d.heads / d.kv_heads) <= (int64_t)d.batch * kFew;
}

// Shares of the keys: one where the row tiles fill the chip, else so many that they do, of 256 keys at least on average
// (few rows: 2048; an upper bound, a share may be empty).  Each share of few rows is a partial row to join, and the join reads
// them eight at a time.  Measured with shares of 2048 / 1024 / 512 keys at least, one new token, us (12.5 is the host's part):
// one sequence of 131071 keys, 16 heads over 2: 17.8 / 19.6 / 21.7; four of 8192, 16 over 8: 19.9 / 20.2 / 23.0; but one of
// 32768, 16 over 2: 17.1 / 12.4 / 12.6, and one of 8192, 16 over 8: 14.2 / 12.7 / 12.8.  Where the tiles fill the chip (64
// sequences) the bound is not reached.
inline int splits(const i2pc_attn_packed_desc& d) {
  if (d.total_k == 0) return 1;
  const bool few = few_rows(d);
  const int64_t tiles = row_tiles(d, few ? kFew : kRows / 2) * d.kv_heads;
  const int64_t most = few ? (d.total_k + 2047) / 2048 : (d.total_k + 255) / 256;
  const int64_t want = few ? 2048 / tiles : key_waves(d) == 1 || tiles >= 512 ? 1 : 1024 / tiles;
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, most, 512}));
}

// The dK / dV call: keys of a workgroup / 32, and whether each query head of a group has workgroups of its own: where
// 128-key tiles alone do not fill the chip's 512 places.  The partial sums are 1 KiB a key and query head, written and read, so
// short sequences lose by them at any number of tiles and long ones gain a little beyond 512 too; between them 512 costs least.
// Measured backward, split / not, us (16 heads over 4, causal): tokens 4097, 2050, 1023, 130, 1 (248 tiles) 201 / 250, 2 x 4096
// (264) 277 / 330, 3 x 4096 (396) 411 / 423, 12 x 1024 (432) 161 / 151, 7 x 2048 (476) 279 / 280; above 512, where it is not
// split: 26 x 512 (520) 130 / 110, 4 x 4096 (528) 518 / 530, 8 x 2048 (544) 316 / 325, 16 x 1024 (576) 211 / 195, 8 x 4096
// (1056) 1015 / 1034, 64 x 512 (1280) 307 / 226.
struct KeySplit {
  int kw, heads;
};
inline int64_t key_tiles(const i2pc_attn_packed_desc& d, int keys) {
  return (int64_t)d.total_k / keys + d.batch + (d.zero_tail ? 1 : 0);
}
inline KeySplit key_split(const i2pc_attn_packed_desc& d) {
  const int G = d.heads / d.kv_heads;
  const int64_t wide = key_tiles(d, 128) * d.kv_heads;
  const int heads = wide < 512 ? G : 1;
  return {wide * heads < 768 ? 2 : 4, heads};
}

// Rows apart (the range checks of the tiles' loads go by the row stride); where they are written heads apart too, and the
// heads of a row all before the next row or the rows of a head all before the next head.  The stride of a single row or head is
// not looked at.
inline bool rows_ok(const void* p, int64_t t, int64_t h, int rows, int heads, bool written) {
  if (rows == 0) return true;
  if (!p || reinterpret_cast<uintptr_t>(p) % 16) return false;
  if (rows > 1 && (t % 8 || t < 64 || t >= (int64_t)1 << 23)) return false;
  if (heads > 1 && (h % 8 || h < 0 || h >= (int64_t)1 << 40)) return false;
  if (!written || heads == 1) return true;
  return h >= 64 && (rows == 1 || t >= (heads - 1) * h + 64 || h >= (rows - 1) * t + 64);
}

int check(const char* what, const i2pc_attn_packed_desc* d) {
  I2PC_REQUIRE(d, "NULL descriptor");
  I2PC_REQUIRE(d->batch >= 0 && d->total_q >= 0 && d->total_k >= 0 && d->heads > 0 && d->kv_heads > 0 &&
                   d->heads % d->kv_heads == 0,
               "%s: batch=%d total_q=%d total_k=%d heads=%d kv_heads=%d (heads a multiple of kv_heads)", what, d->batch,
               d->total_q, d->total_k, d->heads, d->kv_heads);
  if (d->head_dim != 64) return set_error(I2PC_EUNSUPPORTED, "%s: head_dim=%d, the kernels are of 64", what, d->head_dim);
  // grids of 256-thread workgroups hold 2^24 of them
  const int64_t most = (int64_t)1 << 24;
  if ((int64_t)d->total_q * d->heads >= most * 32 || ((int64_t)d->total_q / kRows + 2 * (int64_t)d->batch + 2) * d->heads >= most ||
      ((int64_t)d->total_k / 64 + (int64_t)d->batch + 1) * d->kv_heads >= most)
    return set_error(I2PC_EUNSUPPORTED, "%s: total_q * heads must stay below 2^29, (total_k / 64 + batch) * kv_heads below 2^24", what);
  // lse / scale has to stay finite
  I2PC_REQUIRE(d->scale >= 0x1p-64f && d->scale <= 0x1p64f, "%s: scale=%g must lie within 2^-64 and 2^64", what, (double)d->scale);
  I2PC_REQUIRE(d->batch == 0 || (d->cu_q && d->cu_k), "%s: NULL cu_q or cu_k", what);
  I2PC_REQUIRE(rows_ok(d->q, d->q_t, d->q_h, d->total_q, d->heads, false) &&
                   rows_ok(d->out, d->o_t, d->o_h, d->total_q, d->heads, true) &&
                   rows_ok(d->k, d->k_t, d->k_h, d->total_k, d->kv_heads, false) &&
                   rows_ok(d->v, d->v_t, d->v_h, d->total_k, d->kv_heads, false) &&
                   (d->total_q == 0 || d->lse),
               "%s: q, k, v, out must be 16-byte aligned with strides that are multiples of 8 "
               "(row strides from 64 to 2^23), out without rows that overlap", what);
  return I2PC_OK;
}

// The row stride of an operand of one row is never taken, but the kernels take the end of a tile's rows from it: rows behind the
// first have to lie behind its 64 values.
inline int64_t pitch(int64_t t, int rows) { return rows > 1 ? t : 64; }

Args args_of(const i2pc_attn_packed_desc& d) {
  Args a = {};
  a.q = static_cast<const bf16_t*>(d.q), a.k = static_cast<const bf16_t*>(d.k), a.v = static_cast<const bf16_t*>(d.v);
  a.q_t = pitch(d.q_t, d.total_q), a.q_h = d.q_h, a.k_t = pitch(d.k_t, d.total_k), a.k_h = d.k_h;
  a.v_t = pitch(d.v_t, d.total_k), a.v_h = d.v_h;
  a.out = static_cast<bf16_t*>(d.out), a.o_t = pitch(d.o_t, d.total_q), a.o_h = d.o_h, a.lse = d.lse;
  a.cu_q = d.cu_q, a.cu_k = d.cu_k, a.k_lens = d.k_lens;
  a.B = d.batch, a.Tq = d.total_q, a.Tk = d.total_k, a.H = d.heads, a.Hk = d.kv_heads, a.G = d.heads / d.kv_heads;
  a.zero_tail = d.zero_tail != 0;
  a.scale = d.scale;
  a.c = d.scale * 1.4426950408889634f;
  a.nsplit = 1;
  return a;
}

}  // namespace attnp
}  // namespace i2pc

using namespace i2pc;

extern "C" size_t i2pc_attention_packed_workspace_bytes(const i2pc_attn_packed_desc* d) {
  if (attnp::check("attention_packed", d) != I2PC_OK) return 0;
  const int n = attnp::splits(*d);
  return n == 1 ? 0 : (size_t)n * d->heads * d->total_q * 66 * sizeof(float);
}

extern "C" int i2pc_attention_packed(const i2pc_attn_packed_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (const int rc = attnp::check("attention_packed", d)) return rc;
  if (d->total_q == 0 || (d->batch == 0 && !d->zero_tail)) return I2PC_OK;
  I2PC_REQUIRE(d->batch > 0, "attention_packed: zero_tail without a sequence");
  const size_t need = i2pc_attention_packed_workspace_bytes(d);
  if (need > workspace_bytes || (need && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16)))
    return set_error(I2PC_EWORKSPACE, "attention_packed: workspace of %zu bytes, needs %zu (16-byte aligned)", workspace_bytes, need);
  attnp::Args a = attnp::args_of(*d);
  hipStream_t s = as_stream(stream);
  a.nsplit = attnp::splits(*d);
  const bool few = attnp::few_rows(*d);
  const int kw = attnp::key_waves(*d);
  const dim3 block(256), grid((uint32_t)(attnp::row_tiles(*d, few ? attnp::kFew : attnp::kRows / kw) * a.Hk * a.nsplit));
  if (a.nsplit > 1) {
    a.part_o = static_cast<float*>(workspace);
    a.part_l = reinterpret_cast<float2*>(a.part_o + (size_t)a.nsplit * a.H * a.Tq * 64);
  }
  if (few && d->causal) hipLaunchKernelGGL(attnp::k_attnp_few<true>, grid, block, 0, s, a);
  else if (few) hipLaunchKernelGGL(attnp::k_attnp_few<false>, grid, block, 0, s, a);
  else if (kw == 1 && d->causal) hipLaunchKernelGGL((attnp::k_attnp_fwd<true, false, 1>), grid, block, 0, s, a);
  else if (kw == 1) hipLaunchKernelGGL((attnp::k_attnp_fwd<false, false, 1>), grid, block, 0, s, a);
  else if (a.nsplit == 1 && d->causal) hipLaunchKernelGGL((attnp::k_attnp_fwd<true, false, 2>), grid, block, 0, s, a);
  else if (a.nsplit == 1) hipLaunchKernelGGL((attnp::k_attnp_fwd<false, false, 2>), grid, block, 0, s, a);
  else if (d->causal) hipLaunchKernelGGL((attnp::k_attnp_fwd<true, true, 2>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((attnp::k_attnp_fwd<false, true, 2>), grid, block, 0, s, a);
  const int64_t rows = (int64_t)a.Tq * a.H;
  if (a.nsplit > 32)
    hipLaunchKernelGGL(attnp::k_attnp_join<16>, dim3((uint32_t)rows), dim3(1024), 0, s, a);
  else if (a.nsplit > 1)
    hipLaunchKernelGGL(attnp::k_attnp_join<1>, dim3((uint32_t)((rows + 3) / 4)), block, 0, s, a);
  return check_launch("attention_packed");
}

static int check_grad(const i2pc_attn_packed_grad_desc* g) {
  using attnp::rows_ok;
  I2PC_REQUIRE(g, "NULL descriptor");
  const i2pc_attn_packed_desc& d = g->f;
  if (const int rc = attnp::check("attention_packed_backward", &d)) return rc;
  I2PC_REQUIRE(!d.k_lens, "attention_packed_backward: k_lens is of the forward call only");
  I2PC_REQUIRE(rows_ok(g->dout, g->d_t, g->d_h, d.total_q, d.heads, false) &&
                   rows_ok(g->dq, g->dq_t, g->dq_h, d.total_q, d.heads, true) &&
                   rows_ok(g->dk, g->dk_t, g->dk_h, d.total_k, d.kv_heads, true) &&
                   rows_ok(g->dv, g->dv_t, g->dv_h, d.total_k, d.kv_heads, true),
               "attention_packed_backward: dout, dq, dk, dv must be 16-byte aligned with strides that are multiples of 8 "
               "(row strides from 64 to 2^23), dq, dk, dv without rows that overlap");
  return I2PC_OK;
}

extern "C" size_t i2pc_attention_packed_backward_workspace_bytes(const i2pc_attn_packed_grad_desc* g) {
  if (check_grad(g) != I2PC_OK) return 0;
  // four statistics of every row, and the query heads' partial sums where they are split
  const attnp::KeySplit k = attnp::key_split(g->f);
  return (size_t)4 * g->f.total_q * g->f.heads * sizeof(float) +
         (k.heads == 1 ? 0 : (size_t)k.heads * g->f.total_k * g->f.kv_heads * 128 * sizeof(float));
}

extern "C" int i2pc_attention_packed_backward(const i2pc_attn_packed_grad_desc* g, void* workspace, size_t workspace_bytes,
                                              void* stream) {
  clear_error();
  if (const int rc = check_grad(g)) return rc;
  const i2pc_attn_packed_desc& d = g->f;
  if (d.batch == 0) {
    I2PC_REQUIRE(!d.zero_tail, "attention_packed_backward: zero_tail without a sequence");
    return I2PC_OK;
  }
  const size_t need = i2pc_attention_packed_backward_workspace_bytes(g);
  if (need > workspace_bytes || (need && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16)))
    return set_error(I2PC_EWORKSPACE, "attention_packed_backward: workspace of %zu bytes, needs %zu (16-byte aligned)",
                     workspace_bytes, need);
  attnp::Args a = attnp::args_of(d);
  a.dout = static_cast<const attn::bf16_t*>(g->dout), a.d_t = attnp::pitch(g->d_t, d.total_q), a.d_h = g->d_h;
  a.dq = static_cast<attn::bf16_t*>(g->dq), a.dk = static_cast<attn::bf16_t*>(g->dk), a.dv = static_cast<attn::bf16_t*>(g->dv);
  a.dq_t = attnp::pitch(g->dq_t, d.total_q), a.dq_h = g->dq_h;
  a.dk_t = attnp::pitch(g->dk_t, d.total_k), a.dk_h = g->dk_h;
  a.dv_t = attnp::pitch(g->dv_t, d.total_k), a.dv_h = g->dv_h;
  a.nlse = static_cast<float*>(workspace);
  a.ndelta = a.nlse + (size_t)a.Tq * a.H;
  a.far_m = a.ndelta + (size_t)a.Tq * a.H;
  a.far_l = a.far_m + (size_t)a.Tq * a.H;
  hipStream_t s = as_stream(stream);
  const dim3 block(256);
  if (a.Tq > 0) {
    const int kw = attnp::key_waves(d);
    const dim3 grid((uint32_t)(attnp::row_tiles(d, attnp::kRows / kw) * a.Hk));
    if (kw == 1 && d.causal) hipLaunchKernelGGL((attnp::k_attnp_dq<true, 1>), grid, block, 0, s, a);
    else if (kw == 1) hipLaunchKernelGGL((attnp::k_attnp_dq<false, 1>), grid, block, 0, s, a);
    else if (d.causal) hipLaunchKernelGGL((attnp::k_attnp_dq<true, 2>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((attnp::k_attnp_dq<false, 2>), grid, block, 0, s, a);
  }
  if (a.Tk > 0) {
    const attnp::KeySplit k = attnp::key_split(d);
    a.nsplit = k.heads;
    a.part_o = a.nlse + (size_t)4 * a.Tq * a.H;
    const dim3 grid((uint32_t)(attnp::key_tiles(d, 32 * k.kw) * a.Hk * a.nsplit));
    if (k.kw == 4 && d.causal) hipLaunchKernelGGL((attnp::k_attnp_dkdv<true, 4>), grid, block, 0, s, a);
    else if (k.kw == 4) hipLaunchKernelGGL((attnp::k_attnp_dkdv<false, 4>), grid, block, 0, s, a);
    else if (d.causal) hipLaunchKernelGGL((attnp::k_attnp_dkdv<true, 2>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((attnp::k_attnp_dkdv<false, 2>), grid, block, 0, s, a);
    if (a.nsplit > 1)
      hipLaunchKernelGGL(attnp::k_attnp_sum, dim3((uint32_t)(((int64_t)a.Tk * a.Hk + 7) / 8)), block, 0, s, a);
  }
  return check_launch("attention_packed_backward");
}
