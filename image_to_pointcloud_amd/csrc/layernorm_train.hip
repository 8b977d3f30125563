// LayerNorm's training step (gfx950): forward with its row statistics, backward with the gradients of
// the input, the scale and the offset.
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) r
//   y  = h gamma + beta
//   dx = r (dy gamma - mean(dy gamma) - h mean(dy gamma h)) [+ add]
//   dgamma = sum over rows of dy h,   dbeta = sum over rows of dy
//
// Both directions are bound by HBM: x, dy, add read once, y / dx written once, the row in registers
// between its reductions (two-pass variance in fp32).  The column sums of the backward pass ride on the
// same read: a wave keeps the partial sums of its columns in registers over all the rows it takes, a
// workgroup adds its waves' through LDS and writes one partial row, and k_lnt_cols adds the partial rows
// -- fixed assignment and order, so the result does not change from run to run (no atomics).
// Measured, calls one after the other: 18464 x 1024 fp32 forward 24.6 us (4.6 TB/s), backward with add 54 us (4.9 TB/s; a copy
// of 2 GiB reaches 4.9), the partial rows' sum 5 us of it; 4099 x 1111 bf16 7.2 and 17.1 us (its rows start at odd
// addresses); 5 x 384: the launches.
#include "common.h"

#include <algorithm>

namespace i2pc {
namespace lnt {

typedef uint16_t bf16_t;

constexpr int kThreads = 512;                 // 8 waves
constexpr int kMaxDim = 8192;
constexpr int kCUs = 256;

// The sum over a wave, in every lane: four DPP additions within 16 lanes, two swaps of rows -- all on the vector unit, where
// shuffles through LDS would add their latency six times to every row sum.
template <int CTRL>
__device__ __forceinline__ float plus_dpp(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float wave_sum(float x) {
  x = plus_dpp<0xB1>(x);                           // quad_perm 1, 0, 3, 2
  x = plus_dpp<0x4E>(x);                           // quad_perm 2, 3, 0, 1
  x = plus_dpp<0x141>(x);                          // row_half_mirror
  x = plus_dpp<0x140>(x);                          // row_mirror
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(h[0]) + __uint_as_float(h[1]);
}

// E consecutive elements as floats, from / to an address with the element's own alignment only (rows of
// an odd pitch): global memory takes such vector accesses, and one 16-byte request stays one request.
template <typename T, int E>
struct Vec;
template <int E>
struct Vec<float, E> {
  static __device__ __forceinline__ void load(const float* p, float (&v)[E]) { __builtin_memcpy(v, p, E * 4); }
  static __device__ __forceinline__ void store(float* p, const float (&v)[E]) { __builtin_memcpy(p, v, E * 4); }
};
template <int E>
struct Vec<bf16_t, E> {
  static __device__ __forceinline__ void load(const bf16_t* p, float (&v)[E]) {
    bf16_t u[E];
    __builtin_memcpy(u, p, E * 2);
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] = __uint_as_float((uint32_t)u[j] << 16);
  }
  static __device__ __forceinline__ void store(bf16_t* p, const float (&v)[E]) {
    if constexpr (E == 1) {
      const __bf16 b = (__bf16)v[0];
      __builtin_memcpy(p, &b, 2);
    } else {
      uint32_t u[E / 2];
#pragma unroll
      for (int j = 0; j < E / 2; ++j) u[j] = pk2bf(v[2 * j], v[2 * j + 1]);
      __builtin_memcpy(p, u, E * 2);
    }
  }
};

// E bf16 values as they are in memory, widened where they are used: half the registers of their floats.
template <int E>
struct Packed {
  uint32_t w[(E + 1) / 2];
  __device__ __forceinline__ void load(const bf16_t* p) {
    if constexpr (E == 1) w[0] = *p;
    else __builtin_memcpy(w, p, E * 2);
  }
  // to be widened anew: the floats are not kept from one use to the next
  __device__ __forceinline__ void renew() {
#pragma unroll
    for (int j = 0; j < (E + 1) / 2; ++j) asm volatile("" : "+v"(w[j]));
  }
  __device__ __forceinline__ float operator[](int j) const {
    return __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
  }
};

// E values of T as they are in memory
template <int E>
struct Floats {
  float v[E];
  __device__ __forceinline__ void load(const float* p) { __builtin_memcpy(v, p, E * 4); }
  __device__ __forceinline__ float operator[](int j) const { return v[j]; }
};
template <typename T, int E>
struct Raw {
  typedef Packed<E> type;
};
template <int E>
struct Raw<float, E> {
  typedef Floats<E> type;
};

// A row's columns over WPR waves: chunk i of a lane starts at column (i * 64 * WPR + wave * 64 + lane) * E.
// The last chunk of a row whose width is no multiple of E starts at dim - E instead and repeats columns of
// the chunk before it: every load is a whole vector, and `live` keeps the repeated columns out of the row
// sums.  The forward pass stores them twice with the same value.
template <int E, int V, int WPR>
struct Cols {
  int col[V];
  uint32_t first[V];      // elements below this index repeat another chunk's (E: the whole chunk is off the row)
  __device__ __forceinline__ Cols(int lane, int sub, int dim) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int at = ((i * WPR + sub) * 64 + lane) * E;
      col[i] = min(at, dim - E);
      first[i] = (uint32_t)min(at - col[i], E);
    }
  }
  __device__ __forceinline__ bool live(int i, int j) const { return (uint32_t)j >= first[i]; }
};

// Sums over the row's WPR waves, in every lane of them.  The waves' parts meet in LDS, in one of two slots in turn: a wave
// that writes a slot again has passed the other slot's barrier, which no wave reaches before it has read the first.
template <int WPR>
struct RowSum {
  float2 (*slot)[8];
  int wave, turn;
  __device__ __forceinline__ float2 operator()(float a, float b) {
    a = wave_sum(a);
    b = wave_sum(b);
    if constexpr (WPR > 1) {
      if ((threadIdx.x & 63) == 0) slot[turn][wave] = make_float2(a, b);
      __syncthreads();
      const int w0 = wave / WPR * WPR;
      a = b = 0.f;
#pragma unroll
      for (int w = 0; w < WPR; ++w) {
        const float2 x = slot[turn][w0 + w];
        a += x.x;
        b += x.y;
      }
      turn ^= 1;
    }
    return make_float2(a, b);
  }
};

// One row per WPR waves of a workgroup of four waves (eight for the widest rows).
template <typename T, int E, int V, int WPR>
__global__ __launch_bounds__(WPR == 8 ? 512 : 256) void k_lnt_fwd(const T* __restrict__ x, int64_t ldx, const float* __restrict__ gamma,
                                                 const float* __restrict__ beta, float eps, int rows, int dim,
                                                 bf16_t* __restrict__ y, int64_t ldy, float2* __restrict__ stats) {
  __shared__ float2 red[2][8];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);   // scalar row addresses
  const Cols<E, V, WPR> c(lane, wave % WPR, dim);
  RowSum<WPR> row_sum{red, wave, 0};
  constexpr int R = WPR == 1 ? 4 : 1;              // WPR > 1: one row a workgroup, all its waves or none
  for (int64_t row = (int64_t)blockIdx.x * R + (WPR == 1 ? wave : 0); row < rows; row += (int64_t)gridDim.x * R) {
    const T* xr = x + row * ldx;
    float v[V][E];
#pragma unroll
    for (int i = 0; i < V; ++i) Vec<T, E>::load(xr + c.col[i], v[i]);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < E; ++j) s += c.live(i, j) ? v[i][j] : 0.f;
    const float mean = row_sum(s, 0.f).x / (float)dim;
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < E; ++j) {
        v[i][j] -= mean;
        q += c.live(i, j) ? v[i][j] * v[i][j] : 0.f;
      }
    const float rstd = 1.0f / sqrtf(row_sum(q, 0.f).x / (float)dim + eps);
    if (lane == 0 && wave % WPR == 0) stats[row] = make_float2(mean, rstd);
    bf16_t* yr = y + row * ldy;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float g[E], b[E];
      Vec<float, E>::load(gamma + c.col[i], g);
      Vec<float, E>::load(beta + c.col[i], b);
#pragma unroll
      for (int j = 0; j < E; ++j) v[i][j] = v[i][j] * rstd * g[j] + b[j];
      if (c.first[i] < (uint32_t)E) Vec<bf16_t, E>::store(yr + c.col[i], v[i]);
    }
  }
}

// Rows blockIdx.x * R + k * gridDim.x * R for the R = 8 / WPR rows a workgroup takes at a time.  Partial row p of the
// column sums goes to dgamma + p * 2 * dim and dbeta + p * 2 * dim: with one partial row, the outputs themselves.
template <typename T, int E, int V, int WPR>
__global__ __launch_bounds__(kThreads, E * V <= 8 ? 4 : 2) void k_lnt_bwd(const bf16_t* __restrict__ dy, int64_t lddy, const T* __restrict__ x,
                                                      int64_t ldx, const float2* __restrict__ stats,
                                                      const float* __restrict__ gamma, const T* add, int64_t lda, int rows,
                                                      int dim, T* dx, int64_t lddx, float* __restrict__ dgamma,
                                                      float* __restrict__ dbeta) {
  __shared__ float2 red[2][8];
  extern __shared__ float sums[];                  // [2][dim] (R > 1)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);   // scalar row addresses
  constexpr int R = 8 / WPR;
  const Cols<E, V, WPR> c(lane, wave % WPR, dim);
  RowSum<WPR> row_sum{red, wave, 0};
  float g[V][E], dg[V][E], db[V][E];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    Vec<float, E>::load(gamma + c.col[i], g[i]);
#pragma unroll
    for (int j = 0; j < E; ++j) dg[i][j] = db[i][j] = 0.f;
  }
  const float inv = 1.0f / (float)dim;
  // A row as it is read.  AHEAD: the next row's loads go out before this row's sums (where the registers allow it)
  struct Row {
    typename Raw<T, E>::type x[V], a[V];
    Packed<E> dy[V];
    float2 st;
  };
  constexpr bool AHEAD = E * V <= 8;
  auto load = [&](int64_t row, Row& w) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      w.x[i].load(x + row * ldx + c.col[i]);
      w.dy[i].load(dy + row * lddy + c.col[i]);
    }
    if (add) {
#pragma unroll
      for (int i = 0; i < V; ++i) w.a[i].load(add + row * lda + c.col[i]);
    }
    w.st = stats[row];
  };
  // WPR > 1 meets barriers inside: every wave runs the same number of rounds
  const int64_t step = (int64_t)gridDim.x * R;
  Row next;
  const int64_t row0 = (int64_t)blockIdx.x * R, mine = row0 + wave / WPR;
  if (AHEAD && row0 < rows) load(min(mine, (int64_t)rows - 1), next);
  for (int64_t at = row0; at < rows; at += step) {
    const int64_t row = at + wave / WPR;
    const bool on = row < rows;
    if (WPR == 1 && !on) break;
    Row w;
    if (AHEAD) {
      w = next;
      if (at + step < rows) load(min(row + step, (int64_t)rows - 1), next);
    } else {
      load(on ? row : (int64_t)rows - 1, w);
    }
    const float2 st = w.st;
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float h = (w.x[i][j] - st.x) * st.y, d = w.dy[i][j], gd = d * g[i][j];
        if constexpr (sizeof(T) == 4) w.x[i].v[j] = h;
        a += c.live(i, j) ? gd : 0.f;
        b += c.live(i, j) ? gd * h : 0.f;
        if (WPR == 1 || on) {
          dg[i][j] += d * h;
          db[i][j] += d;
        }
      }
    const float2 ab = row_sum(a, b);
    a = ab.x * inv;
    b = ab.y * inv;
    if (WPR == 1 || on) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float o[E];
        w.dy[i].renew();
        if constexpr (sizeof(T) == 2) w.x[i].renew();
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const float h = sizeof(T) == 4 ? w.x[i][j] : (w.x[i][j] - st.x) * st.y;
          o[j] = st.y * (w.dy[i][j] * g[i][j] - a - h * b);
          if (add) o[j] += w.a[i][j];
        }
        T* to = dx + row * lddx + c.col[i];
        if (c.first[i] == 0) {
          Vec<T, E>::store(to, o);
        } else if (c.first[i] < (uint32_t)E) {
          // dx may be add, and another wave of the row may have stored the repeated columns before this one's add came:
          // they are its alone
#pragma unroll
          for (int j = 1; j < E; ++j)
            if (c.live(i, j)) {
              const float one[1] = {o[j]};
              Vec<T, 1>::store(to + j, one);
            }
        }
      }
    }
  }
  const int64_t p = (int64_t)blockIdx.x * 2 * dim;
  if constexpr (R == 1) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c.first[i] < (uint32_t)E) {
        Vec<float, E>::store(dgamma + p + c.col[i], dg[i]);
        Vec<float, E>::store(dbeta + p + c.col[i], db[i]);
      }
  } else {                                         // the row groups' column sums, one after the other
    for (int w = 0; w < R; ++w) {
      __syncthreads();
      if (wave / WPR == w) {
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
          for (int j = 0; j < E; ++j)
            if (c.live(i, j)) {
              const int at = c.col[i] + j;
              sums[at] = w == 0 ? dg[i][j] : sums[at] + dg[i][j];
              sums[dim + at] = w == 0 ? db[i][j] : sums[dim + at] + db[i][j];
            }
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < dim; i += kThreads) {
      dgamma[p + i] = sums[i];
      dbeta[p + i] = sums[dim + i];
    }
  }
}

// dgamma | dbeta [2 * dim] = the sum of `parts` partial rows: 32 columns a workgroup, 32 row groups, sixteen loads in
// flight each -- 512 partial rows are one round trip.
__global__ __launch_bounds__(1024) void k_lnt_cols(const float* __restrict__ part, int parts, int dim,
                                                   float* __restrict__ dgamma, float* __restrict__ dbeta) {
  __shared__ float s[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + x, n = 2 * dim, cc = min(col, n - 1);
  float a = 0.f;
  for (int p0 = y; p0 < parts; p0 += 512) {
    float v[16];
#pragma unroll
    for (int u = 0; u < 16; ++u) v[u] = part[(int64_t)min(p0 + 32 * u, parts - 1) * n + cc];
#pragma unroll
    for (int u = 0; u < 16; ++u) a += p0 + 32 * u < parts ? v[u] : 0.f;
  }
  s[y][x] = a;
  __syncthreads();
  a = s[x][y];                                     // row group x of column y
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a += __shfl_xor(a, o);
  const int c = blockIdx.x * 32 + y;
  if (x == 0 && c < n) {
    if (c < dim) dgamma[c] = a;
    else dbeta[c - dim] = a;
  }
}

// How a row lies in registers: E elements a load, V loads a lane, WPR waves a row -- the narrowest that holds it.
template <int E_, int V_, int WPR_>
struct Shape {
  static constexpr int E = E_, V = V_, WPR = WPR_;
};
template <bool BACK, class F>
auto with_shape(int dim, F f) {
  if (dim <= 64) return f(Shape<1, 1, 1>{});
  if (dim <= 128) return f(Shape<2, 1, 1>{});
  if (dim <= 256) return f(Shape<4, 1, 1>{});
  if (dim <= 384) return f(Shape<2, 3, 1>{});
  if (dim <= 512) return f(Shape<4, 2, 1>{});
  if constexpr (BACK) {
    // eight columns a lane while eight waves hold the row: the backward pass holds four values and two sums a column, and
    // with sixteen there are two waves a SIMD and no registers to read a row ahead (18464 x 1024, one wave a row: 65 us,
    // two: 54 us; 12000 x 768 bf16 23.5 and 19.5 us)
    if (dim <= 1024) return f(Shape<4, 2, 2>{});
    if (dim <= 2048) return f(Shape<8, 1, 4>{});
    if (dim <= 4096) return f(Shape<8, 1, 8>{});
  } else {
    if (dim <= 768) return f(Shape<4, 3, 1>{});
    if (dim <= 1024) return f(Shape<4, 4, 1>{});
    if (dim <= 1536) return f(Shape<8, 3, 1>{});
    if (dim <= 2048) return f(Shape<8, 4, 1>{});
    if (dim <= 4096) return f(Shape<8, 2, 4>{});
  }
  return f(Shape<8, 2, 8>{});
}

// Workgroups (and partial rows) of the backward pass: as many as fit the CUs at once -- two, one of the widest shape -- or
// as a round of 8 / WPR rows each takes while there are few rows.  (A third and a fourth workgroup a CU that wait, which
// even out the last round, cost more in partial rows than they gave.)
inline int parts_for(int rows, int dim) {
  return with_shape<true>(dim, [&](auto s) {
    typedef decltype(s) H;
    return std::max(1, std::min(H::E * H::V <= 8 ? 2 * kCUs : kCUs, (rows - 1) / (8 / H::WPR) + 1));
  });
}

template <typename T>
void launch_fwd(const T* x, int64_t ldx, const float* gamma, const float* beta, float eps, int rows, int dim, bf16_t* y,
                int64_t ldy, float2* stats, hipStream_t s) {
  with_shape<false>(dim, [&](auto h) {
    typedef decltype(h) H;
    constexpr int R = H::WPR == 1 ? 4 : 1;
    hipLaunchKernelGGL((k_lnt_fwd<T, H::E, H::V, H::WPR>), dim3(std::min((rows - 1) / R + 1, 1 << 22)), dim3(H::WPR == 8 ? 512 : 256),
                       0, s, x, ldx, gamma, beta, eps, rows, dim, y, ldy, stats);
  });
}
template <typename T>
void launch_bwd(const bf16_t* dy, int64_t lddy, const T* x, int64_t ldx, const float2* stats, const float* gamma, const T* add,
                int64_t lda, int rows, int dim, T* dx, int64_t lddx, float* dgamma, float* dbeta, hipStream_t s) {
  with_shape<true>(dim, [&](auto h) {
    typedef decltype(h) H;
    hipLaunchKernelGGL((k_lnt_bwd<T, H::E, H::V, H::WPR>), dim3(parts_for(rows, dim)), dim3(kThreads),
                       H::WPR < 8 ? 2 * dim * sizeof(float) : 0, s, dy, lddy, x, ldx, stats, gamma, add, lda, rows, dim, dx, lddx,
                       dgamma, dbeta);
  });
}

}  // namespace lnt
}  // namespace i2pc

using namespace i2pc;

extern "C" int i2pc_layernorm_train(const void* x, int x_f32, int64_t ldx, const float* gamma, const float* beta, float eps,
                                    int rows, int dim, void* y, int64_t ldy, float* stats, void* stream) {
  clear_error();
  I2PC_REQUIRE(rows >= 0 && dim > 0, "layernorm_train: empty shape");
  I2PC_REQUIRE(dim <= lnt::kMaxDim, "layernorm_train: dim=%d is above %d", dim, lnt::kMaxDim);
  if (rows == 0) return I2PC_OK;
  I2PC_REQUIRE(x && gamma && beta && y && stats, "NULL pointer");
  I2PC_REQUIRE(ldx >= dim && ldy >= dim, "layernorm_train: row strides must be at least dim");
  hipStream_t s = as_stream(stream);
  auto* yy = static_cast<lnt::bf16_t*>(y);
  auto* st = reinterpret_cast<float2*>(stats);
  using namespace lnt;
  if (x_f32)
    launch_fwd(static_cast<const float*>(x), ldx, gamma, beta, eps, rows, dim, yy, ldy, st, s);
  else
    launch_fwd(static_cast<const bf16_t*>(x), ldx, gamma, beta, eps, rows, dim, yy, ldy, st, s);
  return check_launch("layernorm_train");
}

extern "C" size_t i2pc_layernorm_backward_workspace_bytes(int rows, int dim) {
  if (rows < 0 || dim <= 0 || dim > lnt::kMaxDim) return 0;
  const int parts = lnt::parts_for(rows, dim);
  return parts == 1 ? 0 : (size_t)parts * 2 * dim * sizeof(float);
}

extern "C" int i2pc_layernorm_backward(const void* dy, int64_t lddy, const void* x, int x_f32, int64_t ldx,
                                       const float* stats, const float* gamma, const void* add, int64_t lda, int rows,
                                       int dim, void* dx, int64_t lddx, float* dgamma, float* dbeta, void* workspace,
                                       size_t workspace_bytes, void* stream) {
  clear_error();
  I2PC_REQUIRE(rows >= 0 && dim > 0, "layernorm_backward: empty shape");
  I2PC_REQUIRE(dim <= lnt::kMaxDim, "layernorm_backward: dim=%d is above %d", dim, lnt::kMaxDim);
  I2PC_REQUIRE(gamma && dgamma && dbeta && (rows == 0 || (dy && x && stats && dx)), "NULL pointer");
  I2PC_REQUIRE(rows == 0 || (ldx >= dim && lddy >= dim && lddx >= dim && (!add || lda >= dim)),
               "layernorm_backward: row strides must be at least dim");
  const size_t need = i2pc_layernorm_backward_workspace_bytes(rows, dim);
  if (workspace_bytes < need || (need && !workspace))
    return set_error(I2PC_EWORKSPACE, "layernorm_backward: workspace of %zu bytes, needs %zu", workspace_bytes, need);
  hipStream_t s = as_stream(stream);
  float* part = static_cast<float*>(workspace);
  float *pg = need ? part : dgamma, *pb = need ? part + dim : dbeta;
  using namespace lnt;
  auto* g = static_cast<const bf16_t*>(dy);
  auto* st = reinterpret_cast<const float2*>(stats);
  if (x_f32)
    launch_bwd(g, lddy, static_cast<const float*>(x), ldx, st, gamma, static_cast<const float*>(add),
                 lda, rows, dim, static_cast<float*>(dx), lddx, pg, pb, s);
  else
    launch_bwd(g, lddy, static_cast<const bf16_t*>(x), ldx, st, gamma, static_cast<const bf16_t*>(add),
                 lda, rows, dim, static_cast<bf16_t*>(dx), lddx, pg, pb, s);
  if (need)
    hipLaunchKernelGGL(k_lnt_cols, dim3((2 * dim + 31) / 32), dim3(1024), 0, s, part, parts_for(rows, dim), dim, dgamma, dbeta);
  return check_launch("layernorm_backward");
}
