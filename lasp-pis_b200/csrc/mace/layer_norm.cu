// Layer norm with an activation, forward and backward.
//
//   forward   m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), xhat = (x - m) r,
//             y = act(xhat gamma + beta)
//   backward  dz = dy act'(xhat gamma + beta), g = dz gamma,
//             dx = r (g - mean(g) - xhat mean(g xhat)),
//             dgamma = sum over rows of dz xhat, dbeta = sum over rows of dz
//
// One pass over the data: a row stays in the registers of its group of threads (part of a warp, a
// warp, or a block for wide rows) between its statistics and its result.  HBM bounds it, so what
// counts is bytes in flight: a warp holds rows of up to 4 KiB (backward 1 KiB), a block wider ones, and
// where a thread's share of a row is small it takes several rows at once, and loads the next ones
// before the arithmetic of these.  The
// variance is taken about a first mean and corrected for that mean's own rounding, so a row far from
// zero loses nothing.  A group walks the rows with a fixed set of columns per thread, so the
// parameters' gradients stay in registers too; each block writes one partial row of dgamma and
// dbeta, and a second launch adds the partial rows in a fixed order.
//
// bf16 16384 x 4096 forward: 60 us, 4.4 TB/s (0.68 of the measured copy rate); f16 8191 x 2048: 18 us
// forward, 29 backward (3.5 TB/s); f32 84613 x 64 with SiLU: 11.5 and 17.8.
#include "operators.cuh"
#include "tcgen05.cuh"
#include <algorithm>
#include <cfloat>
#include <type_traits>

namespace mace {
namespace op {
namespace {
constexpr int kWarpBlock = 256; // threads of a block whose rows belong to warps or parts of them
constexpr int kSharedChunks = 4; // forward: from as many units per lane on

// A unit of an array, or zeros where it is not live.  The load itself is unconditional, from a place
// inside the array: a load under a branch is waited for where the branches join, which leaves one in
// flight instead of all of a row's (bf16 16384 x 4096: 192 us, 93 without).
template <class T, int U>
__device__ __forceinline__ Unit<T, U> load_unit(const T *row, bool live, int col) {
  Unit<T, U> v = *reinterpret_cast<const Unit<T, U> *>(row + col);
  if constexpr (sizeof(v) >= 4) {
    uint32_t w[sizeof(v) / 4];
    memcpy(w, &v, sizeof v);
#pragma unroll
    for (int i = 0; i < int(sizeof(v) / 4); ++i)
      w[i] = live ? w[i] : 0u;
    memcpy(&v, w, sizeof v);
  } else if (!live)
    v.v[0] = from_float<T>(0.f);
  return v;
}
// A unit of gamma or beta (`none` where there is no array or no column).
template <class T, int U>
__device__ __forceinline__ Unit<T, U> parameter_unit(const void *p, int col, int width, float none) {
  Unit<T, U> v;
  if (p && col < width)
    v = *reinterpret_cast<const Unit<T, U> *>(static_cast<const T *>(p) + col);
  else
#pragma unroll
    for (int u = 0; u < U; ++u)
      v.v[u] = from_float<T>(none);
  return v;
}

// Sums of R pairs of values, each over a row's group: G lanes (G <= 32, power of two), or the block.
template <bool Warp, int R>
__device__ __forceinline__ void group_sum(float2 (&v)[R], int G, float2 (*shared)[32]) {
  for (int o = Warp ? G >> 1 : 16; o; o >>= 1)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      v[r].x += __shfl_xor_sync(0xffffffffu, v[r].x, o);
      v[r].y += __shfl_xor_sync(0xffffffffu, v[r].y, o);
    }
  if (Warp)
    return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if (!lane)
#pragma unroll
    for (int r = 0; r < R; ++r)
      shared[r][warp] = v[r];
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r)
    v[r] = lane < warps ? shared[r][lane] : make_float2(0.f, 0.f);
#pragma unroll
  for (int o = 16; o; o >>= 1)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      v[r].x += __shfl_xor_sync(0xffffffffu, v[r].x, o);
      v[r].y += __shfl_xor_sync(0xffffffffu, v[r].y, o);
    }
}

// Arithmetic on pairs of floats (one instruction for two), where a thread's elements come in pairs.
template <int N> __device__ __forceinline__ float sum_of(const float *v) {
  if constexpr (N % 4 == 0) {
    float2 a = make_float2(v[0], v[1]), b = make_float2(v[2], v[3]);
#pragma unroll
    for (int i = 4; i < N; i += 4) {
      a = __fadd2_rn(a, make_float2(v[i], v[i + 1]));
      b = __fadd2_rn(b, make_float2(v[i + 2], v[i + 3]));
    }
    a = __fadd2_rn(a, b);
    return a.x + a.y;
  } else {
    float s = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i)
      s += v[i];
    return s;
  }
}
// v = v a + b, element by element.
template <int N> __device__ __forceinline__ void scale_shift(float *v, float a, float b) {
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 r = __ffma2_rn(make_float2(v[i], v[i + 1]), make_float2(a, a), make_float2(b, b));
      v[i] = r.x, v[i + 1] = r.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = fmaf(v[i], a, b);
  }
}
// c + sum a b
template <int N> __device__ __forceinline__ float dot_of(const float *a, const float *b, float c) {
  if constexpr (N % 2 == 0) {
    float2 s = make_float2(c, 0.f);
#pragma unroll
    for (int i = 0; i < N; i += 2)
      s = __ffma2_rn(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]), s);
    return s.x + s.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      c = fmaf(a[i], b[i], c);
    return c;
  }
}
// z = z a + b with arrays.
template <int N> __device__ __forceinline__ void fma_all(float *z, const float *a, const float *b) {
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 r = __ffma2_rn(make_float2(z[i], z[i + 1]), make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]));
      z[i] = r.x, z[i + 1] = r.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      z[i] = fmaf(z[i], a[i], b[i]);
  }
}

// A row may lie far from zero against its spread, or have none.  The values centred about a first mean have
// a mean of their own, `fix`, that mean's rounding error; s is the sum of the centred values and that of
// their squares.  Where fix is not small against the spread (a few steps of the type at most, then),
// the difference below loses the variance, and the row is centred once more; so where the squares overflow.
__device__ __forceinline__ float variance(float2 s, float inv_n) {
  const float fix = s.x * inv_n, w = fmaf(-fix, fix, s.y * inv_n);
  return w < 0.f ? 0.f : w; // (NaN stays)
}
__device__ __forceinline__ bool recentre(float fix, float var) { return !(4.f * fix * fix <= var && var <= FLT_MAX); }
// Such a row of floats, from memory: its group centres it twice more and writes its result (mine: whether
// this group's row is one).
template <bool Warp>
__device__ __noinline__ void centre_again(const Norm &a, long long row, bool mine, float mean, int G, int t,
                                          float2 (*shared0)[32], float2 (*shared1)[32]) {
  const float inv_n = 1.f / float(a.width);
  mine = mine && row < a.rows;
  const float *x = static_cast<const float *>(a.x) + (mine ? row : 0) * a.ldx;
  float fix = 0.f;
  float2 s[1];
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    s[0] = make_float2(0.f, 0.f);
    for (long long i = t; mine && i < a.width; i += G) {
      const float d = x[i] - mean - fix;
      s[0].x += d;
      s[0].y = fmaf(d, d, s[0].y);
    }
    __syncwarp();
    group_sum<Warp, 1>(s, G, k ? shared1 : shared0);
    fix += s[0].x * inv_n;
  }
  const float r = 1.f / sqrtf(variance(s[0], inv_n) + a.eps);
  if (!mine)
    return;
  if (a.mean && !t) {
    a.mean[row] = mean + fix;
    a.rstd[row] = r;
  }
  for (long long i = t; i < a.width; i += G) {
    float z = (x[i] - mean - fix) * r;
    if (a.gamma)
      z *= static_cast<const float *>(a.gamma)[i];
    if (a.beta)
      z += static_cast<const float *>(a.beta)[i];
    static_cast<float *>(a.y)[row * a.ldy + i] = activate<false>(z, a.activation);
  }
}

// T elements in units of U, C units per thread (columns (c G + t) U ...), a row per group of G threads
// -- G lanes of a warp (Threads = kWarpBlock), or a block of at most Threads -- and R rows per group
// at once.  Instructions come next after bytes: at 6.5 TB/s an SM has 22 issue slots for each 16-bit
// element, so elements are converted by words and handled in pairs.
template <class T, int U, int C, int R, int Threads>
__global__ void __launch_bounds__(Threads) layer_norm_kernel(const __grid_constant__ Norm a, int lanes) {
  // Lanes with many columns find gamma and beta in shared memory, others in registers.
  constexpr bool Fast = sizeof(T) == 2, Ahead = C * R <= 4, Warp = Threads == kWarpBlock,
                 Shared = Warp && C >= kSharedChunks;
  using Un = Unit<T, U>;
  __shared__ float2 shared[Fast ? 2 : 4][R][32];
  extern __shared__ __align__(16) unsigned char parameters[]; // [2][32 C] units (Shared)
  Un *const common = reinterpret_cast<Un *>(parameters);
  const int G = Warp ? lanes : blockDim.x, t = Warp ? threadIdx.x & (G - 1) : threadIdx.x;
  const int per_block = Warp ? kWarpBlock / G : 1, group = Warp ? threadIdx.x / G : 0, width = int(a.width);
  const T *x = static_cast<const T *>(a.x);
  T *y = static_cast<T *>(a.y);
  const float inv_n = 1.f / float(width);
  const long long step = (long long)gridDim.x * per_block * R;
  long long base = (long long)blockIdx.x * per_block * R;
  auto col = [&](int c) { return (c * G + t) * U; };
  Un own[2][Shared ? 1 : C];
  if (Shared) { // unit by unit
    for (int i = threadIdx.x; i < C * G; i += Threads) {
      common[i] = parameter_unit<T, U>(a.gamma, i * U, width, 1.f);
      common[C * 32 + i] = parameter_unit<T, U>(a.beta, i * U, width, 0.f);
    }
    __syncthreads();
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      own[0][c] = parameter_unit<T, U>(a.gamma, col(c), width, 1.f);
      own[1][c] = parameter_unit<T, U>(a.beta, col(c), width, 0.f);
    }
  }
  float count = 0.f; // of this thread's elements of a row
#pragma unroll
  for (int c = 0; c < C; ++c)
    count += Fast && col(c) < width ? float(U) : 0.f;
  Un next[R][C];
  T next_first[R];
  auto load = [&](long long from) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = from + r * per_block + group;
      const T *p = x + min(row, a.rows - 1) * a.ldx;
      if (Fast)
        next_first[r] = *p;
#pragma unroll
      for (int c = 0; c < C; ++c)
        next[r][c] = load_unit<T, U>(p, col(c) < width, min(col(c), width - U));
    }
  };
  if (Ahead)
    load(base);
  for (; base < a.rows; base += step) {
    if (!Ahead)
      load(base);
    float v[R][C * U], pivot[R];
    float2 s[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int c = 0; c < C; ++c)
        unpack<T, U>(next[r][c], v[r] + c * U);
      pivot[r] = Fast ? to_float(next_first[r]) : 0.f;
      const float sum = sum_of<C * U>(v[r]);
      s[r] = Fast ? make_float2(fmaf(-count, pivot[r], sum), sum) : make_float2(sum, 0.f);
    }
    if (Ahead)
      load(base + step);
    group_sum<Warp, R>(s, G, shared[0]);
    float mean[R], rs[R], rest[R], shift[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      // 16-bit values: the sums' distance from the first value's is exact where values are near each other,
      // so that what the mean's rounding leaves is known.  Where that distance is the larger sum (the
      // first value lies far from the rest), the plain sum has the smaller error.
      const float d = s[r].x * inv_n;
      const bool near = Fast && fabsf(s[r].x) <= fabsf(s[r].y);
      mean[r] = near ? pivot[r] + d : Fast ? s[r].y * inv_n : d;
      rest[r] = near ? (pivot[r] - mean[r]) + d : 0.f;
      scale_shift<C * U>(v[r], 1.f, -mean[r]);
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (col(c) >= width)
#pragma unroll
          for (int u = 0; u < U; ++u)
            v[r][c * U + u] = 0.f;
      s[r] = make_float2(Fast ? 0.f : sum_of<C * U>(v[r]), dot_of<C * U>(v[r], v[r], 0.f));
    }
    group_sum<Warp, R>(s, G, shared[1]);
    unsigned again = 0; // rows
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float fix = Fast ? rest[r] : s[r].x * inv_n, w = fmaf(-fix, fix, s[r].y * inv_n), var = w < 0.f ? 0.f : w;
      const bool later = !Fast && recentre(fix, var);
      again |= unsigned(later) << r;
      rs[r] = Fast ? rsqrtf(var + a.eps) : 1.f / sqrtf(var + a.eps);
      const long long row = base + r * per_block + group;
      if (a.mean && !t && row < a.rows && !later) {
        a.mean[row] = mean[r] + fix;
        a.rstd[row] = Fast ? 1.f / sqrtf(var + a.eps) : rs[r];
      }
      shift[r] = -fix * rs[r]; // (v - fix) rs in one instruction
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float gamma[U], beta[U];
      unpack<T, U>(Shared ? common[c * G + t] : own[0][Shared ? 0 : c], gamma);
      unpack<T, U>(Shared ? common[(32 * C + c * G) + t] : own[1][Shared ? 0 : c], beta);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const long long row = base + r * per_block + group;
        float z[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
          z[u] = v[r][c * U + u];
        scale_shift<U>(z, rs[r], shift[r]);
        fma_all<U>(z, gamma, beta);
        activate_all<Fast>(z, a.activation);
        if (row < a.rows && col(c) < width && !(again >> r & 1))
          *reinterpret_cast<Un *>(y + row * a.ldy + col(c)) = pack<T, U>(z);
      }
    }
    if constexpr (!Fast)
      if (Warp ? __any_sync(0xffffffffu, again) : again)
#pragma unroll
        for (int r = 0; r < R; ++r)
          centre_again<Warp>(a, base + r * per_block + group, again >> r & 1, mean[r], G, t, shared[2], shared[3]);
  }
}

// partial: [gridDim.x][2][width] (dgamma, dbeta), or NULL.
template <class T, int U, int C, int R, int Threads>
__global__ void __launch_bounds__(Threads)
    layer_norm_backward_kernel(const __grid_constant__ NormBackward a, int lanes, float *partial) {
  constexpr bool Fast = sizeof(T) == 2, Warp = Threads == kWarpBlock;
  constexpr int N = C * U;
  using Un = Unit<T, U>;
  __shared__ float2 shared[2][R][32];
  __shared__ float join[Warp ? kWarpBlock * N : 1];
  const int G = Warp ? lanes : blockDim.x, t = Warp ? threadIdx.x & (G - 1) : threadIdx.x;
  const int per_block = Warp ? kWarpBlock / G : 1, group = Warp ? threadIdx.x / G : 0, width = int(a.width);
  const T *x = static_cast<const T *>(a.x), *dy = static_cast<const T *>(a.dy);
  T *dx = static_cast<T *>(a.dx);
  const float inv_n = 1.f / float(width);
  auto col = [&](int c) { return (c * G + t) * U; };
  Un gamma[C], beta[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    gamma[c] = parameter_unit<T, U>(a.gamma, col(c), width, 1.f);
    beta[c] = parameter_unit<T, U>(a.activation != None ? a.beta : nullptr, col(c), width, 0.f);
  }
  float sum_gamma[N] = {}, sum_beta[N] = {};
  const long long step = (long long)gridDim.x * per_block * R;
  long long base = (long long)blockIdx.x * per_block * R;
  Un next_x[R][C], next_dy[R][C];
  float next_mean[R], next_r[R];
  // Rows and columns outside: dy reads as zero, so they add nothing to any sum.
  auto load = [&](long long from) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = from + r * per_block + group, in = min(row, a.rows - 1);
      next_mean[r] = a.mean[in];
      next_r[r] = a.rstd[in];
      const T *px = x + in * a.ldx, *pd = dy + in * a.lddy;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int at = min(col(c), width - U);
        next_x[r][c] = load_unit<T, U>(px, col(c) < width && row < a.rows, at);
        next_dy[r][c] = load_unit<T, U>(pd, col(c) < width && row < a.rows, at);
      }
    }
  };
  load(base);
  for (int k = 0; base < a.rows; base += step, k ^= 1) {
    float xh[R][N], g[R][N], rs[R];
    float2 s[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool mine = base + r * per_block + group < a.rows;
      const float mean = next_mean[r];
      rs[r] = next_r[r];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        unpack<T, U>(next_x[r][c], xh[r] + c * U);
        unpack<T, U>(next_dy[r][c], g[r] + c * U);
      }
      scale_shift<N>(xh[r], 1.f, -mean);
      scale_shift<N>(xh[r], rs[r], 0.f);
#pragma unroll
      for (int c = 0; c < C; ++c) // outside xhat is 0 too: its row's statistics need not be finite
        if (col(c) >= width || !mine)
#pragma unroll
          for (int u = 0; u < U; ++u)
            xh[r][c * U + u] = 0.f;
      float gm[N];
#pragma unroll
      for (int c = 0; c < C; ++c)
        unpack<T, U>(gamma[c], gm + c * U);
      if (a.activation != None) {
        float z[N];
#pragma unroll
        for (int c = 0; c < C; ++c)
          unpack<T, U>(beta[c], z + c * U);
#pragma unroll
        for (int i = 0; i < N; ++i)
          z[i] = fmaf(xh[r][i], gm[i], z[i]);
        slope_all<Fast>(z, a.activation);
#pragma unroll
        for (int i = 0; i < N; ++i)
          g[r][i] *= z[i];
      }
      const float none[N] = {};
      if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
          const float2 d = make_float2(g[r][i], g[r][i + 1]);
          const float2 p = __ffma2_rn(d, make_float2(xh[r][i], xh[r][i + 1]), make_float2(sum_gamma[i], sum_gamma[i + 1]));
          const float2 q = __fadd2_rn(d, make_float2(sum_beta[i], sum_beta[i + 1]));
          sum_gamma[i] = p.x, sum_gamma[i + 1] = p.y;
          sum_beta[i] = q.x, sum_beta[i + 1] = q.y;
        }
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          sum_gamma[i] = fmaf(g[r][i], xh[r][i], sum_gamma[i]);
          sum_beta[i] += g[r][i];
        }
      }
      fma_all<N>(g[r], gm, none);
      s[r] = make_float2(sum_of<N>(g[r]), dot_of<N>(g[r], xh[r], 0.f));
    }
    load(base + step);
    if (!dx)
      continue;
    group_sum<Warp, R>(s, G, shared[k]); // two buffers: sums are read while the next are written
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = base + r * per_block + group;
      const float mg = s[r].x * inv_n, mgx = s[r].y * inv_n;
      scale_shift<N>(xh[r], -mgx, -mg);
      float o[N];
      if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
          const float2 f = __fmul2_rn(__fadd2_rn(make_float2(g[r][i], g[r][i + 1]), make_float2(xh[r][i], xh[r][i + 1])),
                                      make_float2(rs[r], rs[r]));
          o[i] = f.x, o[i + 1] = f.y;
        }
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
          o[i] = rs[r] * (g[r][i] + xh[r][i]);
      }
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (col(c) < width && row < a.rows)
          *reinterpret_cast<Un *>(dx + row * a.lddx + col(c)) = pack<T, U>(o + c * U);
    }
  }
  if (!partial)
    return;
  float *out = partial + (long long)blockIdx.x * 2 * a.width;
#pragma unroll 1
  for (int k = 0; k < 2; ++k, out += a.width) {
    if (Warp) { // the block's groups hold the same columns: add them in group order
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i)
        join[(group * N + i) * G + t] = k ? sum_beta[i] : sum_gamma[i];
      __syncthreads();
      for (int j = threadIdx.x; j < N * G; j += kWarpBlock) {
        const int i = j / G, cc = ((i / U) * G + j % G) * U + i % U;
        float v = 0.f;
        for (int q = 0; q < per_block; ++q)
          v += join[q * N * G + j];
        if (cc < width)
          out[cc] = v;
      }
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (col(c) < width)
#pragma unroll
          for (int u = 0; u < U; ++u)
            out[col(c) + u] = k ? sum_beta[c * U + u] : sum_gamma[c * U + u];
    }
  }
}

// ---------------- rows too wide for registers: loops over the row, read again from L2 ----------------
constexpr int kWideThreads = 1024;
template <class T> __global__ void __launch_bounds__(kWideThreads) wide_norm_kernel(const __grid_constant__ Norm a) {
  constexpr bool Fast = sizeof(T) == 2;
  __shared__ float2 shared[3][1][32];
  const float inv_n = 1.f / float(a.width);
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + row * a.ldx;
    T *y = static_cast<T *>(a.y) + row * a.ldy;
    float2 s[1] = {};
    for (long long i = threadIdx.x; i < a.width; i += kWideThreads)
      s[0].x += to_float(x[i]);
    group_sum<false, 1>(s, 0, shared[0]);
    const float m1 = s[0].x * inv_n;
    s[0] = make_float2(0.f, 0.f);
    for (long long i = threadIdx.x; i < a.width; i += kWideThreads) {
      float d = to_float(x[i]) - m1;
      s[0].x += d;
      s[0].y = fmaf(d, d, s[0].y);
    }
    group_sum<false, 1>(s, 0, shared[1]);
    float fix = s[0].x * inv_n, var = variance(s[0], inv_n);
    if (recentre(fix, var)) { // (the same for all threads)
      s[0] = make_float2(0.f, 0.f);
      for (long long i = threadIdx.x; i < a.width; i += kWideThreads) {
        float d = to_float(x[i]) - m1 - fix;
        s[0].x += d;
        s[0].y = fmaf(d, d, s[0].y);
      }
      group_sum<false, 1>(s, 0, shared[2]);
      fix += s[0].x * inv_n;
      var = variance(s[0], inv_n);
    }
    const float r = 1.f / sqrtf(var + a.eps);
    if (a.mean && !threadIdx.x) {
      a.mean[row] = m1 + fix;
      a.rstd[row] = r;
    }
    for (long long i = threadIdx.x; i < a.width; i += kWideThreads) {
      float z = (to_float(x[i]) - m1 - fix) * r;
      if (a.gamma)
        z *= to_float(static_cast<const T *>(a.gamma)[i]);
      if (a.beta)
        z += to_float(static_cast<const T *>(a.beta)[i]);
      y[i] = from_float<T>(activate<Fast>(z, a.activation));
    }
  }
}
// xhat and dz of one element.
template <class T> __device__ __forceinline__ float2 wide_element(const NormBackward &a, long long row, long long i) {
  constexpr bool Fast = sizeof(T) == 2;
  float xh = (to_float(static_cast<const T *>(a.x)[row * a.ldx + i]) - a.mean[row]) * a.rstd[row];
  float dz = to_float(static_cast<const T *>(a.dy)[row * a.lddy + i]);
  if (a.activation != None)
    dz *= slope<Fast>(fmaf(xh, a.gamma ? to_float(static_cast<const T *>(a.gamma)[i]) : 1.f,
                           a.beta ? to_float(static_cast<const T *>(a.beta)[i]) : 0.f),
                      a.activation);
  return make_float2(xh, dz);
}
template <class T>
__global__ void __launch_bounds__(kWideThreads) wide_norm_backward_kernel(const __grid_constant__ NormBackward a) {
  __shared__ float2 shared[2][1][32];
  const float inv_n = 1.f / float(a.width);
  int k = 0;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, k ^= 1) {
    float2 s[1] = {};
    for (long long i = threadIdx.x; i < a.width; i += kWideThreads) {
      float2 e = wide_element<T>(a, row, i);
      float g = e.y * (a.gamma ? to_float(static_cast<const T *>(a.gamma)[i]) : 1.f);
      s[0].x += g;
      s[0].y = fmaf(g, e.x, s[0].y);
    }
    group_sum<false, 1>(s, 0, shared[k]);
    const float mg = s[0].x * inv_n, mgx = s[0].y * inv_n, r = a.rstd[row];
    // dx may be dy: an element is read and written by the same thread.
    for (long long i = threadIdx.x; i < a.width; i += kWideThreads) {
      float2 e = wide_element<T>(a, row, i);
      float g = e.y * (a.gamma ? to_float(static_cast<const T *>(a.gamma)[i]) : 1.f);
      static_cast<T *>(a.dx)[row * a.lddx + i] = from_float<T>(r * (g - fmaf(e.x, mgx, mg)));
    }
  }
}
// Partial dgamma and dbeta of every gridDim.y-th row, a column per thread.
template <class T>
__global__ void __launch_bounds__(256) wide_params_kernel(const __grid_constant__ NormBackward a, float *partial) {
  long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.width)
    return;
  float sg = 0.f, sb = 0.f;
  for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
    float2 e = wide_element<T>(a, row, i);
    sg = fmaf(e.y, e.x, sg);
    sb += e.y;
  }
  float *out = partial + (long long)blockIdx.y * 2 * a.width;
  out[i] = sg;
  out[a.width + i] = sb;
}

// ---------------- rows that start anywhere ----------------
// Rows that allow no wide loads (odd widths) are copied into shared memory as spans: several rows that
// lie one behind another without gaps, or one row.  One bulk copy brings what of a span lies between
// 16-byte boundaries, single loads its two ends, to a place with the same offset from a boundary; the
// result goes back the same way.  Element by element there, with several blocks to an SM, so that one
// computes while another's copies are under way.  f16 8191 x 2053, backward: single-element loads take
// 105 us, spans 56.
struct Span {
  int rows, bytes; // of a span; bytes: of its place in shared memory
};
struct Ends {
  int head, whole; // elements before the first boundary, and from there to the last one
};
template <class T> __device__ __forceinline__ Ends ends_of(const T *p, int elements) {
  const int off = int(reinterpret_cast<uintptr_t>(p) & 15), head = min(off ? (16 - off) / int(sizeof(T)) : 0, elements);
  return {head, (elements - head) * int(sizeof(T)) / 16 * (16 / int(sizeof(T)))};
}
// A span's first element in its place.
template <class T> __device__ __forceinline__ T *placed(unsigned char *place, const T *p) {
  return reinterpret_cast<T *>(place + (reinterpret_cast<uintptr_t>(p) & 15));
}
// Copies `elements` elements of each of K spans; whether they came.
template <class T, int K>
__device__ __forceinline__ bool bring_spans(const T *const (&from)[K], T *const (&to)[K], int elements, unsigned bar,
                                            unsigned &phase) {
  Ends e[K];
  unsigned bytes = 0;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    e[k] = ends_of(from[k], elements);
    bytes += unsigned(e[k].whole) * unsigned(sizeof(T));
  }
  if (bytes && threadIdx.x == 0) {
    tc::mbar_expect_tx(bar, bytes);
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (e[k].whole)
        tc::bulk_load(tc::smem_u32(to[k] + e[k].head), from[k] + e[k].head, unsigned(e[k].whole) * unsigned(sizeof(T)), bar);
  }
  // (16 / size ends at most on each side)
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = threadIdx.x;
    if (i < e[k].head)
      to[k][i] = from[k][i];
    const int tail = e[k].head + e[k].whole + i;
    if (i < 32 && tail < elements)
      to[k][tail] = from[k][tail];
  }
  bool there = true;
  if (bytes) {
    const long long start = clock64();
    while (!(there = tc::mbar_try(bar, phase)) && clock64() - start < tc::kWaitCycles) {
    }
    phase ^= 1;
  }
  return __syncthreads_and(there);
}
template <class T> __device__ __forceinline__ void send_span(T *to, const T *from, int elements) {
  tc::fence_proxy_async_smem();
  __syncthreads();
  // Bulk where both sides agree about the boundaries (they do, but for rows of different distances).
  Ends e = ends_of(to, elements);
  if ((reinterpret_cast<uintptr_t>(to) ^ reinterpret_cast<uintptr_t>(from)) & 15)
    e = {0, 0};
  if (e.whole && threadIdx.x == 0) {
    tc::bulk_store(to + e.head, tc::smem_u32(from + e.head), unsigned(e.whole) * unsigned(sizeof(T)));
    tc::bulk_commit();
    tc::bulk_wait_read();
  }
  for (int i = threadIdx.x; i < e.head; i += blockDim.x)
    to[i] = from[i];
  for (int i = e.head + e.whole + int(threadIdx.x); i < elements; i += blockDim.x)
    to[i] = from[i];
  __syncthreads();
}
// gamma and beta (1 and 0 where there is none) into shared memory.
template <class T> __device__ __forceinline__ void bring_parameters(const void *gamma, const void *beta, int width, T *to) {
  for (int i = threadIdx.x; i < width; i += blockDim.x) {
    to[i] = gamma ? static_cast<const T *>(gamma)[i] : from_float<T>(1.f);
    to[width + i] = beta ? static_cast<const T *>(beta)[i] : from_float<T>(0.f);
  }
}
// A row of a span belongs to a warp, or to the whole block where a span is a single row (Block):
// its first thread and stride, and sums over it.
template <bool Block> struct Team {
  static __device__ __forceinline__ int first() { return Block ? threadIdx.x : threadIdx.x & 31; }
  static __device__ __forceinline__ int stride() { return Block ? blockDim.x : 32; }
  static __device__ __forceinline__ float2 sum(float2 v, float2 (*shared)[32]) {
    float2 s[1] = {v};
    group_sum<!Block, 1>(s, 32, shared);
    return s[0];
  }
};

template <class T, bool Block>
__global__ void __launch_bounds__(Block ? 1024 : 256) span_norm_kernel(const __grid_constant__ Norm a, Span span) {
  constexpr bool Fast = sizeof(T) == 2;
  extern __shared__ __align__(16) unsigned char parameters[];
  __shared__ uint64_t bar;
  __shared__ float2 shared[3][1][32];
  T *gamma = reinterpret_cast<T *>(parameters + span.bytes), *beta = gamma + a.width;
  const int width = int(a.width), warp = threadIdx.x >> 5, t = Team<Block>::first(), stride = Team<Block>::stride();
  const float inv_n = 1.f / float(width);
  if (threadIdx.x == 0) {
    tc::mbar_init(tc::smem_u32(&bar), 1);
    tc::fence_proxy_async_smem();
  }
  bring_parameters(a.gamma, a.beta, width, gamma);
  __syncthreads();
  unsigned phase = 0;
  for (long long first = (long long)blockIdx.x * span.rows; first < a.rows; first += (long long)gridDim.x * span.rows) {
    const int rows = int(min((long long)span.rows, a.rows - first)), elements = rows * width;
    const T *const from[1] = {static_cast<const T *>(a.x) + first * a.ldx};
    T *const x = placed(parameters, from[0]), *const to[1] = {x};
    const bool there = bring_spans<T, 1>(from, to, elements, tc::smem_u32(&bar), phase);
    for (int r = Block ? 0 : warp; r < rows; r += Block ? 1 : 8) {
      T *row = x + r * width;
      float2 s = make_float2(0.f, 0.f);
#pragma unroll 8
      for (int c = t; c < width; c += stride)
        s.x += to_float(row[c]);
      const float m1 = Team<Block>::sum(s, shared[0]).x * inv_n;
      s = make_float2(0.f, 0.f);
#pragma unroll 8
      for (int c = t; c < width; c += stride) {
        const float d = to_float(row[c]) - m1;
        s.x += d;
        s.y = fmaf(d, d, s.y);
      }
      s = Team<Block>::sum(s, shared[1]);
      float fix = s.x * inv_n, var = variance(s, inv_n);
      if (recentre(fix, var)) { // (the same for the whole team)
        s = make_float2(0.f, 0.f);
        for (int c = t; c < width; c += stride) {
          const float d = to_float(row[c]) - m1 - fix;
          s.x += d;
          s.y = fmaf(d, d, s.y);
        }
        s = Team<Block>::sum(s, shared[2]);
        fix += s.x * inv_n;
        var = variance(s, inv_n);
      }
      // A wait that ran out shows as NaN.
      const float rs = there ? 1.f / sqrtf(var + a.eps) : __uint_as_float(0x7fc00000u);
      if (a.mean && !t) {
        a.mean[first + r] = m1 + fix;
        a.rstd[first + r] = rs;
      }
      // Each thread rewrites the elements that it reads.
      for (int c0 = t; c0 < width; c0 += 8 * stride) {
        float z[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int c = min(c0 + i * stride, width - 1);
          z[i] = c0 + i * stride < width ? fmaf((to_float(row[c]) - m1 - fix) * rs, to_float(gamma[c]), to_float(beta[c])) : 0.f;
        }
        activate_all<Fast>(z, a.activation);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c0 + i * stride < width)
            row[c0 + i * stride] = from_float<T>(z[i]);
      }
    }
    send_span<T>(static_cast<T *>(a.y) + first * a.ldy, x, elements);
  }
}

// Row sums, then dx and the parameters' gradients by columns: thread t has columns t, t + blockDim.x, ...
// (at most C of them).
template <class T, int C, bool Block>
__global__ void __launch_bounds__(Block ? 1024 : 256)
    span_norm_backward_kernel(const __grid_constant__ NormBackward a, Span span, float *partial) {
  constexpr bool Fast = sizeof(T) == 2;
  extern __shared__ __align__(16) unsigned char parameters[];
  __shared__ uint64_t bar;
  __shared__ float2 shared[2][1][32];
  __shared__ float4 stats[Block ? 1 : 256]; // mean, r, mean(g), mean(g xhat) of each row
  T *gamma = reinterpret_cast<T *>(parameters + 2 * span.bytes), *beta = gamma + a.width;
  const int width = int(a.width), warp = threadIdx.x >> 5, t = Team<Block>::first(), stride = Team<Block>::stride();
  const float inv_n = 1.f / float(width);
  if (threadIdx.x == 0) {
    tc::mbar_init(tc::smem_u32(&bar), 1);
    tc::fence_proxy_async_smem();
  }
  bring_parameters(a.gamma, a.activation != None ? a.beta : nullptr, width, gamma);
  __syncthreads();
  float sum_gamma[C] = {}, sum_beta[C] = {};
  unsigned phase = 0;
  int k2 = 0;
  for (long long first = (long long)blockIdx.x * span.rows; first < a.rows; first += (long long)gridDim.x * span.rows) {
    const int rows = int(min((long long)span.rows, a.rows - first)), elements = rows * width;
    const T *const from[2] = {static_cast<const T *>(a.x) + first * a.ldx, static_cast<const T *>(a.dy) + first * a.lddy};
    T *const x = placed(parameters, from[0]), *const dy = placed(parameters + span.bytes, from[1]), *const to[2] = {x, dy};
    const bool there = bring_spans<T, 2>(from, to, elements, tc::smem_u32(&bar), phase);
    auto element = [&](int at, int c, float mean, float r, float &xh) { // dz
      xh = (to_float(x[at]) - mean) * r;
      float dz = to_float(dy[at]);
      if (a.activation != None)
        dz *= slope<Fast>(fmaf(xh, to_float(gamma[c]), to_float(beta[c])), a.activation);
      return dz;
    };
    for (int r = Block ? 0 : warp; r < rows; r += Block ? 1 : 8) {
      const float mean = a.mean[first + r], rs = there ? a.rstd[first + r] : __uint_as_float(0x7fc00000u);
      float2 s = make_float2(0.f, 0.f);
#pragma unroll 8
      for (int c = t; c < width; c += stride) {
        float xh;
        const float g = element(r * width + c, c, mean, rs, xh) * to_float(gamma[c]);
        s.x += g;
        s.y = fmaf(g, xh, s.y);
      }
      s = Team<Block>::sum(s, shared[k2 ^= 1]);
      if (!t)
        stats[r] = make_float4(mean, rs, s.x * inv_n, s.y * inv_n);
    }
    __syncthreads();
    // dx over dy's place where it lies like dy, else over x's: both are read by their thread only.
    T *const out = a.dx && ((reinterpret_cast<uintptr_t>(static_cast<T *>(a.dx) + first * a.lddx) ^ reinterpret_cast<uintptr_t>(dy)) & 15) == 0 ? dy : x;
#pragma unroll
    for (int k = 0; k < C; ++k) {
      const int c = k * int(blockDim.x) + int(threadIdx.x);
      if (c < width) {
        const float gm = to_float(gamma[c]);
#pragma unroll 4
        for (int r = 0; r < rows; ++r) {
          const float4 st = stats[r];
          float xh;
          const float dz = element(r * width + c, c, st.x, st.y, xh);
          sum_gamma[k] = fmaf(dz, xh, sum_gamma[k]);
          sum_beta[k] += dz;
          if (a.dx) // (else nothing may write here: the next span's copies are not ordered after such writes)
            out[r * width + c] = from_float<T>(st.y * (dz * gm - fmaf(xh, st.w, st.z)));
        }
      }
    }
    if (a.dx)
      send_span<T>(static_cast<T *>(a.dx) + first * a.lddx, out, elements);
    else
      __syncthreads();
  }
  if (!partial)
    return;
  float *sums = partial + (long long)blockIdx.x * 2 * width;
#pragma unroll
  for (int k = 0; k < C; ++k) {
    const int c = k * int(blockDim.x) + int(threadIdx.x);
    if (c < width) {
      sums[c] = sum_gamma[k];
      sums[width + c] = sum_beta[k];
    }
  }
}

// How a row is laid over threads: units of `unit` elements, `chunks` of them per thread.  Part of a warp
// or a warp holds it where that leaves a lane at most 8 units, or backward, where every column has two
// sums in registers as well, 2; else a block, as small as its chunks allow, so that several share an SM
// and one computes while another waits at its barrier.  Rows that allow no wide loads: below 128
// elements, 1 or 8 per lane (longer ones are spans, see span_of).
struct Shape {
  int unit, chunks, threads, most; // threads: lanes of a warp, or the block's threads; most: its class
  bool wide;
};
constexpr int kShort = 128; // single elements
Shape shape_of(int type, long long width, bool vectors, bool backward) {
  Shape s{vectors ? 16 / bytes_of(type) : 1, 0, 1, kWarpBlock, false};
  const long long units = (width + s.unit - 1) / s.unit;
  static constexpr int kLane[4][5] = {{1, 8}, {1, 8}, {1, 2, 4, 8}, {1, 2}}; // [vectors][backward]
  static constexpr int kBlock[2][3] = {{4}, {1, 2}};                          // [backward]
  for (const int *c = kLane[2 * vectors + backward]; *c; ++c)
    if (units <= 32 * *c && (vectors || width < kShort)) {
      s.chunks = *c;
      while ((long long)s.threads * *c < units)
        s.threads *= 2;
      return s;
    }
  for (int most : {512, 1024})
    for (const int *c = kBlock[backward]; vectors && *c; ++c)
      if (units <= (long long)most * *c) {
        s.chunks = *c;
        s.threads = int((units + 32 * *c - 1) / (32 * *c) * 32);
        s.most = most;
        return s;
      }
  s.wide = true;
  return s;
}
// Rows at once: several where a thread's share of one is small.
template <bool Backward> constexpr int rows_of(int share, int most) {
  return most == 1024 ? 1 : Backward ? (share <= 4 ? 4 : share <= 8 ? 2 : 1) : (share <= 8 ? 4 : 1);
}
// launch(unit, chunks, most) with the shape's values as constants.
template <bool Backward, int V, class F> void with_shape(const Shape &s, F &&launch) {
  bool done = false;
  auto is = [&](auto u, auto c, auto most) {
    if (done || s.chunks != decltype(c)::value || s.most != decltype(most)::value || (s.unit > 1) != (decltype(u)::value > 1))
      return;
    launch(u, c, most);
    done = true;
  };
  using std::integral_constant;
  integral_constant<int, V> v;
  integral_constant<int, 1> one;
  integral_constant<int, 2> two;
  integral_constant<int, 4> four;
  integral_constant<int, 8> eight;
  integral_constant<int, kWarpBlock> warps;
  integral_constant<int, 512> small;
  integral_constant<int, 1024> large;
  is(v, one, warps), is(v, two, warps), is(one, one, warps), is(one, eight, warps);
  if constexpr (Backward)
    is(v, one, small), is(v, two, small), is(v, two, large);
  else
    is(v, four, warps), is(v, eight, warps), is(v, four, small), is(v, four, large);
  if (!done)
    throw lapis::Error("Layer norm has no kernel for this row length");
}
// Blocks that fit on the device at once (asked once per kernel, block size and thread).
template <auto Kernel> int resident_blocks(int threads, int shared = 0) {
  static thread_local int known[33] = {};
  int &b = known[threads / 32];
  if (!b) {
    lapis::check(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&b, Kernel, threads, shared));
    b = std::max(b, 1);
  }
  return b * sm_count();
}
// Upper bound of a backward pass's partial rows (its grid): 148 SMs hold at most 8 blocks of 256
// threads each; other devices may hold more blocks, the grid is cut at this number.
constexpr int kMostParts = 1184;
constexpr int kSpanColumns = 12; // of a thread, backward
int wide_parts(long long rows) { return int(std::min<long long>(rows, 32)); }
// Whether spans are used, for rows that allow no wide loads: from 128 elements on, as far as their
// place (and gamma and beta) fits in shared memory.  Rows that lie without gaps form spans of up to 64
// KiB a block, a multiple of 8 rows with a warp each, while two blocks fit an SM; other rows, and longer
// ones, are a span each for a block of 512 or 1024 threads.
bool span_of(int type, long long rows, long long width, bool contiguous, int arrays, Span &s, int &shared, bool &block) {
  const int b = bytes_of(type);
  const long long row = width * b;
  if (width < kShort)
    return false;
  block = !contiguous || 8 * row * arrays + 2 * row > 110000;
  // (As few rows to a span as give every SM four.)
  s.rows = block ? 1 : int(8 * std::max(1ll, std::min({32ll, 65536 / (row * 8 * arrays), rows / (32ll * sm_count())})));
  const long long place = (s.rows * row + 31) / 16 * 16, all = place * arrays + 2 * row;
  s.bytes = int(std::min(place, 1ll << 30));
  shared = int(std::min(all, 1ll << 30));
  return all <= 216 * 1024 && (arrays == 1 || width <= kSpanColumns * (block ? 1024 : 256));
}
template <auto Kernel> int span_blocks(int shared, int threads) {
  static thread_local int device = -1;
  int now = 0;
  lapis::check(cudaGetDevice(&now));
  if (device != now) {
    lapis::check(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 216 * 1024));
    device = now;
  }
  // Per SM: shared memory (228 KiB, some of them each block's own) and registers.
  return std::max(1, std::min(1536 / threads, 233472 / (shared + 6144))) * sm_count();
}
} // namespace

void layer_norm(const Norm &a, cudaStream_t stream) {
  with_type(a.type, [&](auto tag) {
    using T = decltype(tag);
    constexpr int V = 16 / int(sizeof(T));
    bool vectors = a.width % V == 0 && aligned16(a.x) && aligned16(a.y) && aligned16(a.gamma) &&
                   aligned16(a.beta) && (a.rows == 1 || (a.ldx % V == 0 && a.ldy % V == 0));
    Shape s = shape_of(a.type, a.width, vectors, false);
    Span span;
    int shared = 0;
    bool block = false;
    if (!vectors && span_of(a.type, a.rows, a.width, a.ldx == a.width && a.ldy == a.width, 1, span, shared, block)) {
      auto go = [&](auto whole) {
        constexpr bool Block = decltype(whole)::value;
        constexpr auto kernel = span_norm_kernel<T, Block>;
        const int threads = !Block ? 256 : a.width <= 8192 ? 512 : 1024;
        const int grid = int(std::min<long long>((a.rows + span.rows - 1) / span.rows, span_blocks<kernel>(shared, threads)));
        lapis::launch(kernel, grid, threads, shared, stream, a, span);
      };
      block ? go(std::true_type{}) : go(std::false_type{});
    } else if (s.wide) {
      int grid = int(std::min<long long>(a.rows, resident_blocks<wide_norm_kernel<T>>(kWideThreads)));
      lapis::launch(wide_norm_kernel<T>, grid, kWideThreads, 0, stream, a);
    } else {
      with_shape<false, V>(s, [&](auto unit, auto chunks, auto most) {
        constexpr int U = decltype(unit)::value, C = decltype(chunks)::value, M = decltype(most)::value;
        constexpr int R = rows_of<false>(C * U, M);
        constexpr auto kernel = layer_norm_kernel<T, U, C, R, M>;
        const int threads = M == kWarpBlock ? kWarpBlock : s.threads;
        const long long high = (long long)R * (M == kWarpBlock ? kWarpBlock / s.threads : 1);
        constexpr int shared = M == kWarpBlock && C >= kSharedChunks ? 2 * C * 32 * U * int(sizeof(T)) : 0;
        const int grid = int(std::min<long long>((a.rows + high - 1) / high, resident_blocks<kernel>(threads, shared)));
        lapis::launch(kernel, grid, threads, shared, stream, a, s.threads);
      });
    }
    lapis::check(cudaGetLastError());
  });
}

long long layer_norm_backward_workspace(int type, long long rows, long long width) {
  // Partial rows: never more than one per row of x, nor than a grid's blocks.  Rows longer than registers
  // (2048 units) and spans (12 columns a thread) hold, whatever their alignment, have few.
  const bool wide = width > std::max(2048 * (16 / bytes_of(type)), kSpanColumns * 1024);
  return (wide ? wide_parts(rows) : std::min<long long>(rows, kMostParts)) * 2 * width * 4;
}

void layer_norm_backward(const NormBackward &a, void *workspace, cudaStream_t stream) {
  if (!a.dx && !a.dgamma && !a.dbeta)
    return;
  with_type(a.type, [&](auto tag) {
    using T = decltype(tag);
    constexpr int V = 16 / int(sizeof(T));
    bool params = a.dgamma || a.dbeta;
    float *partial = params ? static_cast<float *>(workspace) : nullptr;
    int parts = 0;
    if (a.rows) {
      bool vectors = a.width % V == 0 && aligned16(a.x) && aligned16(a.dy) && aligned16(a.dx) &&
                     aligned16(a.gamma) && aligned16(a.beta) &&
                     (a.rows == 1 || (a.ldx % V == 0 && a.lddy % V == 0 && a.lddx % V == 0));
      Shape s = shape_of(a.type, a.width, vectors, true);
      Span span;
      int shared = 0;
      bool block = false;
      const bool contiguous = a.ldx == a.width && a.lddy == a.width && (!a.dx || a.lddx == a.width);
      if (!vectors && span_of(a.type, a.rows, a.width, contiguous, 2, span, shared, block)) {
        auto go = [&](auto columns, auto whole) {
          constexpr bool Block = decltype(whole)::value;
          constexpr auto kernel = span_norm_backward_kernel<T, decltype(columns)::value, Block>;
          const int threads = !Block ? 256 : a.width <= 6144 ? 512 : 1024;
          parts = int(std::min<long long>({(a.rows + span.rows - 1) / span.rows,
                                           (long long)span_blocks<kernel>(shared, threads), (long long)kMostParts}));
          lapis::launch(kernel, parts, threads, shared, stream, a, span, partial);
        };
        using std::integral_constant;
        const bool narrow = a.width <= 4 * (block ? 512 : 256);
        if (block)
          narrow ? go(integral_constant<int, 4>{}, std::true_type{}) : go(integral_constant<int, kSpanColumns>{}, std::true_type{});
        else
          narrow ? go(integral_constant<int, 4>{}, std::false_type{}) : go(integral_constant<int, kSpanColumns>{}, std::false_type{});
      } else if (s.wide) {
        if (a.dx) {
          int grid = int(std::min<long long>(a.rows, resident_blocks<wide_norm_backward_kernel<T>>(kWideThreads)));
          if (params && a.dx == a.dy)
            grid = 0; // the parameters' gradients read dy first
          if (grid)
            lapis::launch(wide_norm_backward_kernel<T>, grid, kWideThreads, 0, stream, a);
        }
        if (params) {
          parts = wide_parts(a.rows);
          lapis::launch(wide_params_kernel<T>, dim3(unsigned((a.width + 255) / 256), unsigned(parts)), 256, 0, stream,
                        a, partial);
          if (a.dx && a.dx == a.dy)
            lapis::launch(wide_norm_backward_kernel<T>,
                          int(std::min<long long>(a.rows, resident_blocks<wide_norm_backward_kernel<T>>(kWideThreads))),
                          kWideThreads, 0, stream, a);
        }
      } else {
        with_shape<true, V>(s, [&](auto unit, auto chunks, auto most) {
          constexpr int U = decltype(unit)::value, C = decltype(chunks)::value, M = decltype(most)::value;
          constexpr int R = rows_of<true>(C * U, M);
          constexpr auto kernel = layer_norm_backward_kernel<T, U, C, R, M>;
          const int threads = M == kWarpBlock ? kWarpBlock : s.threads;
          const long long high = (long long)R * (M == kWarpBlock ? kWarpBlock / s.threads : 1);
          parts = int(std::min<long long>(
              {(a.rows + high - 1) / high, (long long)resident_blocks<kernel>(threads), (long long)kMostParts}));
          lapis::launch(kernel, parts, threads, 0, stream, a, s.threads, partial);
        });
      }
      lapis::check(cudaGetLastError());
    }
    if (params) {
      dim3 grid(unsigned((a.width + 31) / 32), 2);
      lapis::launch(column_sum_kernel<T>, grid, 1024, 0, stream, partial, parts, 2, a.width,
                    static_cast<T *>(a.dgamma), static_cast<T *>(a.dbeta));
      lapis::check(cudaGetLastError());
    }
  });
}
} // namespace op
} // namespace mace
