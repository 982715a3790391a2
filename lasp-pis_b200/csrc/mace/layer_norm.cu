// Layer norm with an activation, forward and backward.
//
//   forward   m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), xhat = (x - m) r,
//             y = act(xhat gamma + beta)
//   backward  dz = dy act'(xhat gamma + beta), g = dz gamma,
//             dx = r (g - mean(g) - xhat mean(g xhat)),
//             dgamma = sum over rows of dz xhat, dbeta = sum over rows of dz
//
// One pass over the data: a row stays in the registers of its group of threads (part of a warp,
// or a block for wide rows) between its statistics and its result, and each row's loads are
// issued before the arithmetic of the row before.  The variance is taken about a first mean and
// corrected for that mean's own rounding, so a row far from zero loses nothing.  A group walks
// the rows with a fixed set of columns per thread, so gamma, beta and the parameters' gradients
// stay in registers too; each block writes one partial row of dgamma and dbeta, and a second
// launch adds the partial rows in a fixed order.
#include "operators.cuh"
#include <algorithm>
#include <type_traits>

namespace mace {
namespace op {
namespace {
constexpr int kWarpBlock = 256; // threads of a block whose rows belong to parts of warps

// Sum of two values over a row's group: G lanes (G <= 32, power of two), or the block.
template <bool Warp> __device__ __forceinline__ float2 group_sum(float2 v, int G, float2 *shared) {
  int top = Warp ? G >> 1 : 16;
  for (int o = top; o; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if (Warp)
    return v;
  int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if (!lane)
    shared[warp] = v;
  __syncthreads();
  v = lane < warps ? shared[lane] : make_float2(0.f, 0.f);
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  return v;
}

// T elements in units of U, C units per thread (columns (c G + t) U ...), a row per group of G
// threads: G lanes of a warp (Warp), or the block.
template <class T, int U, int C, bool Warp>
__global__ void __launch_bounds__(Warp ? kWarpBlock : 1024) layer_norm_kernel(const __grid_constant__ Norm a, int lanes) {
  constexpr bool Fast = sizeof(T) == 2;
  using Un = Unit<T, U>;
  __shared__ float2 shared[2][32];
  const int G = Warp ? lanes : blockDim.x, t = Warp ? threadIdx.x & (G - 1) : threadIdx.x;
  const int per_block = Warp ? kWarpBlock / G : 1, group = Warp ? threadIdx.x / G : 0;
  const T *x = static_cast<const T *>(a.x);
  T *y = static_cast<T *>(a.y);
  const float inv_n = 1.f / float(a.width);
  Un gamma[C], beta[C];
  long long col[C];
  bool live[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    col[c] = (long long)(c * G + t) * U;
    live[c] = col[c] < a.width;
    if (live[c] && a.gamma)
      gamma[c] = *reinterpret_cast<const Un *>(static_cast<const T *>(a.gamma) + col[c]);
    if (live[c] && a.beta)
      beta[c] = *reinterpret_cast<const Un *>(static_cast<const T *>(a.beta) + col[c]);
  }
  const long long step = (long long)gridDim.x * per_block;
  long long base = (long long)blockIdx.x * per_block;
  Un next[C];
  auto load = [&](long long row) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (live[c] && row < a.rows)
        next[c] = *reinterpret_cast<const Un *>(x + row * a.ldx + col[c]);
  };
  load(base + group);
  for (; base < a.rows; base += step) {
    const long long row = base + group;
    const bool mine = row < a.rows;
    float v[C * U];
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        v[c * U + u] = live[c] && mine ? to_float(next[c].v[u]) : 0.f;
        s.x += v[c * U + u];
      }
    load(row + step);
    const float m1 = group_sum<Warp>(s, G, shared[0]).x * inv_n;
    s = make_float2(0.f, 0.f);
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (live[c])
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float d = v[c * U + u] -= m1;
          s.x += d;
          s.y = fmaf(d, d, s.y);
        }
    s = group_sum<Warp>(s, G, shared[1]);
    // The first mean's rounding error, and the variance about the corrected mean.
    const float fix = s.x * inv_n;
    const float var = fmaxf(fmaf(-fix, fix, s.y * inv_n), 0.f) + (s.y != s.y ? s.y : 0.f);
    const float r = Fast ? rsqrtf(var + a.eps) : 1.f / sqrtf(var + a.eps);
    if (!mine)
      continue;
    if (a.mean && !t) {
      a.mean[row] = m1 + fix;
      a.rstd[row] = Fast ? 1.f / sqrtf(var + a.eps) : r;
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (!live[c])
        continue;
      Un o;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float z = (v[c * U + u] - fix) * r;
        if (a.gamma)
          z *= to_float(gamma[c].v[u]);
        if (a.beta)
          z += to_float(beta[c].v[u]);
        o.v[u] = from_float<T>(activate<Fast>(z, a.activation));
      }
      *reinterpret_cast<Un *>(y + row * a.ldy + col[c]) = o;
    }
  }
}

// partial: [gridDim.x][2][width] (dgamma, dbeta), or NULL.
template <class T, int U, int C, bool Warp>
__global__ void __launch_bounds__(Warp ? kWarpBlock : 1024)
    layer_norm_backward_kernel(const __grid_constant__ NormBackward a, int lanes, float *partial) {
  constexpr bool Fast = sizeof(T) == 2;
  using Un = Unit<T, U>;
  __shared__ float2 shared[2][32];
  __shared__ float join[Warp ? kWarpBlock * C * U : 1];
  const int G = Warp ? lanes : blockDim.x, t = Warp ? threadIdx.x & (G - 1) : threadIdx.x;
  const int per_block = Warp ? kWarpBlock / G : 1, group = Warp ? threadIdx.x / G : 0;
  const T *x = static_cast<const T *>(a.x), *dy = static_cast<const T *>(a.dy);
  T *dx = static_cast<T *>(a.dx);
  const float inv_n = 1.f / float(a.width);
  Un gamma[C], beta[C];
  long long col[C];
  bool live[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    col[c] = (long long)(c * G + t) * U;
    live[c] = col[c] < a.width;
    if (live[c] && a.gamma)
      gamma[c] = *reinterpret_cast<const Un *>(static_cast<const T *>(a.gamma) + col[c]);
    if (live[c] && a.beta && a.activation != None)
      beta[c] = *reinterpret_cast<const Un *>(static_cast<const T *>(a.beta) + col[c]);
  }
  float sum_gamma[C * U] = {}, sum_beta[C * U] = {};
  const long long step = (long long)gridDim.x * per_block;
  long long base = (long long)blockIdx.x * per_block;
  Un next_x[C], next_dy[C];
  float next_mean = 0.f, next_r = 0.f;
  auto load = [&](long long row) {
    if (row >= a.rows)
      return;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (live[c]) {
        next_x[c] = *reinterpret_cast<const Un *>(x + row * a.ldx + col[c]);
        next_dy[c] = *reinterpret_cast<const Un *>(dy + row * a.lddy + col[c]);
      }
    next_mean = a.mean[row];
    next_r = a.rstd[row];
  };
  load(base + group);
  for (int k = 0; base < a.rows; base += step, k ^= 1) {
    const long long row = base + group;
    const bool mine = row < a.rows;
    const float mean = next_mean, r = next_r;
    float xh[C * U], g[C * U];
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = c * U + u;
        xh[i] = g[i] = 0.f;
        if (live[c] && mine) {
          xh[i] = (to_float(next_x[c].v[u]) - mean) * r;
          float gm = a.gamma ? to_float(gamma[c].v[u]) : 1.f, dz = to_float(next_dy[c].v[u]);
          if (a.activation != None)
            dz *= slope<Fast>(fmaf(xh[i], gm, a.beta ? to_float(beta[c].v[u]) : 0.f), a.activation);
          sum_gamma[i] = fmaf(dz, xh[i], sum_gamma[i]);
          sum_beta[i] += dz;
          g[i] = dz * gm;
          s.x += g[i];
          s.y = fmaf(g[i], xh[i], s.y);
        }
      }
    load(row + step);
    if (!dx)
      continue;
    s = group_sum<Warp>(s, G, shared[k]); // two buffers: a row's sums are read while the next are written
    if (!mine)
      continue;
    const float mg = s.x * inv_n, mgx = s.y * inv_n;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (!live[c])
        continue;
      Un o;
#pragma unroll
      for (int u = 0; u < U; ++u)
        o.v[u] = from_float<T>(r * (g[c * U + u] - fmaf(xh[c * U + u], mgx, mg)));
      *reinterpret_cast<Un *>(dx + row * a.lddx + col[c]) = o;
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
      for (int i = 0; i < C * U; ++i) // group-major: [group][c][u][t]
        join[(group * C * U + i) * G + t] = k ? sum_beta[i] : sum_gamma[i];
      __syncthreads();
      for (int j = threadIdx.x; j < C * U * G; j += kWarpBlock) {
        int i = j / G, tt = j % G;
        long long cc = (long long)((i / U) * G + tt) * U + i % U;
        float v = 0.f;
        for (int q = 0; q < per_block; ++q)
          v += join[q * C * U * G + j];
        if (cc < a.width)
          out[cc] = v;
      }
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (live[c])
#pragma unroll
          for (int u = 0; u < U; ++u)
            out[col[c] + u] = k ? sum_beta[c * U + u] : sum_gamma[c * U + u];
    }
  }
}

// ---------------- rows too wide for registers: loops over the row, read again from L2 ----------------
constexpr int kWideThreads = 1024;
template <class T> __global__ void __launch_bounds__(kWideThreads) wide_norm_kernel(const __grid_constant__ Norm a) {
  constexpr bool Fast = sizeof(T) == 2;
  __shared__ float2 shared[2][32];
  const float inv_n = 1.f / float(a.width);
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + row * a.ldx;
    T *y = static_cast<T *>(a.y) + row * a.ldy;
    float2 s = make_float2(0.f, 0.f);
    for (long long i = threadIdx.x; i < a.width; i += kWideThreads)
      s.x += to_float(x[i]);
    const float m1 = group_sum<false>(s, 0, shared[0]).x * inv_n;
    s = make_float2(0.f, 0.f);
    for (long long i = threadIdx.x; i < a.width; i += kWideThreads) {
      float d = to_float(x[i]) - m1;
      s.x += d;
      s.y = fmaf(d, d, s.y);
    }
    s = group_sum<false>(s, 0, shared[1]);
    const float fix = s.x * inv_n;
    const float var = fmaxf(fmaf(-fix, fix, s.y * inv_n), 0.f) + (s.y != s.y ? s.y : 0.f);
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
  __shared__ float2 shared[2][32];
  const float inv_n = 1.f / float(a.width);
  int k = 0;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, k ^= 1) {
    float2 s = make_float2(0.f, 0.f);
    for (long long i = threadIdx.x; i < a.width; i += kWideThreads) {
      float2 e = wide_element<T>(a, row, i);
      float g = e.y * (a.gamma ? to_float(static_cast<const T *>(a.gamma)[i]) : 1.f);
      s.x += g;
      s.y = fmaf(g, e.x, s.y);
    }
    s = group_sum<false>(s, 0, shared[k]);
    const float mg = s.x * inv_n, mgx = s.y * inv_n, r = a.rstd[row];
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

// How a row is laid over threads.
struct Shape {
  int unit, chunks, threads; // threads: lanes of a warp, or the block's threads
  bool warp, wide;
};
Shape shape_of(int type, long long width, bool vectors) {
  int unit = vectors ? 16 / bytes_of(type) : 1;
  long long units = (width + unit - 1) / unit;
  int most = vectors ? 4 : 16;
  Shape s{unit, 1, 0, false, false};
  if (units <= 32 * most) { // part of a warp, or a warp
    while (units > 32ll * s.chunks)
      s.chunks *= vectors ? 2 : 4;
    s.warp = true;
    s.threads = 1;
    while ((long long)s.threads * s.chunks < units)
      s.threads *= 2;
    return s;
  }
  s.chunks = vectors ? (units <= 1024 ? 1 : units <= 2048 ? 2 : 4) : (units <= 4096 ? 4 : 16);
  long long threads = (units + s.chunks - 1) / s.chunks;
  if (threads > 1024) {
    s.wide = true;
    return s;
  }
  s.threads = int((threads + 31) / 32 * 32);
  return s;
}
template <class F> void with_shape(const Shape &s, F &&f) {
  auto chunks = [&](auto warp) {
    using std::integral_constant;
    if (s.unit > 1) {
      if (s.chunks == 1)
        f(std::true_type{}, integral_constant<int, 1>{}, warp);
      else if (s.chunks == 2)
        f(std::true_type{}, integral_constant<int, 2>{}, warp);
      else
        f(std::true_type{}, integral_constant<int, 4>{}, warp);
    } else {
      if (s.chunks == 1)
        f(std::false_type{}, integral_constant<int, 1>{}, warp);
      else if (s.chunks == 4)
        f(std::false_type{}, integral_constant<int, 4>{}, warp);
      else
        f(std::false_type{}, integral_constant<int, 16>{}, warp);
    }
  };
  if (s.warp)
    chunks(std::true_type{});
  else
    chunks(std::false_type{});
}
// Blocks that fit on the device at once (asked once per kernel, block size and thread).
template <auto Kernel> int resident_blocks(int threads) {
  static thread_local int known[33] = {};
  int &b = known[threads / 32];
  if (!b) {
    lapis::check(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&b, Kernel, threads, 0));
    b = std::max(b, 1);
  }
  return b * sm_count();
}
// Upper bound of a backward pass's partial rows (its grid): 148 SMs hold at most 8 blocks of 256
// threads each; other devices may hold more blocks, the grid is cut at this number.
constexpr int kMostParts = 1184;
int wide_parts(long long rows) { return int(std::min<long long>(rows, 32)); }
} // namespace

void layer_norm(const Norm &a, cudaStream_t stream) {
  with_type(a.type, [&](auto tag) {
    using T = decltype(tag);
    constexpr int V = 16 / int(sizeof(T));
    bool vectors = a.width % V == 0 && aligned16(a.x) && aligned16(a.y) && aligned16(a.gamma) &&
                   aligned16(a.beta) && (a.rows == 1 || (a.ldx % V == 0 && a.ldy % V == 0));
    Shape s = shape_of(a.type, a.width, vectors);
    if (s.wide) {
      int grid = int(std::min<long long>(a.rows, resident_blocks<wide_norm_kernel<T>>(kWideThreads)));
      lapis::launch(wide_norm_kernel<T>, grid, kWideThreads, 0, stream, a);
    } else {
      with_shape(s, [&](auto vec, auto chunks, auto warp) {
        constexpr auto kernel =
            layer_norm_kernel<T, decltype(vec)::value ? V : 1, decltype(chunks)::value, decltype(warp)::value>;
        int threads = s.warp ? kWarpBlock : s.threads;
        long long blocks = s.warp ? (a.rows + kWarpBlock / s.threads - 1) / (kWarpBlock / s.threads) : a.rows;
        int grid = int(std::min<long long>(blocks, resident_blocks<kernel>(threads)));
        lapis::launch(kernel, grid, threads, 0, stream, a, s.threads);
      });
    }
    lapis::check(cudaGetLastError());
  });
}

long long layer_norm_backward_workspace(int, long long rows, long long width) {
  // Partial rows: never more than one per row of x, nor than a grid's blocks.
  return std::min<long long>(rows, kMostParts) * 2 * width * 4;
}

void layer_norm_backward(const NormBackward &a, void *workspace, cudaStream_t stream) {
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
      Shape s = shape_of(a.type, a.width, vectors);
      if (s.wide) {
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
        with_shape(s, [&](auto vec, auto chunks, auto warp) {
          constexpr auto kernel =
              layer_norm_backward_kernel<T, decltype(vec)::value ? V : 1, decltype(chunks)::value, decltype(warp)::value>;
          int threads = s.warp ? kWarpBlock : s.threads;
          long long blocks = s.warp ? (a.rows + kWarpBlock / s.threads - 1) / (kWarpBlock / s.threads) : a.rows;
          parts = int(std::min<long long>({blocks, (long long)resident_blocks<kernel>(threads), (long long)kMostParts}));
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
