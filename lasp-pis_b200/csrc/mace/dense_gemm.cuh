// Tensor maps, tiles and the epilogue shared by the dense layer's matrix products.
#pragma once
#include "operators.cuh"
#include "tcgen05.cuh"
#include <algorithm>
#include <mutex>
#include <string>

namespace mace {
namespace op {
// out(i, j) = sum_k P(i, k) Q(j, k), i < I, j < J, k < K, then the epilogue.  An operand is an
// array with row distance ld: [I][K] (k contiguous), or [K][I] (turned).
struct Operand {
  const void *p;
  long long ld;
  bool turned;
};
struct Epilogue {
  const void *bias; // [J]
  int activation;
  const void *residual;
  long long ldr;
  void *out;
  long long ldo;
  void *z;
  long long ldz;
  int vectors; // every array's rows start on 16-byte boundaries and J is a multiple of 16 bytes
};
struct Product {
  int type;
  long long I, J, K;
  Operand p, q;
  Epilogue e;
};

// Output tiles in groups of kBand rows of tiles, column by column within a group: the tiles that
// run together share their operands in L2.
struct Tiles {
  long long nI, nJ, count;
  __host__ __device__ Tiles(long long I, long long J, int bi, int bj)
      : nI((I + bi - 1) / bi), nJ((J + bj - 1) / bj), count(nI * nJ) {}
  __device__ __forceinline__ void at(long long t, long long &i, long long &j) const {
    constexpr long long kBand = 16;
    long long band = t / (kBand * nJ), first = band * kBand, rows = min(kBand, nI - first), r = t - first * nJ;
    i = first + r % rows;
    j = r / rows;
  }
};

// One value of the product through the epilogue: z, then the output value.
template <class T>
__device__ __forceinline__ void finish(const Epilogue &e, long long row, long long col, float v) {
  constexpr bool Fast = sizeof(T) == 2;
  if (e.bias)
    v += to_float(static_cast<const T *>(e.bias)[col]);
  if (e.z)
    static_cast<T *>(e.z)[row * e.ldz + col] = from_float<T>(v);
  v = activate<Fast>(v, e.activation);
  if (e.residual)
    v += to_float(static_cast<const T *>(e.residual)[row * e.ldr + col]);
  static_cast<T *>(e.out)[row * e.ldo + col] = from_float<T>(v);
}
// N neighbouring values (N a multiple of a 16-byte unit), for arrays that allow vectors.
template <class T, int N>
__device__ __forceinline__ void finish_row(const Epilogue &e, long long row, long long col, float (&v)[N]) {
  constexpr bool Fast = sizeof(T) == 2;
  constexpr int U = 16 / int(sizeof(T));
  using Un = Unit<T, U>;
#pragma unroll
  for (int k = 0; k < N; k += U) {
    if (e.bias) {
      Un b = *reinterpret_cast<const Un *>(static_cast<const T *>(e.bias) + col + k);
#pragma unroll
      for (int u = 0; u < U; ++u)
        v[k + u] += to_float(b.v[u]);
    }
    if (e.z) {
      Un z;
#pragma unroll
      for (int u = 0; u < U; ++u)
        z.v[u] = from_float<T>(v[k + u]);
      *reinterpret_cast<Un *>(static_cast<T *>(e.z) + row * e.ldz + col + k) = z;
    }
    if (e.activation != None)
#pragma unroll
      for (int u = 0; u < U; ++u)
        v[k + u] = activate<Fast>(v[k + u], e.activation);
    if (e.residual) {
      Un r = *reinterpret_cast<const Un *>(static_cast<const T *>(e.residual) + row * e.ldr + col + k);
#pragma unroll
      for (int u = 0; u < U; ++u)
        v[k + u] += to_float(r.v[u]);
    }
    Un o;
#pragma unroll
    for (int u = 0; u < U; ++u)
      o.v[u] = from_float<T>(v[k + u]);
    *reinterpret_cast<Un *>(static_cast<T *>(e.out) + row * e.ldo + col + k) = o;
  }
}

// A warp's 32 x 32 block of the product: lane = row, v = its columns from col0.  Rows that allow
// no vectors go through `stage` (32 x 33 floats), so that neighbouring lanes write neighbouring
// columns.  partial != NULL: the float values go to partial[row * J + col] instead.
template <class T>
__device__ __forceinline__ void finish_block(const Epilogue &e, float *partial, long long I, long long J,
                                             long long row0, long long col0, float (&v)[32], float *stage) {
  const int lane = threadIdx.x & 31;
  if (partial ? J % 4 == 0 : e.vectors) {
    long long row = row0 + lane;
    if (row < I) {
      if (partial) {
#pragma unroll
        for (int k = 0; k < 32; k += 4)
          if (col0 + k < J)
            *reinterpret_cast<float4 *>(partial + row * J + col0 + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
      } else if (col0 + 32 <= J) {
        finish_row<T>(e, row, col0, v);
      } else {
        constexpr int U = 16 / int(sizeof(T));
#pragma unroll
        for (int k = 0; k < 32; k += U)
          if (col0 + k < J) {
            float w[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
              w[u] = v[k + u];
            finish_row<T>(e, row, col0 + k, w);
          }
      }
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 32; ++k)
    stage[lane * 33 + k] = v[k];
  __syncwarp();
  long long col = col0 + lane;
  int rows = int(min(32ll, I - row0));
  if (col < J)
    for (int r = 0; r < rows; ++r) {
      if (partial)
        partial[(row0 + r) * J + col] = stage[r * 33 + lane];
      else
        finish<T>(e, row0 + r, col, stage[r * 33 + lane]);
    }
  __syncwarp();
}

// ---------------- host ----------------
inline long long round_up(long long n, long long to) { return (n + to - 1) / to * to; }

// Tensor map of a [rows][cols] array of 16-bit or float elements with row distance ld, in boxes of
// box_rows rows by 128 bytes, SWIZZLE_128B; elements outside the array read as zero.
CUtensorMap tile_map(int type, const void *base, long long rows, long long cols, long long ld, int box_rows);
// Whether TMA can read the array in place: 16-byte aligned rows.
inline bool tma_ready(int type, const void *p, long long rows, long long ld) {
  return aligned16(p) && (rows <= 1 || ld * bytes_of(type) % 16 == 0);
}

// The products of 16-bit types (dense_gemm16.cu): operands that TMA can read; workspace of
// product16_workspace bytes.
long long product16_workspace(long long I, long long J, long long K);
void product16(const Product &, void *workspace, cudaStream_t);
// Sum of `parts` float products [parts][I][J], through the epilogue.
void finish_parts(int type, const Epilogue &, const float *partial, int parts, long long I, long long J, cudaStream_t);
} // namespace op
} // namespace mace
