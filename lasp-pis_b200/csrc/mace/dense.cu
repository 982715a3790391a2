// Dense layer, forward and backward: y = act(x W^T + b) + r; dx = dz W, dW = dz^T x, db = sum dz.
//
// The three products are one kernel over operands with two strides each:
//   out(i, j) = sum_k P(i, k) Q(j, k)
//   forward  P = x (rows, inputs),  Q = W   (outputs, inputs)
//   dx       P = dz (rows, outputs), Q = W^T (inputs, outputs)
//   dW       P = dz^T (outputs, rows), Q = x^T (inputs, rows)
// 64 x 64 output tiles, 4 x 4 per thread, float accumulation.
#include "operators.cuh"
#include <algorithm>

namespace mace {
namespace op {
namespace {
struct Product {
  long long I, J, K;
  const void *p;
  long long pi, pk; // strides of P in elements
  const void *q;
  long long qj, qk;
  const void *bias; // [J]
  int activation;
  const void *residual;
  long long ldr;
  void *out;
  long long ldo;
  void *z;
  long long ldz;
};

template <class T> __global__ void __launch_bounds__(256) product_kernel(const __grid_constant__ Product a) {
  constexpr bool Fast = sizeof(T) == 2;
  __shared__ float ps[16][65], qs[16][65];
  const T *p = static_cast<const T *>(a.p), *q = static_cast<const T *>(a.q);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const long long i0 = (long long)blockIdx.x * 64, j0 = (long long)blockIdx.y * 64;
  float acc[4][4] = {};
  for (long long k0 = 0; k0 < a.K; k0 += 16) {
    for (int e = threadIdx.x; e < 64 * 16; e += 256) {
      // Consecutive threads walk the contiguous index.
      int kp = a.pk == 1 ? e & 15 : e >> 6, ip = a.pk == 1 ? e >> 4 : e & 63;
      int kq = a.qk == 1 ? e & 15 : e >> 6, jq = a.qk == 1 ? e >> 4 : e & 63;
      ps[kp][ip] = i0 + ip < a.I && k0 + kp < a.K ? to_float(p[(i0 + ip) * a.pi + (k0 + kp) * a.pk]) : 0.f;
      qs[kq][jq] = j0 + jq < a.J && k0 + kq < a.K ? to_float(q[(j0 + jq) * a.qj + (k0 + kq) * a.qk]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = fmaf(ps[k][ty + 16 * i], qs[k][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      long long r = i0 + ty + 16 * i, c = j0 + tx + 16 * j;
      if (r >= a.I || c >= a.J)
        continue;
      float v = acc[i][j] + (a.bias ? to_float(static_cast<const T *>(a.bias)[c]) : 0.f);
      if (a.z)
        static_cast<T *>(a.z)[r * a.ldz + c] = from_float<T>(v);
      v = activate<Fast>(v, a.activation);
      if (a.residual)
        v += to_float(static_cast<const T *>(a.residual)[r * a.ldr + c]);
      static_cast<T *>(a.out)[r * a.ldo + c] = from_float<T>(v);
    }
}

// dz = dy act'(z) into dz [rows][outputs] (NULL: not written) and the partial column sums of its
// float values, [gridDim.y][outputs] (NULL: not wanted).
template <class T>
__global__ void __launch_bounds__(256) gradient_kernel(const __grid_constant__ DenseBackward a, T *dz, float *partial) {
  constexpr bool Fast = sizeof(T) == 2;
  long long c = (long long)blockIdx.x * 256 + threadIdx.x;
  if (c >= a.outputs)
    return;
  float sum = 0.f;
  for (long long r = blockIdx.y; r < a.rows; r += gridDim.y) {
    float v = to_float(static_cast<const T *>(a.dy)[r * a.lddy + c]);
    if (a.activation != None)
      v *= slope<Fast>(to_float(static_cast<const T *>(a.z)[r * a.ldz + c]), a.activation);
    sum += v;
    if (dz)
      dz[r * a.outputs + c] = from_float<T>(v);
  }
  if (partial)
    partial[blockIdx.y * a.outputs + c] = sum;
}

int parts_of(long long rows) { return int(std::min<long long>(rows, 256)); }
long long round16(long long n) { return (n + 15) / 16 * 16; }

void product(int type, const Product &p, cudaStream_t stream) {
  with_type(type, [&](auto tag) {
    dim3 grid(unsigned((p.I + 63) / 64), unsigned((p.J + 63) / 64));
    lapis::launch(product_kernel<decltype(tag)>, grid, 256, 0, stream, p);
    lapis::check(cudaGetLastError());
  });
}
} // namespace

long long dense_workspace(const Dense &) { return 0; }
void dense(const Dense &d, void *, cudaStream_t stream) {
  product(d.type,
          {d.rows, d.outputs, d.inputs, d.x, d.ldx, 1, d.weight, d.ldw, 1, d.bias, d.activation, d.residual, d.ldr,
           d.y, d.ldy, d.z, d.ldz},
          stream);
}

long long dense_backward_workspace(const DenseBackward &d) {
  return round16(parts_of(d.rows) * d.outputs * 4) +
         (d.activation != None ? round16(d.rows * d.outputs * bytes_of(d.type)) : 0);
}
void dense_backward(const DenseBackward &d, void *workspace, cudaStream_t stream) {
  with_type(d.type, [&](auto tag) {
    using T = decltype(tag);
    int parts = parts_of(d.rows);
    float *partial = d.dbias ? static_cast<float *>(workspace) : nullptr;
    T *dz = d.activation != None && (d.dx || d.dweight)
                ? reinterpret_cast<T *>(static_cast<char *>(workspace) + round16(parts * d.outputs * 4))
                : nullptr;
    if (d.rows && (dz || partial))
      lapis::launch(gradient_kernel<T>, dim3(unsigned((d.outputs + 255) / 256), unsigned(parts)), 256, 0, stream, d, dz,
                    partial);
    if (d.dbias)
      lapis::launch(column_sum_kernel<T>, dim3(unsigned((d.outputs + 31) / 32), 1), 1024, 0, stream, partial, parts, 1,
                    d.outputs, static_cast<T *>(d.dbias), static_cast<T *>(nullptr));
    if (d.dbias || (d.rows && dz))
      lapis::check(cudaGetLastError());
    const void *g = dz ? dz : d.dy;
    long long ldg = dz ? d.outputs : d.lddy;
    if (d.dx && d.rows)
      product(d.type, {d.rows, d.inputs, d.outputs, g, ldg, 1, d.weight, 1, d.ldw, nullptr, None, nullptr, 0, d.dx,
                       d.lddx, nullptr, 0},
              stream);
    if (d.dweight)
      product(d.type, {d.outputs, d.inputs, d.rows, g, 1, ldg, d.x, 1, d.ldx, nullptr, None, nullptr, 0, d.dweight,
                       d.lddw, nullptr, 0},
              stream);
  });
}
} // namespace op
} // namespace mace
