// Dense layer and layer norm: the launches behind include/mace/operators.h.  Arguments have
// been checked by the C entries (operators.cpp).
#pragma once
#include "lapis/runtime.hpp"

namespace mace {
namespace op {
enum Type { F32 = 0, BF16 = 1, F16 = 2 };
enum Activation { None = 0, Silu = 1, Gelu = 2, Relu = 3 };
inline int bytes_of(int type) { return type == F32 ? 4 : 2; }

struct Dense {
  int type;
  long long rows, inputs, outputs;
  const void *x;
  long long ldx;
  const void *weight;
  long long ldw;
  const void *bias;
  int activation;
  const void *residual;
  long long ldr;
  void *y;
  long long ldy;
  void *z;
  long long ldz;
};
struct DenseBackward {
  int type;
  long long rows, inputs, outputs;
  const void *dy;
  long long lddy;
  const void *x;
  long long ldx;
  const void *weight;
  long long ldw;
  int activation;
  const void *z;
  long long ldz;
  void *dx;
  long long lddx;
  void *dweight;
  long long lddw;
  void *dbias;
};
struct Norm {
  int type;
  long long rows, width;
  const void *x;
  long long ldx;
  const void *gamma, *beta;
  float eps;
  int activation;
  void *y;
  long long ldy;
  float *mean, *rstd;
};
struct NormBackward {
  int type;
  long long rows, width;
  const void *dy;
  long long lddy;
  const void *x;
  long long ldx;
  const float *mean, *rstd;
  const void *gamma, *beta;
  int activation;
  void *dx;
  long long lddx;
  void *dgamma, *dbeta;
};

long long dense_workspace(const Dense &);
void dense(const Dense &, void *workspace, cudaStream_t);
long long dense_backward_workspace(const DenseBackward &);
void dense_backward(const DenseBackward &, void *workspace, cudaStream_t);
void layer_norm(const Norm &, cudaStream_t);
long long layer_norm_backward_workspace(int type, long long rows, long long width);
void layer_norm_backward(const NormBackward &, void *workspace, cudaStream_t);
} // namespace op
} // namespace mace
