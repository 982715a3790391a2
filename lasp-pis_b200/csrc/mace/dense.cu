// Dense layer, forward and backward: y = act(x W^T + b) + r; dx = dz W, dW = dz^T x, db = sum dz
// with dz = dy act'(z).
//
// The three products are out(i, j) = sum_k P(i, k) Q(j, k):
//   forward  P = x (rows, inputs),   Q = W (outputs, inputs)
//   dx       P = dz (rows, outputs), Q = W turned (inputs, outputs)
//   dW       P = dz turned (outputs, rows), Q = x turned (inputs, rows)
// 16-bit types run on dense_gemm16.cu, floats on dense_gemm32.cu.  Around them: a copy of
// operands whose rows TMA cannot read in place, and one pass over dy (and z) that writes dz and sums
// its columns.
#include "dense_gemm.cuh"

namespace mace {
namespace op {
namespace {
// ---------------- few inputs ----------------
// y for few inputs (the radial network's first layer has 10), rows of any alignment: float arithmetic,
// 64 x 64 tiles, 4 rows x 4 columns per thread, x and W in shared memory.  The tensor cores' slab of 64
// would be mostly padding, and rows that TMA cannot read would be copied first: 5417 x 10 -> 64 f32 takes
// 3.4 us here and 13 us there.
constexpr int kNarrow = 32;
// Up to 32 inputs while the result is small (5417 x 32 -> 64: 4.5 us, 6.7 with 40 inputs on the tensor
// cores; 84613 x 32 -> 64: 19 us against 16), and up to 12 for floats (84613 x 8 -> 1280: 168 us
// against 195; bf16: 145 against 76).
bool is_narrow(const Dense &d) {
  return (d.inputs <= kNarrow && d.rows <= (1 << 20) / d.outputs) || (d.type == F32 && d.inputs <= 12);
}
template <class T> __global__ void __launch_bounds__(256) narrow_kernel(const __grid_constant__ Dense d, int vectors) {
  constexpr bool Fast = sizeof(T) == 2;
  using Un = Unit<T, 4>;
  __shared__ float xs[kNarrow][68], ws[kNarrow][68];
  const int K = int(d.inputs), tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const unsigned across = unsigned((d.outputs + 63) / 64);
  const long long i0 = (long long)(blockIdx.x / across) * 64, j0 = (long long)(blockIdx.x % across) * 64;
  for (int e = threadIdx.x; e < 64 * K; e += 256) {
    const int r = e / K, k = e - r * K;
    xs[k][r] = i0 + r < d.rows ? to_float(static_cast<const T *>(d.x)[(i0 + r) * d.ldx + k]) : 0.f;
    ws[k][r] = j0 + r < d.outputs ? to_float(static_cast<const T *>(d.weight)[(j0 + r) * d.ldw + k]) : 0.f;
  }
  __syncthreads();
  float acc[4][4] = {};
#pragma unroll 4
  for (int k = 0; k < K; ++k) {
    const float4 w = *reinterpret_cast<const float4 *>(&ws[k][4 * tx]), v = *reinterpret_cast<const float4 *>(&xs[k][4 * ty]);
    const float a[4] = {v.x, v.y, v.z, v.w}, b[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
  }
  const long long col = j0 + 4 * tx;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long row = i0 + 4 * ty + i;
    if (row >= d.rows || col >= d.outputs)
      continue;
    if (!vectors) {
      const Epilogue e{d.bias, d.activation, d.residual, d.ldr, d.y, d.ldy, d.z, d.ldz};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col + j < d.outputs)
          finish<T>(e, row, col + j, acc[i][j]);
      continue;
    }
    float v[4], r[4];
    if (d.bias) {
      unpack<T, 4>(*reinterpret_cast<const Un *>(static_cast<const T *>(d.bias) + col), r);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        acc[i][j] += r[j];
    }
    if (d.z)
      *reinterpret_cast<Un *>(static_cast<T *>(d.z) + row * d.ldz + col) = pack<T, 4>(acc[i]);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      v[j] = acc[i][j];
    activate_all<Fast>(v, d.activation);
    if (d.residual) {
      unpack<T, 4>(*reinterpret_cast<const Un *>(static_cast<const T *>(d.residual) + row * d.ldr + col), r);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[j] += r[j];
    }
    *reinterpret_cast<Un *>(static_cast<T *>(d.y) + row * d.ldy + col) = pack<T, 4>(v);
  }
}
void narrow(const Dense &d, cudaStream_t stream) {
  const int bytes = 4 * bytes_of(d.type);
  auto fits = [&](const void *p, long long ld) {
    return !p || (reinterpret_cast<uintptr_t>(p) % unsigned(bytes) == 0 && (d.rows <= 1 || ld % 4 == 0));
  };
  const bool vectors = d.outputs % 4 == 0 && fits(d.y, d.ldy) && fits(d.z, d.ldz) && fits(d.residual, d.ldr) && fits(d.bias, 4);
  const double blocks = double((d.rows + 63) / 64) * double((d.outputs + 63) / 64);
  if (blocks > 2e9)
    throw lapis::Error("The product has too many tiles");
  with_type(d.type, [&](auto tag) {
    lapis::launch(narrow_kernel<decltype(tag)>, dim3(unsigned(blocks)), 256, 0, stream, d, int(vectors));
    lapis::check(cudaGetLastError());
  });
}

// ---------------- few rows ----------------
// y for up to kFew rows (a token, or a few): W is read once and HBM bounds the call, so the warps only
// stream it.  A warp has four rows of W under way, eight 16-byte loads per lane in flight, finds x in
// L1, and `ks` warps of a block share them along k where there are few outputs.  Float
// sums: lanes, then the warps in order.  M: d.rows or a little more (rows past the last read it).
// Turned: the same for a few outputs, with x in W's place and W in x's.  gridDim.y: further groups of M
// rows (see is_small).
constexpr int kFew = 8, kFewOutputs = 4;
// A unit that is read once, in the order written (all of a step's loads before the first use).
template <class T, int U> __device__ __forceinline__ Unit<T, U> stream_unit(const T *p) {
  Unit<T, U> u;
  if constexpr (sizeof(u) == 16) {
    uint4 w;
    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                 : "l"(p));
    memcpy(&u, &w, 16);
  } else {
    u = *reinterpret_cast<const Unit<T, U> *>(p);
  }
  return u;
}
template <class T, int U, int M, bool Turned>
__global__ void __launch_bounds__(256) few_rows_kernel(const __grid_constant__ Dense d, int ks) {
  constexpr int R = kFewOutputs;
  const long long many = Turned ? d.rows : d.outputs, few = Turned ? d.outputs : d.rows, ldm = Turned ? d.ldx : d.ldw,
                  ldf = Turned ? d.ldw : d.ldx;
  using Un = Unit<T, U>;
  __shared__ float parts[8][R * M];
  const T *const x = static_cast<const T *>(Turned ? d.weight : d.x);
  const long long few0 = (long long)blockIdx.y * M;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = warp % ks, slot = warp / ks, slots = 8 / ks;
  // Groups of four outputs go round the blocks first, so that every SM reads as much.
  const long long groups = (many + R - 1) / R;
  for (long long first = 0; first < groups; first += (long long)gridDim.x * slots) {
    const long long group = first + (long long)slot * gridDim.x + blockIdx.x;
    const long long n0 = group * R; // rows past the end: the last row, not written
    const long long units = group < groups ? d.inputs / U : 0;
    const T *w[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
      w[r] = static_cast<const T *>(Turned ? d.x : d.weight) + min(n0 + r, many - 1) * ldm;
    float acc[R][M] = {};
    auto add = [&](const Un (&u)[R], const Un (&v)[M]) {
#pragma unroll
      for (int m = 0; m < M; ++m) {
        float xv[U];
        unpack<T, U>(v[m], xv);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float wv[U];
          unpack<T, U>(u[r], wv);
#pragma unroll
          for (int i = 0; i < U; ++i)
            acc[r][m] = fmaf(wv[i], xv[i], acc[r][m]);
        }
      }
    };
    const int step = 32 * ks;
    long long at = sub * 32 + lane;
    for (; at + step < units; at += 2 * step) {
      Un a[R], b[R], v[M], u[M];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        a[r] = stream_unit<T, U>(w[r] + at * U);
        b[r] = stream_unit<T, U>(w[r] + (at + step) * U);
      }
#pragma unroll
      for (int m = 0; m < M; ++m) {
        v[m] = *reinterpret_cast<const Un *>(x + min(few0 + m, few - 1) * ldf + at * U);
        u[m] = *reinterpret_cast<const Un *>(x + min(few0 + m, few - 1) * ldf + (at + step) * U);
      }
      add(a, v);
      add(b, u);
    }
    if (at < units) {
      Un a[R], v[M];
#pragma unroll
      for (int r = 0; r < R; ++r)
        a[r] = stream_unit<T, U>(w[r] + at * U);
#pragma unroll
      for (int m = 0; m < M; ++m)
        v[m] = *reinterpret_cast<const Un *>(x + min(few0 + m, few - 1) * ldf + at * U);
      add(a, v);
    }
    __syncwarp();
    float mine = 0.f; // lane i has output i / M of the group, row i % M
#pragma unroll
    for (int i = 0; i < R * M; ++i) {
      float v = acc[i / M][i % M];
#pragma unroll
      for (int o = 16; o; o >>= 1)
        v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane == i)
        mine = v;
    }
    if (ks > 1) {
      if (lane < R * M)
        parts[warp][lane] = mine;
      __syncthreads();
      if (!sub && lane < R * M)
        for (int s = 1; s < ks; ++s)
          mine += parts[warp + s][lane];
      __syncthreads();
    }
    const long long at_many = n0 + lane / M, at_few = few0 + lane % M;
    if (!sub && lane < R * M && at_many < many && at_few < few) {
      const Epilogue e{d.bias, d.activation, d.residual, d.ldr, d.y, d.ldy, d.z, d.ldz};
      finish<T>(e, Turned ? at_many : at_few, Turned ? at_few : at_many, mine);
    }
  }
}
bool few_vectors(const Dense &d) {
  const int V = 16 / bytes_of(d.type);
  return d.inputs % V == 0 && aligned16(d.weight) && (d.outputs <= 1 || d.ldw % V == 0) && aligned16(d.x) &&
         (d.rows <= 1 || d.ldx % V == 0);
}
// bf16 1 x 4096 -> 16384 takes 24.5 us here (5.5 TB/s) and 28.5 on the tensor cores, 4 x 1024 -> 1024 3.5
// and 7.5, f32 4 x 4096 -> 16384 56 and 124; but 16-bit weights of that size from two rows on 33 to
// 36 and 28.9: the conversions and products of each weight then take longer than its bytes.
bool is_few(const Dense &d) {
  return d.rows <= kFew && (d.rows == 1 || d.type == F32 || !few_vectors(d) || d.inputs <= (1ll << 24) / d.outputs);
}
// Few outputs: the tensor cores' tiles would be mostly empty, and x is what streams.
bool is_few_outputs(const Dense &d) { return d.outputs <= kFew; }
// Small products whose operands TMA cannot read: every warp forms its 4 x 8 sums, the operands come from
// L2, and nothing is copied or cut first.  f32 and bf16 393 x 1235 -> 27: 7.5 and 7.7 us here, 19.7 and
// 16.1 with copies and the tensor cores; but bf16 1000 x 565 -> 110 (62 million products) 18.4 and 13.6, and
// 10000 x 65 -> 64 (640,000 sums, whose joining over a warp bounds it) 25.8 and 9.5.
constexpr long long kSmallSums = 1ll << 17, kSmallProducts = 1ll << 25;
bool is_small(const Dense &d) {
  return d.rows * d.outputs <= std::min(kSmallSums, kSmallProducts / d.inputs) &&
         !(tma_ready(d.type, d.x, d.rows, d.ldx) && tma_ready(d.type, d.weight, d.outputs, d.ldw));
}
template <class T, int U, int M, bool Turned> void launch_few(const Dense &d, cudaStream_t stream) {
  const long long rest = ((Turned ? d.outputs : d.rows) + M - 1) / M;
  const long long groups = ((Turned ? d.rows : d.outputs) + kFewOutputs - 1) / kFewOutputs;
  // Warps share a group while there are fewer groups than warps and each keeps two steps of k.
  int ks = 1;
  while (ks < 8 && groups * rest * ks < 16ll * sm_count() && d.inputs / U >= 128ll * ks)
    ks *= 2;
  const long long blocks = (groups + 8 / ks - 1) / (8 / ks);
  // As many blocks as fit, so that groups spread evenly over the SMs; fewer where they are not filled.
  lapis::launch(few_rows_kernel<T, U, M, Turned>, dim3(unsigned(std::min<long long>(blocks, 4ll * sm_count())), unsigned(rest)),
                256, 0, stream, d, ks);
  lapis::check(cudaGetLastError());
}
void few_rows(const Dense &d, bool turned, cudaStream_t stream) {
  with_type(d.type, [&](auto tag) {
    using T = decltype(tag);
    const long long few = turned ? d.outputs : d.rows;
    auto rows = [&](auto unit, auto way) {
      constexpr int U = decltype(unit)::value;
      constexpr bool Turned = decltype(way)::value;
      if (few == 1)
        launch_few<T, U, 1, Turned>(d, stream);
      else if (few == 2)
        launch_few<T, U, 2, Turned>(d, stream);
      else if (few <= 4)
        launch_few<T, U, 4, Turned>(d, stream);
      else
        launch_few<T, U, 8, Turned>(d, stream);
    };
    auto units = [&](auto way) {
      if (few_vectors(d))
        rows(std::integral_constant<int, 16 / int(sizeof(T))>{}, way);
      else
        rows(std::integral_constant<int, 1>{}, way);
    };
    if (turned)
      units(std::true_type{});
    else
      units(std::false_type{});
  });
}

// ---------------- up to 16 outputs, many rows that TMA cannot read ----------------
// Floats, rows of x that start anywhere: copying x for the tensor cores moves it three times, where the
// call's floor is to read it once.  A block has 64 rows and all outputs; a slab of 32 k comes by single
// loads (a warp a row: 128 bytes at any offset), on its way in registers while the slab before it is
// summed from shared memory, 4 rows by 2 outputs a thread, in floats, a slab at a time.  Rows of shared memory
// are 36 floats apart, so that its 16-byte reads have no bank conflicts; these reads bound it.  With
// few rows the blocks do not fill the device.  Here, with a copy and the tensor cores, and as a plain
// product (us): 80000 x 301 -> 16 53, 85, 67; 80000 x 33 -> 16 16, 32, 27; 57901 x 911 -> 10 115, 169, 121;
// 20000 x 1001 -> 12 64, 85, 66; but 9472 x 1237 -> 16 55 and 45.  With more outputs shared memory is read
// more often (20000 x 1001 -> 48: 128, and 87 with a copy).  4-byte asynchronous copies: 74 at 1001 -> 12.
constexpr int kOddOutputs = 16, kOddRows = 64, kOddSlab = 32, kOddPitch = 36, kOddThreads = 128;
__global__ void __launch_bounds__(kOddThreads, 5) odd_rows_kernel(const __grid_constant__ Dense d) {
  constexpr int N = kOddOutputs, kWarps = kOddThreads / 32, R = 4, C = 2, kAcross = N / C, kHigh = kOddRows / R;
  static_assert(kAcross * kHigh == kOddThreads, "a thread has R rows and C outputs");
  constexpr int kMine = kOddRows / kWarps, kMineW = N / kWarps; // rows of x and W that a warp brings
  __shared__ __align__(16) float slabs[2][kOddRows + N][kOddPitch];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, cx = threadIdx.x % kAcross, ry = threadIdx.x / kAcross;
  const long long row0 = (long long)blockIdx.x * kOddRows;
  const float *const x = static_cast<const float *>(d.x), *const w = static_cast<const float *>(d.weight);
  const long long count = (d.inputs + kOddSlab - 1) / kOddSlab;
  float next[kMine + kMineW];
  auto load = [&](long long slab) { // columns and rows past the end: the last ones (as zeros; not written)
    const long long in = min(slab * kOddSlab + lane, d.inputs - 1);
#pragma unroll
    for (int r = 0; r < kMine; ++r)
      next[r] = x[min(row0 + warp + kWarps * r, d.rows - 1) * d.ldx + in];
#pragma unroll
    for (int n = 0; n < kMineW; ++n)
      next[kMine + n] = w[min((long long)(warp + kWarps * n), d.outputs - 1) * d.ldw + in];
  };
  float sum[R][C] = {};
  load(0);
  for (long long slab = 0; slab < count; ++slab) {
    float(*const at)[kOddPitch] = slabs[slab & 1];
    const bool there = slab * kOddSlab + lane < d.inputs;
#pragma unroll
    for (int r = 0; r < kMine + kMineW; ++r)
      at[r < kMine ? warp + kWarps * r : kOddRows + warp + kWarps * (r - kMine)][lane] = there ? next[r] : 0.f;
    __syncthreads(); // (who writes this place next has passed the next barrier, and with it all of its readers)
    load(min(slab + 1, count - 1));
    const float *const xs = at[ry], *const ws = at[kOddRows + cx];
    float part[R][C] = {};
#pragma unroll
    for (int k = 0; k < kOddSlab; k += 4) {
      float4 a[R], b[C];
#pragma unroll
      for (int i = 0; i < R; ++i)
        a[i] = *reinterpret_cast<const float4 *>(xs + i * kHigh * kOddPitch + k);
#pragma unroll
      for (int j = 0; j < C; ++j)
        b[j] = *reinterpret_cast<const float4 *>(ws + j * kAcross * kOddPitch + k);
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < C; ++j)
          part[i][j] = fmaf(a[i].w, b[j].w, fmaf(a[i].z, b[j].z, fmaf(a[i].y, b[j].y, fmaf(a[i].x, b[j].x, part[i][j]))));
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < C; ++j)
        sum[i][j] += part[i][j];
  }
  const Epilogue e{d.bias, d.activation, d.residual, d.ldr, d.y, d.ldy, d.z, d.ldz};
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const long long row = row0 + ry + i * kHigh;
      const int col = cx + j * kAcross;
      if (row < d.rows && col < d.outputs)
        finish<float>(e, row, col, sum[i][j]);
    }
}
bool is_odd(const Dense &d) {
  return d.type == F32 && d.outputs > kFew && d.outputs <= kOddOutputs && d.inputs > 12 && d.rows >= 128ll * sm_count() &&
         !tma_ready(d.type, d.x, d.rows, d.ldx);
}
void odd(const Dense &d, cudaStream_t stream) {
  lapis::launch(odd_rows_kernel, dim3(unsigned((d.rows + kOddRows - 1) / kOddRows)), kOddThreads, 0, stream, d);
  lapis::check(cudaGetLastError());
}

// ---------------- one pass over dy ----------------
// A block is `lanes` columns units wide (a power of two up to 32) and 256 / lanes rows high; it walks
// rows by gridDim.y blocks' heights, writes dz = dy act'(z) (dz NULL: not wanted) and adds its columns:
// partial [gridDim.y][outputs] (NULL: not wanted).  Memory-bound: every value is read once.
template <class T, int U>
__global__ void __launch_bounds__(256)
    gradient_kernel(const __grid_constant__ DenseBackward a, T *dz, long long lddz, float *partial, int lanes) {
  constexpr bool Fast = sizeof(T) == 2;
  constexpr int kAhead = 4; // rows in flight per thread; rows past the end read the last one
  using Un = Unit<T, U>;
  __shared__ float join[256 * U];
  const int tx = threadIdx.x & (lanes - 1), ty = threadIdx.x / lanes, high = 256 / lanes;
  const long long col = ((long long)blockIdx.x * lanes + tx) * U;
  const bool live = col < a.outputs;
  const long long step = (long long)gridDim.y * high;
  float sum[U] = {};
  if (live)
    for (long long r0 = (long long)blockIdx.y * high + ty; r0 < a.rows; r0 += step * kAhead) {
      Un dy[kAhead], z[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        dy[k] = *reinterpret_cast<const Un *>(static_cast<const T *>(a.dy) + min(r0 + k * step, a.rows - 1) * a.lddy + col);
      if (a.activation != None)
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
          z[k] = *reinterpret_cast<const Un *>(static_cast<const T *>(a.z) + min(r0 + k * step, a.rows - 1) * a.ldz + col);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const long long r = r0 + k * step;
        float v[U], s[U];
        unpack<T, U>(dy[k], v);
        if (a.activation != None) {
          unpack<T, U>(z[k], s);
          slope_all<Fast>(s, a.activation);
#pragma unroll
          for (int u = 0; u < U; ++u)
            v[u] *= s[u];
        }
        if (r < a.rows) {
#pragma unroll
          for (int u = 0; u < U; ++u)
            sum[u] += v[u];
          if (dz)
            *reinterpret_cast<Un *>(dz + r * lddz + col) = pack<T, U>(v);
        }
      }
    }
  if (!partial)
    return;
#pragma unroll
  for (int u = 0; u < U; ++u)
    join[(ty * lanes + tx) * U + u] = sum[u];
  __syncthreads();
  const long long c0 = (long long)blockIdx.x * lanes * U;
  for (int c = threadIdx.x; c < lanes * U; c += 256) {
    float s = 0.f;
    for (int y = 0; y < high; ++y)
      s += join[y * lanes * U + c];
    if (c0 + c < a.outputs)
      partial[blockIdx.y * a.outputs + c0 + c] = s;
  }
}

// ---------------- small gradients ----------------
// All gradients of a layer with few weights, any alignment, float arithmetic: a block takes kSmallRows rows
// or fewer (as shared memory allows) at a time, forms their dz (in float, not rounded) beside x and W in
// shared memory, writes their dx, and adds to dW and db -- x has one more column of ones for db -- in
// registers.  Many rows: each block writes a partial [outputs][inputs + 1], which a second launch adds.
// Launches are what bound such calls, one or two here and 4 to 8 with the tensor cores (f32 with SiLU,
// here and there: 12 x 9 -> 7 4.4 and 22 us, 18081 x 8 -> 24 11.7 and 40, 295 x 338 -> 12 18 and 41; bf16
// 4096 x 63 -> 64 26 and 29).  What bounds large ones is shared memory, two reads for each product, so
// steps are short where there are many weights, and blocks many; bf16 1000 x 1000 -> 4, whose steps are
// short and wide, takes 27 us and 17.
constexpr int kSmallRows = 64, kSmallWeights = 4096, kSmallWidth = 512, kSmallFloats = 16384;
constexpr long long kSmallWork = 1ll << 24; // products of a pair of values, for dW
struct SmallGradients {
  int rows, blocks; // of a step; of the grid
  unsigned shared;
};
bool is_small(const DenseBackward &d) {
  return d.outputs + d.inputs < kSmallWidth && d.outputs * (d.inputs + 1) <= kSmallWeights &&
         d.rows <= kSmallWork / (d.outputs * (d.inputs + 1));
}
SmallGradients small_gradients(const DenseBackward &d) {
  SmallGradients s;
  const int width = int(d.outputs + d.inputs + 1);
  s.rows = std::min({kSmallRows, kSmallFloats / width, std::max(8, 32768 / int(d.outputs * (d.inputs + 1)))});
  s.shared = unsigned(std::max(s.rows * width + int(d.outputs * d.inputs), 256)) * 4u; // (256: the groups' sums)
  s.blocks = int(std::min<long long>((d.rows + s.rows - 1) / s.rows, std::min(4ll, 200000ll / (s.shared + 1024)) * sm_count()));
  return s;
}
// Value e of [outputs][inputs + 1] (dW, db) to its place.
template <class T> __device__ __forceinline__ void small_result(const DenseBackward &a, int e, float v) {
  const int W = int(a.inputs) + 1, o = e / W, i = e - o * W;
  if (i < W - 1) {
    if (a.dweight)
      static_cast<T *>(a.dweight)[o * a.lddw + i] = from_float<T>(v);
  } else if (a.dbias) {
    static_cast<T *>(a.dbias)[o] = from_float<T>(v);
  }
}
template <class T>
__global__ void __launch_bounds__(256)
    small_gradient_kernel(const __grid_constant__ DenseBackward a, int step, float *partial) {
  constexpr bool Fast = sizeof(T) == 2;
  constexpr int kMine = kSmallWeights / 256;
  extern __shared__ float shared[];
  const int I = int(a.inputs), O = int(a.outputs), W = I + 1, n = O * W;
  float *const xs = shared, *const dz = xs + step * W, *const ws = dz + step * O; // [step][W], [step][O], [O][I]
  const int t = threadIdx.x;
  if (a.dx)
    for (int e = t; e < O * I; e += 256)
      ws[e] = to_float(static_cast<const T *>(a.weight)[(long long)(e / I) * a.ldw + e % I]);
  // Fewer sums than threads: groups of threads take every groups-th row.
  const int groups = n < 256 ? 256 / n : 1, group = n < 256 ? t / n : 0, mine = n < 256 ? t % n : t;
  float acc[kMine] = {};
  for (long long r0 = (long long)blockIdx.x * step; r0 < a.rows; r0 += (long long)gridDim.x * step) {
    const int rows = int(min((long long)step, a.rows - r0));
    __syncthreads();
    if (a.dweight)
      for (int e = t; e < rows * I; e += 256) {
        const int r = e / I, i = e - r * I;
        xs[r * W + i] = to_float(static_cast<const T *>(a.x)[(r0 + r) * a.ldx + i]);
      }
    for (int r = t; r < rows; r += 256)
      xs[r * W + I] = 1.f;
    for (int e = t; e < rows * O; e += 256) {
      const int r = e / O, o = e - r * O;
      float v = to_float(static_cast<const T *>(a.dy)[(r0 + r) * a.lddy + o]);
      if (a.activation != None)
        v *= slope<Fast>(to_float(static_cast<const T *>(a.z)[(r0 + r) * a.ldz + o]), a.activation);
      dz[e] = v;
    }
    __syncthreads();
    if (a.dx)
      for (int e = t; e < rows * I; e += 256) {
        const int r = e / I, i = e - r * I;
        float s = 0.f;
#pragma unroll 4
        for (int o = 0; o < O; ++o)
          s = fmaf(dz[r * O + o], ws[o * I + i], s);
        static_cast<T *>(a.dx)[(r0 + r) * a.lddx + i] = from_float<T>(s);
      }
    if ((a.dweight || a.dbias) && group < groups) {
#pragma unroll
      for (int k = 0; k < kMine; ++k) {
        const int e = mine + 256 * k;
        if (e < n && (k == 0 || groups == 1)) {
          const int o = e / W;
          const float *const g = dz + o, *const x = xs + (e - o * W);
          float s = acc[k];
          if (a.dweight || e - o * W == I)
#pragma unroll 4
            for (int r = group; r < rows; r += groups)
              s = fmaf(g[r * O], x[r * W], s);
          acc[k] = s;
        }
      }
    }
  }
  if (!a.dweight && !a.dbias)
    return;
  if (groups > 1) { // the groups' sums in order
    __syncthreads();
    shared[t] = acc[0];
    __syncthreads();
    float s = 0.f;
    if (t < n)
      for (int k = 0; k < groups; ++k)
        s += shared[k * n + t];
    acc[0] = s;
  }
#pragma unroll
  for (int k = 0; k < kMine; ++k) {
    const int e = t + 256 * k;
    if (e < n) {
      if (partial)
        partial[(long long)blockIdx.x * n + e] = acc[k];
      else
        small_result<T>(a, e, acc[k]);
    }
  }
}
// The partials' sums: 32 values per block, in a fixed order.
template <class T>
__global__ void __launch_bounds__(1024)
    small_sum_kernel(const __grid_constant__ DenseBackward a, const float *partial, int parts) {
  __shared__ float sum[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, n = int(a.outputs * (a.inputs + 1)), e = int(blockIdx.x) * 32 + x;
  float s = 0.f;
  if (e < n)
    for (int p = y; p < parts; p += 32)
      s += partial[(long long)p * n + e];
  sum[y][x] = s;
  __syncthreads();
  float v = sum[x][y];
#pragma unroll
  for (int o = 16; o; o >>= 1)
    v += __shfl_xor_sync(0xffffffffu, v, o);
  if (!x && int(blockIdx.x) * 32 + y < n)
    small_result<T>(a, int(blockIdx.x) * 32 + y, v);
}

// Copy of a [rows][cols] array with any row distance and alignment into rows of ldo elements (a multiple
// of 16 bytes): a lane gathers 16 bytes of a row by single elements, all in flight, and stores them at
// once; what lies behind cols in a row's last 16 bytes is zero.  A warp takes 32 neighbouring units.
template <class T>
__global__ void __launch_bounds__(256) pack_kernel(const T *in, long long ldi, T *out, long long ldo, long long rows,
                                                   long long cols) {
  constexpr int U = 16 / int(sizeof(T));
  const long long units = ldo / U, total = rows * units;
  for (long long x = (long long)blockIdx.x * 256 + threadIdx.x; x < total; x += 256ll * gridDim.x) {
    const long long r = x / units, c = (x - r * units) * U;
    const T *p = in + r * ldi;
    Unit<T, U> u;
#pragma unroll
    for (int i = 0; i < U; ++i)
      u.v[i] = p[min(c + i, cols - 1)];
#pragma unroll
    for (int i = 0; i < U; ++i)
      u.v[i] = c + i < cols ? u.v[i] : T(0);
    *reinterpret_cast<Unit<T, U> *>(out + r * ldo + c) = u;
  }
}

// The pass's grid: about 8 blocks per SM.
struct Pass {
  int unit, lanes, grid_x, parts;
};
Pass pass_of(const DenseBackward &d, bool vectors) {
  Pass p{vectors ? 16 / bytes_of(d.type) : 1, 1, 0, 0};
  long long units = (d.outputs + p.unit - 1) / p.unit;
  while (p.lanes < 32 && p.lanes < units)
    p.lanes *= 2;
  p.grid_x = int((units + p.lanes - 1) / p.lanes);
  long long high = 256 / p.lanes, blocks = (d.rows + 4 * high - 1) / (4 * high);
  p.parts = int(std::min<long long>({blocks, std::max(1ll, 8ll * sm_count() / p.grid_x), 2048}));
  return p;
}
bool vectors_of(const DenseBackward &d) {
  const int U = 16 / bytes_of(d.type);
  return d.outputs % U == 0 && aligned16(d.dy) && (d.rows <= 1 || d.lddy % U == 0) &&
         (d.activation == None || (aligned16(d.z) && (d.rows <= 1 || d.ldz % U == 0)));
}
// z's alignment is not known to the workspace call: the larger of both passes.
long long partial_bytes(const DenseBackward &d) {
  return round_up(std::max(pass_of(d, true).parts, pass_of(d, false).parts) * d.outputs * 4, 16);
}

// Where an operand lies once TMA can read it: in place, or copied behind `used` bytes of the workspace.
struct Place {
  long long at = -1, ld = 0, bytes = 0;
};
Place place(int type, const void *p, long long rows, long long cols, long long ld, long long &used) {
  Place w;
  w.ld = ld;
  if (tma_ready(type, p, rows, ld))
    return w;
  w.at = used;
  w.ld = round_up(cols, 16 / bytes_of(type));
  w.bytes = round_up(rows * w.ld * bytes_of(type), 16);
  used += w.bytes;
  return w;
}
Operand bring(int type, const Place &w, const void *p, long long rows, long long cols, long long ld, bool turned,
              void *workspace, cudaStream_t stream) {
  if (w.at < 0)
    return {p, ld, turned};
  void *to = static_cast<char *>(workspace) + w.at;
  const long long units = rows * (w.ld * bytes_of(type) / 16);
  const dim3 grid(unsigned(std::min<long long>((units + 255) / 256, 16ll * sm_count())));
  auto copy = [&](auto tag) {
    using U = decltype(tag);
    lapis::launch(pack_kernel<U>, grid, 256, 0, stream, static_cast<const U *>(p), ld, static_cast<U *>(to), w.ld, rows, cols);
  };
  if (type == F32)
    copy(0u);
  else
    copy((unsigned short)0);
  lapis::check(cudaGetLastError());
  return {to, w.ld, turned};
}

void product(const Product &p, void *workspace, cudaStream_t stream, float *sums = nullptr) {
  if (p.type == F32)
    product32(p, workspace, stream, sums);
  else
    product16(p, workspace, stream);
}
long long product_workspace(int type, long long I, long long J, long long K) {
  return parts_workspace(type == F32 ? plan32(I, J, K) : plan16(I, J, K), I, J);
}

struct ForwardLayout {
  Place x, w;
  long long product, total;
  explicit ForwardLayout(const Dense &d) {
    long long used = 0;
    x = place(d.type, d.x, d.rows, d.inputs, d.ldx, used);
    w = place(d.type, d.weight, d.outputs, d.inputs, d.ldw, used);
    product = used;
    total = used + product_workspace(d.type, d.rows, d.outputs, d.inputs);
  }
};
struct BackwardLayout {
  Place dz, x, w;
  bool write_dz; // by the pass over dy: the activation's slope, or a copy that TMA can read
  long long partial, product, total;
  explicit BackwardLayout(const DenseBackward &d) {
    long long used = 0;
    partial = used;
    used += std::max(partial_bytes(d), d.type == F32 ? round_up(plan32(d.outputs, d.inputs, d.rows).parts * d.outputs * 8, 16) : 0);
    write_dz = d.activation != None || !tma_ready(d.type, d.dy, d.rows, d.lddy);
    dz.ld = d.lddy;
    if (write_dz) {
      dz.at = used;
      dz.ld = round_up(d.outputs, 16 / bytes_of(d.type));
      used += round_up(d.rows * dz.ld * bytes_of(d.type), 16);
    }
    x = place(d.type, d.x, d.rows, d.inputs, d.ldx, used);
    w = place(d.type, d.weight, d.outputs, d.inputs, d.ldw, used);
    product = used;
    total = used + std::max(product_workspace(d.type, d.rows, d.inputs, d.outputs),
                            product_workspace(d.type, d.outputs, d.inputs, d.rows));
  }
};
} // namespace

long long dense_workspace(const Dense &d) {
  return is_narrow(d) || is_few(d) || is_few_outputs(d) || is_small(d) || is_odd(d) ? 0 : ForwardLayout(d).total;
}
void dense(const Dense &d, void *workspace, cudaStream_t stream) {
  if (is_odd(d)) {
    odd(d, stream);
    return;
  }
  if (is_narrow(d)) {
    narrow(d, stream);
    return;
  }
  if (is_few(d) || is_few_outputs(d) || is_small(d)) {
    few_rows(d, !is_few(d) && is_few_outputs(d), stream);
    return;
  }
  const ForwardLayout l(d);
  const Epilogue e{d.bias, d.activation, d.residual, d.ldr, d.y, d.ldy, d.z, d.ldz};
  Product p{d.type, d.rows, d.outputs, d.inputs,
            bring(d.type, l.x, d.x, d.rows, d.inputs, d.ldx, false, workspace, stream),
            bring(d.type, l.w, d.weight, d.outputs, d.inputs, d.ldw, false, workspace, stream), e};
  product(p, static_cast<char *>(workspace) + l.product, stream);
}

long long dense_backward_workspace(const DenseBackward &d) {
  if (is_small(d)) {
    const int blocks = small_gradients(d).blocks;
    return blocks > 1 ? round_up(blocks * d.outputs * (d.inputs + 1) * 4, 16) : 0;
  }
  return BackwardLayout(d).total;
}
namespace {
void small_backward(const DenseBackward &d, float *partial, cudaStream_t stream) {
  const SmallGradients s = small_gradients(d);
  with_type(d.type, [&](auto tag) {
    using T = decltype(tag);
    static thread_local int configured = -1;
    int device = 0;
    lapis::check(cudaGetDevice(&device));
    if (configured != device) {
      lapis::check(cudaFuncSetAttribute(small_gradient_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (kSmallFloats + kSmallWeights) * 4));
      configured = device;
    }
    const bool sums = s.blocks > 1 && (d.dweight || d.dbias);
    lapis::launch(small_gradient_kernel<T>, dim3(unsigned(s.blocks)), 256, s.shared, stream, d, s.rows, sums ? partial : nullptr);
    if (sums)
      lapis::launch(small_sum_kernel<T>, dim3(unsigned((d.outputs * (d.inputs + 1) + 31) / 32)), 1024, 0, stream, d, partial, s.blocks);
    lapis::check(cudaGetLastError());
  });
}
} // namespace
void dense_backward(const DenseBackward &d, void *workspace, cudaStream_t stream) {
  if (!d.rows) { // sums of nothing
    if (d.dweight)
      lapis::check(cudaMemset2DAsync(d.dweight, size_t(d.lddw) * bytes_of(d.type), 0, size_t(d.inputs) * bytes_of(d.type),
                                     size_t(d.outputs), stream));
    if (d.dbias)
      lapis::check(cudaMemsetAsync(d.dbias, 0, size_t(d.outputs) * bytes_of(d.type), stream));
    return;
  }
  if (is_small(d)) {
    if (d.dx || d.dweight || d.dbias)
      small_backward(d, static_cast<float *>(workspace), stream);
    return;
  }
  const BackwardLayout l(d);
  char *ws = static_cast<char *>(workspace);
  const bool products = d.dx || d.dweight, write_dz = products && l.write_dz;
  // Without a pass that writes dz, the product for dweight adds dz's columns while it splits them
  // (floats; the pass alone would read dz once more: 71 of 430 us at 84613 x 64 -> 1280).
  const bool fused = d.dbias && d.dweight && d.type == F32 && !write_dz;
  float *const sums = d.dbias ? reinterpret_cast<float *>(ws + l.partial) : nullptr, *partial = fused ? nullptr : sums;
  void *dz = write_dz ? ws + l.dz.at : nullptr;
  if (dz || partial)
    with_type(d.type, [&](auto tag) {
      using T = decltype(tag);
      constexpr int V = 16 / int(sizeof(T));
      const bool vectors = vectors_of(d);
      const Pass p = pass_of(d, vectors);
      dim3 grid(unsigned(p.grid_x), unsigned(p.parts));
      if (vectors)
        lapis::launch(gradient_kernel<T, V>, grid, 256, 0, stream, d, static_cast<T *>(dz), l.dz.ld, partial, p.lanes);
      else
        lapis::launch(gradient_kernel<T, 1>, grid, 256, 0, stream, d, static_cast<T *>(dz), l.dz.ld, partial, p.lanes);
      if (partial)
        lapis::launch(column_sum_kernel<T>, dim3(unsigned((d.outputs + 31) / 32), 1), 1024, 0, stream, partial, p.parts, 1,
                      d.outputs, static_cast<T *>(d.dbias), static_cast<T *>(nullptr));
      lapis::check(cudaGetLastError());
    });
  const void *g = dz ? dz : d.dy;
  const long long ldg = dz ? l.dz.ld : d.lddy;
  if (d.dx)
    product({d.type, d.rows, d.inputs, d.outputs, {g, ldg, false},
             bring(d.type, l.w, d.weight, d.outputs, d.inputs, d.ldw, true, workspace, stream),
             Epilogue{nullptr, None, nullptr, 0, d.dx, d.lddx}},
            ws + l.product, stream);
  if (d.dweight)
    product({d.type, d.outputs, d.inputs, d.rows, {g, ldg, true},
             bring(d.type, l.x, d.x, d.rows, d.inputs, d.ldx, true, workspace, stream),
             Epilogue{nullptr, None, nullptr, 0, d.dweight, d.lddw}},
            ws + l.product, stream, fused ? sums : nullptr);
  if (fused) {
    const int parts = 2 * plan32(d.outputs, d.inputs, d.rows).parts;
    lapis::launch(column_sum_kernel<float>, dim3(unsigned((d.outputs + 31) / 32), 1), 1024, 0, stream, sums, parts, 1,
                  d.outputs, static_cast<float *>(d.dbias), static_cast<float *>(nullptr));
    lapis::check(cudaGetLastError());
  }
}
} // namespace op
} // namespace mace
