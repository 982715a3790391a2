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
};
// How the finished blocks reach memory.  on: as boxes of 32 rows through TMA, where y, z and the
// residual (or the parts) have 16-byte aligned rows; columns past J are clipped.
struct Boxes {
  CUtensorMap y, z, residual; // y: the parts, when K is cut
  int on;
  int sectors; // rows of all of them begin and end with whole 32-byte sectors
};
struct Product {
  int type;
  long long I, J, K;
  Operand p, q;
  Epilogue e;
};

// Output tiles in bands of kBand rows of tiles, column by column within a band: the tiles that run
// together share their operands in L2.  32-bit indices: products that large in memory have fewer
// than 2^31 tiles and parts of tiles (checked on the host).
struct Tiles {
  unsigned nI, nJ, count;
  Tiles() = default;
  Tiles(long long I, long long J, int bi, int bj)
      : nI(unsigned((I + bi - 1) / bi)), nJ(unsigned((J + bj - 1) / bj)), count(nI * nJ) {}
  __device__ __forceinline__ void at(unsigned t, long long &i, long long &j) const {
    constexpr unsigned kBand = 16;
    const unsigned band = t / (kBand * nJ), first = band * kBand, rows = min(kBand, nI - first), r = t - first * nJ;
    const unsigned c = r / rows;
    i = first + (r - c * rows);
    j = c;
  }
};
inline void check_tiles(long long I, long long J, int bi, int bj, long long parts) {
  if (double((I + bi - 1) / bi) * double((J + bj - 1) / bj) * double(parts) > 2e9)
    throw lapis::Error("The product has too many tiles");
}

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
// A box of 32 rows by 128 bytes in shared memory, a warp's, and the mbarrier of its residual.
constexpr int kBoxBytes = 32 * 128;
struct Box {
  unsigned char *at; // 1024-byte aligned
  unsigned bar;
};
// Starts the load of a residual box (one lane; the box's last store has read it).
__device__ __forceinline__ void fetch_residual(const Boxes &m, const Box &w, long long row0, long long col0) {
  tc::mbar_expect_tx(w.bar, kBoxBytes);
  tc::tma_load_3d(tc::smem_u32(w.at), &m.residual, int(col0), int(row0), 0, w.bar);
}

// `count` (a multiple of 32) values of the bias from column col0 into a warp's shared memory.
template <class T>
__device__ __forceinline__ void fetch_bias(const Epilogue &e, long long J, long long col0, int count, T *to) {
  if (!e.bias)
    return;
  __syncwarp();
  for (int c = threadIdx.x & 31; c < count; c += 32)
    to[c] = col0 + c < J ? static_cast<const T *>(e.bias)[col0 + c] : T(0.f);
  __syncwarp();
}

// 32 rows by 128 bytes of the result from (row0, col0), rows = lanes.  get(c, v) gives the product's
// columns col0 + c .. + 31, bias their bias in shared memory (NULL: they have it).  part >= 0 (T float): the
// values as they are, to plane `part`.  ready: the box's last store has read it, and the residual is on
// its way; phase: of its barrier.  Rows are swizzled in shared memory, so that neither side has bank
// conflicts; TMA writes whole lines.  Bare: the epilogue is empty (the gradients' products).
template <class T, bool Bare, class Get>
__device__ __forceinline__ void finish_box(const Epilogue &e, const Boxes &m, long long row0, long long col0, int part,
                                           const Box &w, unsigned &phase, bool ready, const T *bias, Get &&get) {
  constexpr bool Fast = sizeof(T) == 2;
  constexpr int U = 16 / int(sizeof(T)), W = 128 / int(sizeof(T));
  using Un = Unit<T, U>;
  const int lane = threadIdx.x & 31;
  unsigned char *mine = w.at + lane * 128;
  const bool plain = Bare || part >= 0;
  auto block = [&](int c, float (&v)[32]) {
    get(c, v);
    if (!bias)
      return;
#pragma unroll
    for (int i = 0; i < 32; i += U) {
      const Un b = *reinterpret_cast<const Un *>(bias + c + i);
#pragma unroll
      for (int u = 0; u < U; ++u)
        v[i + u] += to_float(b.v[u]);
    }
  };
  auto free_box = [&] { // its last store has read it
    if (lane == 0)
      tc::bulk_wait_read();
    __syncwarp();
  };
  auto send = [&](const CUtensorMap &map, int plane) {
    tc::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      tc::tma_store_3d(&map, tc::smem_u32(w.at), int(col0), int(row0), plane);
      tc::bulk_commit();
    }
  };
  if (!plain && e.z) {
    free_box();
#pragma unroll
    for (int c = 0; c < W; c += 32) {
      float v[32];
      block(c, v);
#pragma unroll
      for (int i = 0; i < 32; i += U) {
        Un o;
#pragma unroll
        for (int u = 0; u < U; ++u)
          o.v[u] = from_float<T>(v[i + u]);
        *reinterpret_cast<Un *>(mine + ((((c + i) / U) ^ (lane & 7)) << 4)) = o;
      }
    }
    send(m.z, 0);
  }
  const bool residual = !plain && e.residual;
  if (!ready) {
    free_box();
    if (residual && lane == 0)
      fetch_residual(m, w, row0, col0);
  }
  bool there = true;
#pragma unroll
  for (int c = 0; c < W; c += 32) {
    float v[32];
    block(c, v);
    if (!plain)
      activate_all<Fast>(v, e.activation);
    if (residual && c == 0) {
      const long long start = clock64();
      while (!(there = tc::mbar_try(w.bar, phase)) && clock64() - start < tc::kWaitCycles) {
      }
      phase ^= 1;
    }
#pragma unroll
    for (int i = 0; i < 32; i += U) {
      Un *at = reinterpret_cast<Un *>(mine + ((((c + i) / U) ^ (lane & 7)) << 4));
      Un o;
      if (residual) {
        o = *at;
#pragma unroll
        for (int u = 0; u < U; ++u) // a wait that ran out shows as NaN
          v[i + u] = there ? v[i + u] + to_float(o.v[u]) : __uint_as_float(0x7fc00000u);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        o.v[u] = from_float<T>(v[i + u]);
      *at = o;
    }
  }
  send(m.y, max(part, 0));
}

// 32 bytes at once (aligned to 32).
__device__ __forceinline__ void store32(void *p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
               "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
__device__ __forceinline__ void load32(const void *p, uint32_t (&w)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p)
               : "memory");
}
// The residual of 32 columns of a lane's row, for finish_row.
template <class T> struct Sectors {
  static constexpr int S = 32 / int(sizeof(T)); // elements of a sector
  uint32_t w[32 / S][8];
  __device__ __forceinline__ void load(const Epilogue &e, long long I, long long J, long long row, long long col0) {
#pragma unroll
    for (int k = 0; k < 32; k += S)
      if (row < I && col0 + k < J)
        load32(static_cast<const T *>(e.residual) + row * e.ldr + col0 + k, w[k / S]);
  }
};
// 32 columns of a lane's row from col0, for rows of whole sectors (Boxes::sectors): each lane writes its
// row 32 bytes at a time, a sector each, with nothing staged and nothing waited for (bf16 84613 x 64
// -> 1280: 50 us, 62 through boxes; float rows, twice as long, take longer this way: 227 us, 195).
// bias: in shared memory.  part: the float values as they are, to that array.
template <class T>
__device__ __forceinline__ void finish_row(const Epilogue &e, float *part, long long I, long long J, long long row,
                                           long long col0, float (&v)[32], const T *bias, const Sectors<T> &residual) {
  constexpr bool Fast = sizeof(T) == 2;
  if (part) {
    if (row < I)
#pragma unroll
      for (int k = 0; k < 32; k += 8)
        if (col0 + k < J) {
          uint32_t w[8];
          memcpy(w, v + k, 32);
          store32(part + row * J + col0 + k, w);
        }
    return;
  }
  constexpr int S = Sectors<T>::S;
  if (e.bias) {
    constexpr int U = 16 / int(sizeof(T));
#pragma unroll
    for (int i = 0; i < 32; i += U) {
      float b[U];
      unpack<T, U>(*reinterpret_cast<const Unit<T, U> *>(bias + i), b);
#pragma unroll
      for (int u = 0; u < U; ++u)
        v[i + u] += b[u];
    }
  }
  auto write = [&](void *out, long long ld) {
#pragma unroll
    for (int k = 0; k < 32; k += S)
      if (row < I && col0 + k < J) {
        const Unit<T, S> o = pack<T, S>(v + k);
        uint32_t w[8];
        memcpy(w, &o, 32);
        store32(static_cast<T *>(out) + row * ld + col0 + k, w);
      }
  };
  if (e.z)
    write(e.z, e.ldz);
  activate_all<Fast>(v, e.activation);
  if (e.residual)
#pragma unroll
    for (int k = 0; k < 32; k += S) {
      Unit<T, S> o;
      memcpy(&o, residual.w[k / S], 32);
      float f[S];
      unpack<T, S>(o, f);
#pragma unroll
      for (int u = 0; u < S; ++u)
        v[k + u] += f[u];
    }
  write(e.out, e.ldo);
}

// A warp's 32 x 32 block where rows allow no boxes: through its box (columns permuted by row), so that
// neighbouring lanes write neighbouring columns, with several rows' residuals in flight (as registers
// allow).  bias: it is added here.  partial != NULL: the float values go to partial[row * J + col] instead.
template <class T>
__device__ __forceinline__ void finish_block(const Epilogue &e, float *partial, long long I, long long J,
                                             long long row0, long long col0, const float *v, bool bias, unsigned char *box) {
  constexpr bool Fast = sizeof(T) == 2;
  constexpr int kRows = Fast ? 16 : 8; // at once
  const int lane = threadIdx.x & 31, rows = int(min(32ll, I - row0));
  float *stage = reinterpret_cast<float *>(box);
  __syncwarp();
#pragma unroll
  for (int k = 0; k < 32; ++k)
    stage[lane * 32 + (k ^ lane)] = v[k];
  __syncwarp();
  const long long col = col0 + lane;
  if (col < J) {
    // Pointers that go down the column: a row costs what its instructions do (f16 1237 x 64 -> 2055: 19.5
    // us with an address formed for each row, 9.2 so).
    if (partial) {
      float *to = partial + row0 * J + col;
#pragma unroll 8
      for (int r = 0; r < rows; ++r, to += J)
        *to = stage[r * 32 + (lane ^ r)];
    } else {
      const float add = bias ? to_float(static_cast<const T *>(e.bias)[col]) : 0.f;
      const T *from = e.residual ? static_cast<const T *>(e.residual) + row0 * e.ldr + col : nullptr;
      T *z = e.z ? static_cast<T *>(e.z) + row0 * e.ldz + col : nullptr, *to = static_cast<T *>(e.out) + row0 * e.ldo + col;
#pragma unroll 1
      for (int r0 = 0; r0 < rows; r0 += kRows) {
        float x[kRows];
        T res[kRows];
        if (from)
#pragma unroll
          for (int i = 0; i < kRows; ++i, from += e.ldr)
            if (r0 + i < rows)
              res[i] = *from;
#pragma unroll
        for (int i = 0; i < kRows; ++i)
          x[i] = stage[(r0 + i) * 32 + (lane ^ (r0 + i))] + add;
        if (z)
#pragma unroll
          for (int i = 0; i < kRows; ++i, z += e.ldz)
            if (r0 + i < rows)
              *z = from_float<T>(x[i]);
        activate_all<Fast>(x, e.activation);
        if (from)
#pragma unroll
          for (int i = 0; i < kRows; ++i)
            x[i] += to_float(res[i]);
#pragma unroll
        for (int i = 0; i < kRows; ++i, to += e.ldo)
          if (r0 + i < rows)
            *to = from_float<T>(x[i]);
      }
    }
  }
  __syncwarp();
}

// ---------------- host ----------------
inline long long round_up(long long n, long long to) { return (n + to - 1) / to * to; }

// Tensor map of a [rows][cols] array of 16-bit or float elements with row distance ld, in boxes of
// box_rows rows by 128 bytes, SWIZZLE_128B; elements outside the array read as zero.
// planes: a third dimension of `rows` rows each (0: a map of two dimensions).
CUtensorMap tile_map(int type, const void *base, long long rows, long long cols, long long ld, int box_rows,
                     int planes = 0);
// The boxes of a product's results, or of its parts.
Boxes boxes_of(const Product &, float *partial, int parts);
// Whether TMA can read the array in place: 16-byte aligned rows.
inline bool tma_ready(int type, const void *p, long long rows, long long ld) {
  return aligned16(p) && (rows <= 1 || ld * bytes_of(type) % 16 == 0);
}

// Tile width and parts of K of a product.
struct Plan {
  int bn, parts;
};
// Workspace of a product: the float values of its parts.
inline long long parts_workspace(const Plan &p, long long I, long long J) {
  return p.parts > 1 ? round_up(p.parts * I * J * 4, 16) : 0;
}
// The products of 16-bit types (dense_gemm16.cu) and of floats
// (dense_gemm32.cu); the operands are as TMA can read them.
Plan plan16(long long I, long long J, long long K);
void product16(const Product &, void *workspace, cudaStream_t);
Plan plan32(long long I, long long J, long long K);
// sums (p turned; NULL: not wanted): partial sums over k of P's rows, [2 parts][I].
void product32(const Product &, void *workspace, cudaStream_t, float *sums = nullptr);
// Sum of `parts` float products [parts][I][J], through the epilogue.
void finish_parts(int type, const Epilogue &, const float *partial, int parts, long long I, long long J, cudaStream_t);
} // namespace op
} // namespace mace
