// The dense layer's matrix products of floats on the tensor cores (tcgen05, kind::f16), with the
// error of float arithmetic.
//
//   out(i, j) = sum_k P(i, k) Q(j, k)
//
// Both operands are split on the way into shared memory: per row and 64-wide slab of k, with 2^e the
// power of two that brings the largest magnitude into [2^14, 2^15), v 2^e = hi + lo, both fp16
// rounded to nearest (22 significant bits for values down to 2^-18 of the largest).  A slab's
// products lo*hi + hi*lo + hi*hi (lo*lo is below 2^-22) accumulate fresh in TMEM, are scaled back
// by the two exact powers of two and added to float registers: the tensor pipe truncates, which
// must not add up over long k.  A slab's result is first moved one ulp away from zero, which
// cancels the mean of that truncation (the same measure as in tc_gemm.cu).
//
// Operands are read by plain coalesced loads, so any row distance and alignment will do, and the
// split turns a [K][I] operand for free: the slab in shared memory is always k-major.  16 warps (128
// registers each; a 17th for the MMAs would leave 96 and spill):
//   0..7    load and split: four for P, four for Q; the loads of the next slab are issued as the
//           registers of this one are split.  Warp 0 also issues the MMAs of a slab, after its
//           own part of the next one, when the other warps' parts are long there.
//   8..15   drain: lane = output row, two warps per TMEM lane quadrant, BN / 2 columns each
// Infinities and NaN make every result of their row (of P or Q) NaN in this scheme; results that
// are not finite are summed again, one product at a time.
#include "dense_gemm.cuh"

namespace mace {
namespace op {
namespace {
using namespace tc;
constexpr int kBM = 128, kBK = 64, kStages = 3;
constexpr int kThreads = 512, kSplitThreads = 256, kDrainThreads = 256;
// The split of slab g runs after the MMAs of g - 3, which waited for the drain of g - 5.
constexpr int kSlots = 6;
constexpr int kBoxBytes = 32 * 64; // a third stage leaves room for no more
template <int BN> constexpr int stage_bytes() { return 2 * (kBM + BN) * kBK * 2; }
template <int BN> constexpr int smem_bytes() {
  return 1024 + kStages * stage_bytes<BN>() + 8 * kBoxBytes + 8 * 128 + kSlots * (kBM + BN) * 4 + 256;
}
static_assert(smem_bytes<128>() + 64 <= 232448, "shared memory budget");

struct Gemm32 {
  long long I, J, K;
  const float *p, *q;
  long long ldp, ldq;
  int slabs, parts;
  uint32_t idesc;
  float *partial;
  Epilogue e;
  Boxes boxes;
};

// 2^e for the split of a row whose largest magnitude has these bits, e within normal powers.
__device__ __forceinline__ int split_power(uint32_t bits) {
  int ex = int(bits >> 23); // sign is clear
  int e = ex ? 141 - ex : (bits ? 126 : 0);
  return min(max(e, -126), 126);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(uint32_t(127 + e) << 23); }
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// Two neighbouring values: hi and lo halves.
__device__ __forceinline__ void split2(float a, float b, float scale, uint32_t &hi, uint32_t &lo) {
  a *= scale, b *= scale;
  __half2 h = __floats2half2_rn(a, b);
  float2 f = __half22float2(h);
  __half2 l = __floats2half2_rn(a - f.x, b - f.y);
  hi = *reinterpret_cast<uint32_t *>(&h);
  lo = *reinterpret_cast<uint32_t *>(&l);
}

// Predicated loads that leave zero where they are off.  Written out, so that each lands in its own
// register and none waits for another: a load under a branch is waited for where the branches join,
// and a second load into the same register waits for the first even if only one of them is on.
__device__ __forceinline__ float load_if(const float *p, bool on) {
  float v;
  asm volatile("{\n\t.reg .pred a;\n\tsetp.ne.u32 a, %2, 0;\n\tmov.b32 %0, 0;\n\t@a ld.global.nc.f32 %0, [%1];\n\t}"
               : "=f"(v)
               : "l"(p), "r"(unsigned(on)));
  return v;
}
__device__ __forceinline__ void load_pair_if(const float *p, bool on, float &x, float &y) {
  asm volatile("{\n\t.reg .pred a;\n\tsetp.ne.u32 a, %3, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\t"
               "@a ld.global.nc.v2.f32 {%0, %1}, [%2];\n\t}"
               : "=f"(x), "=f"(y)
               : "l"(p), "r"(unsigned(on)));
}

// The walk over (tile, slab): the same for all warps.
struct Walk {
  long long u, units, tiles;
  int k, end, slabs, parts;
  __device__ Walk(const Gemm32 &g, const Tiles &t)
      : u(blockIdx.x), units(t.count * g.parts), tiles(t.count), k(0), end(0), slabs(g.slabs), parts(g.parts) {
    open();
  }
  __device__ __forceinline__ void open() {
    if (u < units) {
      const long long s = u / tiles;
      k = int(s * slabs / parts);
      end = int((s + 1) * slabs / parts);
    }
  }
  __device__ __forceinline__ bool live() const { return u < units; }
  __device__ __forceinline__ void next() {
    if (++k >= end) {
      u += gridDim.x;
      open();
    }
  }
};

// 16 rows of an operand's slab in a warp's registers, 32 values per lane.  k-major: lane = two
// neighbouring k, v[2 r], v[2 r + 1] of row r; a row's largest magnitude by one warp reduction.
// Turned: lane = row lane % 16 and half of the slab's k, v[k].  A warp keeps two batches: one is
// split while the other's loads are in flight, and each batch's loads are issued together (loads
// interleaved with the split would share the few scoreboards that it waits on: 9x slower).
template <bool Turned> struct Batch {
  float v[32];
  __device__ __forceinline__ void load(const float *base, long long ld, bool pairs, long long row0, long long rows,
                                       long long k0, long long K) {
    const int lane = threadIdx.x & 31;
    if (Turned) {
      const long long row = row0 + (lane & 15), kf = k0 + 32 * (lane >> 4);
      const float *p = base + kf * ld + row;
      const int most = row < rows ? int(min(32ll, max(0ll, K - kf))) : 0;
#pragma unroll
      for (int i = 0; i < 32; ++i, p += ld)
        v[i] = load_if(p, i < most);
    } else {
      const long long k = k0 + 2 * lane;
      const float *p = base + row0 * ld + k;
      const int most = int(min(16ll, max(0ll, rows - row0)));
      if (pairs) {
#pragma unroll
        for (int r = 0; r < 16; ++r, p += ld)
          load_pair_if(p, k < K && r < most, v[2 * r], v[2 * r + 1]);
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r, p += ld) {
          v[2 * r] = load_if(p, k < K && r < most);
          v[2 * r + 1] = load_if(p + 1, k + 1 < K && r < most);
        }
      }
    }
  }
  // Splits into hi and lo (k-major, SWIZZLE_128B; the batch's first row at `row` of the tile) and
  // writes the rows' 2^-e.
  __device__ __forceinline__ void split(unsigned char *hi, unsigned char *lo, int row, float *unscale) {
    const int lane = threadIdx.x & 31;
    if (Turned) {
      uint32_t m[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        m[k] = magnitude(v[k]);
#pragma unroll
      for (int k = 8; k < 32; ++k)
        m[k & 7] = max(m[k & 7], magnitude(v[k]));
#pragma unroll
      for (int w = 4; w; w >>= 1)
#pragma unroll
        for (int j = 0; j < w; ++j)
          m[j] = max(m[j], m[j + w]);
      const int e = split_power(max(m[0], __shfl_xor_sync(0xffffffffu, m[0], 16))), r = row + (lane & 15);
      const float scale = pow2(e);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t h[4], l[4];
#pragma unroll
        for (int p = 0; p < 4; ++p)
          split2(v[8 * c + 2 * p], v[8 * c + 2 * p + 1], scale, h[p], l[p]);
        const int at = r * 128 + (((c + 4 * (lane >> 4)) ^ (r & 7)) << 4);
        *reinterpret_cast<uint4 *>(hi + at) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4 *>(lo + at) = make_uint4(l[0], l[1], l[2], l[3]);
      }
      if (lane < 16)
        unscale[r] = pow2(-e);
    } else {
      // All maxima before the first of them is used: the reductions' latencies overlap.
      uint32_t m[16];
#pragma unroll
      for (int r = 0; r < 16; ++r)
        m[r] = __reduce_max_sync(0xffffffffu, max(magnitude(v[2 * r]), magnitude(v[2 * r + 1])));
      float mine = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int e = split_power(m[r]);
        uint32_t h, l;
        split2(v[2 * r], v[2 * r + 1], pow2(e), h, l);
        const int at = (row + r) * 128 + (((lane >> 2) ^ ((row + r) & 7)) << 4) + ((lane & 3) << 2);
        *reinterpret_cast<uint32_t *>(hi + at) = h;
        *reinterpret_cast<uint32_t *>(lo + at) = l;
        if (lane == r)
          mine = pow2(-e);
      }
      if (lane < 16)
        unscale[row + lane] = mine;
    }
  }
};

// sum_k P(i, k) Q(j, k) for k in [k0, k1) by a whole warp, one product at a time; ends early at NaN.
__device__ __noinline__ float plain_sum(const float *p, long long pk, const float *q, long long qk, long long k0,
                                        long long k1) {
  float s = 0.f;
  for (long long k = k0; k < k1; k += 128) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long kk = k + 32 * i + (threadIdx.x & 31);
      if (kk < k1)
        s = fmaf(p[kk * pk], q[kk * qk], s);
    }
    if (__any_sync(0xffffffffu, s != s))
      return __uint_as_float(0x7fc00000u);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1)
    s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

template <int BN, bool PT, bool QT>
__global__ void __launch_bounds__(kThreads, 1) gemm32_kernel(const __grid_constant__ Gemm32 g) {
  constexpr int kPBytes = kBM * kBK * 2, kQBytes = BN * kBK * 2, kStageBytes = stage_bytes<BN>();
  constexpr int kTmemCols = 2 * BN;
  extern __shared__ unsigned char smem_raw[];
  unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char *staging = smem + kStages * kStageBytes; // a box per drain warp, then its bias
  float *scales = reinterpret_cast<float *>(staging + 8 * kBoxBytes + 8 * 128); // [kSlots][kBM + BN]: 2^-e of P's rows, then of Q's
  uint64_t *bars = reinterpret_cast<uint64_t *>(scales + kSlots * (kBM + BN));
  // ready[S] | empty[S] | tfull[2] | tfree[2] | done | scaled[kSlots] | residual[8]
  __shared__ uint32_t tmem_base;
  __shared__ volatile int abort_flag;
  __shared__ int mma_done_issued;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned ready0 = smem_u32(bars), empty0 = ready0 + 8 * kStages, tfull0 = empty0 + 8 * kStages,
                 tfree0 = tfull0 + 16, done = tfree0 + 16, scaled0 = done + 8, residual0 = scaled0 + 8 * kSlots;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    mma_done_issued = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(ready0 + 8 * s, kSplitThreads);
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull0 + 8 * b, 1);
      mbar_init(tfree0 + 8 * b, kDrainThreads);
    }
    mbar_init(done, 1);
    for (int x = 0; x < kSlots; ++x)
      mbar_init(scaled0 + 8 * x, 8);
    for (int x = 0; x < 8; ++x)
      mbar_init(residual0 + 8 * x, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async_smem();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  const Tiles tiles(g.I, g.J, kBM, BN);

  // The MMAs of slab n (one thread).
  auto multiply = [&](int n) {
    const int st = n % kStages, b = n & 1;
    if (!mbar_wait(ready0 + 8 * st, unsigned(n / kStages) & 1, &abort_flag) ||
        (n >= 2 && !mbar_wait(tfree0 + 8 * b, unsigned(n / 2 - 1) & 1, &abort_flag)))
      return false;
    tc_fence_after();
    const unsigned ph = smem_u32(smem + st * kStageBytes), pl = ph + kPBytes, qh = pl + kPBytes, ql = qh + kQBytes;
    const uint32_t d = tmem + uint32_t(b * BN);
#pragma unroll
    for (int m = 0; m < kBK / 16; ++m) { // the small terms first
      umma_f16_desc(d, smem_desc(pl + 32 * m), smem_desc(qh + 32 * m), g.idesc, m ? 1u : 0u);
      umma_f16_desc(d, smem_desc(ph + 32 * m), smem_desc(ql + 32 * m), g.idesc, 1u);
    }
#pragma unroll
    for (int m = 0; m < kBK / 16; ++m)
      umma_f16_desc(d, smem_desc(ph + 32 * m), smem_desc(qh + 32 * m), g.idesc, 1u);
    umma_commit(empty0 + 8 * st);
    umma_commit(tfull0 + 8 * b);
    return true;
  };
  // A split warp: `high` (16 or 32) rows of every tile's P or Q from row `first` of the tile.
  auto split_warp = [&](auto turned, auto high, int first, bool of_q) {
    constexpr bool Turned = decltype(turned)::value;
    constexpr int kHigh = decltype(high)::value;
    const float *base = of_q ? g.q : g.p;
    const long long ld = of_q ? g.ldq : g.ldp, rows = of_q ? g.J : g.I;
    // 8-byte loads: aligned, and none crosses the end of a row.
    const bool pairs = reinterpret_cast<uintptr_t>(base) % 8 == 0 && (rows <= 1 || ld % 2 == 0) && g.K % 2 == 0;
    Batch<Turned> batch[2];
    // The walk of the loads, and the first row of its tile; it leads by the two batches.
    Walk ahead(g, tiles);
    long long row0 = 0, row_u = -1;
    auto load = [&](Batch<Turned> &b, int row) {
      if (!ahead.live())
        return;
      if (ahead.u != row_u) {
        long long i, j;
        tiles.at(ahead.u % tiles.count, i, j);
        row0 = (of_q ? j * BN : i * kBM) + first;
        row_u = ahead.u;
      }
      b.load(base, ld, pairs, row0 + row, rows, (long long)ahead.k * kBK, g.K);
      if (row + 16 == kHigh)
        ahead.next();
    };
    load(batch[0], 0);
    load(batch[1], kHigh == 32 ? 16 : 0);
    bool ok = true, issued = true; // ok: the same in the whole warp
    int n = 0;
    auto slab = [&](auto one) { // slab n from both batches (32 rows) or from batch[one]
      const int st = n % kStages;
      ok = issued && (n < kStages || mbar_wait(empty0 + 8 * st, unsigned(n / kStages - 1) & 1, &abort_flag));
      if (!(ok = __all_sync(0xffffffffu, ok)))
        return;
      unsigned char *hi = smem + st * kStageBytes + (of_q ? 2 * kPBytes : 0), *lo = hi + (of_q ? kQBytes : kPBytes);
      float *unscale = scales + n % kSlots * (kBM + BN) + (of_q ? kBM : 0);
      if (kHigh == 32) {
        batch[0].split(hi, lo, first, unscale);
        load(batch[0], 0);
        batch[1].split(hi, lo, first + 16, unscale);
        load(batch[1], 16);
      } else {
        constexpr int k = decltype(one)::value;
        batch[k].split(hi, lo, first, unscale);
        load(batch[k], 0);
      }
      fence_proxy_async_smem();
      mbar_arrive(ready0 + 8 * st);
      __syncwarp();
      if (lane == 0) // this warp's scales, for the drain
        mbar_arrive(scaled0 + 8 * (n % kSlots));
      if (warp == 0 && lane == 0 && n)
        issued = multiply(n - 1);
      ++n;
    };
    Walk w(g, tiles);
    while (w.live() && ok) {
      slab(std::integral_constant<int, 0>{});
      w.next();
      if (kHigh == 16 && w.live() && ok) {
        slab(std::integral_constant<int, 1>{});
        w.next();
      }
    }
    if (warp == 0 && lane == 0) {
      if (ok && issued && n)
        multiply(n - 1);
      umma_commit(done);
      mma_done_issued = 1;
    }
  };

  using std::integral_constant;
  if (warp < 4)
    split_warp(integral_constant<bool, PT>{}, integral_constant<int, 32>{}, 32 * warp, false);
  else if (warp < 8)
    split_warp(integral_constant<bool, QT>{}, integral_constant<int, BN / 4>{}, BN / 4 * (warp - 4), true);
  else {
    constexpr int kCols = BN / 2;
    const int quarter = warp & 3, half = (warp - 8) >> 2;
    const int me = warp - 8;
    Warp box{staging + me * kBoxBytes, reinterpret_cast<float *>(staging + 8 * kBoxBytes + me * 128), residual0 + 8 * me, 0};
    float acc[kCols];
    bool ok = true;
    int n = 0;
    for (Walk w(g, tiles); w.live();) {
      const long long u = w.u, s = u / tiles.count;
      const long long k0 = (long long)w.k * kBK, k1 = min(g.K, (long long)w.end * kBK);
      long long i, j;
      tiles.at(u - s * tiles.count, i, j);
#pragma unroll
      for (int c = 0; c < kCols; ++c)
        acc[c] = 0.f;
      for (; w.live() && w.u == u; w.next(), ++n) {
        const int b = n & 1;
        ok = ok && mbar_wait(tfull0 + 8 * b, unsigned(n / 2) & 1, &abort_flag) &&
             mbar_wait(scaled0 + 8 * (n % kSlots), unsigned(n / kSlots) & 1, &abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok)
          continue;
        tc_fence_after();
        const float *scale = scales + n % kSlots * (kBM + BN);
        const float fp = scale[32 * quarter + lane];
        const float *fq = scale + kBM + half * kCols;
#pragma unroll
        for (int c0 = 0; c0 < kCols; c0 += 32) {
          uint32_t r[32];
          tmem_ld32_async(tmem + (uint32_t(quarter * 32) << 16) + uint32_t(b * BN + half * kCols + c0), r);
          tmem_wait_ld();
          tmem_anchor(r);
          if (c0 + 32 == kCols) {
            tc_fence_before();
            mbar_arrive(tfree0 + 8 * b);
          }
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            const float4 f = *reinterpret_cast<const float4 *>(fq + c0 + c);
            const float fs[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const uint32_t bits = r[c + x];
              // One ulp away from zero (not zero itself, infinities and NaN); then the two exact
              // scalings.
              const uint32_t away = bits + ((bits << 1) - 1u < 0xfeffffffu);
              acc[c0 + c + x] = fmaf(__uint_as_float(away) * fs[x], fp, acc[c0 + c + x]);
            }
          }
        }
      }
      float *partial = g.partial ? g.partial + s * g.I * g.J : nullptr;
      const long long row0 = i * kBM + 32 * quarter, row = row0 + lane;
#pragma unroll
      for (int c0 = 0; c0 < kCols; c0 += 32) {
        const long long col0 = j * BN + half * kCols + c0;
        if (row0 >= g.I || col0 >= g.J)
          continue;
        bool odd = false;
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          if (!ok) // a wait that ran out shows as NaN
            acc[c0 + c] = __uint_as_float(0x7fc00000u);
          odd |= !(fabsf(acc[c0 + c]) < INFINITY);
        }
        if (__any_sync(0xffffffffu, odd && ok)) {
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            unsigned todo = __ballot_sync(0xffffffffu, !(fabsf(acc[c0 + c]) < INFINITY) && row < g.I && col0 + c < g.J);
            while (todo) {
              const int at = __ffs(todo) - 1;
              todo &= todo - 1;
              const float x = plain_sum(g.p + (row0 + at) * (PT ? 1 : g.ldp), PT ? g.ldp : 1,
                                        g.q + (col0 + c) * (QT ? 1 : g.ldq), QT ? g.ldq : 1, k0, k1);
              if (lane == at)
                acc[c0 + c] = x;
            }
          }
        }
        if (g.boxes.on)
#pragma unroll
          for (int h = 0; h < 32; h += 16) {
            if (col0 + h < g.J)
              finish_box<float, 64>(g.e, g.boxes, g.J, row0, col0 + h, g.partial ? int(s) : -1, box,
                                    [&](int, float (&v)[16]) {
#pragma unroll
                                      for (int c = 0; c < 16; ++c)
                                        v[c] = acc[c0 + h + c];
                                    });
          }
        else
          finish_block<float>(g.e, partial, g.I, g.J, row0, col0, acc + c0, reinterpret_cast<float *>(box.box));
      }
    }
    if (lane == 0)
      bulk_wait();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    if (abort_flag && mma_done_issued) { // bounded wait for the MMAs in flight before TMEM goes
      long long start = clock64();
      while (!mbar_try(done, 0) && clock64() - start < kWaitCycles) {
      }
    }
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

template <int BN, bool PT, bool QT> void launch_gemm32(const Gemm32 &g, cudaStream_t stream) {
  static thread_local int configured = -1;
  int device = 0;
  lapis::check(cudaGetDevice(&device));
  if (configured != device) {
    lapis::check(cudaFuncSetAttribute(gemm32_kernel<BN, PT, QT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      smem_bytes<BN>()));
    configured = device;
  }
  long long units = Tiles(g.I, g.J, kBM, BN).count * g.parts;
  lapis::launch(gemm32_kernel<BN, PT, QT>, dim3(unsigned(std::min<long long>(units, sm_count()))), kThreads,
                smem_bytes<BN>(), stream, g);
  lapis::check(cudaGetLastError());
}
} // namespace

// 128-wide tiles, 64-wide ones for at most 64 columns; few tiles are cut along k until they fill the
// device, parts of at least two slabs.
Plan plan32(long long I, long long J, long long K) {
  Plan p{J <= 64 ? 64 : 128, 1};
  const long long tiles = Tiles(I, J, kBM, p.bn).count, slabs = (K + kBK - 1) / kBK;
  p.parts = int(std::min<long long>({std::max(1ll, sm_count() / tiles), std::max(1ll, slabs / 2), 148}));
  return p;
}

void product32(const Product &p, void *workspace, cudaStream_t stream) {
  const Plan plan = plan32(p.I, p.J, p.K);
  Gemm32 g{p.I, p.J, p.K, static_cast<const float *>(p.p.p), static_cast<const float *>(p.q.p), p.p.ld, p.q.ld};
  g.slabs = int((p.K + kBK - 1) / kBK);
  g.parts = plan.parts;
  g.idesc = idesc_f16(kBM, plan.bn);
  g.partial = plan.parts > 1 ? static_cast<float *>(workspace) : nullptr;
  g.e = p.e;
  g.boxes = boxes_of(p, g.partial, plan.parts, 64);
  auto width = [&](auto bn) {
    constexpr int BN = decltype(bn)::value;
    if (!p.p.turned && !p.q.turned)
      launch_gemm32<BN, false, false>(g, stream);
    else if (!p.p.turned)
      launch_gemm32<BN, false, true>(g, stream);
    else
      launch_gemm32<BN, true, true>(g, stream);
  };
  if (plan.bn == 128)
    width(std::integral_constant<int, 128>{});
  else
    width(std::integral_constant<int, 64>{});
  if (plan.parts > 1)
    finish_parts(F32, p.e, g.partial, plan.parts, p.I, p.J, stream);
}
} // namespace op
} // namespace mace
