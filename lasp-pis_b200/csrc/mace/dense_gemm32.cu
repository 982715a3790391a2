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
// must not add up over long k.  A slab's result comes out 8.7e-8 too small in the mean (tc_gemm.cu),
// so three slabs of four are scaled by 1 + 2^-23: 8.9e-8.
//
// TMA brings the slab's floats into the place of the split (128 rows of 64 floats are as large as two
// fp16 planes), whichever index is contiguous; the split reads a row per thread and leaves it k-major,
// hi over the first half and lo over the second.  16 warps, 128 registers each:
//   0..7    split, a row per thread: four warps P, four Q (two in 64-wide tiles).  The warp that
//           finishes a slab last issues its MMAs.
//   8..15   drain: lane = output row, two warps per TMEM lane quadrant, BN / 2 columns each, and the
//           epilogue.  A slab that has reached TMEM has left its stage: warp 8 then starts the
//           loads of the slab three ahead.
// (Loading by plain loads straight into the registers of the split was 5 times slower: the loads of
// 64 KB per slab stalled the split warps.)
// Infinities and NaN make every result of their row (of P or Q) NaN in this scheme; results that
// are not finite are summed again, one product at a time.
#include "dense_gemm.cuh"

namespace mace {
namespace op {
namespace {
using namespace tc;
constexpr int kBM = 128, kBK = 64, kStages = 3;
constexpr int kThreads = 512, kDrainThreads = 256;
// The split of slab g runs after the MMAs of g - 3, which waited for the drain of g - 5.
constexpr int kSlots = 5;
template <int BN> constexpr int stage_bytes() { return 2 * (kBM + BN) * kBK * 2; }
template <int BN> constexpr int smem_bytes() {
  return kStages * stage_bytes<BN>() + 8 * kBoxBytes + kSlots * (kBM + 2 * BN) + 384;
}
static_assert(smem_bytes<128>() <= 232448, "shared memory budget");

struct Gemm32 {
  CUtensorMap mp, mq;
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
  int ex = int(bits >> 23) & 0xff;
  int e = ex ? 141 - ex : (bits ? 126 : 0);
  return min(max(e, -126), 126);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(uint32_t(127 + e) << 23); }
// Two neighbouring values: hi and lo halves (the remainder v 2^e - hi is exact).
__device__ __forceinline__ void split2(float2 v, float2 scale, uint32_t &hi, uint32_t &lo) {
  const float2 x = __fmul2_rn(v, scale);
  const __half2 h = __float22half2_rn(x);
  const __half2 l = __float22half2_rn(__ffma2_rn(__half22float2(h), make_float2(-1.f, -1.f), x));
  hi = *reinterpret_cast<const uint32_t *>(&h);
  lo = *reinterpret_cast<const uint32_t *>(&l);
}

// The walk over (tile, slab): the same for all warps.
struct Walk {
  long long u, units, tiles;
  int k, end, slabs, parts;
  Walk() = default;
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

// The walk's state of the loads, and what the warps share.
struct Shared {
  Walk ahead;
  uint32_t tmem_base;
  volatile int abort_flag;
  int arrived[kSlots]; // split warps that are through with a slab
};

// Splits row r of an operand's slab (ROWS rows, floats at `base`) in place.  k-major: two boxes of
// ROWS rows by 32 k; a thread's row is its own.  Turned: boxes of 64 k by 32 rows; the rows of a box
// are read by a warp's lanes together, and all of the operand's threads have read before any
// writes (named barrier `id` of ROWS threads).  Returns the power of two that scales back, biased.
template <int ROWS, bool Turned>
__device__ __forceinline__ unsigned split_row(unsigned char *base, int r, int id) {
  float v[64];
  if (Turned) {
    const unsigned char *box = base + (r >> 5) * 8192 + (r & 3) * 4;
    const int chunk = r >> 2 & 7;
#pragma unroll
    for (int k = 0; k < 64; ++k)
      v[k] = *reinterpret_cast<const float *>(box + k * 128 + ((chunk ^ (k & 7)) << 4));
  } else {
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      const float4 x = *reinterpret_cast<const float4 *>(base + (c >> 3) * (ROWS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
      v[4 * c] = x.x, v[4 * c + 1] = x.y, v[4 * c + 2] = x.z, v[4 * c + 3] = x.w;
    }
  }
  // The largest magnitude; NaN does not count, and stays NaN in the split.
  float m[8];
#pragma unroll
  for (int k = 0; k < 8; ++k)
    m[k] = fabsf(v[k]);
#pragma unroll
  for (int k = 8; k < 64; ++k)
    m[k & 7] = fmaxf(m[k & 7], fabsf(v[k]));
#pragma unroll
  for (int w = 4; w; w >>= 1)
#pragma unroll
    for (int j = 0; j < w; ++j)
      m[j] = fmaxf(m[j], m[j + w]);
  const int e = split_power(__float_as_uint(m[0]));
  const float2 scale = make_float2(pow2(e), pow2(e));
  if (Turned)
    asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(ROWS) : "memory");
  unsigned char *hi = base + r * 128, *lo = hi + ROWS * 128;
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int p = 0; p < 4; ++p)
      split2(make_float2(v[8 * c + 2 * p], v[8 * c + 2 * p + 1]), scale, h[p], l[p]);
    const int at = (c ^ (r & 7)) << 4;
    *reinterpret_cast<uint4 *>(hi + at) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4 *>(lo + at) = make_uint4(l[0], l[1], l[2], l[3]);
  }
  return unsigned(127 - e);
}

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
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char *staging = smem + kStages * kStageBytes; // a box per drain warp
  // [kSlots][2 BN + kBM]: 2^-e of Q's rows (the upper halves of floats), then 127 - e of P's
  unsigned char *scales = staging + 8 * kBoxBytes;
  constexpr int kSlotBytes = 2 * BN + kBM;
  uint64_t *bars = reinterpret_cast<uint64_t *>(scales + kSlots * kSlotBytes);
  // full[S] | tfull[2] | tfree[2] | scaled[kSlots] | residual[8]
  constexpr int kBars = kStages + 4 + kSlots + 8;
  static_assert(kBars * 8 + sizeof(Shared) <= 384, "barriers and state");
  Shared &sh = *reinterpret_cast<Shared *>(bars + kBars);
  volatile int &abort_flag = sh.abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned full0 = smem_u32(bars), tfull0 = full0 + 8 * kStages, tfree0 = tfull0 + 16, scaled0 = tfree0 + 16,
                 residual0 = scaled0 + 8 * kSlots;
  constexpr int kSplitWarps = 4 + BN / 32;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < kStages; ++s)
      mbar_init(full0 + 8 * s, 1);
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull0 + 8 * b, 1);
      mbar_init(tfree0 + 8 * b, kDrainThreads);
    }
    for (int x = 0; x < kSlots; ++x) {
      mbar_init(scaled0 + 8 * x, kSplitWarps);
      sh.arrived[x] = 0;
    }
    for (int x = 0; x < 8; ++x)
      mbar_init(residual0 + 8 * x, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async_smem();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem_base;
  const Tiles tiles(g.I, g.J, kBM, BN);

  // The MMAs of slab n (one thread).
  auto multiply = [&](int n) {
    const int b = n & 1;
    if (n >= 2 && !mbar_wait(tfree0 + 8 * b, unsigned(n / 2 - 1) & 1, &sh.abort_flag))
      return;
    tc_fence_after();
    const unsigned ph = smem_u32(smem + n % kStages * kStageBytes), pl = ph + kPBytes, qh = pl + kPBytes, ql = qh + kQBytes;
    const uint32_t d = tmem + uint32_t(b * BN);
#pragma unroll
    for (int m = 0; m < kBK / 16; ++m) { // the small terms first
      umma_f16_desc(d, smem_desc(pl + 32 * m), smem_desc(qh + 32 * m), g.idesc, m ? 1u : 0u);
      umma_f16_desc(d, smem_desc(ph + 32 * m), smem_desc(ql + 32 * m), g.idesc, 1u);
    }
#pragma unroll
    for (int m = 0; m < kBK / 16; ++m)
      umma_f16_desc(d, smem_desc(ph + 32 * m), smem_desc(qh + 32 * m), g.idesc, 1u);
    umma_commit(tfull0 + 8 * b);
  };
  // The loads of slab n at walk w (one thread; the MMAs of slab n - 3 are done).
  auto fetch = [&](int n, const Walk &w) {
    long long i, j;
    tiles.at(w.u % tiles.count, i, j);
    const int i0 = int(i * kBM), j0 = int(j * BN), k0 = w.k * kBK;
    const unsigned base = smem_u32(smem + n % kStages * kStageBytes), full = full0 + 8 * (n % kStages);
    mbar_expect_tx(full, kStageBytes);
    if (PT) {
#pragma unroll
      for (int h = 0; h < kBM / 32; ++h)
        tma_load_2d(base + 8192 * h, &g.mp, i0 + 32 * h, k0, full);
    } else {
      tma_load_2d(base, &g.mp, k0, i0, full);
      tma_load_2d(base + kPBytes, &g.mp, k0 + 32, i0, full);
    }
    if (QT) {
#pragma unroll
      for (int h = 0; h < BN / 32; ++h)
        tma_load_2d(base + 2 * kPBytes + 8192 * h, &g.mq, j0 + 32 * h, k0, full);
    } else {
      tma_load_2d(base + 2 * kPBytes, &g.mq, k0, j0, full);
      tma_load_2d(base + 2 * kPBytes + kQBytes, &g.mq, k0 + 32, j0, full);
    }
  };

  if (warp < kSplitWarps) {
    const bool of_q = warp >= 4;
    const int r = threadIdx.x & 127;
    bool ok = true; // the same in the whole warp
    int n = 0;
    for (Walk w(g, tiles); w.live(); w.next(), ++n) {
      ok = __all_sync(0xffffffffu, ok && mbar_wait(full0 + 8 * (n % kStages), unsigned(n / kStages) & 1, &sh.abort_flag));
      if (!ok) { // the other warps of the operand may wait at this slab's barrier
        if (of_q ? QT : PT)
          asm volatile("bar.sync %0, %1;" ::"r"(of_q ? 2 : 1), "r"(of_q ? BN : kBM) : "memory");
        continue;
      }
      unsigned char *stage = smem + n % kStages * kStageBytes, *scale = scales + n % kSlots * kSlotBytes;
      if (of_q)
        reinterpret_cast<unsigned short *>(scale)[r] =
            static_cast<unsigned short>(split_row<BN, QT>(stage + 2 * kPBytes, r, 2) << 7);
      else
        scale[2 * BN + r] = static_cast<unsigned char>(split_row<kBM, PT>(stage, r, 1));
      // Each lane's stores, then the warp's, are visible before the warp counts as arrived; the
      // last to arrive sees all of them.
      fence_proxy_async_smem();
      __threadfence_block();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(scaled0 + 8 * (n % kSlots)); // this warp's scales, for the drain
        if (atomicAdd(&sh.arrived[n % kSlots], 1) == kSplitWarps - 1) {
          sh.arrived[n % kSlots] = 0;
          __threadfence_block();
          fence_proxy_async_smem();
          multiply(n);
        }
      }
    }
  } else if (warp >= 8) {
    constexpr int kCols = BN / 2;
    const int quarter = warp & 3, half = (warp - 8) >> 2;
    const int me = warp - 8;
    Warp box{staging + me * kBoxBytes, residual0 + 8 * me, 0};
    // The residual of a tile's first box is on its way while the tile accumulates (a kept z needs the
    // box first).
    const bool early = g.boxes.on && !g.partial && g.e.residual && !g.e.z;
    Walk &ahead = sh.ahead; // of the loads: warp 8's first lane
    if (me == 0 && lane == 0) {
      ahead = Walk(g, tiles);
      for (int x = 0; x < kStages && ahead.live(); ++x, ahead.next())
        fetch(x, ahead);
    }
    float acc[kCols];
    bool ok = true;
    int n = 0;
    for (Walk w(g, tiles); w.live();) {
      const long long u = w.u, s = u / tiles.count;
      const long long k0 = (long long)w.k * kBK, k1 = min(g.K, (long long)w.end * kBK);
      long long i, j;
      tiles.at(u - s * tiles.count, i, j);
      const long long row0 = i * kBM + 32 * quarter, row = row0 + lane, cols0 = j * BN + half * kCols;
      const bool any = row0 < g.I && cols0 < g.J;
      float bias[kCols / 32];
#pragma unroll
      for (int c = 0; c < kCols / 32; ++c)
        bias[c] = g.e.bias && cols0 + 32 * c + lane < g.J ? static_cast<const float *>(g.e.bias)[cols0 + 32 * c + lane] : 0.f;
      if (early && any && lane == 0) {
        bulk_wait_read();
        fetch_residual(g.boxes, box, row0, cols0);
      }
#pragma unroll
      for (int c = 0; c < kCols; ++c)
        acc[c] = 0.f;
      for (; w.live() && w.u == u; w.next(), ++n) {
        const int b = n & 1;
        ok = ok && mbar_wait(tfull0 + 8 * b, unsigned(n / 2) & 1, &sh.abort_flag) &&
             mbar_wait(scaled0 + 8 * (n % kSlots), unsigned(n / kSlots) & 1, &sh.abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok)
          continue;
        if (me == 0 && lane == 0 && ahead.live()) {
          fetch(n + kStages, ahead);
          ahead.next();
        }
        tc_fence_after();
        const unsigned char *scale = scales + n % kSlots * kSlotBytes;
        const unsigned char *fq = scale + 2 * (half * kCols);
        // 2^-e of P's row, one ulp more in three slabs of four.
        const float fp = __uint_as_float((uint32_t(scale[2 * BN + 32 * quarter + lane]) << 23) + ((n & 3) != 3));
        const float2 fp2 = make_float2(fp, fp);
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
            const uint2 f = *reinterpret_cast<const uint2 *>(fq + 2 * (c0 + c));
            const uint32_t fs[2] = {f.x, f.y};
#pragma unroll
            for (int y = 0; y < 2; ++y) { // the two scalings, and the float sum
              const int x = c0 + c + 2 * y;
              const float2 s = make_float2(__uint_as_float(fs[y] << 16), __uint_as_float(fs[y] & 0xffff0000u));
              const float2 a = __ffma2_rn(
                  __fmul2_rn(make_float2(__uint_as_float(r[c + 2 * y]), __uint_as_float(r[c + 2 * y + 1])), s), fp2,
                  make_float2(acc[x], acc[x + 1]));
              acc[x] = a.x, acc[x + 1] = a.y;
            }
          }
        }
      }
      float *partial = g.partial ? g.partial + s * g.I * g.J : nullptr;
#pragma unroll
      for (int c0 = 0; c0 < kCols; c0 += 32) {
        const long long col0 = cols0 + c0;
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
          finish_box<float>(
              g.e, g.boxes, row0, col0, g.partial ? int(s) : -1, box, early && c0 == 0,
              [&](int, float (&v)[32]) {
#pragma unroll
                for (int c = 0; c < 32; ++c)
                  v[c] = acc[c0 + c];
              },
              [&](int) { return bias[c0 / 32]; });
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
    if (abort_flag) { // bounded pause for copies and MMAs in flight before TMEM and the CTA go
      long long start = clock64();
      while (clock64() - start < kWaitCycles / 100) {
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
  Gemm32 g{};
  g.I = p.I, g.J = p.J, g.K = p.K;
  g.p = static_cast<const float *>(p.p.p), g.ldp = p.p.ld;
  g.q = static_cast<const float *>(p.q.p), g.ldq = p.q.ld;
  g.mp = p.p.turned ? tile_map(F32, p.p.p, p.K, p.I, p.p.ld, kBK) : tile_map(F32, p.p.p, p.I, p.K, p.p.ld, kBM);
  g.mq = p.q.turned ? tile_map(F32, p.q.p, p.K, p.J, p.q.ld, kBK) : tile_map(F32, p.q.p, p.J, p.K, p.q.ld, plan.bn);
  g.slabs = int((p.K + kBK - 1) / kBK);
  g.parts = plan.parts;
  g.idesc = idesc_f16(kBM, plan.bn);
  g.partial = plan.parts > 1 ? static_cast<float *>(workspace) : nullptr;
  g.e = p.e;
  g.boxes = boxes_of(p, g.partial, plan.parts);
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
