// The dense layer's matrix products of floats on the tensor cores (tcgen05, kind::f16), with an error
// like that of float arithmetic.
//
//   out(i, j) = sum_k P(i, k) Q(j, k)
//
// Both operands are split on the way to the tensor cores: per row and 64-wide slab of k, with 2^e the
// power of two that brings the largest magnitude into [2^14, 2^15), v 2^e = hi + 2^-12 lo, both fp16
// rounded to nearest.  Scaled so, lo is as large as hi, and values down to 2^-29 of the largest keep 22
// bits (2^-23 of themselves), smaller ones 2^-52 of the largest.  A slab's products lo*hi + hi*lo
// accumulate fresh in TMEM, the first product of hi*hi scales them by 2^-12 (lo*lo is below 2^-22), and
// the sum is scaled back by the two exact powers of two and added to float registers: the tensor pipe
// truncates, which must not add up over long k.  A slab's result comes out too small by that, 9e-8 in the
// mean for values of both signs, 2e-7 for values of one; no factor makes up for it, since sums that are
// exact in floats (small integers, one product) come out exact.  2-norm errors against 64 bits: 1.3e-7
// to 2.1e-7, where float sums in order have 1.2e-7 to 1.6e-6.
//
// TMA brings the slab's floats into shared memory, whichever index is contiguous; the split reads a row
// per thread.  P's rows go to TMEM, the first operand's other place; Q's over their floats, k-major
// (64 floats are as long as two rows of fp16), hi over the first half and lo over the second.  16 warps,
// 128 registers each at launch:
//   0..7    split.  64-wide tiles: two groups take the slabs in turn, a row of P and (half of them) one
//           of Q per thread; the latencies of a split, not its instructions, take its time, and so
//           two are under way (gradients of 84613 x 64 -> 1280: 351 -> 291 us).  128-wide ones have
//           only two stages, which one group uses better (61 us against 67 for 10000 x 512 -> 512):
//           four warps P, four Q.  The warp that finishes a slab last issues its MMAs, all operands
//           uniform (84613 x 64 -> 1280: 182 -> 172 us).
//   8..15   drain: lane = output row, two warps per TMEM lane quadrant, BN / 2 columns each, and the
//           epilogue.  A slab that has reached TMEM has left its stage: one of them (in turn) then
//           starts the loads of the slab that takes its place.
// What bounds it: no unit (gradients of 84613 x 64 -> 1280, 284 us: issue slots 47% busy, DRAM 41%, tensor
// pipe 17%), but the chain load, split, multiply, drain of a slab at one CTA per SM (10000 x 512 -> 512: 57
// us); with one slab per tile (84613 x 64 -> 1280: 155 us, 2.9 TB/s) the drain, by its instructions'
// latencies: the bias as the sums' first value, prefetched, and scales as whole floats took it from 200 us
// to 179.  Measured and not kept: plain loads
// straight into the split's registers (10000 x 512 -> 512: 174 us, then 104 with TMA), P split in place
// (358 us where TMEM gave 351), L2 prefetches of P (no change), three stages and one box of results for
// 128-wide tiles (84613 x 64 -> 1280: 245 us), results written from registers by sectors (227 us).
// Infinities and NaN make every result of their row (of P or Q) NaN in this scheme; results that
// are not finite are summed again, one product at a time.
#include "dense_gemm.cuh"

namespace mace {
namespace op {
namespace {
using namespace tc;
constexpr int kBM = 128, kBK = 64;
constexpr int kThreads = 512, kDrainThreads = 256;
constexpr int kLoBits = 12; // lo halves hold (v 2^e - hi) 2^12: up to 2^15, as hi
template <int BN> constexpr int stage_bytes() { return 2 * (kBM + BN) * kBK * 2; }
// 64-wide tiles: three stages, and a box of results per drain warp; 128-wide ones: two and two.  TMEM
// holds P's split slabs, 64 columns for each stage, and as many accumulators as then fit.
template <int BN> constexpr int stages() { return BN == 64 ? 3 : 2; }
template <int BN> constexpr int buffers() { return BN == 64 ? 4 : 3; }
static_assert(buffers<64>() * 64 + stages<64>() * 64 <= 512 && buffers<128>() * 128 + stages<128>() * 64 <= 512, "TMEM");
// Scales of a slab's rows, from its split to its drain.  The split of slab n writes them after the MMAs of
// n - stages, which wait until every drain warp has read TMEM for n - stages - buffers.  A warp reads
// the last of that slab's scales after that, but those of the slab before ahead of it: a slot more than
// buffers + stages.
template <int BN> constexpr int slots() { return buffers<BN>() + stages<BN>() + 1; }
template <int BN> constexpr int slot_bytes() { return 4 * BN + kBM; }
template <int BN> constexpr int smem_bytes() {
  return stages<BN>() * stage_bytes<BN>() + 8 * (BN / 64) * kBoxBytes + 8 * (BN / 2) * 4 + slots<BN>() * slot_bytes<BN>() + 512;
}
static_assert(smem_bytes<128>() <= 232448 && smem_bytes<64>() <= 232448, "shared memory budget");

struct Gemm32 {
  CUtensorMap mp, mq;
  long long I, J, K;
  const float *p, *q;
  long long ldp, ldq;
  Tiles tiles;
  unsigned units; // tiles x parts
  int slabs, parts;
  uint32_t idesc;
  float *partial;
  float *sums; // of P's rows over each part's k, [parts][2][I] (turned P; NULL: not wanted)
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
// Two neighbouring values: hi and lo halves (the remainder v 2^e - hi is exact; its half is scaled by 2^kLoBits).
__device__ __forceinline__ void split2(float2 v, float2 scale, uint32_t &hi, uint32_t &lo) {
  constexpr float kUp = float(1 << kLoBits);
  const float2 x = __fmul2_rn(v, scale);
  const __half2 h = __float22half2_rn(x);
  const float2 rest = __ffma2_rn(__half22float2(h), make_float2(-1.f, -1.f), x);
  const __half2 l = __float22half2_rn(__fmul2_rn(rest, make_float2(kUp, kUp)));
  hi = *reinterpret_cast<const uint32_t *>(&h);
  lo = *reinterpret_cast<const uint32_t *>(&l);
}

// The walk over (part of a tile, slab): the same for all warps.  Unit u is part u / tiles of tile
// u % tiles, slabs [k, end).
struct Walk {
  unsigned u, tile;
  int k, end, part;
  __device__ __forceinline__ explicit Walk(const Gemm32 &g) : u(blockIdx.x) { open(g); }
  __device__ __forceinline__ void open(const Gemm32 &g) {
    part = 0;
    tile = u;
    k = 0;
    end = g.slabs;
    if (g.parts > 1) {
      part = int(u / g.tiles.count);
      tile = u - unsigned(part) * g.tiles.count;
      k = int((long long)part * g.slabs / g.parts);
      end = int((part + 1ll) * g.slabs / g.parts);
    }
  }
  __device__ __forceinline__ bool live(const Gemm32 &g) const { return u < g.units; }
  // Whether the next slab opens another unit.
  __device__ __forceinline__ bool next(const Gemm32 &g) {
    if (++k < end)
      return false;
    skip(g);
    return true;
  }
  __device__ __forceinline__ void skip(const Gemm32 &g) {
    u += gridDim.x;
    open(g);
  }
};

// What the warps share.
struct Shared {
  uint32_t tmem_base;
  volatile int abort_flag;
  volatile int progress; // of sums that a drain warp adds again
  int arrived[8]; // per slot: split warps that are through with a slab
};

// Bounded wait, as mbar_wait; but results that are summed again may take a drain warp longer than that (a
// finite number of them, each ends), and while their count grows the others wait on.
__device__ __forceinline__ bool wait_for(unsigned bar, unsigned parity, Shared &sh) {
  long long start = clock64();
  int seen = sh.progress;
  for (unsigned it = 1;; ++it) {
    if (mbar_try(bar, parity))
      return true;
    if (sh.abort_flag)
      return false;
    if (it & 255)
      continue;
    if (sh.progress != seen) {
      seen = sh.progress;
      start = clock64();
    } else if (clock64() - start > kWaitCycles) {
      sh.abort_flag = 1;
      return false;
    }
  }
}

// Row r of an operand's slab (ROWS rows, floats at `base`).  k-major: two boxes of ROWS rows by 32 k; a
// thread's row is its own.  Turned: boxes of 64 k by 32 rows, which a warp's lanes read together.
template <int ROWS, bool Turned> __device__ __forceinline__ void read_row(const unsigned char *base, int r, float (&v)[64]) {
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
}
// The exponent that scales a row, from its largest magnitude; NaN does not count, and stays NaN in the
// split.
__device__ __forceinline__ int row_power(const float (&v)[64]) {
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
  return split_power(__float_as_uint(m[0]));
}
__device__ __forceinline__ float row_sum(const float (&v)[64]) {
  float2 s[4] = {};
#pragma unroll
  for (int k = 0; k < 64; k += 2)
    s[k / 2 & 3] = __fadd2_rn(s[k / 2 & 3], make_float2(v[k], v[k + 1]));
  s[0] = __fadd2_rn(__fadd2_rn(s[0], s[1]), __fadd2_rn(s[2], s[3]));
  return s[0].x + s[0].y;
}
// 16 columns of this warp's 32 lanes.
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
               "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
// P's row r to TMEM, lane = row: hi in 32 columns from `taddr` (two k each), lo in the next 32.  Returns
// the power of two that scales back, biased.  sum (not NULL) grows by the row's values.
template <bool Turned>
__device__ __forceinline__ unsigned split_p(const unsigned char *base, int r, uint32_t taddr, float *sum) {
  float v[64];
  read_row<kBM, Turned>(base, r, v);
  if (Turned && sum)
    *sum += row_sum(v);
  const int e = row_power(v);
  const float2 scale = make_float2(pow2(e), pow2(e));
#pragma unroll
  for (int c = 0; c < 32; c += 16) {
    uint32_t h[16], l[16];
#pragma unroll
    for (int p = 0; p < 16; ++p)
      split2(make_float2(v[2 * (c + p)], v[2 * (c + p) + 1]), scale, h[p], l[p]);
    tmem_st16(taddr + c, h);
    tmem_st16(taddr + 32 + c, l);
  }
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
  tc_fence_before();
  return unsigned(127 - e);
}
// Q's row r in place.  Turned: all of its threads have read before any writes (named barrier `id` of
// ROWS threads).
template <int ROWS, bool Turned> __device__ __forceinline__ unsigned split_q(unsigned char *base, int r, int id) {
  float v[64];
  read_row<ROWS, Turned>(base, r, v);
  const int e = row_power(v);
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
// True in one thread of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
// D (TMEM) = A (TMEM) B (shared memory) + 2^-Down D, D's old value where Add.
template <bool Add, int Down = 0>
__device__ __forceinline__ void umma_f16_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
  if constexpr (Down == 0)
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "n"(int(Add)));
  else
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p, %5;\n\t}" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "n"(int(Add)), "n"(Down));
}

// sum_k P(i, k) Q(j, k) for k in [k0, k1) by a whole warp, one product at a time, 8 per lane under way;
// ends early at NaN.
__device__ __forceinline__ float plain_sum(const float *p, long long pk, const float *q, long long qk, long long k0,
                                           long long k1) {
  float s = 0.f;
#pragma unroll 1
  for (; k0 < k1; k0 += 256) {
    float a[8], b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const long long k = k0 + 32 * i + (threadIdx.x & 31), in = min(k, k1 - 1);
      a[i] = p[in * pk];
      b[i] = k < k1 ? q[in * qk] : 0.f;
      a[i] = k < k1 ? a[i] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      s = fmaf(a[i], b[i], s);
    if (__any_sync(0xffffffffu, s != s))
      break;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1)
    s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

template <int BN, bool PT, bool QT, bool Act>
__global__ void __launch_bounds__(kThreads, 1) gemm32_kernel(const __grid_constant__ Gemm32 g) {
  constexpr int kPBytes = kBM * kBK * 2, kQBytes = BN * kBK * 2, kStageBytes = stage_bytes<BN>();
  constexpr int kStages = stages<BN>(), kSlots = slots<BN>(), kSlotBytes = slot_bytes<BN>(), kBoxes = BN / 64,
                kBuffers = buffers<BN>(), kTmemCols = 512;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char *staging = smem + kStages * kStageBytes; // the drain warps' boxes, then their bias
  float *biases = reinterpret_cast<float *>(staging + 8 * kBoxes * kBoxBytes);
  // [kSlots][4 BN + kBM]: 2^-e of Q's rows (floats), then 127 - e of P's (bytes)
  unsigned char *scales = reinterpret_cast<unsigned char *>(biases + 8 * (BN / 2));
  uint64_t *bars = reinterpret_cast<uint64_t *>(scales + kSlots * kSlotBytes);
  // full[S] | tfull[B] | tfree[B] | scaled[kSlots] | residual[8 x boxes]
  constexpr int kBars = kStages + 2 * kBuffers + kSlots + 8 * kBoxes;
  static_assert(kBars * 8 + sizeof(Shared) <= 512 && kSlots <= 8, "barriers and state");
  Shared &sh = *reinterpret_cast<Shared *>(bars + kBars);
  volatile int &abort_flag = sh.abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned full0 = smem_u32(bars), tfull0 = full0 + 8 * kStages, tfree0 = tfull0 + 8 * kBuffers, scaled0 = tfree0 + 8 * kBuffers,
                 residual0 = scaled0 + 8 * kSlots;
  constexpr bool kInTurn = BN == 64;             // two groups of split warps take the slabs in turn
  constexpr int kSplitWarps = kInTurn ? 4 : 8; // of each slab
  if (threadIdx.x == 0) {
    abort_flag = 0;
    sh.progress = 0;
    for (int s = 0; s < kStages; ++s)
      mbar_init(full0 + 8 * s, 1);
    for (int b = 0; b < kBuffers; ++b) {
      mbar_init(tfull0 + 8 * b, 1);
      mbar_init(tfree0 + 8 * b, kDrainThreads);
    }
    for (int x = 0; x < kSlots; ++x) {
      mbar_init(scaled0 + 8 * x, kSplitWarps);
      sh.arrived[x] = 0;
    }
    for (int x = 0; x < 8 * kBoxes; ++x)
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

  // P's split slab n: 64 columns behind the accumulators, a place for each stage.
  auto p_columns = [&](int n) { return tmem + uint32_t(kBuffers * BN + n % kStages * 64); };
  // The MMAs of slab n (one warp, one of its threads: what the warp computes together is uniform, which
  // the instructions' operands have to be).
  auto multiply = [&](int n) {
    const int b = n % kBuffers;
    if (!__all_sync(0xffffffffu, n < kBuffers || wait_for(tfree0 + 8 * b, unsigned(n / kBuffers - 1) & 1, sh)))
      return;
    tc_fence_after();
    // Few instructions per MMA: while one thread issues, its warp's share of the next slab waits.  A
    // 16-wide step is 32 bytes (2 descriptor units) of Q, 8 columns of P.
    const uint64_t qh = smem_desc(smem_u32(smem + n % kStages * kStageBytes) + 2 * kPBytes), ql = qh + (kQBytes >> 4);
    const uint32_t d = tmem + uint32_t(b * BN), ph = p_columns(n), pl = ph + 32, idesc = g.idesc;
    if (!elect_one())
      return;
    umma_f16_tmem<false>(d, pl, qh, idesc); // the small terms first
    umma_f16_tmem<true>(d, ph, ql, idesc);
#pragma unroll
    for (int m = 1; m < kBK / 16; ++m) {
      umma_f16_tmem<true>(d, pl + 8 * m, qh + 2 * m, idesc);
      umma_f16_tmem<true>(d, ph + 8 * m, ql + 2 * m, idesc);
    }
    umma_f16_tmem<true, kLoBits>(d, ph, qh, idesc); // scales them back
#pragma unroll
    for (int m = 1; m < kBK / 16; ++m)
      umma_f16_tmem<true>(d, ph + 8 * m, qh + 2 * m, idesc);
    umma_commit(tfull0 + 8 * b);
  };
  // The loads of slab n at w (one thread; the MMAs of slab n - kStages are done).
  auto fetch = [&](int n, const Walk &w) {
    long long i, j;
    g.tiles.at(w.tile, i, j);
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

  // Registers: 128 each at launch; the 256 threads that split give some to the 256 that drain (2 x 128
  // in all).  84613 x 64 -> 1280 and its gradients with 96: 186 and 292 us, 112: 184 and 275, 128: 191 and 277.
  constexpr int kSplitRegs = 112;
  if (warp < 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kSplitRegs));
    const int group = warp >> 2, r = threadIdx.x & 127;
    const bool has_p = kInTurn || group == 0, has_q = kInTurn ? r < BN : group == 1;
    bool ok = true; // the same in the whole warp
    float sum = 0.f;
    int n = 0;
    for (Walk w(g); w.live(g); ++n) {
      if (!kInTurn || (n & 1) == group) {
        ok = __all_sync(0xffffffffu, ok && wait_for(full0 + 8 * (n % kStages), unsigned(n / kStages) & 1, sh));
        if (!ok) { // Q's other warps may wait at this slab's barrier
          if (QT && has_q)
            asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(BN) : "memory");
          sum = __uint_as_float(0x7fc00000u);
        } else {
          unsigned char *stage = smem + n % kStages * kStageBytes, *scale = scales + n % kSlots * kSlotBytes;
          if (has_p)
            scale[4 * BN + r] = static_cast<unsigned char>(
                split_p<PT>(stage, r, p_columns(n) + (uint32_t(32 * (warp & 3)) << 16), PT && g.sums ? &sum : nullptr));
          if (has_q)
            reinterpret_cast<unsigned *>(scale)[r] = split_q<BN, QT>(stage + 2 * kPBytes, r, 1 + group) << 23;
          // Each lane's stores, then the warp's, are visible before the warp counts as arrived; the
          // last to arrive sees all of them.
          fence_proxy_async_smem();
          __threadfence_block();
          __syncwarp();
          int before = 0;
          if (lane == 0) {
            mbar_arrive(scaled0 + 8 * (n % kSlots)); // this warp's scales, for the drain
            before = atomicAdd(&sh.arrived[n % kSlots], 1);
            if (before == kSplitWarps - 1)
              sh.arrived[n % kSlots] = 0;
            __threadfence_block();
          }
          if (__shfl_sync(0xffffffffu, before, 0) == kSplitWarps - 1) {
            fence_proxy_async_smem();
            multiply(n);
          }
        }
      }
      const unsigned tile = w.tile;
      const int part = w.part;
      if (w.next(g) && PT && g.sums && has_p) { // the unit is done: the tiles of the first column have the sums
        long long i, j;
        g.tiles.at(tile, i, j);
        if (j == 0 && i * kBM + r < g.I) {
          g.sums[(2ll * part + group) * g.I + i * kBM + r] = sum;
          if (!kInTurn)
            g.sums[(2ll * part + 1) * g.I + i * kBM + r] = 0.f;
        }
        sum = 0.f;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(256 - kSplitRegs));
    constexpr int kCols = BN / 2;
    Epilogue ep = g.e;
    if (!Act)
      ep.activation = None;
    const int quarter = warp & 3, half = (warp - 8) >> 2;
    const int me = warp - 8;
    Box boxes[kBoxes];
    unsigned phase[kBoxes] = {};
#pragma unroll
    for (int x = 0; x < kBoxes; ++x)
      boxes[x] = {staging + (kBoxes * me + x) * kBoxBytes, residual0 + 8 * (kBoxes * me + x)};
    float *bias = biases + me * kCols;
    // A tile's residual is on its way while the tile accumulates (a kept z needs the boxes first).
    const bool early = !QT && g.boxes.on && !g.partial && g.e.residual && !g.e.z;
    Walk ahead(g); // of the loads
    for (int x = 0; x < kStages && ahead.live(g); ++x) {
      if (me == x && lane == 0)
        fetch(x, ahead);
      ahead.next(g);
    }
    // A unit's tile and its bias are ready before the unit: the drain's latencies are what a unit takes.
    int next_i = 0, next_j = 0; // its rows' and columns' tile
    float next_bias[kCols / 32] = {};
    auto prepare = [&](unsigned tile) {
      long long i, j;
      g.tiles.at(tile, i, j);
      next_i = int(i), next_j = int(j);
      if (!QT && g.e.bias && !g.partial)
#pragma unroll
        for (int h = 0; h < kCols / 32; ++h)
          next_bias[h] = static_cast<const float *>(g.e.bias)[min(j * BN + half * kCols + 32 * h + lane, g.J - 1)];
    };
    float acc[kCols];
    bool ok = true;
    int n = 0;
    Walk w(g);
    if (w.live(g))
      prepare(w.tile);
    while (w.live(g)) {
      const int s = w.part;
      const long long i = next_i, j = next_j;
      const long long row0 = i * kBM + 32 * quarter, row = row0 + lane, cols0 = j * BN + half * kCols;
      const bool any = row0 < g.I && cols0 < g.J;
      // The sums start with the bias (the gradients' products have none).
      if (QT) {
#pragma unroll
        for (int c = 0; c < kCols; ++c)
          acc[c] = 0.f;
      } else {
#pragma unroll
        for (int h = 0; h < kCols / 32; ++h)
          bias[32 * h + lane] = next_bias[h];
        __syncwarp();
#pragma unroll
        for (int c = 0; c < kCols; c += 4) {
          const float4 f = *reinterpret_cast<const float4 *>(bias + c);
          acc[c] = f.x, acc[c + 1] = f.y, acc[c + 2] = f.z, acc[c + 3] = f.w;
        }
        __syncwarp();
      }
      {
        Walk after = w;
        after.skip(g);
        if (after.live(g))
          prepare(after.tile);
      }
      if (early && any && lane == 0) {
        bulk_wait_read();
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c)
          if (cols0 + 32 * c < g.J)
            fetch_residual(g.boxes, boxes[c], row0, cols0 + 32 * c);
      }
      for (bool same = true; same; same = !w.next(g), ++n) {
        const int b = n % kBuffers;
        ok = ok && wait_for(tfull0 + 8 * b, unsigned(n / kBuffers) & 1, sh) &&
             wait_for(scaled0 + 8 * (n % kSlots), unsigned(n / kSlots) & 1, sh);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok)
          continue;
        if (me == (n & 7) && lane == 0 && ahead.live(g)) // in turn: no warp falls behind by all of them
          fetch(n + kStages, ahead);
        ahead.next(g);
        tc_fence_after();
        const unsigned char *scale = scales + n % kSlots * kSlotBytes;
        const float *fq = reinterpret_cast<const float *>(scale) + half * kCols;
        // 2^-e of P's row.
        const float fp = __uint_as_float(uint32_t(scale[4 * BN + 32 * quarter + lane]) << 23);
        const float2 fp2 = make_float2(fp, fp);
#pragma unroll
        for (int h = 0; h < kCols; h += 32) {
          uint32_t r[32];
          tmem_ld32_async(tmem + (uint32_t(quarter * 32) << 16) + uint32_t(b * BN + half * kCols + h), r);
          tmem_wait_ld();
          tmem_anchor(r);
          if (h + 32 == kCols) {
            tc_fence_before();
            mbar_arrive(tfree0 + 8 * b);
          }
#pragma unroll
          for (int c = 0; c < 32; c += 4) { // the two scalings, and the float sum
            const float4 f = *reinterpret_cast<const float4 *>(fq + h + c);
            const float2 v = make_float2(__uint_as_float(r[c]), __uint_as_float(r[c + 1]));
            const float2 u = make_float2(__uint_as_float(r[c + 2]), __uint_as_float(r[c + 3]));
            const int x = h + c;
            const float2 a = __ffma2_rn(__fmul2_rn(v, make_float2(f.x, f.y)), fp2, make_float2(acc[x], acc[x + 1]));
            const float2 d = __ffma2_rn(__fmul2_rn(u, make_float2(f.z, f.w)), fp2, make_float2(acc[x + 2], acc[x + 3]));
            acc[x] = a.x, acc[x + 1] = a.y, acc[x + 2] = d.x, acc[x + 3] = d.y;
          }
        }
      }
      float *partial = g.partial ? g.partial + s * g.I * g.J : nullptr;
#pragma unroll
      for (int c0 = 0; c0 < kCols; c0 += 32) {
        const long long col0 = cols0 + c0;
        if (row0 >= g.I || col0 >= g.J)
          continue;
        if (!ok) { // a wait that ran out shows as NaN
#pragma unroll
          for (int c = 0; c < 32; ++c)
            acc[c0 + c] = __uint_as_float(0x7fc00000u);
        }
        // 0 x: NaN where x is not finite.
        float2 probe[4] = {};
#pragma unroll
        for (int c = 0; c < 32; c += 2)
          probe[c / 2 & 3] = __ffma2_rn(make_float2(acc[c0 + c], acc[c0 + c + 1]), make_float2(0.f, 0.f), probe[c / 2 & 3]);
        const float2 p01 = __fadd2_rn(__fadd2_rn(probe[0], probe[1]), __fadd2_rn(probe[2], probe[3]));
        uint32_t odd = 0; // this lane's columns that are not finite
        if (__any_sync(0xffffffffu, p01.x + p01.y != 0.f) && ok) {
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (!(fabsf(acc[c0 + c]) < INFINITY) && row < g.I && col0 + c < g.J)
              odd |= 1u << c;
        }
        while (const unsigned lanes = __ballot_sync(0xffffffffu, odd != 0)) {
          const int at = __ffs(lanes) - 1, c = __ffs(__shfl_sync(0xffffffffu, odd, at)) - 1;
          float x = plain_sum(g.p + (row0 + at) * (PT ? 1 : g.ldp), PT ? g.ldp : 1,
                                    g.q + (col0 + c) * (QT ? 1 : g.ldq), QT ? g.ldq : 1,
                                    (long long)s * g.slabs / g.parts * kBK,
                                    min(g.K, (s + 1ll) * g.slabs / g.parts * kBK));
          if (!QT && g.e.bias && !g.partial)
            x += static_cast<const float *>(g.e.bias)[col0 + c];
          if (lane == 0)
            sh.progress = sh.progress + 1;
          if (lane == at) {
            odd &= odd - 1;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i == c)
                acc[c0 + i] = x;
          }
        }
        if (g.boxes.on)
          finish_box<float, QT>(
              ep, g.boxes, row0, col0, g.partial ? s : -1, boxes[c0 / 32], phase[c0 / 32], early || (c0 && !g.e.z), nullptr,
              [&](int, float (&v)[32]) {
#pragma unroll
                for (int c = 0; c < 32; ++c)
                  v[c] = acc[c0 + c];
              });
        else
          finish_block<float>(ep, partial, g.I, g.J, row0, col0, acc + c0, false, boxes[0].at);
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

template <int BN, bool PT, bool QT, bool Act> void launch_gemm32(const Gemm32 &g, cudaStream_t stream) {
  static thread_local int configured = -1;
  int device = 0;
  lapis::check(cudaGetDevice(&device));
  if (configured != device) {
    lapis::check(cudaFuncSetAttribute(gemm32_kernel<BN, PT, QT, Act>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      smem_bytes<BN>()));
    configured = device;
  }
  lapis::launch(gemm32_kernel<BN, PT, QT, Act>, dim3(std::min(g.units, unsigned(sm_count()))), kThreads, smem_bytes<BN>(),
                stream, g);
  lapis::check(cudaGetLastError());
}
} // namespace

// 128-wide tiles, 64-wide ones for at most 64 columns; few tiles are cut along k until they fill the
// device, parts of at least two slabs.
Plan plan32(long long I, long long J, long long K) {
  Plan p{J <= 64 ? 64 : 128, 1};
  const long long tiles = (I + kBM - 1) / kBM * ((J + p.bn - 1) / p.bn), slabs = (K + kBK - 1) / kBK;
  p.parts = int(std::min<long long>({std::max(1ll, sm_count() / tiles), std::max(1ll, slabs / 2), 148}));
  return p;
}

void product32(const Product &p, void *workspace, cudaStream_t stream, float *sums) {
  const Plan plan = plan32(p.I, p.J, p.K);
  Gemm32 g{};
  g.I = p.I, g.J = p.J, g.K = p.K;
  g.p = static_cast<const float *>(p.p.p), g.ldp = p.p.ld;
  g.q = static_cast<const float *>(p.q.p), g.ldq = p.q.ld;
  g.mp = p.p.turned ? tile_map(F32, p.p.p, p.K, p.I, p.p.ld, kBK) : tile_map(F32, p.p.p, p.I, p.K, p.p.ld, kBM);
  g.mq = p.q.turned ? tile_map(F32, p.q.p, p.K, p.J, p.q.ld, kBK) : tile_map(F32, p.q.p, p.J, p.K, p.q.ld, plan.bn);
  g.slabs = int((p.K + kBK - 1) / kBK);
  g.parts = plan.parts;
  check_tiles(p.I, p.J, kBM, plan.bn, plan.parts);
  g.tiles = Tiles(p.I, p.J, kBM, plan.bn);
  g.units = g.tiles.count * unsigned(plan.parts);
  g.idesc = idesc_f16(kBM, plan.bn);
  g.partial = plan.parts > 1 ? static_cast<float *>(workspace) : nullptr;
  g.sums = sums;
  g.e = p.e;
  g.boxes = boxes_of(p, g.partial, plan.parts);
  auto width = [&](auto bn) {
    constexpr int BN = decltype(bn)::value;
    // Without the activations' code the drain is the faster one (84613 x 64 -> 1280: 155 us, 167 with it).
    if (!p.p.turned && !p.q.turned && p.e.activation != None && !g.partial)
      launch_gemm32<BN, false, false, true>(g, stream);
    else if (!p.p.turned && !p.q.turned)
      launch_gemm32<BN, false, false, false>(g, stream);
    else if (!p.p.turned)
      launch_gemm32<BN, false, true, false>(g, stream);
    else
      launch_gemm32<BN, true, true, false>(g, stream);
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
