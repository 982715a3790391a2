// The dense layer's matrix products of 16-bit types on the tensor cores (tcgen05, kind::f16).
//
//   out(i, j) = sum_k P(i, k) Q(j, k), accumulated in float in TMEM
//
// An operand may be k-major ([I][K]) or turned ([K][I], the gradients' products): TMA brings 64-wide
// slabs of k into shared memory in the layout that it has in global memory (SWIZZLE_128B), and the
// matrix descriptor says which of the two it is.
//
// Persistent: one CTA per SM walks 128 x BN tiles.  10 warps: TMA producer, MMA issuer (one elected
// thread), and eight that move a finished tile out of TMEM, through the epilogue and to global
// memory while the next tile accumulates in TMEM's other half.  With too few tiles for the
// device, K is cut into parts whose float products a second launch adds in order.
//
// bf16, back to back: 8192 x 4096 -> 16384 in 813 us (1.35 PFLOP/s, 0.98 of the measured sustained rate;
// with bias, GELU and z kept 931), 4096 x 2048 -> 8192 in 123 us (1.1 PFLOP/s).  84613 x 64 -> 1280 in 50 us
// (4.5 TB/s written and read): one slab per tile, so the epilogue bounds it.
#include "dense_gemm.cuh"

namespace mace {
namespace op {
namespace {
using namespace tc;
constexpr int kBM = 128, kBK = 64;
constexpr int kThreads = 320, kEpilogueThreads = 256;
constexpr int kStageRing = 192 * 1024; // bytes of the operand ring
constexpr int kBiasBytes = 8 * 128 * 2; // each epilogue warp's columns
constexpr int kSmem = kStageRing + 8 * kBoxBytes + kBiasBytes + 256;
static_assert(kSmem <= 232448, "shared memory budget");

struct Gemm16 {
  CUtensorMap p, q;
  long long I, J;
  Tiles tiles;
  unsigned units; // tiles x parts
  int slabs, parts, p_rows, q_rows; // rows of a k-major operand's boxes
  uint32_t idesc;
  float *partial;
  Epilogue e;
  Boxes boxes;
};

// Shared-memory descriptor of a turned operand (MN-major, SWIZZLE_128B): 64-wide blocks 8 KiB apart,
// groups of 8 k 1024 bytes apart.
__device__ __forceinline__ uint64_t turned_desc(unsigned addr) {
  return uint64_t((addr >> 4) & 0x3fff) | uint64_t(8192 >> 4) << 16 | uint64_t(1024 >> 4) << 32 | uint64_t(1) << 46 |
         uint64_t(2) << 61;
}

template <class T, int BN, bool PT, bool QT>
__global__ void __launch_bounds__(kThreads, 1) gemm16_kernel(const __grid_constant__ Gemm16 g) {
  constexpr int kPBytes = kBM * kBK * 2, kQBytes = BN * kBK * 2, kStageBytes = kPBytes + kQBytes;
  constexpr int kStages = kStageRing / kStageBytes;
  constexpr int kTmemCols = 2 * BN;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char *staging = smem + kStageRing; // a box per epilogue warp, then its bias
  uint64_t *bars = reinterpret_cast<uint64_t *>(staging + 8 * kBoxBytes + kBiasBytes);
  // full[S] | empty[S] | tfull[2] | tfree[2] | done | residual[8]
  constexpr int kBars = 2 * kStages + 5 + 8;
  static_assert(kBars * 8 + 12 <= 256, "barriers and state");
  uint32_t &tmem_base = *reinterpret_cast<uint32_t *>(bars + kBars);
  volatile int &abort_flag = *reinterpret_cast<volatile int *>(&tmem_base + 1);
  int &mma_done_issued = *reinterpret_cast<int *>(&tmem_base + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned full0 = smem_u32(bars), empty0 = full0 + 8 * kStages, tfull0 = empty0 + 8 * kStages,
                 tfree0 = tfull0 + 16, done = tfree0 + 16, residual0 = done + 8;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    mma_done_issued = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull0 + 8 * b, 1);
      mbar_init(tfree0 + 8 * b, kEpilogueThreads);
    }
    mbar_init(done, 1);
    for (int x = 0; x < 8; ++x)
      mbar_init(residual0 + 8 * x, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  const Tiles &tiles = g.tiles;
  const unsigned units = g.units;
  // Unit u is part s = u / tiles of tile u % tiles: slabs [first_slab(s), first_slab(s + 1)).
  auto first_slab = [&](unsigned s) { return g.parts > 1 ? int((long long)s * g.slabs / g.parts) : s ? g.slabs : 0; };
  auto part_of = [&](unsigned u) { return g.parts > 1 ? u / tiles.count : 0u; };

  if (warp == 0) {
    if (lane == 0) {
      unsigned n = 0;
      bool ok = true;
      const unsigned bytes = (PT ? kPBytes : g.p_rows * 128) + (QT ? kQBytes : g.q_rows * 128);
      for (unsigned u = blockIdx.x; u < units && ok; u += gridDim.x) {
        const unsigned s = part_of(u);
        long long i, j;
        tiles.at(u - s * tiles.count, i, j);
        const int i0 = int(i * kBM), j0 = int(j * BN);
        for (int k = first_slab(s), end = first_slab(s + 1); k < end; ++k, ++n) {
          const int st = int(n % kStages);
          if (n >= kStages && !(ok = mbar_wait(empty0 + 8 * st, unsigned(n / kStages - 1) & 1, &abort_flag)))
            break;
          const unsigned base = smem_u32(smem + st * kStageBytes), full = full0 + 8 * st;
          mbar_expect_tx(full, bytes);
          if (PT) {
#pragma unroll
            for (int h = 0; h < kBM / 64; ++h)
              tma_load_2d(base + 8192 * h, &g.p, i0 + 64 * h, k * kBK, full);
          } else {
            tma_load_2d(base, &g.p, k * kBK, i0, full);
          }
          if (QT) {
#pragma unroll
            for (int h = 0; h < BN / 64; ++h)
              tma_load_2d(base + kPBytes + 8192 * h, &g.q, j0 + 64 * h, k * kBK, full);
          } else {
            tma_load_2d(base + kPBytes, &g.q, k * kBK, j0, full);
          }
        }
      }
      if (!ok) // copies in flight end (bounded wait) before the CTA does
        for (unsigned m = n > kStages ? n - kStages : 0; m < n; ++m) {
          long long start = clock64();
          while (!mbar_try(full0 + 8 * int(m % kStages), unsigned(m / kStages) & 1) && clock64() - start < kWaitCycles) {
          }
        }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      unsigned n = 0;
      int tile = 0;
      bool ok = true;
      for (unsigned u = blockIdx.x; u < units && ok; u += gridDim.x, ++tile) {
        const int b = tile & 1;
        const unsigned s = part_of(u);
        const uint32_t d = tmem + uint32_t(b * BN);
        if (tile >= 2 && !(ok = mbar_wait(tfree0 + 8 * b, unsigned(tile / 2 - 1) & 1, &abort_flag)))
          break;
        tc_fence_after();
        const int first = first_slab(s), end = first_slab(s + 1);
        for (int k = first; k < end; ++k, ++n) {
          const int st = int(n % kStages);
          if (!(ok = mbar_wait(full0 + 8 * st, unsigned(n / kStages) & 1, &abort_flag)))
            break;
          tc_fence_after();
          const unsigned base = smem_u32(smem + st * kStageBytes);
          // 16-wide k steps: 32 bytes into k-major rows, two groups of 8 rows into turned ones.
#pragma unroll
          for (int m = 0; m < kBK / 16; ++m)
            umma_f16_desc(d, PT ? turned_desc(base + 2048 * m) : smem_desc(base + 32 * m),
                          QT ? turned_desc(base + kPBytes + 2048 * m) : smem_desc(base + kPBytes + 32 * m), g.idesc,
                          k > first || m ? 1u : 0u);
          umma_commit(empty0 + 8 * st);
        }
        if (ok)
          umma_commit(tfull0 + 8 * b);
      }
      umma_commit(done);
      mma_done_issued = 1;
    }
  } else {
    // Two warps per TMEM lane quadrant, each with half of the columns.
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const int me = warp - 2;
    const Box w{staging + me * kBoxBytes, residual0 + 8 * me};
    T *bias = reinterpret_cast<T *>(staging + 8 * kBoxBytes) + me * 128;
    unsigned phase = 0;
    bool ok = true;
    int tile = 0;
    for (unsigned u = blockIdx.x; u < units; u += gridDim.x, ++tile) {
      const int b = tile & 1;
      const unsigned s = part_of(u);
      long long i, j;
      tiles.at(u - s * tiles.count, i, j);
      if (!g.partial)
        fetch_bias<T>(g.e, g.J, j * BN + (BN >= 128 ? half * (BN / 2) : 0), BN >= 128 ? BN / 2 : 64, bias);
      const long long row0 = i * kBM + 32 * quarter;
      Sectors<T> residual; // of the next 32 columns, on its way before they are
      if (g.boxes.sectors && BN >= 128 && g.e.residual && !g.partial)
        residual.load(g.e, g.I, g.J, row0 + lane, j * BN + half * (BN / 2));
      ok = ok && mbar_wait(tfull0 + 8 * b, unsigned(tile / 2) & 1, &abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      const uint32_t d = tmem + (uint32_t(quarter * 32) << 16) + uint32_t(b * BN);
      auto get = [&](int c, float (&v)[32]) { // the tile's columns c ..
        uint32_t r[32];
        tmem_ld32_async(d + uint32_t(c), r);
        tmem_wait_ld();
        tmem_anchor(r);
#pragma unroll
        for (int k = 0; k < 32; ++k) // a wait that ran out shows as NaN
          v[k] = ok ? __uint_as_float(r[k]) : __uint_as_float(0x7fc00000u);
      };
      const int first = half * (BN / 2), end = first + BN / 2;
      if (row0 < g.I) {
        if (g.boxes.sectors && BN >= 128) {
          float *partial = g.partial ? g.partial + s * g.I * g.J : nullptr;
#pragma unroll 1
          for (int c = first; c < end && j * BN + c < g.J; c += 32) {
            const Sectors<T> now = residual;
            if (g.e.residual && !partial && c + 32 < end)
              residual.load(g.e, g.I, g.J, row0 + lane, j * BN + c + 32);
            float v[32];
            get(c, v);
            finish_row<T>(g.e, partial, g.I, g.J, row0 + lane, j * BN + c, v, bias + c - first, now);
          }
        } else if (g.boxes.on && g.partial) {
#pragma unroll 1
          for (int c = first; c < end && j * BN + c < g.J; c += 32)
            finish_box<float, true>(g.e, g.boxes, row0, j * BN + c, int(s), w, phase, false,
                              nullptr, [&](int k, float (&v)[32]) { get(c + k, v); });
        } else if (g.boxes.on) {
          // 64 columns to a box: where the tile has no more, the first of a quarter's two warps has it.
          const int step = BN >= 128 ? 1 : 2;
#pragma unroll
          for (int x = 0; x < (BN + 127) / 128; ++x) {
            const int c = first * step + 64 * x;
            if (c < end && j * BN + c < g.J)
              finish_box<T, QT>(g.e, g.boxes, row0, j * BN + c, -1, w, phase, false,
                            g.e.bias ? bias + 64 * x : nullptr, [&](int k, float (&v)[32]) { get(c + k, v); });
          }
        } else {
          float *partial = g.partial ? g.partial + s * g.I * g.J : nullptr;
#pragma unroll 1
          for (int c = first; c < end && j * BN + c < g.J; c += 32) {
            float v[32];
            get(c, v);
            finish_block<T>(g.e, partial, g.I, g.J, row0, j * BN + c, v, g.e.bias && !partial, w.at);
          }
        }
      }
      tc_fence_before();
      mbar_arrive(tfree0 + 8 * b);
    }
    if (lane == 0)
      bulk_wait();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    if (abort_flag && mma_done_issued) { // bounded wait for the MMAs in flight before TMEM goes
      long long start = clock64();
      while (!mbar_try(done, 0) && clock64() - start < kWaitCycles) {
      }
    }
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

template <class T>
__global__ void __launch_bounds__(256) finish_parts_kernel(const __grid_constant__ Epilogue e, const float *partial,
                                                           int parts, long long I, long long J) {
  const long long plane = I * J;
  if (J % 4 == 0) {
    for (long long x = 4 * ((long long)blockIdx.x * 256 + threadIdx.x); x < plane; x += 1024ll * gridDim.x) {
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int p = 0; p < parts; ++p) {
        const float4 v = *reinterpret_cast<const float4 *>(partial + p * plane + x);
        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
      }
      const long long row = x / J, col = x - row * J;
      finish<T>(e, row, col, s.x), finish<T>(e, row, col + 1, s.y);
      finish<T>(e, row, col + 2, s.z), finish<T>(e, row, col + 3, s.w);
    }
    return;
  }
  for (long long x = (long long)blockIdx.x * 256 + threadIdx.x; x < plane; x += 256ll * gridDim.x) {
    float s = 0.f;
    for (int p = 0; p < parts; ++p)
      s += partial[p * plane + x];
    finish<T>(e, x / J, x % J, s);
  }
}

} // namespace

// The cheapest of the tile widths, in units of a 128 x 256 tile's slab (0.43 us at K = 4096).  A narrower
// tile saves little: a 128 x 128 one takes 0.85 of that (P's shared-memory reads bound both); but with
// one row of tiles Q comes from HBM, and a slab costs what its bytes do (1.7 for 256 columns).  Few tiles
// are cut along K until they fill the device, parts of at least four slabs; a second launch then
// reads the parts.
Plan plan16(long long I, long long J, long long K) {
  const int sms = sm_count();
  const long long slabs = (K + kBK - 1) / kBK;
  Plan best{0, 1};
  double cost = 0;
  for (int bn : {256, 128, 64}) {
    const long long tiles = (I + kBM - 1) / kBM * ((J + bn - 1) / bn);
    const double slab = std::max(bn == 256 ? 1. : bn == 128 ? .85 : .75, I <= kBM ? 1.7 * bn / 256 : 0.);
    for (int cut : {0, 1}) {
      const int parts = cut ? int(std::min<long long>({std::max(1ll, sms / tiles), std::max(1ll, slabs / 4), 64})) : 1;
      const long long waves = (tiles * parts + sms - 1) / sms;
      const double c = double(waves) * double((slabs + parts - 1) / parts) * slab +
                       (parts > 1 ? 8. + double(parts) * double(I) * double(J) * 3e-6 : 0.);
      if (!best.bn || c < cost)
        best = {bn, parts}, cost = c;
    }
  }
  return best;
}
namespace {
using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                              const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encoder() {
  static EncodeFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeFn>(p);
  });
  if (!fn)
    throw lapis::Error("cuTensorMapEncodeTiled is unavailable");
  return fn;
}

template <class T, int BN, bool PT, bool QT> void launch_gemm16(const Gemm16 &g, cudaStream_t stream) {
  static thread_local int configured = -1;
  int device = 0;
  lapis::check(cudaGetDevice(&device));
  if (configured != device) {
    lapis::check(cudaFuncSetAttribute(gemm16_kernel<T, BN, PT, QT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    configured = device;
  }
  lapis::launch(gemm16_kernel<T, BN, PT, QT>, dim3(std::min(g.units, unsigned(sm_count()))), kThreads, kSmem, stream, g);
  lapis::check(cudaGetLastError());
}
} // namespace

CUtensorMap tile_map(int type, const void *base, long long rows, long long cols, long long ld, int box_rows,
                     int planes) {
  const int b = bytes_of(type);
  if (rows <= 1)
    ld = round_up(cols, 16 / b);
  CUtensorMap map;
  cuuint64_t dims[3] = {cuuint64_t(cols), cuuint64_t(rows), cuuint64_t(planes)};
  cuuint64_t strides[2] = {cuuint64_t(ld) * unsigned(b), cuuint64_t(ld) * cuuint64_t(rows) * unsigned(b)};
  cuuint32_t box[3] = {cuuint32_t(128 / b), cuuint32_t(box_rows), 1}, elem[3] = {1, 1, 1};
  CUresult r = encoder()(&map,
                         type == F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                         : type == BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                        : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                         planes ? 3 : 2, const_cast<void *>(base), dims, strides, box, elem,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    throw lapis::Error("cuTensorMapEncodeTiled failed (" + std::to_string(int(r)) + ")");
  return map;
}

Boxes boxes_of(const Product &p, float *partial, int parts) {
  Boxes b{};
  const Epilogue &e = p.e;
  auto sectors = [&](const void *a, long long ld) {
    return !a || (reinterpret_cast<uintptr_t>(a) % 32 == 0 && (p.I <= 1 || ld * bytes_of(p.type) % 32 == 0));
  };
  b.sectors = partial ? p.J % 8 == 0 && reinterpret_cast<uintptr_t>(partial) % 32 == 0
                      : p.J * bytes_of(p.type) % 32 == 0 && sectors(e.out, e.ldo) && sectors(e.z, e.ldz) &&
                            sectors(e.residual, e.ldr);
  if (partial) {
    b.on = p.J % 4 == 0;
    if (b.on)
      b.y = tile_map(F32, partial, p.I, p.J, p.J, 32, parts);
    return b;
  }
  b.on = tma_ready(p.type, e.out, p.I, e.ldo) && (!e.z || tma_ready(p.type, e.z, p.I, e.ldz)) &&
         (!e.residual || tma_ready(p.type, e.residual, p.I, e.ldr));
  if (!b.on)
    return b;
  b.y = tile_map(p.type, e.out, p.I, p.J, e.ldo, 32, 1);
  if (e.z)
    b.z = tile_map(p.type, e.z, p.I, p.J, e.ldz, 32, 1);
  if (e.residual)
    b.residual = tile_map(p.type, e.residual, p.I, p.J, e.ldr, 32, 1);
  return b;
}

void product16(const Product &p, void *workspace, cudaStream_t stream) {
  const Plan plan = plan16(p.I, p.J, p.K);
  Gemm16 g{};
  g.I = p.I, g.J = p.J;
  g.slabs = int((p.K + kBK - 1) / kBK);
  g.parts = plan.parts;
  check_tiles(p.I, p.J, kBM, plan.bn, plan.parts);
  g.tiles = Tiles(p.I, p.J, kBM, plan.bn);
  g.units = g.tiles.count * unsigned(plan.parts);
  // Boxes of a short k-major operand end with its rows (in groups of 8): what lies behind them in
  // shared memory reaches no output that is written.
  g.p_rows = int(std::min<long long>(kBM, round_up(p.I, 8)));
  g.q_rows = int(std::min<long long>(plan.bn, round_up(p.J, 8)));
  g.p = p.p.turned ? tile_map(p.type, p.p.p, p.K, p.I, p.p.ld, kBK) : tile_map(p.type, p.p.p, p.I, p.K, p.p.ld, g.p_rows);
  g.q = p.q.turned ? tile_map(p.type, p.q.p, p.K, p.J, p.q.ld, kBK) : tile_map(p.type, p.q.p, p.J, p.K, p.q.ld, g.q_rows);
  const uint32_t format = p.type == BF16 ? 1 : 0;
  g.idesc = idesc_f16(kBM, plan.bn) | format << 7 | format << 10 | uint32_t(p.p.turned) << 15 | uint32_t(p.q.turned) << 16;
  g.partial = plan.parts > 1 ? static_cast<float *>(workspace) : nullptr;
  g.e = p.e;
  g.boxes = boxes_of(p, g.partial, plan.parts);
  auto run = [&](auto tag) {
    using T = decltype(tag);
    auto width = [&](auto bn) {
      constexpr int BN = decltype(bn)::value;
      if (!p.p.turned && !p.q.turned)
        launch_gemm16<T, BN, false, false>(g, stream);
      else if (!p.p.turned)
        launch_gemm16<T, BN, false, true>(g, stream);
      else
        launch_gemm16<T, BN, true, true>(g, stream);
    };
    if (plan.bn == 256)
      width(std::integral_constant<int, 256>{});
    else if (plan.bn == 128)
      width(std::integral_constant<int, 128>{});
    else
      width(std::integral_constant<int, 64>{});
  };
  if (p.type == BF16)
    run(__nv_bfloat16{});
  else
    run(__half{});
  if (plan.parts > 1)
    finish_parts(p.type, p.e, g.partial, plan.parts, p.I, p.J, stream);
}

void finish_parts(int type, const Epilogue &e, const float *partial, int parts, long long I, long long J,
                  cudaStream_t stream) {
  with_type(type, [&](auto tag) {
    long long blocks = (I * J + 1023) / 1024;
    lapis::launch(finish_parts_kernel<decltype(tag)>, dim3(unsigned(std::min<long long>(blocks, 8ll * sm_count()))), 256,
                  0, stream, e, partial, parts, I, J);
    lapis::check(cudaGetLastError());
  });
}
} // namespace op
} // namespace mace
