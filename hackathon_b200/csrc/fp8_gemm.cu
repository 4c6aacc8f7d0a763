// 8-bit projection: e4m3 operands, float32 scales for each 128 columns of an
// activation row and each 128 x 128 block of the weight.
//
//   y[m, n] = act( sum_g xs[m, g] ws[n / 128, g] * (sum_{k in g} x[m, k] w[n, k]) + bias[n] )
//
// The inner sum over a group's 128 products is four tcgen05.mma of kind f8f6f4
// into a fresh TMEM accumulator (float32); the epilogue warps read it, multiply
// by the two scales and add it to float32 registers while the next group's MMAs
// run into the other accumulator. The products of e4m3 values are exact in
// float32. One K step of the pipeline is one scale group: 128 bytes, one
// swizzled row.
//
// Two shapes of the same pipeline:
//  - rows kernel: M = 128 activation rows (a thread's TMEM lane is a row, so both
//    scales are one scalar a thread and group), N = BN output features;
//    persistent CTAs. Bound by the exchange of the accumulators: a group of BN =
//    256 keeps the tensor cores busy for 515 cycles of some 1,070 at 10000 x 4096 x
//    2048 (48%, starts and stores of the tiles included); its sums are read from TMEM
//    and scaled by eight warps, 128 scalar FMAs a thread.
//    18944 x 4096 x 4096 to bf16 takes 322 us (1.97 PFLOP/s), 10000 x 4096 x 2048 103
//    us (1.63), where a last round of whole tiles over the SMs would leave most of
//    them idle: tiles that would are taken in halves (104 us without when 101 with;
//    4096 x 256 x 1280 13.5 us for 14.8, 300 x 2048 x 8448 18.0 for 19.4).
//  - few-rows kernel, where there are not tiles for every SM: M = 128 output
//    features, N = BR rows (16, 32 or 64; a grid of them above 64); the groups are
//    shared out over a cluster of up to 8 CTAs, whose float32 sums meet through
//    distributed shared memory in rank order (the same result every time). Bound
//    by latency at the sizes it is for: 1 x 2048 x 8448 takes 7.3 us, 2.7 of them
//    its weight's bytes, the rest the first load, the joining and the launch.
#include <algorithm>
#include <cooperative_groups.h>
#include <type_traits>

#include "seqops.cuh"
#include "tc.cuh"

namespace b2e {
namespace {

namespace cg = cooperative_groups;

constexpr uint32_t kKB = kFp8Group;           // bytes of a K step
enum Fp8Error : int { kFp8TimeoutTma = 121, kFp8TimeoutMma = 122, kFp8TimeoutEpi = 123 };

// Instruction descriptor of kind f8f6f4: float32 accumulator, e4m3 x e4m3, both
// K-major, M = 128, N = n.
__host__ __device__ constexpr uint32_t idesc_f8(int n) {
  return (1u << 4) | (uint32_t(n >> 3) << 17) | (uint32_t(128 >> 4) << 24);
}

__device__ __forceinline__ void mma_f8(uint32_t tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
      "l"(a), "l"(b), "r"(idesc), "r"(acc));
}

struct Args {
  const float* xs;
  const float* ws;
  const float* bias;
  void* y;
  long long ldy;
  int m, n, groups, wgroups;  // wgroups: scale columns of ws
  int relu, y_type, vec;      // vec: rows of y may take 32-byte stores
  int tiles_m, tiles_n;
  int whole;  // rows kernel: tiles behind the first `whole` are taken in two halves
  int* err;
};

// ReLU that keeps a NaN.
__device__ __forceinline__ float2 activate(float2 v, int relu) {
  if (relu) {
    v.x = v.x < 0.f ? 0.f : v.x;
    v.y = v.y < 0.f ? 0.f : v.y;
  }
  return v;
}

// Sixteen results (two and two) to a row of y, all inside, 32-byte aligned.
template <int Y>
__device__ __forceinline__ void store16_y(void* y, long long at, const float2* v) {
  if constexpr (Y == kF32) {
    float* p = reinterpret_cast<float*>(y) + at;
#pragma unroll
    for (int i = 0; i < 8; i += 4)
      asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p + 2 * i), "f"(v[i].x), "f"(v[i].y), "f"(v[i + 1].x),
                   "f"(v[i + 1].y), "f"(v[i + 2].x), "f"(v[i + 2].y), "f"(v[i + 3].x), "f"(v[i + 3].y)
                   : "memory");
  } else {
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (Y == kBF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[i].x, v[i].y);
        u[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(v[i].x, v[i].y);
        u[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(reinterpret_cast<uint16_t*>(y) + at), "r"(u[0]),
                 "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
                 : "memory");
  }
}

// ------------------------------------------------------------- rows kernel

// Row scales come in blocks of kXB groups through shared memory, group-major: a
// row's scales are contiguous in memory, so a load for every row of a tile takes
// a line a lane, which per group cost more than the group's MMAs.
constexpr int kXB = 16, kXStride = 128 + 1;

template <int BN>
struct RowsCfg {
  static constexpr uint32_t TILE_X = 128 * kKB, TILE_W = BN * kKB, STAGE = TILE_X + TILE_W;
  static constexpr int STAGES = BN == 256 ? 4 : 3;
  static constexpr int CTAS = BN == 256 ? 1 : 2;  // resident on an SM
  // Eight epilogue warps behind a warpgroup of TMA, MMA and two idle warps. The
  // registers are split by warpgroup: 4 x 32 x LOW + 8 x 32 x HIGH are the launch's
  // 384 x 168 (80 where two CTAs share an SM).
  static constexpr int EPI = 8, THREADS = 128 + 32 * EPI, HN = BN / 2;
  static constexpr int LOW = BN == 256 ? 40 : 24, HIGH = BN == 256 ? 232 : 104;
  static_assert(4 * LOW + 8 * HIGH <= 12 * (BN == 256 ? 168 : 80), "register shares exceed the launch's");
  static constexpr uint32_t TMEM = 2 * BN;
  static constexpr uint32_t SCALES = kXB * kXStride * 4;  // row scales of kXB groups
  static constexpr size_t SMEM = size_t(STAGES) * STAGE + SCALES + 1024 + 256;
};

// Item `i` of the rows kernel: a tile, or half of one (its first or second 128 features).
struct RowsItem {
  int m0, n0;
  bool half;
};
template <int BN>
__device__ __forceinline__ RowsItem rows_item(const Args& e, int i) {
  const bool half = BN == 256 && i >= e.whole;
  const int t = half ? e.whole + (i - e.whole) / 2 : i;
  return {(t % e.tiles_m) * 128, (t / e.tiles_m) * BN + (half ? (i - e.whole) % 2 * 128 : 0), half};
}

template <int BN, int Y>
__global__ void __launch_bounds__(RowsCfg<BN>::THREADS, RowsCfg<BN>::CTAS)
    k_fp8_rows(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw, const Args e) {
  using K = RowsCfg<BN>;
  constexpr int S = K::STAGES, HN = K::HN;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  float* xsm = reinterpret_cast<float*>(smem + size_t(S) * K::STAGE);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + size_t(S) * K::STAGE + K::SCALES);
  uint64_t* empty = full + S;
  uint64_t* pfull = empty + S;   // a group's sum is in TMEM buffer b
  uint64_t* pempty = pfull + 2;  // its epilogue has read it
  uint64_t* done = pempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&pfull[b], 1);
      mbar_init(&pempty[b], K::EPI);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
    tc::prefetch_map(&tx);
    tc::prefetch_map(&tw);
  }
  if (warp == 1) tc::tmem_alloc(tmem_slot, K::TMEM);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;
  const int items = BN == 256 ? 2 * e.tiles_m * e.tiles_n - e.whole : e.tiles_m * e.tiles_n;

  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(K::LOW));
  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      for (int t = blockIdx.x; t < items && !*abort_flag; t += gridDim.x) {
        const RowsItem w = rows_item<BN>(e, t);
        for (int g = 0; g < e.groups; ++g, ++it) {
          const int s = it % S;
          if (it >= S && !mbar_wait(&empty[s], ((it / S) & 1) ^ 1, abort_flag)) {
            if (!*abort_flag) atomicExch(e.err, kFp8TimeoutTma);
            *abort_flag = 1;
            break;
          }
          uint8_t* st = smem + size_t(s) * K::STAGE;
          mbar_expect_tx(&full[s], w.half ? K::TILE_X + K::TILE_W / 2 : K::STAGE);
          tc::tma_load_2d(st, &tx, g * int(kKB), w.m0, &full[s]);
          tc::tma_load_2d(st + K::TILE_X, &tw, g * int(kKB), w.n0, &full[s]);
          if (BN == 256 && !w.half) tc::tma_load_2d(st + K::TILE_X + 128 * kKB, &tw, g * int(kKB), w.n0 + 128, &full[s]);
        }
      }
      if (*abort_flag) {  // every load issued lands before the CTA leaves (bounded)
        volatile int never = 0;
        for (int i = max(0, it - S); i < it; ++i) mbar_wait(&full[i % S], (i / S) & 1, &never);
      }
    }
  } else if (warp == 1) {
    const uint64_t dx0 = tc::desc_k(smem_u32(smem)), dw0 = tc::desc_k(smem_u32(smem) + K::TILE_X);
    int it = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < items && ok; t += gridDim.x) {
      const uint32_t idesc = BN == 256 && t >= e.whole ? idesc_f8(BN / 2) : idesc_f8(BN);
#pragma unroll 1
      for (int g = 0; g < e.groups; ++g, ++it) {
        const int s = it % S, b = it & 1;
        ok = (it < 2 || mbar_wait(&pempty[b], ((it >> 1) & 1) ^ 1, abort_flag)) && mbar_wait(&full[s], (it / S) & 1, abort_flag);
        if (!(ok = __all_sync(0xffffffffu, ok))) {
          if (lane == 0 && !*abort_flag) atomicExch(e.err, kFp8TimeoutMma);
          *abort_flag = 1;
          break;
        }
        tc::fence_after();
        const uint64_t dx = tc::desc_at(dx0, s * K::STAGE), dw = tc::desc_at(dw0, s * K::STAGE);
        if (tc::elect()) {
#pragma unroll
          for (int k = 0; k < 4; ++k)  // K = 32 an instruction: 32 bytes further in the swizzled row
            mma_f8(tmem + b * BN, tc::desc_at(dx, k * 32), tc::desc_at(dw, k * 32), idesc, k != 0);
          tc::commit(&empty[s]);
          tc::commit(&pfull[b]);
        }
        __syncwarp();
      }
    }
    if (tc::elect()) tc::commit(done);  // the CTA leaves (and frees its TMEM) after the last MMA
    __syncwarp();
    volatile int never = 0;
    mbar_wait(done, 0, &never);
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(K::HIGH));
    const int q = warp & 3, part = (warp - 4) >> 2;  // TMEM lanes q*32.., columns part*HN..
    // this warp's share of a block of scales: rows 16 ew .. 16 ew + 15, two a load
    const int ew = warp - 4, fg = lane % kXB, fr = ew * 16 + lane / kXB;
    float fetched[8];
    const auto fetch = [&](int t, int g0) {
      const int m0 = rows_item<BN>(e, t).m0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = m0 + fr + 2 * i;
        fetched[i] = r < e.m && g0 + fg < e.groups ? e.xs[(long long)r * e.groups + g0 + fg] : 0.f;
      }
    };
    if (int(blockIdx.x) < items) fetch(blockIdx.x, 0);
    int it = 0;
    bool ok = true;  // false: this warp computes and stores nothing more, but keeps to the barriers
    const auto item = [&](int t, auto columns) {  // of this warp
      constexpr int HN = decltype(columns)::value;
      const RowsItem w = rows_item<BN>(e, t);
      const int row = w.m0 + q * 32 + lane, c0 = w.n0 + part * HN;
      const bool in = row < e.m;
      const float* ws = e.ws + (long long)(min(c0, e.n - 1) / kFp8Group) * e.wgroups;
      float2 acc[HN / 2];
#pragma unroll
      for (int j = 0; j < HN / 2; ++j) acc[j] = make_float2(0.f, 0.f);
      float wn = ws[0];  // the next group's scale, in flight beside this group
#pragma unroll 1
      for (int g = 0; g < e.groups; ++g, ++it) {
        const int b = it & 1;
        if (g % kXB == 0) {
          named_bar(1, 32 * K::EPI);  // everyone has used the block before
#pragma unroll
          for (int i = 0; i < 8; ++i) xsm[fg * kXStride + fr + 2 * i] = fetched[i];
          named_bar(1, 32 * K::EPI);
          if (g + kXB < e.groups)
            fetch(t, g + kXB);
          else if (t + int(gridDim.x) < items)
            fetch(t + gridDim.x, 0);
        }
        const float f = xsm[(g % kXB) * kXStride + q * 32 + lane] * wn;
        wn = ws[min(g + 1, e.groups - 1)];
        if (ok) {
          ok = mbar_wait(&pfull[b], (it >> 1) & 1, abort_flag);
          if (!(ok = __all_sync(0xffffffffu, ok))) {
            if (lane == 0 && !*abort_flag) atomicExch(e.err, kFp8TimeoutEpi);
            *abort_flag = 1;
          }
        }
        if (!ok) continue;
        tc::fence_after();
        // LD columns arrive while the LD before them are added
        constexpr int LD = BN == 256 ? 32 : 16;
        const uint32_t at = tmem + (uint32_t(q * 32) << 16) + uint32_t(b * BN + part * HN);
        uint32_t r[2][LD];
        const auto load = [&](int j) {
          if constexpr (LD == 32)
            tc::tmem_ld32(at + j * LD, r[j & 1]);
          else
            tc::tmem_ld16(at + j * LD, r[j & 1]);
        };
        load(0);
#pragma unroll
        for (int j = 0; j < HN / LD; ++j) {
          tc::tmem_wait_ld();
          tc::landed(r[j & 1]);
          if (j + 1 < HN / LD) {
            load(j + 1);
          } else {  // read: the next group but one may overwrite it
            tc::fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&pempty[b]);
          }
#pragma unroll
          for (int i = 0; i < LD / 2; ++i) {
            acc[j * (LD / 2) + i].x = fmaf(__uint_as_float(r[j & 1][2 * i]), f, acc[j * (LD / 2) + i].x);
            acc[j * (LD / 2) + i].y = fmaf(__uint_as_float(r[j & 1][2 * i + 1]), f, acc[j * (LD / 2) + i].y);
          }
        }
      }
      // The accumulators' registers fix the unrolling, so the stores are kept to a
      // few instructions a column: as one general path they were 25 KB of code, and
      // fetching it once a tile took as long as twelve groups.
      if (ok && in) {
        const long long at = (long long)row * e.ldy + c0;
        if (e.vec && c0 + HN <= e.n) {
          if (e.bias || e.relu) {
#pragma unroll
            for (int j = 0; j < HN / 2; j += 2) {
              const float4 w = e.bias ? *reinterpret_cast<const float4*>(e.bias + c0 + 2 * j) : make_float4(0.f, 0.f, 0.f, 0.f);
              acc[j] = activate(make_float2(acc[j].x + w.x, acc[j].y + w.y), e.relu);
              acc[j + 1] = activate(make_float2(acc[j + 1].x + w.z, acc[j + 1].y + w.w), e.relu);
            }
          }
#pragma unroll
          for (int j = 0; j < HN / 2; j += 8) store16_y<Y>(e.y, at + 2 * j, acc + j);
        } else {
#pragma unroll
          for (int j = 0; j < HN; ++j) {
            if (c0 + j < e.n) {
              float v = j & 1 ? acc[j / 2].y : acc[j / 2].x;
              if (e.bias) v += e.bias[c0 + j];
              if (e.relu) v = v < 0.f ? 0.f : v;
              LowP<Y>::store(e.y, size_t(at + j), v);
            }
          }
        }
      }
    };
    for (int t = blockIdx.x; t < items; t += gridDim.x) {
      if (BN == 256 && t >= e.whole)
        item(t, std::integral_constant<int, HN / 2>{});
      else
        item(t, std::integral_constant<int, HN>{});
    }
  }
  tc::fence_before();
  __syncthreads();
  if (warp == 1) tc::tmem_free(tmem, K::TMEM);
}

// --------------------------------------------------------- few-rows kernel

constexpr int kFewStages = 4;  // 8, one CTA an SM, left clusters to a second round: 1 x 16384 x 2048 21.5 us against 12.4
constexpr int kFewBufs = 4;  // accumulators in TMEM, so that the MMAs need not wait for each one's reading: 3% to 5% over two
constexpr int kFewThreads = 64 + 128, kFewSplit = 8;  // CTAs of a cluster at most

template <int BR>
struct FewCfg {
  static constexpr uint32_t TILE_W = 128 * kKB, TILE_X = BR * kKB, STAGE = TILE_W + TILE_X;
  static constexpr uint32_t TMEM = kFewBufs * BR;
  // the ring; the float32 sums of the CTA's tile reuse it; then the row scales
  static size_t smem(int stages, int local_groups) {
    return 1024 + size_t(std::max(stages * int(STAGE), 128 * BR * 4)) + size_t(local_groups) * BR * 4 + 512;
  }
};

template <int BR>
__global__ void __launch_bounds__(kFewThreads)
    k_fp8_few(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw, const Args e, int stages) {
  using K = FewCfg<BR>;
  cg::cluster_group cl = cg::this_cluster();
  const int nsplit = int(cl.num_blocks()), rank = int(cl.block_rank());
  const int n0 = (blockIdx.x / nsplit) * 128, m0 = blockIdx.y * BR;
  const int per = ceil_div(e.groups, nsplit), g0 = min(rank * per, e.groups), g1 = min(g0 + per, e.groups), ng = g1 - g0;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int ring = max(stages * int(K::STAGE), 128 * BR * 4);
  float* xsc = reinterpret_cast<float*>(smem + ring);  // [group][row]
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + ring + size_t(per) * BR * 4);
  uint64_t* empty = full + kFewStages;
  uint64_t* pfull = empty + kFewStages;
  uint64_t* pempty = pfull + kFewBufs;
  uint64_t* done = pempty + kFewBufs;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < kFewBufs; ++b) {
      mbar_init(&pfull[b], 1);
      mbar_init(&pempty[b], 4);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
    tc::prefetch_map(&tx);
    tc::prefetch_map(&tw);
  }
  if (warp == 1) tc::tmem_alloc(tmem_slot, K::TMEM);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;
  float acc[BR];
#pragma unroll
  for (int j = 0; j < BR; ++j) acc[j] = 0.f;

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      for (; it < ng; ++it) {
        const int s = it % stages;
        if (it >= stages && !mbar_wait(&empty[s], ((it / stages) & 1) ^ 1, abort_flag)) {
          if (!*abort_flag) atomicExch(e.err, kFp8TimeoutTma);
          *abort_flag = 1;
          break;
        }
        uint8_t* st = smem + size_t(s) * K::STAGE;
        mbar_expect_tx(&full[s], K::STAGE);
        tc::tma_load_2d(st, &tw, (g0 + it) * int(kKB), n0, &full[s]);
        tc::tma_load_2d(st + K::TILE_W, &tx, (g0 + it) * int(kKB), m0, &full[s]);
      }
      if (*abort_flag) {
        volatile int never = 0;
        for (int i = max(0, it - stages); i < it; ++i) mbar_wait(&full[i % stages], (i / stages) & 1, &never);
      }
    }
  } else if (warp == 1) {
    const uint64_t dw0 = tc::desc_k(smem_u32(smem)), dx0 = tc::desc_k(smem_u32(smem) + K::TILE_W);
#pragma unroll 1
    for (int it = 0; it < ng; ++it) {
      const int s = it % stages, b = it % kFewBufs;
      bool ok = (it < kFewBufs || mbar_wait(&pempty[b], ((it / kFewBufs) & 1) ^ 1, abort_flag)) && mbar_wait(&full[s], (it / stages) & 1, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) {
        if (lane == 0 && !*abort_flag) atomicExch(e.err, kFp8TimeoutMma);
        *abort_flag = 1;
        break;
      }
      tc::fence_after();
      const uint64_t dx = tc::desc_at(dx0, s * K::STAGE), dw = tc::desc_at(dw0, s * K::STAGE);
      if (tc::elect()) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_f8(tmem + b * BR, tc::desc_at(dw, k * 32), tc::desc_at(dx, k * 32), idesc_f8(BR), k != 0);
        tc::commit(&empty[s]);
        tc::commit(&pfull[b]);
      }
      __syncwarp();
    }
    if (tc::elect()) tc::commit(done);
    __syncwarp();
    volatile int never = 0;
    mbar_wait(done, 0, &never);
  } else {
    const int q = warp & 3, tid = threadIdx.x - 64;
    // the products of scales of this CTA's rows and groups, while the first tiles arrive
    const float* ws = e.ws + (long long)(n0 / kFp8Group) * e.wgroups + g0;
    for (int i = tid; i < ng * BR; i += 128) {
      const int r = m0 + i % BR;
      xsc[i] = r < e.m ? ws[i / BR] * e.xs[(long long)r * e.groups + g0 + i / BR] : 0.f;
    }
    named_bar(1, 128);
    for (int it = 0; it < ng; ++it) {
      const int b = it % kFewBufs;
      const bool ok = mbar_wait(&pfull[b], (it / kFewBufs) & 1, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) {
        if (lane == 0 && !*abort_flag) atomicExch(e.err, kFp8TimeoutEpi);
        *abort_flag = 1;
        break;
      }
      tc::fence_after();
#pragma unroll
      for (int j = 0; j < BR; j += 16) {
        uint32_t r[16];
        tc::tmem_ld16(tmem + (uint32_t(q * 32) << 16) + uint32_t(b * BR + j), r);
        tc::tmem_wait_ld();
        tc::landed(r);
        if (j + 16 >= BR) {
          tc::fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&pempty[b]);
        }
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const float4 x4 = *reinterpret_cast<const float4*>(xsc + it * BR + j + i);
          acc[j + i] = fmaf(__uint_as_float(r[i]), x4.x, acc[j + i]);
          acc[j + i + 1] = fmaf(__uint_as_float(r[i + 1]), x4.y, acc[j + i + 1]);
          acc[j + i + 2] = fmaf(__uint_as_float(r[i + 2]), x4.z, acc[j + i + 2]);
          acc[j + i + 3] = fmaf(__uint_as_float(r[i + 3]), x4.w, acc[j + i + 3]);
        }
      }
    }
  }
  tc::fence_before();
  __syncthreads();  // every MMA and load of this CTA is complete: the ring is free
  if (warp == 1) tc::tmem_free(tmem, K::TMEM);
  float* part = reinterpret_cast<float*>(smem);  // [row][feature]
  if (warp >= 2) {
    const int f = (warp & 3) * 32 + lane;
#pragma unroll
    for (int j = 0; j < BR; ++j) part[j * 128 + f] = acc[j];
  }
  cl.sync();
  // Rank r sums the rows r, r + nsplit, ... over the ranks in order, a warp a row,
  // with the sums of all ranks in flight together (one read after the other, 64
  // rows took 9 us more than one).
  const int rows = min(BR, e.m - m0);
#pragma unroll 1
  for (int r = rank + nsplit * warp; r < rows; r += nsplit * (kFewThreads / 32)) {
    float v[kFewSplit][4];
#pragma unroll
    for (int k = 0; k < kFewSplit; ++k)
      if (k < nsplit) {
        const float* from = cl.map_shared_rank(part, k) + r * 128 + lane;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[k][j] = from[32 * j];
      }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + 32 * j + lane;
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < kFewSplit; ++k)
        if (k < nsplit) sum += v[k][j];
      if (n >= e.n) continue;
      if (e.bias) sum += e.bias[n];
      if (e.relu) sum = sum < 0.f ? 0.f : sum;
      store_as(e.y_type, e.y, size_t((long long)(m0 + r) * e.ldy + n), sum);
    }
  }
  cl.sync();  // peers' sums stay until everyone has read them
}

constexpr size_t kSmemMax = 227 * 1024;

// Tiles of 256 features left for a last round over the SMs that may as well be
// taken in halves, because twice as many items still fit in it.
int halved(long long tiles) {
  const int left = int(tiles % 148);
  return left * 2 <= 148 ? left : 0;
}

template <int BN, int Y>
void launch_rows_y(const Fp8GemmParams& p, Args e, cudaStream_t s) {
  using K = RowsCfg<BN>;
  CUtensorMap tx, tw;
  tc::make_map(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.x, p.k, p.m, p.ldx, kKB, 128);
  tc::make_map(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.w, p.k, p.n, p.ldw, kKB, 128);
  e.tiles_m = ceil_div(p.m, 128);
  e.tiles_n = ceil_div(p.n, BN);
  static std::atomic<unsigned long long> allowed{0};
  tc::allow_smem(k_fp8_rows<BN, Y>, K::SMEM, allowed);
  const int tiles = e.tiles_m * e.tiles_n;
  e.whole = BN == 256 ? tiles - halved(tiles) : tiles;
  const int grid = int(std::min<long long>(2LL * tiles - e.whole, 148LL * K::CTAS));
  k_fp8_rows<BN, Y><<<grid, K::THREADS, K::SMEM, s>>>(tx, tw, e);
  B2E_CUDA(cudaGetLastError());
}

template <int BN>
void launch_rows(const Fp8GemmParams& p, const Args& e, cudaStream_t s) {
  if (p.y_type == kF32) return launch_rows_y<BN, kF32>(p, e, s);
  if (p.y_type == kBF16) return launch_rows_y<BN, kBF16>(p, e, s);
  launch_rows_y<BN, kF16>(p, e, s);
}

// False where the rows kernel takes less time. With one round of tiles over the SMs
// that kernel takes 3 + 0.385 us a group, and this one 4 (one row) to 5.4 (64 rows)
// + 0.5 us a group of its share, which is the comparison below. Rows against few:
// 1 x 256 x 1280 3.8 / 4.2 us, 1 x 2048 x 8448 9.4 / 7.3, 64 x 2048 x 8448 9.7 /
// 10.5, 64 x 4096 x 1024 15.5 / 7.3, 400 x 4096 x 1024 16.1 / 13.9, 1000 x 4096 x
// 1024 16.7 / 25.4, 1 x 4096 x 40000 (more than L2) 42.4 / 43.4.
// False too where the scales of a CTA's groups would not fit beside the ring.
template <int BR>
bool launch_few(const Fp8GemmParams& p, const Args& e, cudaStream_t s) {
  using K = FewCfg<BR>;
  const int tn = ceil_div(p.n, 128), tm = ceil_div(p.m, BR);
  // as many CTAs of a cluster as fill the SMs and still have a group each
  int split = 1;
  while (split < kFewSplit && split * 2 <= e.groups && (long long)tn * tm * split * 2 <= 148) split *= 2;
  const int per = ceil_div(e.groups, split), stages = std::min(kFewStages, per);
  if (3LL * e.groups - 4LL * per < 8 + std::min(p.m, 64) / 7) return false;
  const size_t smem = K::smem(stages, per);
  if (smem > kSmemMax) return false;
  CUtensorMap tx, tw;
  tc::make_map(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.x, p.k, p.m, p.ldx, kKB, BR);
  tc::make_map(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.w, p.k, p.n, p.ldw, kKB, 128);
  static std::atomic<unsigned long long> allowed{0};
  tc::allow_smem(k_fp8_few<BR>, kSmemMax, allowed);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(tn * split, tm);
  cfg.blockDim = dim3(kFewThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {unsigned(split), 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 1;
  B2E_CUDA(cudaLaunchKernelEx(&cfg, k_fp8_few<BR>, tx, tw, e, stages));
  return true;
}

}  // namespace

void fp8_gemm(const Fp8GemmParams& p, cudaStream_t s) {
  if (p.m == 0) return;
  const int esz = int(dtype_size(p.y_type));
  Args e{p.xs, p.ws, p.bias, p.y, p.ldy, p.m, p.n, ceil_div(p.k, kFp8Group), ceil_div(p.k, kFp8Group),
         p.relu, p.y_type, 0, 0, 0, 0, p.err};
  e.vec = reinterpret_cast<uintptr_t>(p.y) % 32 == 0 && (p.ldy * esz) % 32 == 0 && reinterpret_cast<uintptr_t>(p.bias) % 16 == 0;
  if (p.m <= 16 && launch_few<16>(p, e, s)) return;
  if (p.m > 16 && p.m <= 32 && launch_few<32>(p, e, s)) return;
  if (p.m > 32 && launch_few<64>(p, e, s)) return;
  const long long tm = ceil_div(p.m, 128), t128 = tm * ceil_div(p.n, 128), t256 = tm * ceil_div(p.n, 256);
  B2E_CHECK(t128 <= 0x3fffffffLL, kErrInvalid, "fp8_linear: too many tiles");
  // Tiles of 128 features run two CTAs an SM; tiles of 256 read less shared memory
  // a product. The wider tile where its rounds over the SMs, a last one of halves
  // counted half, cost no more.
  const long long h128 = (t128 + 295) / 296 * 2, h256 = (t256 + 147) / 148 * 2 - (halved(t256) > 0);
  if (h256 <= h128)
    launch_rows<256>(p, e, s);
  else
    launch_rows<128>(p, e, s);
}

namespace tc {

void make_map(CUtensorMap* m, CUtensorMapDataType type, int size, const void* base, uint64_t inner, uint64_t rows,
              uint64_t ld, uint32_t box_inner, uint32_t box_rows) {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  B2E_CHECK(fn != nullptr, kErrCuda, "cuTensorMapEncodeTiled is unavailable");
  const cuuint64_t dims[2] = {inner, rows};
  const cuuint64_t strides[1] = {ld * uint64_t(size)};
  const cuuint32_t box[2] = {box_inner, box_rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(m, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  B2E_CHECK(r == CUDA_SUCCESS, kErrCuda, "cuTensorMapEncodeTiled failed (" + std::to_string(int(r)) + ")");
}

}  // namespace tc
}  // namespace b2e
