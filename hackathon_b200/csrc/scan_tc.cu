// Chunked selective scan on the tensor cores (tcgen05), for bf16 operands, heads
// of 64 rows and states of 64 or 128 columns.
//
// A sequence (or one segment of it) is walked in chunks of 128 tokens by one CTA
// for a pair of heads. With c[t] = sum of a dt over the chunk up to token t, and
// H the pair's state [2 x 64, N] at the chunk's start,
//
//   G = C B^T                                   (once for both heads)
//   S[t, s] = G[t, s] exp(c[t] - c[s]) dt[s],   s <= t
//   Y = exp(c[t]) (C H^T) + S X
//   H <- exp(c[T]) H + (exp(c[T] - c[s]) dt[s] X)^T B
//
// which is the recurrence written out over a chunk (with a above zero it overflows
// where the sum of a dt over a chunk passes 88). Five products a chunk, all
// M = 128 in float32 TMEM accumulators: G, C H^T and the state's with N = 128
// columns (both heads at once, so the shared-memory operands are read at the
// rate the MMA can take), S X with its left operand in TMEM.
//
// Roundings: S and the copy of H that multiplies C are rounded once to bf16, as
// y itself is: they are the MMA's operands, and a second half of either would not fit
// (TMEM is full, and shared memory but for 3 KB). y is then 0.0022 to 0.0023 from 64
// bits (relative 2-norm) where its own rounding alone is 0.0017. The
// state must not drift: its operand exp() dt x is split exactly over three bf16
// values (24 bits), three products into the float32 state that stays in TMEM
// over the whole walk. Sums of a dt are carried as float32 pairs (hi, lo), so
// that differences of far sums keep their low bits after a token with a very
// large step; rows of S take one factor a row block times one a column where
// blocks of 32 tokens do not touch, and the exponential of the difference inside
// the diagonal blocks, so nothing overflows for decays below one.
//
// Twenty-eight warps: 0 TMA loads; 1 the state's MMAs; 2 the decays, a half-warp a
// head; 3 the MMAs of G and y (and zeros in B behind a sequence's end); 4-11 S from
// G; 12-19 the state: its decay, its bf16 copy, the split operand (and zeros in x
// behind the end); 20-27 y: exp(c) on C H^T, skip, gate and stores. The chain of a
// chunk is state ready -> C H^T -> scaled -> + S X -> y; the state's products, G of
// the next chunk, decays up to three chunks ahead and the gate run beside it. There
// are two MMA issuers because the state's chain must not queue behind y's.
//
// What bounds it: the handoffs along that chain and instruction latency (seven
// warps a scheduler issue in 53% of the cycles); the tensor cores, with 6 x 128 x 128 x
// 128 products a chunk and pair, are active in 21%, and DRAM is at 23%. 37 sequences of
// 4096 tokens, 16 heads, state 128: 437 to 443 us with the gate, 343 to 348 without (755
// and 608 with sixteen warps and one MMA issuer); 64 sequences of 512 tokens, 64 heads:
// 530 us; one chunk alone 18 us.
#include <algorithm>

#include "packed.cuh"
#include "scan.cuh"
#include "tc.cuh"

namespace b2e {
namespace {

constexpr int Q = 128;                       // tokens of a chunk
constexpr uint32_t kTile = Q * 128;          // 128 rows of 128 bytes
constexpr int kXSlots = 3;
constexpr int kTcThreads = 896;
constexpr int kVecs = 3;                     // chunks whose decays are held
enum ScanError : int { kScanTimeout = 131 };
// Registers by warpgroup, out of the launch's 28 warps x 72. The shared memory
// leaves almost no L1, so that a spilled register is a trip to L2: with 72 for
// everyone the y warps spilled and a chunk took three times as long.
constexpr int kRegLaunch = 72, kRegMisc = 72, kRegS = 56, kRegX = 72, kRegY = 88;
static_assert(4 * kRegMisc + 8 * kRegS + 8 * kRegX + 8 * kRegY <= 28 * kRegLaunch, "register shares exceed the launch's");
template <bool ENDS, int N>
__device__ __forceinline__ void shares() {
  if constexpr (!ENDS) {
    if constexpr (N < kRegLaunch)
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
    else if constexpr (N > kRegLaunch)
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
  }
}

// TMEM columns (of 512): G, and S of both heads in its place (each 16 columns of
// G become 8 of either head's S in bf16 pairs); the buffers of the state's
// operand; Y and H of both heads.
constexpr uint32_t cG = 0, cXW = 128, cY = 256, cH = 384;
__device__ __forceinline__ uint32_t s_col(int h, int k) { return cG + k * 16 + h * 8; }  // tokens 16 k..

// kind::f16, bf16 x bf16, float32 accumulator, M = 128.
__host__ __device__ constexpr uint32_t idesc_bf16(int n, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(b_mn) << 16) | (uint32_t(n >> 3) << 17) | (uint32_t(128 >> 4) << 24);
}

// Operand whose contiguous axis is not the summed one: rows of 128 bytes (64
// values of M or N) along K, swizzled by 8-row atoms of 1024 bytes; the next 64
// values of M or N are `chunk` bytes away.
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr, uint32_t chunk) {
  return uint64_t((addr & 0x3FFFF) >> 4) | (uint64_t(chunk >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
         (uint64_t(2) << 61);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc));
}

// A sum kept as hi + lo.
struct Pair {
  float hi, lo;
};
__device__ __forceinline__ Pair add(Pair a, Pair b) {
  const float s = a.hi + b.hi, bb = s - a.hi;
  const float e = (a.hi - (s - bb)) + (b.hi - bb) + (a.lo + b.lo);
  const float h = s + e;
  return {h, e - (h - s)};
}
__device__ __forceinline__ float diff(Pair a, Pair b) { return (a.hi - b.hi) + (a.lo - b.lo); }
// log(1 + exp(x)) = max(x, 0) + log1p(e), e = exp(-|x|), with log1p(e) = 2 atanh(s),
// s = e / (2 + e) <= 1 / 3, by its series to s^17 (the next term is below 2^-31 of
// the first): relative accuracy for any x, in a third of the library's instructions.
__device__ __forceinline__ float softplus_fast(float x) {
  const float e = ex2(fabsf(x) * -1.4426950408889634f), s = e * rcp(2.0f + e), q = s * s;
  float r = 2.0f / 17.0f;
  r = fmaf(r, q, 2.0f / 15.0f);
  r = fmaf(r, q, 2.0f / 13.0f);
  r = fmaf(r, q, 2.0f / 11.0f);
  r = fmaf(r, q, 2.0f / 9.0f);
  r = fmaf(r, q, 2.0f / 7.0f);
  r = fmaf(r, q, 2.0f / 5.0f);
  r = fmaf(r, q, 2.0f / 3.0f);
  r = fmaf(r, q, 2.0f);
  return fmaf(s, r, x < 0.f ? 0.f : x);
}

// The place in a ring of `size`, and its phase, after `n` uses.
struct Turn {
  int size, at = 0, phase = 0;
  __device__ __forceinline__ Turn(int ring, int n = 0) : size(ring), at(n % ring), phase((n / ring) & 1) {}
  __device__ __forceinline__ void next(int n = 1) {
    at += n;
    if (at >= size) {
      at -= size;
      phase ^= 1;
    }
  }
};

// Decays of one head and chunk; c in powers of two.
struct Vec {
  float neg[Q];   // -(c[s] - base[s / 32])
  float dt[Q];
  float w[Q];     // exp(c[T] - c[s]) dt[s]
  float col[192]; // exp(base[i] - c[s]) dt[s] for s before block i: 32 values for i = 1, 64, 96
  float base[4];  // c before each block of 32 tokens
  float total;    // exp(c[T])
  float pad[3];
};

template <int NB>
struct TcCfg {
  static constexpr uint32_t CB = NB * kTile;  // bytes of a chunk of C (or B)
  static constexpr uint32_t oC = 0, oB = CB, STAGE = 2 * CB;
  static constexpr uint32_t oX = 2 * STAGE, oH = oX + kXSlots * kTile, oV = oH + NB * kTile;
  static constexpr uint32_t oBad = oV + kVecs * 2 * sizeof(Vec);    // [kVecs][2][128] first token that is not finite, [kVecs][8] flags
  static constexpr uint32_t oBar = oBad + kVecs * (2 * 128 + 8 * 4);
  static constexpr size_t SMEM = oBar + 512 + 1024;
};

struct TcArgs {
  ScanParams p;
  ScanWork wk;
  int seg, pairs;
};

// ENDS: only the segment's own contribution to the state, from a zero start.
template <int NB, bool ENDS>
__global__ void __launch_bounds__(kTcThreads, 1)
    k_scan_tc(const __grid_constant__ CUtensorMap mx, const __grid_constant__ CUtensorMap mb, const __grid_constant__ CUtensorMap mc,
              const __grid_constant__ TcArgs g) {
  using K = TcCfg<NB>;
  constexpr int N = 64 * NB;
  const ScanParams& p = g.p;
  const int tile = blockIdx.x / g.pairs, h0 = (blockIdx.x % g.pairs) * 2;
  SeqTile t;
  if (g.seg > 0) {
    t = seq_tile(p.plan, tile, g.seg);
  } else {
    t = seq_whole(p.plan, tile);
  }
  if (threadIdx.x == kTcThreads - 1 && h0 == 0) seq_report(p.plan, tile, g.seg == 0, p.err);
  if (!t.live) return;
  const int slot = p.plan.slots ? p.plan.slots[t.seq] : t.seq;
  if (slot < 0 || slot >= p.plan.state_rows) {
    if (threadIdx.x == 0) *p.err = 1;
    return;
  }
  const int end = g.seg > 0 && t.end - t.first > g.seg ? t.first + g.seg : t.end;
  if (ENDS && end == t.end) return;
  const int chunks = (end - t.first + Q - 1) / Q;
  const long long place = g.seg > 0 ? work_place(g.wk, p.plan, g.seg, t.seq, t.start, t.k) : 0;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // What the first chunk waits for from HBM, on its way while the CTA sets up: dt,
  // and the state's rows (half a row a thread).
  if (warp == 2) {
#pragma unroll
    for (int k = 0; k < Q; k += 32)
      if (t.first + k + lane < end)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(p.dt + (long long)(t.first + k + lane) * p.lddt + h0));
  } else if (!ENDS && warp >= 12 && warp < 20) {
    const int row = (warp & 3) * 32 + lane, half = warp >= 16;
    if (h0 + (row >> 6) < p.heads) {
      const bool joined = g.seg > 0 && t.end - t.start > g.seg;
      const float* f = (joined ? g.wk.state + (place * p.heads + h0) * 64 * N : p.ssm + ((long long)slot * p.heads + h0) * 64 * N) +
                       (long long)row * N + half * (N / 2);
#pragma unroll
      for (int k = 0; k < N / 2; k += 32) asm volatile("prefetch.global.L2 [%0];" ::"l"(f + k));
    }
  }

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sbase = smem_u32(smem);
  Vec* vec = reinterpret_cast<Vec*>(smem + K::oV);  // [chunk % kVecs][head]
  uint8_t* bad = smem + K::oBad;
  int* anybad = reinterpret_cast<int*>(bad + kVecs * 2 * 128);
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + K::oBar);
  uint64_t *cbfull = bar, *cbempty = bar + 2, *xfull = bar + 4, *xempty = bar + 7, *vfull = bar + 10, *vempty = bar + 13,
           *xwfull = bar + 16, *xwempty = bar + 18, *xscan = bar + 20, *gfull = bar + 23, *sfull = bar + 24, *y2full = bar + 25,
           *y2scaled = bar + 26, *yfull = bar + 27, *yfree = bar + 28, *hready = bar + 29, *hdone = bar + 30, *done = bar + 31,
           *bzero = bar + 32;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + 33);
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&cbfull[i], 1);
      mbar_init(&cbempty[i], ENDS ? 1 : 2);
      mbar_init(&xwfull[i], 4);
      mbar_init(&xwempty[i], 1);
    }
    for (int i = 0; i < kVecs; ++i) {
      mbar_init(&vfull[i], 1);
      mbar_init(&vempty[i], ENDS ? 8 : 24);
      mbar_init(&xscan[i], 8);
    }
    for (int i = 0; i < kXSlots; ++i) {
      mbar_init(&xfull[i], 1);
      mbar_init(&xempty[i], ENDS ? 4 : 9);  // four warps of the state's, S X, four warps of y's
    }
    mbar_init(gfull, 1);
    mbar_init(sfull, 8);
    mbar_init(y2full, 1);
    mbar_init(y2scaled, 8);
    mbar_init(yfull, 1);
    mbar_init(yfree, 8);
    mbar_init(hready, 8);
    mbar_init(hdone, 1);
    mbar_init(done, ENDS ? 1 : 2);
    mbar_init(bzero, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
    tc::prefetch_map(&mx);
    tc::prefetch_map(&mb);
    tc::prefetch_map(&mc);
  }
  if (warp == 1) tc::tmem_alloc(tmem_slot, 512);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;  // this warp's TMEM lanes

  // The roles' code runs beside one another out of one instruction cache, so it is
  // kept short: loops stay rolled and a wait is a handful of instructions. A wait
  // is bounded by its polls (a poll suspends the thread for a while; 2^22 are from
  // a tenth of a second to seconds), and its role winds down when they run out; the
  // roles that wait for it do so by their own bounds, once each. (A flag of the first
  // one's that ends the others' waits made every wait longer: 343 us to 365 for
  // 37 x 4096 tokens, 16 heads.)
  auto poll = [&](uint64_t* b, uint32_t parity) -> bool {
    int n = 0;
    while (!mbar_try(b, parity))
      if (++n == 1 << 22) return false;
    return true;
  };
  auto failed = [&] { atomicCAS(p.err, 0, kScanTimeout); };  // an earlier code stays
  // Every thread of a warp waits, with one answer for all of them.
  auto wait = [&](uint64_t* b, uint32_t parity) -> bool { return __all_sync(0xffffffffu, poll(b, parity)); };
  auto arrive = [&](uint64_t* b) {
    __syncwarp();
    if (lane == 0) mbar_arrive(b);
  };

  if (warp < 4) {
    shares<ENDS, kRegMisc>();
  if (warp == 0) {
    // ---- loads
    if (lane == 0) {
      Turn ct(2), xt(kXSlots);
      bool ok = true;
      int c = 0, u = 0, cbs = 0;
#pragma unroll 1
      for (int i = 0; i < 3 * chunks; ++i) {  // B and C, x of either head
        const int row = t.first + c * Q, h = u & 1;
        const bool cb = i - 3 * c == 0;
        uint64_t *full = cb ? &cbfull[ct.at] : &xfull[xt.at], *empty = cb ? &cbempty[ct.at] : &xempty[xt.at];
        if ((cb ? c >= 2 : u >= kXSlots) && !(ok = poll(empty, (cb ? ct.phase : xt.phase) ^ 1))) break;
        mbar_expect_tx(full, cb ? (ENDS ? 1 : 2) * K::CB : kTile);
        if (cb) {
          uint8_t* s = smem + ct.at * K::STAGE;
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            tc::tma_load_2d(s + K::oB + n * kTile, &mb, n * 64, row, full);
            if (!ENDS) tc::tma_load_2d(s + K::oC + n * kTile, &mc, n * 64, row, full);
          }
          ct.next();
          ++cbs;
        } else {
          tc::tma_load_2d(smem + K::oX + xt.at * kTile, &mx, (h0 + h) * 64, row, full);
          xt.next();
          ++u;
          c += h;
        }
      }
      if (!ok) failed();
      // After a wait that ran out, here or in another role, the loads that were
      // issued land before the CTA leaves (bounded); otherwise they have.
#pragma unroll 1
      for (int i = max(0, u - kXSlots); i < u; ++i) poll(&xfull[i % kXSlots], (i / kXSlots) & 1);
#pragma unroll 1
      for (int i = max(0, cbs - 2); i < cbs; ++i) poll(&cbfull[i & 1], (i >> 1) & 1);
    }
  } else if (warp == 1) {
    // ---- the state's MMAs: H += (32 tokens of the split operand)^T B
    bool ok = true;
#pragma unroll 1
    for (int c = 0; c < chunks; ++c) {
      const int st = c & 1;
      const uint64_t dB = desc_mn(sbase + st * K::STAGE + K::oB, kTile);
      if (!(ok = wait(hready, c & 1) && wait(&cbfull[st], (c >> 1) & 1))) break;
      if (end - t.first - c * Q < Q && !(ok = wait(bzero, 0))) break;  // the last chunk's, a short one
#pragma unroll 1
      for (int j = 0; j < 4; ++j) {
        if (!(ok = wait(&xwfull[j & 1], j >> 1))) break;
        tc::fence_after();
        const uint64_t dj = tc::desc_at(dB, j * 32 * 128);
        if (tc::elect()) {
#pragma unroll
          for (int k = 0; k < 6; ++k)  // three splits, two steps of 16 tokens each
            mma_ts(tmem + cH, tmem + cXW + (j & 1) * 64 + (k >> 1) * 16 + (k & 1) * 8, tc::desc_at(dj, (k & 1) * 16 * 128),
                   idesc_bf16(N, true), 1);
          tc::commit(&xwempty[j & 1]);
        }
        __syncwarp();
      }
      if (!ok) break;
      if (tc::elect()) {
        tc::commit(hdone);
        tc::commit(&cbempty[st]);
      }
      __syncwarp();
    }
    if (tc::elect()) tc::commit(done);  // the CTA leaves (and frees its TMEM) after the last MMA
    __syncwarp();
    poll(done, 0);
    if (!ok && lane == 0) failed();
  } else if (warp == 3) {
    // ---- y's MMAs: G = C B^T, Y = C H^T, Y += S X
    if (!ENDS) {
      const uint64_t dC0 = tc::desc_k(sbase + K::oC), dB0 = tc::desc_k(sbase + K::oB), dH = tc::desc_k(sbase + K::oH),
                     dX0 = desc_mn(sbase + K::oX, kTile);
      bool ok = true;
      Turn vt(kVecs), xscanned(kVecs), xt(kXSlots);
#pragma unroll 1
      for (int i = 0; i <= chunks; ++i, vt.next()) {
        // Y of chunk i - 1, then G of chunk i
        const int c = i - 1, st = c & 1;
        if (i > 0) {
          const uint64_t dC = tc::desc_at(dC0, st * K::STAGE);
          if (!(ok = wait(hready, c & 1) && wait(&cbfull[st], (c >> 1) & 1) && (c == 0 || wait(yfree, (c - 1) & 1)))) break;
          tc::fence_after();
          if (tc::elect()) {
#pragma unroll 2
            for (int k = 0; k < N / 16; ++k) {
              const uint32_t off = (k / 4) * kTile + (k % 4) * 32;
              mma_ss(tmem + cY, tc::desc_at(dC, off), tc::desc_at(dH, off), idesc_bf16(Q, false), k != 0);
            }
            tc::commit(y2full);
          }
          __syncwarp();
          if (!(ok = wait(sfull, c & 1) && wait(&xscan[xscanned.at], xscanned.phase) && wait(y2scaled, c & 1))) break;
#pragma unroll 1
          for (int h = 0; h < 2; ++h, xt.next()) {
            if (!(ok = wait(&xfull[xt.at], xt.phase))) break;
            tc::fence_after();
            const uint64_t dX = tc::desc_at(dX0, xt.at * kTile);
            if (tc::elect()) {
#pragma unroll 4
              for (int k = 0; k < 8; ++k)
                mma_ts(tmem + cY + h * 64, tmem + s_col(h, k), tc::desc_at(dX, k * 16 * 128), idesc_bf16(64, true), 1);
              tc::commit(&xempty[xt.at]);
            }
            __syncwarp();
          }
          xscanned.next();
          if (!ok) break;
          if (tc::elect()) {
            tc::commit(yfull);
            tc::commit(&cbempty[st]);
          }
          __syncwarp();
        }
        if (i < chunks) {
          if (!(ok = wait(&vfull[vt.at], vt.phase) && wait(&cbfull[i & 1], (i >> 1) & 1))) break;
          tc::fence_after();
          const uint64_t a = tc::desc_at(dC0, (i & 1) * K::STAGE), b = tc::desc_at(dB0, (i & 1) * K::STAGE);
          if (tc::elect()) {
#pragma unroll 2
            for (int k = 0; k < N / 16; ++k) {
              const uint32_t off = (k / 4) * kTile + (k % 4) * 32;
              mma_ss(tmem + cG, tc::desc_at(a, off), tc::desc_at(b, off), idesc_bf16(Q, false), k != 0);
            }
            tc::commit(gfull);
          }
          __syncwarp();
          const int valid = end - t.first - i * Q;
          if (valid < Q) {
            // Behind the sequence's end lie other sequences' rows of B: zeros before the
            // state's products, so that nothing of them meets one (G's columns there
            // are masked in S, and the state's warps do the same for x). Here, because
            // this warp takes every phase of these barriers in turn: a parity cannot
            // tell a phase from the one two before it.
            if (!(ok = wait(gfull, i & 1))) break;
            uint8_t* bt = smem + (i & 1) * K::STAGE + K::oB;
#pragma unroll 4
            for (int k = valid * 8 + lane; k < Q * 8; k += 32)
#pragma unroll
              for (int n = 0; n < NB; ++n) *reinterpret_cast<uint4*>(bt + n * kTile + k * 16) = make_uint4(0, 0, 0, 0);
            fence_proxy_async();
            arrive(bzero);
          }
        }
      }
      if (tc::elect()) tc::commit(done);
      __syncwarp();
      poll(done, 0);
      if (!ok && lane == 0) failed();
    }
  } else if (warp == 2) {
    // ---- decays: a half-warp a head, eight tokens a lane
    const int hh = lane >> 4, l = lane & 15;
    const bool has = h0 + hh < p.heads;
    const float a2 = has ? p.a[h0 + hh] * 1.4426950408889634f : 0.f;
    const float* at = p.dt + (long long)(t.first + 8 * l) * p.lddt + h0 + hh;
    float dt[8];
    const auto fetch = [&](int left) {  // dt of the chunk at `at`, `left` tokens
#pragma unroll
      for (int k = 0; k < 8; ++k) dt[k] = has && 8 * l + k < left ? at[k * p.lddt] : 0.f;
    };
    fetch(end - t.first);
    bool ok = true;
    Turn vt(kVecs);
#pragma unroll 1
    for (int c = 0; c < chunks; ++c, vt.next()) {
      const int vs = vt.at, valid = min(Q, end - t.first - c * Q);
      Pair cum[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const bool in = has && 8 * l + k < valid;
        if (p.softplus) dt[k] = softplus_fast(dt[k]);
        dt[k] = in ? dt[k] : 0.f;
        // Below 2^-200 a decay is zero in float32 whatever it multiplies; the
        // bound keeps the sums small (and keeps a NaN).
        float x = in ? a2 * dt[k] : 0.f;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(x) : "f"(x), "f"(-200.f));
        cum[k] = k ? add(cum[k - 1], {x, 0.f}) : Pair{x, 0.f};
      }
      Pair sum = cum[7];
#pragma unroll 1
      for (int o = 1; o < 16; o <<= 1) {
        const Pair x = {__shfl_up_sync(0xffffffffu, sum.hi, o, 16), __shfl_up_sync(0xffffffffu, sum.lo, o, 16)};
        if (l >= o) sum = add(x, sum);
      }
      Pair before = {__shfl_up_sync(0xffffffffu, sum.hi, 1, 16), __shfl_up_sync(0xffffffffu, sum.lo, 1, 16)};
      if (l == 0) before = {0.f, 0.f};
      const auto upto = [&](int src) { return Pair{__shfl_sync(0xffffffffu, sum.hi, src, 16), __shfl_sync(0xffffffffu, sum.lo, src, 16)}; };
      const Pair b1 = upto(3), b2 = upto(7), b3 = upto(11), total = upto(15);
      const int blk = l >> 2;
      const Pair base = blk == 0 ? Pair{0.f, 0.f} : blk == 1 ? b1 : blk == 2 ? b2 : b3;
      if (c >= kVecs && !(ok = wait(&vempty[vs], vt.phase ^ 1))) break;
      Vec& v = vec[vs * 2 + hh];
#pragma unroll
      for (int k0 = 0; k0 < 8; k0 += 4) {
        float o[5][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const Pair x = add(before, cum[k0 + k]);
          const float d = dt[k0 + k];
          o[0][k] = diff(base, x);
          o[1][k] = ex2(diff(total, x)) * d;
          o[2][k] = ex2(diff(b1, x)) * d;
          o[3][k] = ex2(diff(b2, x)) * d;
          o[4][k] = ex2(diff(b3, x)) * d;
        }
        const auto put = [&](float* to, const float* f) { *reinterpret_cast<float4*>(to + 8 * l + k0) = make_float4(f[0], f[1], f[2], f[3]); };
        put(v.neg, o[0]);
        put(v.dt, dt + k0);
        put(v.w, o[1]);
        if (blk < 1) put(v.col, o[2]);
        if (blk < 2) put(v.col + 32, o[3]);
        if (blk < 3) put(v.col + 96, o[4]);
      }
      if ((l & 3) == 0) v.base[blk] = base.hi + base.lo;
      if (l == 0) v.total = ex2(total.hi + total.lo);
      at += Q * p.lddt;
      fetch(end - t.first - (c + 1) * Q);
      arrive(&vfull[vt.at]);
    }
    if (!ok && lane == 0) failed();
  }
  } else if (warp < 12) {
    shares<ENDS, kRegS>();
    // ---- S of both heads from G, in its place: lane = token t, the blocks of 16 tokens s in turn
    if (!ENDS) {
      const int q = warp & 3, row = q * 32 + lane, odd = (warp >> 2) & 1;
      bool ok = true;
      Turn vt(kVecs);
#pragma unroll 1
      for (int c = 0; c < chunks; ++c, vt.next()) {
        const int vs = vt.at;
        if (!(ok = wait(&vfull[vs], vt.phase) && wait(gfull, c & 1))) break;
        tc::fence_after();
        const int colbase = (q == 1 ? 0 : q == 2 ? 32 : 96);
#pragma unroll 1
        for (int k = odd; k < 8; k += 2) {
          const uint32_t at = tmem + lanes + cG + k * 16;
          uint32_t r[16];
          if (k >> 1 <= q) {
            tc::tmem_ld16(at, r);
            tc::tmem_wait_ld();
            tc::landed(r);
          }
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            const Vec& v = vec[vs * 2 + h];
            uint32_t o[8];
            if (k >> 1 < q) {
              const float rw = ex2(-v.neg[row]);
              const F2 rw2 = f2(rw, rw);
              const float* col = v.col + colbase + k * 16;
#pragma unroll
              for (int i = 0; i < 16; i += 4) {
                const float4 f = *reinterpret_cast<const float4*>(col + i);
                o[i / 2] = pack_bf16(mul2(f2(r[i], r[i + 1]), mul2(f2(f.x, f.y), rw2)));
                o[i / 2 + 1] = pack_bf16(mul2(f2(r[i + 2], r[i + 3]), mul2(f2(f.z, f.w), rw2)));
              }
            } else if (k >> 1 == q) {
              // 32 tokens' sums stay below 6400, so a difference is exact to 2^-11, below S's own rounding
              const float me = -v.neg[row];
              const F2 me2 = f2(me, me);
              const int last = lane - (k & 1) * 16;  // the row's own token in this block
#pragma unroll
              for (int i = 0; i < 16; i += 4) {
                const float4 sn = *reinterpret_cast<const float4*>(v.neg + k * 16 + i);
                const float4 sd = *reinterpret_cast<const float4*>(v.dt + k * 16 + i);
                float e[4], w[4];
                split(add2(me2, f2(sn.x, sn.y)), e[0], e[1]);
                split(add2(me2, f2(sn.z, sn.w)), e[2], e[3]);
                split(mul2(mul2(f2(ex2(e[0]), ex2(e[1])), f2(sd.x, sd.y)), f2(r[i], r[i + 1])), w[0], w[1]);
                split(mul2(mul2(f2(ex2(e[2]), ex2(e[3])), f2(sd.z, sd.w)), f2(r[i + 2], r[i + 3])), w[2], w[3]);
#pragma unroll
                for (int n = 0; n < 4; ++n) w[n] = i + n <= last ? w[n] : 0.f;  // s <= t, whatever G holds
                o[i / 2] = pack_bf16(w[0], w[1]);
                o[i / 2 + 1] = pack_bf16(w[2], w[3]);
              }
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i) o[i] = 0;
            }
            tc::tmem_st8(at + h * 8, o);
          }
        }
        tc::tmem_wait_st();
        tc::fence_before();
        arrive(sfull);
        arrive(&vempty[vs]);
      }
      if (!ok && lane == 0) failed();
    }
  } else if (warp < 20) {
    shares<ENDS, kRegX>();
    // ---- the state: lane = row of the pair's 2 x 64; its columns, and blocks of 32 tokens, in two halves
    const int q = warp & 3, half = (warp >> 2) & 1 ? 0 : 1, hh = q >> 1, pr = (q & 1) * 32 + lane, prow = q * 32 + lane, head = h0 + hh;
    const bool has = head < p.heads;
    const long long hp = 64LL * N;
    float* own = p.ssm + ((long long)slot * p.heads + head) * hp + (long long)pr * N;
    float* part = g.wk.state + (place * p.heads + head) * hp + (long long)pr * N;
    const float* from = g.seg > 0 && t.end - t.start > g.seg ? part : own;
    uint8_t* hrow = smem + K::oH + prow * 128;
    // the state that the segment starts from, while the first chunk's decays are made
#pragma unroll 1
    for (int j = half * (N / 32); j < (half + 1) * (N / 32); ++j) {
      uint32_t r[16];
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const float4 f = !ENDS && has ? *reinterpret_cast<const float4*>(from + j * 16 + i) : make_float4(0.f, 0.f, 0.f, 0.f);
        r[i] = __float_as_uint(f.x);
        r[i + 1] = __float_as_uint(f.y);
        r[i + 2] = __float_as_uint(f.z);
        r[i + 3] = __float_as_uint(f.w);
      }
      tc::tmem_st16(tmem + lanes + cH + j * 16, r);
    }
    tc::tmem_wait_st();
    bool ok = true;
    Turn vt(kVecs), xt(kXSlots, hh);
#pragma unroll 1
    for (int c = 0; c < chunks; ++c, vt.next(), xt.next(2)) {
      const int vs = vt.at, sl = xt.at;
      if (!(ok = wait(&vfull[vs], vt.phase) && (c == 0 || (wait(hdone, (c - 1) & 1) && (ENDS || wait(y2full, (c - 1) & 1)))))) break;
      tc::fence_after();
      const Vec& v = vec[vs * 2 + hh];
      const F2 total = f2(v.total, v.total);
#pragma unroll 1
      for (int j = half * (N / 32); j < (half + 1) * (N / 32); ++j) {
        uint32_t r[16];
        tc::tmem_ld16(tmem + lanes + cH + j * 16, r);
        tc::tmem_wait_ld();
        tc::landed(r);
        if (!ENDS) {
#pragma unroll
          for (int i = 0; i < 16; i += 8) {
            uint4 o;
            o.x = pack_bf16(__uint_as_float(r[i]), __uint_as_float(r[i + 1]));
            o.y = pack_bf16(__uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
            o.z = pack_bf16(__uint_as_float(r[i + 4]), __uint_as_float(r[i + 5]));
            o.w = pack_bf16(__uint_as_float(r[i + 6]), __uint_as_float(r[i + 7]));
            const int chunk = (j & 3) * 2 + i / 8;
            *reinterpret_cast<uint4*>(hrow + (j >> 2) * kTile + ((chunk ^ (prow & 7)) << 4)) = o;
          }
        }
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          float x, y;
          split(mul2(f2(r[i], r[i + 1]), total), x, y);
          r[i] = __float_as_uint(x);
          r[i + 1] = __float_as_uint(y);
        }
        tc::tmem_st16(tmem + lanes + cH + j * 16, r);
      }
      tc::tmem_wait_st();
      if (!ENDS) fence_proxy_async();
      tc::fence_before();
      arrive(hready);
      // exp(c[T] - c[s]) dt[s] x[s], split over three bf16 values, tokens along the columns
      if (!(ok = wait(&xfull[sl], xt.phase))) break;
      uint8_t* xs = smem + K::oX + sl * kTile + (pr & 7) * 2;
      const int valid = end - t.first - c * Q;
      if (valid < Q) {  // behind the sequence's end: zeros (the warp's 32 rows, four 16-byte vectors of a token, and its half's tokens)
#pragma unroll 1
        for (int i = lane; i < Q / 2 * 4; i += 32) {
          const int s = (i >> 7) * 64 + half * 32 + ((i >> 2) & 31), v16 = (q & 1) * 4 + (i & 3);
          if (s >= valid) *reinterpret_cast<uint4*>(smem + K::oX + sl * kTile + s * 128 + ((v16 ^ (s & 7)) << 4)) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async();
        __syncwarp();
      }
      F2 finite = f2(0.f, 0.f);
      const F2 zero = finite, minus = f2(-1.f, -1.f);
#pragma unroll 1
      for (int i4 = 0; i4 < 4; ++i4) {  // 16 tokens; 32 fill a buffer
        const int j = half * 2 + (i4 >> 1) * 4 + (i4 & 1);  // of the chunk's eight
        if (!(i4 & 1)) {
          if ((c > 0 || i4 > 0) && !(ok = wait(&xwempty[half], (i4 >> 1) ^ 1))) break;
          tc::fence_after();
        }
        uint32_t o[3][8];
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const int s = j * 16 + 2 * i;
          const float4 w = *reinterpret_cast<const float4*>(v.w + s);
          float x[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)  // s is a multiple of four: the swizzle of row s + k by constants alone
            x[k] = __uint_as_float(uint32_t(*reinterpret_cast<const uint16_t*>(xs + (s + k) * 128 + (((pr >> 3) ^ ((2 * i + k) & 7)) << 4))) << 16);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const F2 xx = f2(x[2 * k], x[2 * k + 1]);
            finite = fma2(xx, zero, finite);
            F2 f = mul2(xx, k ? f2(w.z, w.w) : f2(w.x, w.y));
            const uint32_t a = pack_bf16(f);
            f = fma2(f2(bf_lo(a), bf_hi(a)), minus, f);
            const uint32_t b = pack_bf16(f);
            f = fma2(f2(bf_lo(b), bf_hi(b)), minus, f);
            o[0][i + k] = a;
            o[1][i + k] = b;
            o[2][i + k] = pack_bf16(f);
          }
        }
#pragma unroll
        for (int k = 0; k < 3; ++k) tc::tmem_st8(tmem + lanes + cXW + half * 64 + k * 16 + (i4 & 1) * 8, o[k]);
        if (i4 & 1) {
          tc::tmem_wait_st();
          tc::fence_before();
          arrive(&xwfull[half]);
        }
      }
      if (!ok) break;
      if (!ENDS) {
        // A value of x that is not finite would reach earlier tokens' y through
        // the zeros of S: it leaves the tile, and y from its token on is NaN.
        int first = Q;
        float f0, f1;
        split(finite, f0, f1);
        if (f0 + f1 != 0.f) {
#pragma unroll 1
          for (int s = Q - 1; s >= 0; --s) {
            if (((s >> 5) & 1) != half) continue;
            uint16_t* e = reinterpret_cast<uint16_t*>(xs + s * 128 + (((pr >> 3) ^ (s & 7)) << 4));
            if ((*e & 0x7f80) == 0x7f80) {
              first = s;
              *e = 0;
            }
          }
          fence_proxy_async();
        }
        bad[(vs * 2 + half) * 128 + prow] = uint8_t(first);
        const bool any = __any_sync(0xffffffffu, first < Q);
        if (lane == 0) anybad[vs * 8 + half * 4 + q] = any;
        arrive(&xscan[vs]);
      }
      arrive(&xempty[sl]);
      arrive(&vempty[vs]);
    }
    if (ok) ok = wait(hdone, (chunks - 1) & 1);
    if (!ok && lane == 0) failed();
    if (ok && (ENDS || end == t.end)) {
      tc::fence_after();
      float* to = ENDS ? part : own;
#pragma unroll 1
      for (int j = half * (N / 32); j < (half + 1) * (N / 32); ++j) {
        uint32_t r[16];
        tc::tmem_ld16(tmem + lanes + cH + j * 16, r);
        tc::tmem_wait_ld();
        tc::landed(r);
        if (has) {
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<float4*>(to + j * 16 + i) =
                make_float4(__uint_as_float(r[i]), __uint_as_float(r[i + 1]), __uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
        }
      }
    }
  } else if (!ENDS) {
    shares<ENDS, kRegY>();
    // ---- y of one head: lane = token
    const int q = warp & 3, row = q * 32 + lane, h = (warp - 20) >> 2, head = h0 + h;
    const bool has = head < p.heads;
    const float d = has && p.d ? p.d[head] : 0.f;
    const F2 d2 = f2(d, d);
    const uint32_t ycol = tmem + lanes + cY + h * 64;
    bool ok = true;
    Turn vt(kVecs), xt(kXSlots, h);
#pragma unroll 1
    for (int c = 0; c < chunks; ++c, vt.next(), xt.next(2)) {
      const int vs = vt.at, sl = xt.at;
      const long long tok = t.first + c * Q + row;
      const bool in = has && t.first + c * Q + row < end;
      uint32_t z[32];
      if (p.z && in) {  // in flight while the products run
        const uint16_t* zp = reinterpret_cast<const uint16_t*>(p.z) + tok * p.ldz + head * 64;
#pragma unroll
        for (int i = 0; i < 32; i += 8)
          asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                       : "=r"(z[i]), "=r"(z[i + 1]), "=r"(z[i + 2]), "=r"(z[i + 3]), "=r"(z[i + 4]), "=r"(z[i + 5]),
                         "=r"(z[i + 6]), "=r"(z[i + 7])
                       : "l"(zp + 2 * i));
      }
      if (!(ok = wait(&vfull[vs], vt.phase) && wait(&xfull[sl], xt.phase) && wait(y2full, c & 1))) break;
      tc::fence_after();
      const Vec& v = vec[vs * 2 + h];
      const float f = ex2(v.base[q] - v.neg[row]);
      const F2 ff = f2(f, f);
      const uint8_t* xr = smem + K::oX + sl * kTile + row * 128;
#pragma unroll 1
      for (int j = 0; j < 4; ++j) {  // exp(c[t]) C H^T + d x
        uint32_t r[16];
        tc::tmem_ld16(ycol + j * 16, r);
        const uint4 x0 = *reinterpret_cast<const uint4*>(xr + (((j * 2) ^ (row & 7)) << 4));
        const uint4 x1 = *reinterpret_cast<const uint4*>(xr + (((j * 2 + 1) ^ (row & 7)) << 4));
        const uint32_t xw[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
        tc::tmem_wait_ld();
        tc::landed(r);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float x, y;
          split(fma2(f2(r[2 * i], r[2 * i + 1]), ff, mul2(d2, f2(bf_lo(xw[i]), bf_hi(xw[i])))), x, y);
          r[2 * i] = __float_as_uint(x);
          r[2 * i + 1] = __float_as_uint(y);
        }
        tc::tmem_st16(ycol + j * 16, r);
      }
      tc::tmem_wait_st();
      tc::fence_before();
      arrive(y2scaled);
      arrive(&xempty[sl]);
      int spoilt = 0;
#pragma unroll 1
      for (int j = 0; j < 4; ++j) {
        // The gate of 16 columns ahead of their sums: the first while the products
        // still run.
        F2 gate[8];
        if (p.z) {
#pragma unroll
          for (int k = 0; k < 8; ++k) gate[k] = silu2(f2(bf_lo(z[k]), bf_hi(z[k])));
#pragma unroll
          for (int i = 0; i < 24; ++i) z[i] = z[i + 8];
        }
        if (j == 0) {
          if (!(ok = wait(yfull, c & 1) && wait(&xscan[vs], vt.phase))) break;
          tc::fence_after();
          spoilt = anybad[vs * 8 + 2 * h] | anybad[vs * 8 + 2 * h + 1] | anybad[vs * 8 + 4 + 2 * h] | anybad[vs * 8 + 4 + 2 * h + 1];
        }
        uint32_t r[16];
        tc::tmem_ld16(ycol + j * 16, r);
        tc::tmem_wait_ld();
        tc::landed(r);
        if (j == 3) {
          tc::fence_before();
          arrive(yfree);
        }
        uint32_t o[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const F2 y = f2(r[2 * k], r[2 * k + 1]);
          o[k] = pack_bf16(p.z ? mul2(y, gate[k]) : y);
        }
        if (spoilt) {
#pragma unroll 1
          for (int i = 0; i < 16; ++i) {
            const int first = min(bad[vs * 256 + h * 64 + j * 16 + i], bad[vs * 256 + 128 + h * 64 + j * 16 + i]);
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (k == i / 2 && row >= first) o[k] |= i & 1 ? 0x7fff0000u : 0x7fffu;
          }
        }
        if (in)
          asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(reinterpret_cast<uint16_t*>(p.y) + tok * p.ldy +
                                                                                head * 64 + j * 16),
                       "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7])
                       : "memory");
      }
      if (!ok) break;
      arrive(&vempty[vs]);
    }
    if (!ok && lane == 0) failed();
  }
  // log of the segment's decay, for the join: pairs as in the chunks, with the library's
  // softplus, which this small part of the work can afford. Below e^-200 a decay is zero
  // in float32; the bound keeps infinite steps (and no NaN) out of the pairs.
  if (ENDS && warp >= 20 && warp < 22) {
    const int head = h0 + warp - 20;
    if (head < p.heads) {
      Pair s{0.f, 0.f};
      for (int i = t.first + lane; i < end; i += 32) {
        const float raw = p.dt[(long long)i * p.lddt + head], dt = p.softplus ? softplusf_(raw) : raw;
        float x = p.a[head] * dt;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(x) : "f"(x), "f"(-200.f));
        s = add(s, {x, 0.f});
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s = add(s, {__shfl_xor_sync(0xffffffffu, s.hi, o), __shfl_xor_sync(0xffffffffu, s.lo, o)});
      if (lane == 0) g.wk.log_decay[place * p.heads + head] = s.hi + s.lo;
    }
  }
  tc::fence_before();
  __syncthreads();
  if (warp == 1) tc::tmem_free(tmem, 512);
}

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

template <int NB, bool ENDS>
void launch(const ScanParams& p, const ScanWork& wk, int seg, cudaStream_t s) {
  using K = TcCfg<NB>;
  CUtensorMap mx, mb, mc;
  const uint64_t rows = uint64_t(p.plan.tokens);
  tc::make_map(&mx, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p.x, uint64_t(p.heads) * 64, rows, p.ldx, 64, Q);
  tc::make_map(&mb, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p.b, uint64_t(p.state), rows, p.ldb, 64, Q);
  tc::make_map(&mc, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p.c, uint64_t(p.state), rows, p.ldc, 64, Q);
  TcArgs g{p, wk, seg, (p.heads + 1) / 2};
  const long long tiles = seg > 0 ? seq_tiles(p.plan, seg) : p.plan.seqs;
  B2E_CHECK(tiles * g.pairs <= 0x7fffffffLL, kErrInvalid, "mamba2_scan: too many (segment, head) pairs");
  static std::atomic<unsigned long long> allowed{0};
  tc::allow_smem(k_scan_tc<NB, ENDS>, K::SMEM, allowed);
  k_scan_tc<NB, ENDS><<<unsigned(tiles * g.pairs), kTcThreads, K::SMEM, s>>>(mx, mb, mc, g);
  B2E_CUDA(cudaGetLastError());
}

template <int NB>
void run(const ScanParams& p, int seg, cudaStream_t s) {
  ScanWork wk{};
  if (seg > 0) {
    wk = scan_work(p, seg);
    launch<NB, true>(p, wk, seg, s);
    scan_join(p, wk, seg, s);
  }
  launch<NB, false>(p, wk, seg, s);
}

}  // namespace

// A chunk costs this kernel the same for 1 token as for 128, the recurrence kernel
// by the token. While all CTAs run at once the longest sequence decides: 4
// sequences, 8 heads, of 16, 24, 32 tokens take 14.5 us here, 12.1, 16.4, 20.1
// there. Beyond that the mean does: 256 sequences of 16, 20, 24 tokens take 99 us
// here, 84, 104, 115 there.
bool scan_tc_eligible(const ScanParams& p) {
  const bool long_enough = (long long)p.plan.seqs * ((p.heads + 1) / 2) <= 148 ? p.plan.longest >= 24 : p.plan.tokens >= 20LL * p.plan.seqs;
  return long_enough && p.type == kBF16 && p.size == 64 && (p.state == 64 || p.state == 128) && aligned(p.x, 16) &&
         aligned(p.b, 16) && aligned(p.c, 16) && aligned(p.y, 32) && p.ldx % 8 == 0 && p.ldb % 8 == 0 && p.ldc % 8 == 0 &&
         p.ldy % 16 == 0 && (!p.z || (aligned(p.z, 32) && p.ldz % 16 == 0));
}

void scan_tc(const ScanParams& p, int seg, cudaStream_t s) {
  if (p.state == 128)
    run<2>(p, seg, s);
  else
    run<1>(p, seg, s);
}

}  // namespace b2e
