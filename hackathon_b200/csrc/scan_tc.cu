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
// which is the recurrence written out over a chunk. Five products a chunk, all
// M = 128 in float32 TMEM accumulators: G, C H^T and the state's with N = 128
// columns (both heads at once, so the shared-memory operands are read at the
// rate the MMA can take), S X with its left operand in TMEM.
//
// Roundings: S and the copy of H that multiplies C are rounded once to bf16, as
// y itself is; together they move y by about as much as y's own rounding. The
// state must not drift: its operand exp() dt x is split exactly over three bf16
// values (24 bits), three products into the float32 state that stays in TMEM
// over the whole walk. Sums of a dt are carried as float32 pairs (hi, lo), so
// that differences of far sums keep their low bits after a token with a very
// large step; rows of S take one factor a row block times one a column where
// blocks of 32 tokens do not touch, and the exponential of the difference inside
// the diagonal blocks, so nothing overflows for decays below one.
//
// Sixteen warps: 0 TMA loads; 1 issues the MMAs; 2-3 the decays of one head each
// (and zeros behind a sequence's end); 4-7 S from G; 8-11 the state: its decay,
// its bf16 copy and the split operand; 12-15 y: exp(c) on C H^T, skip, gate and
// stores. The chain of a chunk is state ready -> C H^T -> scaled -> + S X -> y;
// the state's products, G of the next chunk and the elementwise work of the other
// warps run beside it.
//
// What bounds it: instruction issue (the elementwise work of 2 x 128 x 64 values
// of x, y, z and 2 x 128 x 128 pairs) and HBM are close; the tensor cores need
// 6 x 128 x 128 x 128 products a chunk and pair.
#include <algorithm>

#include "scan.cuh"
#include "tc.cuh"

namespace b2e {
namespace {

constexpr int Q = 128;                       // tokens of a chunk
constexpr uint32_t kTile = Q * 128;          // 128 rows of 128 bytes
constexpr int kXSlots = 3;
constexpr int kTcThreads = 512;
enum ScanError : int { kScanTimeout = 131 };

// TMEM columns (of 512): G, and S of the second head in its place; S of the
// first; two buffers of the state's operand; Y and H of both heads.
constexpr uint32_t cG = 0, cS1 = 0, cS0 = 128, cXW = 192, cY = 256, cH = 384;

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

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float bf_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

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
__device__ __forceinline__ Pair shfl_up(Pair a, int d) {
  return {__shfl_up_sync(0xffffffffu, a.hi, d), __shfl_up_sync(0xffffffffu, a.lo, d)};
}
__device__ __forceinline__ Pair shfl(Pair a, int src) {
  return {__shfl_sync(0xffffffffu, a.hi, src), __shfl_sync(0xffffffffu, a.lo, src)};
}

// Decays of one head and chunk, exponents in powers of two.
struct Vec {
  float4 tok[Q];    // c[s] (hi, lo), dt[s], exp(c[T] - c[s]) dt[s]
  float start[Q];   // exp(c[t])
  float row[Q];     // exp(c[t] - c[first token of its 32-block, exclusive])
  float col[192];   // exp(c[before block i] - c[s]) dt[s] for s before block i: 32 values for i = 1, 64, 96
  float total;      // exp(c[T])
  float pad[3];
};

template <int NB>
struct TcCfg {
  static constexpr uint32_t CB = NB * kTile;  // bytes of a chunk of C (or B)
  static constexpr uint32_t oC = 0, oB = CB, STAGE = 2 * CB;
  static constexpr uint32_t oX = 2 * STAGE, oH = oX + kXSlots * kTile, oV = oH + NB * kTile;
  static constexpr uint32_t oBad = oV + 4 * sizeof(Vec);            // [2][128] first token that is not finite, [2][4] flags
  static constexpr uint32_t oBar = oBad + 2 * 128 * 4 + 2 * 4 * 4;
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
    t.seq = tile;
    t.start = t.first = p.plan.starts[tile];
    t.end = p.plan.starts[tile + 1];
    t.live = t.start >= 0 && t.end <= p.plan.tokens && t.start < t.end;
  }
  if (!t.live) return;
  const int slot = p.plan.slots ? p.plan.slots[t.seq] : t.seq;
  if (slot < 0 || slot >= p.plan.state_rows) {
    if (threadIdx.x == 0 && p.err) *p.err = 1;
    return;
  }
  const int end = g.seg > 0 ? min(t.end, t.first + g.seg) : t.end;
  if (ENDS && end == t.end) return;
  const int chunks = (end - t.first + Q - 1) / Q;

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sbase = smem_u32(smem);
  Vec* vec = reinterpret_cast<Vec*>(smem + K::oV);  // [chunk parity][head]
  int* bad = reinterpret_cast<int*>(smem + K::oBad);
  int* anybad = bad + 2 * 128;
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + K::oBar);
  uint64_t *cbfull = bar, *cbempty = bar + 2, *xfull = bar + 4, *xempty = bar + 7, *vfull = bar + 10, *vempty = bar + 12,
           *gfull = bar + 14, *sfull = bar + 15, *y2full = bar + 17, *y2scaled = bar + 18, *yfull = bar + 19, *yfree = bar + 20,
           *hready = bar + 21, *hdone = bar + 22, *xwfull = bar + 23, *xwempty = bar + 25, *xscan = bar + 27, *done = bar + 29;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + 30);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&cbfull[i], 1);
      mbar_init(&cbempty[i], 1);
      mbar_init(&vfull[i], 2);
      mbar_init(&vempty[i], ENDS ? 4 : 12);
      mbar_init(&sfull[i], 4);
      mbar_init(&xwfull[i], 4);
      mbar_init(&xwempty[i], 1);
      mbar_init(&xscan[i], 4);
    }
    for (int i = 0; i < kXSlots; ++i) {
      mbar_init(&xfull[i], 1);
      mbar_init(&xempty[i], ENDS ? 2 : 7);  // two warps of the state's, S X, four warps of y's
    }
    mbar_init(gfull, 1);
    mbar_init(y2full, 1);
    mbar_init(y2scaled, 4);
    mbar_init(yfull, 1);
    mbar_init(yfree, 4);
    mbar_init(hready, 4);
    mbar_init(hdone, 1);
    mbar_init(done, 1);
    *abort_flag = 0;
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

  // Every thread of a warp waits; false (for all of them) once a wait anywhere ran out.
  auto wait = [&](uint64_t* b, uint32_t parity) -> bool {
    const bool ok = mbar_wait(b, parity, abort_flag);
    if (__all_sync(0xffffffffu, ok)) return true;
    if (lane == 0) {
      if (!*abort_flag) atomicExch(p.err, kScanTimeout);
      *abort_flag = 1;
    }
    return false;
  };
  auto arrive = [&](uint64_t* b) {
    __syncwarp();
    if (lane == 0) mbar_arrive(b);
  };

  if (warp == 0) {
    // ---- loads
    if (lane == 0) {
      int c = 0, u = 0;
      auto wait1 = [&](uint64_t* b, uint32_t parity) {
        if (mbar_wait(b, parity, abort_flag)) return true;
        if (!*abort_flag) atomicExch(p.err, kScanTimeout);
        *abort_flag = 1;
        return false;
      };
      for (; c < chunks; ++c) {
        const int st = c & 1, row = t.first + c * Q;
        if (c >= 2 && !wait1(&cbempty[st], ((c >> 1) & 1) ^ 1)) break;
        uint8_t* s = smem + st * K::STAGE;
        mbar_expect_tx(&cbfull[st], (ENDS ? 1 : 2) * K::CB);
        for (int i = 0; i < NB; ++i) {
          tc::tma_load_2d(s + K::oB + i * kTile, &mb, i * 64, row, &cbfull[st]);
          if (!ENDS) tc::tma_load_2d(s + K::oC + i * kTile, &mc, i * 64, row, &cbfull[st]);
        }
        for (int h = 0; h < 2; ++h) {
          const int sl = u % kXSlots;
          if (u >= kXSlots && !wait1(&xempty[sl], ((u / kXSlots) & 1) ^ 1)) break;
          mbar_expect_tx(&xfull[sl], kTile);
          tc::tma_load_2d(smem + K::oX + sl * kTile, &mx, (h0 + h) * 64, row, &xfull[sl]);
          ++u;
        }
        if (*abort_flag) {
          ++c;
          break;
        }
      }
      if (*abort_flag) {  // every load issued lands before the CTA leaves (bounded)
        volatile int never = 0;
        for (int i = max(0, c - 2); i < c; ++i) mbar_wait(&cbfull[i & 1], (i >> 1) & 1, &never);
        for (int i = max(0, u - kXSlots); i < u; ++i) mbar_wait(&xfull[i % kXSlots], (i / kXSlots) & 1, &never);
      }
    }
  } else if (warp == 1) {
    // ---- MMAs
    if (lane == 0) {
      auto wait1 = [&](uint64_t* b, uint32_t parity) {
        if (mbar_wait(b, parity, abort_flag)) return true;
        if (!*abort_flag) atomicExch(p.err, kScanTimeout);
        *abort_flag = 1;
        return false;
      };
      auto scores = [&](int c) {  // G = C B^T
        const int st = c & 1;
        if (!wait1(&vfull[st], (c >> 1) & 1) || !wait1(&cbfull[st], (c >> 1) & 1)) return false;
        tc::fence_after();
        const uint32_t a = sbase + st * K::STAGE + K::oC, b = sbase + st * K::STAGE + K::oB;
#pragma unroll
        for (int k = 0; k < N / 16; ++k) {
          const uint32_t off = (k / 4) * kTile + (k % 4) * 32;
          mma_ss(tmem + cG, tc::desc_k(a + off), tc::desc_k(b + off), idesc_bf16(Q, false), k != 0);
        }
        tc::commit(gfull);
        return true;
      };
      bool ok = ENDS || scores(0);
      for (int c = 0; c < chunks && ok; ++c) {
        const int st = c & 1;
        const uint32_t sC = sbase + st * K::STAGE + K::oC, sB = sbase + st * K::STAGE + K::oB;
        if (!wait1(hready, c & 1) || !wait1(&cbfull[st], (c >> 1) & 1)) break;
        if (!ENDS) {
          if (c > 0 && !wait1(yfree, (c - 1) & 1)) break;
          tc::fence_after();
#pragma unroll
          for (int k = 0; k < N / 16; ++k) {  // Y = C H^T
            const uint32_t off = (k / 4) * kTile + (k % 4) * 32;
            mma_ss(tmem + cY, tc::desc_k(sC + off), tc::desc_k(sbase + K::oH + off), idesc_bf16(Q, false), k != 0);
          }
          tc::commit(y2full);
        }
        for (int j = 0; j < 6; ++j) {  // H += (split operand, half j / 3 of the tokens)^T B
          const int n = 3 * c + (j >> 1);
          if (!(ok = wait1(&xwfull[j & 1], n & 1))) break;
          tc::fence_after();
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_ts(tmem + cH, tmem + cXW + (j & 1) * 32 + k * 8, desc_mn(sB + (j / 3) * 64 * 128 + k * 16 * 128, kTile),
                   idesc_bf16(N, true), 1);
          tc::commit(&xwempty[j & 1]);
        }
        if (!ok) break;
        tc::commit(hdone);
        if (ENDS) {
          tc::commit(&cbempty[st]);
          continue;
        }
        if (!(ok = wait1(y2scaled, c & 1) && wait1(&xscan[st], (c >> 1) & 1))) break;
        for (int h = 0; h < 2 && ok; ++h) {  // Y += S X
          const int u = 2 * c + h, sl = u % kXSlots;
          if (!(ok = wait1(&sfull[h], c & 1) && wait1(&xfull[sl], (u / kXSlots) & 1))) break;
          tc::fence_after();
#pragma unroll
          for (int k = 0; k < 8; ++k)
            mma_ts(tmem + cY + h * 64, tmem + (h ? cS1 : cS0) + k * 8, desc_mn(sbase + K::oX + sl * kTile + k * 16 * 128, kTile),
                   idesc_bf16(64, true), 1);
          tc::commit(&xempty[sl]);
        }
        if (!ok) break;
        tc::commit(yfull);
        tc::commit(&cbempty[st]);
        if (c + 1 < chunks) ok = scores(c + 1);
      }
      tc::commit(done);  // the CTA leaves (and frees its TMEM) after the last MMA
      volatile int never = 0;
      mbar_wait(done, 0, &never);
    }
  } else if (warp < 4) {
    // ---- decays of head h0 + hh
    const int hh = warp - 2, head = h0 + hh;
    const bool has = head < p.heads;
    const float a2 = has ? p.a[head] * 1.4426950408889634f : 0.f;
    float raw[4];
    auto fetch = [&](int c) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = c * Q + 4 * lane + k;
        raw[k] = has && t.first + i < end ? p.dt[(long long)(t.first + i) * p.lddt + head] : 0.f;
      }
    };
    fetch(0);
    for (int c = 0; c < chunks; ++c) {
      const int st = c & 1, valid = min(Q, end - t.first - c * Q);
      float dt[4];
      Pair cum[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool in = has && 4 * lane + k < valid;
        dt[k] = in ? (p.softplus ? softplusf_(raw[k]) : raw[k]) : 0.f;
        const Pair v{in ? a2 * dt[k] : 0.f, 0.f};
        cum[k] = k ? add(cum[k - 1], v) : v;
      }
      if (c + 1 < chunks) fetch(c + 1);
      Pair sum = cum[3];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const Pair v = shfl_up(sum, o);
        if (lane >= o) sum = add(v, sum);
      }
      Pair before = shfl_up(sum, 1);
      if (lane == 0) before = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 4; ++k) cum[k] = add(before, cum[k]);
      const Pair total = shfl(sum, 31), b1 = shfl(sum, 7), b2 = shfl(sum, 15), b3 = shfl(sum, 23);
      const int blk = lane >> 3;
      const Pair base = blk == 0 ? Pair{0.f, 0.f} : blk == 1 ? b1 : blk == 2 ? b2 : b3;
      if (c >= 2 && !wait(&vempty[st], ((c >> 1) & 1) ^ 1)) break;
      Vec& v = vec[st * 2 + hh];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int s = 4 * lane + k;
        v.tok[s] = make_float4(cum[k].hi, cum[k].lo, dt[k], ex2(diff(total, cum[k])) * dt[k]);
        v.start[s] = ex2(cum[k].hi + cum[k].lo);
        v.row[s] = ex2(diff(cum[k], base));
        if (blk < 1) v.col[s] = ex2(diff(b1, cum[k])) * dt[k];
        if (blk < 2) v.col[32 + s] = ex2(diff(b2, cum[k])) * dt[k];
        if (blk < 3) v.col[96 + s] = ex2(diff(b3, cum[k])) * dt[k];
      }
      if (lane == 0) v.total = ex2(total.hi + total.lo);
      if (valid < Q) {
        // Behind the sequence's end lie other sequences' rows: zeros, so that
        // nothing of them meets a product.
        const int u = 2 * c + hh, sl = u % kXSlots;
        if (!wait(&cbfull[st], (c >> 1) & 1) || !wait(&xfull[sl], (u / kXSlots) & 1)) break;
        uint4* xr = reinterpret_cast<uint4*>(smem + K::oX + sl * kTile);
        for (int i = valid * 8 + lane; i < Q * 8; i += 32) xr[i] = make_uint4(0, 0, 0, 0);
        if (hh < NB) {
          uint4* br = reinterpret_cast<uint4*>(smem + st * K::STAGE + K::oB + hh * kTile);
          for (int i = valid * 8 + lane; i < Q * 8; i += 32) br[i] = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async();
      }
      arrive(&vfull[st]);
    }
  } else if (warp < 8) {
    // ---- S from G
    if (!ENDS) {
      const int q = warp & 3, row = q * 32 + lane;
      for (int c = 0; c < chunks; ++c) {
        const int st = c & 1;
        if (!wait(&vfull[st], (c >> 1) & 1) || !wait(gfull, c & 1)) break;
        tc::fence_after();
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          const Vec& v = vec[st * 2 + h];
          const float rowf = v.row[row];
          const float4 me = v.tok[row];
          const float* col = v.col + (q == 1 ? 0 : q == 2 ? 32 : 96);
          const uint32_t dst = tmem + lanes + (h ? cS1 : cS0);
#pragma unroll 1
          for (int j = 0; j < 4; ++j) {
            uint32_t o[16];
            if (j <= q) {
              uint32_t r[32];
              tc::tmem_ld32(tmem + lanes + cG + j * 32, r);
              tc::tmem_wait_ld();
              tc::landed(r);
              if (j < q) {
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                  const float4 f = *reinterpret_cast<const float4*>(col + j * 32 + i);
                  o[i / 2] = pack_bf16(__uint_as_float(r[i]) * (f.x * rowf), __uint_as_float(r[i + 1]) * (f.y * rowf));
                  o[i / 2 + 1] = pack_bf16(__uint_as_float(r[i + 2]) * (f.z * rowf), __uint_as_float(r[i + 3]) * (f.w * rowf));
                }
              } else {
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                  float e[2];
#pragma unroll
                  for (int k = 0; k < 2; ++k) {
                    const float4 s = v.tok[j * 32 + i + k];
                    const float w = ex2((me.x - s.x) + (me.y - s.y)) * s.z;
                    e[k] = i + k <= lane ? __uint_as_float(r[i + k]) * w : 0.f;
                  }
                  o[i / 2] = pack_bf16(e[0], e[1]);
                }
              }
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = 0;
            }
            tc::tmem_st16(dst + j * 16, o);
          }
          tc::tmem_wait_st();
          tc::fence_before();
          arrive(&sfull[h]);
        }
        arrive(&vempty[st]);
      }
    }
  } else if (warp < 12) {
    // ---- the state: lane = row of the pair's 2 x 64
    const int q = warp & 3, hh = q >> 1, pr = (q & 1) * 32 + lane, prow = q * 32 + lane, head = h0 + hh;
    const bool has = head < p.heads;
    const long long hp = 64LL * N;
    float* own = p.ssm + ((long long)slot * p.heads + head) * hp + (long long)pr * N;
    float* part = g.wk.state + ((long long)tile * p.heads + head) * hp + (long long)pr * N;
    const float* from = g.seg > 0 ? part : own;
    uint8_t* hrow = smem + K::oH + prow * 128;
    bool ok = true;
    for (int c = 0; c < chunks; ++c) {
      const int st = c & 1, u = 2 * c + hh, sl = u % kXSlots;
      if (!(ok = wait(&vfull[st], (c >> 1) & 1))) break;
      if (c > 0 && !(ok = wait(hdone, (c - 1) & 1))) break;
      if (c > 0 && !ENDS && !(ok = wait(y2full, (c - 1) & 1))) break;
      tc::fence_after();
      const Vec& v = vec[st * 2 + hh];
      const float total = v.total;
#pragma unroll 1
      for (int j = 0; j < N / 32; ++j) {
        uint32_t r[32];
        if (c > 0) {
          tc::tmem_ld32(tmem + lanes + cH + j * 32, r);
          tc::tmem_wait_ld();
          tc::landed(r);
        } else {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 f = !ENDS && has ? *reinterpret_cast<const float4*>(from + j * 32 + i) : make_float4(0.f, 0.f, 0.f, 0.f);
            r[i] = __float_as_uint(f.x);
            r[i + 1] = __float_as_uint(f.y);
            r[i + 2] = __float_as_uint(f.z);
            r[i + 3] = __float_as_uint(f.w);
          }
        }
        if (!ENDS) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint4 o;
            o.x = pack_bf16(__uint_as_float(r[i]), __uint_as_float(r[i + 1]));
            o.y = pack_bf16(__uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
            o.z = pack_bf16(__uint_as_float(r[i + 4]), __uint_as_float(r[i + 5]));
            o.w = pack_bf16(__uint_as_float(r[i + 6]), __uint_as_float(r[i + 7]));
            const int chunk = (j & 1) * 4 + i / 8;
            *reinterpret_cast<uint4*>(hrow + (j >> 1) * kTile + ((chunk ^ (prow & 7)) << 4)) = o;
          }
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * total);
        tc::tmem_st32(tmem + lanes + cH + j * 32, r);
      }
      tc::tmem_wait_st();
      if (!ENDS) fence_proxy_async();
      tc::fence_before();
      arrive(hready);
      // exp(c[T] - c[s]) dt[s] x[s], split over three bf16 values, tokens along the columns
      if (!(ok = wait(&xfull[sl], (u / kXSlots) & 1))) break;
      const uint8_t* xs = smem + K::oX + sl * kTile + (pr & 7) * 2;
      float finite = 0.f;
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        uint32_t o[3][32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const int s = half * 64 + 2 * i;
          const float x0 = __uint_as_float(uint32_t(*reinterpret_cast<const uint16_t*>(xs + s * 128 + (((pr >> 3) ^ (s & 7)) << 4))) << 16);
          const float x1 =
              __uint_as_float(uint32_t(*reinterpret_cast<const uint16_t*>(xs + (s + 1) * 128 + (((pr >> 3) ^ ((s + 1) & 7)) << 4))) << 16);
          finite = fmaf(x0, 0.f, finite);
          finite = fmaf(x1, 0.f, finite);
          float f0 = x0 * v.tok[s].w, f1 = x1 * v.tok[s + 1].w;
          o[0][i] = pack_bf16(f0, f1);
          f0 -= bf_lo(o[0][i]);
          f1 -= bf_hi(o[0][i]);
          o[1][i] = pack_bf16(f0, f1);
          f0 -= bf_lo(o[1][i]);
          f1 -= bf_hi(o[1][i]);
          o[2][i] = pack_bf16(f0, f1);
        }
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          const int j = 3 * half + k, n = 3 * c + (j >> 1);  // n: uses of buffer j & 1 before this one
          if (n > 0 && !(ok = wait(&xwempty[j & 1], (n - 1) & 1))) break;
          tc::fence_after();
          tc::tmem_st32(tmem + lanes + cXW + (j & 1) * 32, o[k]);
          tc::tmem_wait_st();
          tc::fence_before();
          arrive(&xwfull[j & 1]);
        }
        if (!ok) break;
      }
      if (!ok) break;
      if (!ENDS) {
        // A value of x that is not finite would reach earlier tokens' y through
        // the zeros of S: it leaves the tile, and y from its token on is NaN.
        int first = Q;
        if (finite != 0.f) {
          for (int s = Q - 1; s >= 0; --s) {
            uint16_t* e = reinterpret_cast<uint16_t*>(const_cast<uint8_t*>(xs) + s * 128 + (((pr >> 3) ^ (s & 7)) << 4));
            if ((*e & 0x7f80) == 0x7f80) {
              first = s;
              *e = 0;
            }
          }
          fence_proxy_async();
        }
        bad[st * 128 + prow] = first;
        const bool any = __any_sync(0xffffffffu, first < Q);
        if (lane == 0) anybad[st * 4 + q] = any;
        arrive(&xscan[st]);
      }
      arrive(&xempty[sl]);
      arrive(&vempty[st]);
    }
    if (ok && wait(hdone, (chunks - 1) & 1) && (ENDS || end == t.end)) {
      tc::fence_after();
      float* to = ENDS ? part : own;
#pragma unroll 1
      for (int j = 0; j < N / 32; ++j) {
        uint32_t r[32];
        tc::tmem_ld32(tmem + lanes + cH + j * 32, r);
        tc::tmem_wait_ld();
        tc::landed(r);
        if (has) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4*>(to + j * 32 + i) =
                make_float4(__uint_as_float(r[i]), __uint_as_float(r[i + 1]), __uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
        }
      }
    }
  } else if (!ENDS) {
    // ---- y: lane = token
    const int q = warp & 3, row = q * 32 + lane;
    for (int c = 0; c < chunks; ++c) {
      const int st = c & 1, valid = min(Q, end - t.first - c * Q);
      const long long tok = t.first + c * Q + row;
      if (!wait(&vfull[st], (c >> 1) & 1) || !wait(y2full, c & 1)) break;
      tc::fence_after();
#pragma unroll 1
      for (int j = 0; j < 4; ++j) {
        const float f = vec[st * 2 + (j >> 1)].start[row];
        uint32_t r[32];
        tc::tmem_ld32(tmem + lanes + cY + j * 32, r);
        tc::tmem_wait_ld();
        tc::landed(r);
#pragma unroll
        for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * f);
        tc::tmem_st32(tmem + lanes + cY + j * 32, r);
      }
      tc::tmem_wait_st();
      tc::fence_before();
      arrive(y2scaled);
      bool ok = true;
#pragma unroll 1
      for (int j = 0; j < 4; ++j) {  // 32 columns: half j & 1 of head j >> 1
        const int h = j >> 1, head = h0 + h, u = 2 * c + h, sl = u % kXSlots;
        const bool in = row < valid && head < p.heads;
        uint4 z[4];
        if (p.z && in) {  // in flight while the products finish
          const uint4* zp = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.z) + tok * p.ldz + head * 64 + (j & 1) * 32);
#pragma unroll
          for (int i = 0; i < 4; ++i) z[i] = __ldcs(zp + i);
        }
        if (j == 0 && !(ok = wait(yfull, c & 1) && wait(&xscan[st], (c >> 1) & 1))) break;
        if (!(j & 1) && !(ok = wait(&xfull[sl], (u / kXSlots) & 1))) break;
        tc::fence_after();
        uint32_t r[32];
        tc::tmem_ld32(tmem + lanes + cY + j * 32, r);
        tc::tmem_wait_ld();
        tc::landed(r);
        if (j == 3) {
          tc::fence_before();
          arrive(yfree);
        }
        if (p.d && head < p.heads) {
          const float d = p.d[head];
          const uint8_t* xr = smem + K::oX + sl * kTile + row * 128;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint4 x = *reinterpret_cast<const uint4*>(xr + ((((j & 1) * 4 + i) ^ (row & 7)) << 4));
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              r[i * 8 + k * 2] = __float_as_uint(fmaf(d, bf_lo(w[k]), __uint_as_float(r[i * 8 + k * 2])));
              r[i * 8 + k * 2 + 1] = __float_as_uint(fmaf(d, bf_hi(w[k]), __uint_as_float(r[i * 8 + k * 2 + 1])));
            }
          }
        }
        if (j & 1) arrive(&xempty[sl]);
        if (p.z && in) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t w[4] = {z[i].x, z[i].y, z[i].z, z[i].w};
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float zz = k & 1 ? bf_hi(w[k / 2]) : bf_lo(w[k / 2]);
              r[i * 8 + k] = __float_as_uint(__uint_as_float(r[i * 8 + k]) * __fdividef(zz, 1.0f + __expf(-zz)));
            }
          }
        }
        if (anybad[st * 4 + 2 * h] | anybad[st * 4 + 2 * h + 1]) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (row >= bad[st * 128 + j * 32 + i]) r[i] = 0x7fc00000u;
        }
        if (in) {
          uint16_t* yp = reinterpret_cast<uint16_t*>(p.y) + tok * p.ldy + head * 64 + (j & 1) * 32;
#pragma unroll
          for (int i = 0; i < 32; i += 16) {
            uint32_t o[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) o[k] = pack_bf16(__uint_as_float(r[i + 2 * k]), __uint_as_float(r[i + 2 * k + 1]));
            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(yp + i), "r"(o[0]), "r"(o[1]), "r"(o[2]),
                         "r"(o[3]), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7])
                         : "memory");
          }
        }
      }
      if (!ok) break;
      arrive(&vempty[st]);
    }
  }
  // log of the segment's decay, for the join: the same float32 sums, segment-wide
  if (ENDS && warp >= 2 && warp < 4) {
    const int head = h0 + warp - 2;
    if (head < p.heads) {
      Pair s{0.f, 0.f};
      for (int i = t.first + lane; i < end; i += 32) {
        const float raw = p.dt[(long long)i * p.lddt + head], dt = p.softplus ? softplusf_(raw) : raw;
        s = add(s, {p.a[head] * dt, 0.f});
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s = add(s, {__shfl_xor_sync(0xffffffffu, s.hi, o), __shfl_xor_sync(0xffffffffu, s.lo, o)});
      if (lane == 0) g.wk.log_decay[(long long)tile * p.heads + head] = s.hi + s.lo;
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
  B2E_CUDA(cudaFuncSetAttribute(k_scan_tc<NB, ENDS>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(K::SMEM)));
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

bool scan_tc_eligible(const ScanParams& p) {
  return p.type == kBF16 && p.size == 64 && (p.state == 64 || p.state == 128) && p.plan.longest >= 32 && aligned(p.x, 16) &&
         aligned(p.b, 16) && aligned(p.c, 16) && aligned(p.y, 32) && p.ldx % 8 == 0 && p.ldb % 8 == 0 && p.ldc % 8 == 0 &&
         p.ldy % 16 == 0 && (!p.z || (aligned(p.z, 16) && p.ldz % 8 == 0));
}

void scan_tc(const ScanParams& p, int seg, cudaStream_t s) {
  if (p.state == 128)
    run<2>(p, seg, s);
  else
    run<1>(p, seg, s);
}

}  // namespace b2e
