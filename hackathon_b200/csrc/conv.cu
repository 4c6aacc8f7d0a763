// Depthwise causal convolution over packed sequences with a window of the last
// taps - 1 inputs a state row (CausalConv1d, model/modules.py:37-41, applied to
// every token of a sequence instead of one).
//
//   v = window[slot] ++ x[sequence];  y[t] = act(bias + sum_j w[j] v[t + j]);  window[slot] <- last taps - 1 of v
//
// Bound by HBM: each x and y once, a window once each way. A warp takes 32
// vectors of channels (16 bytes of x a lane) over a tile of tokens and keeps the
// last taps - 1 inputs in registers, so a token is read once and a tile reads
// only taps - 1 inputs of its neighbour's again; the next few tokens are in flight
// while one batch is computed, channels in packed pairs. The tile that starts a
// sequence is the only one that reads the window, and it writes it too: no other
// tile can see the new one.
//
// 10000 x 4352 with SiLU: float32 60 us (5.9 TB/s), bf16 45 us (3.9 TB/s; 4.8 on
// four times the tokens), where half the bytes meet the same arithmetic: 39 us
// without SiLU. Sixteen tokens in flight in shared memory instead of four in
// registers changed nothing (46 to 48 us); tiles of 24 or 64 tokens were slower.
// Single tokens, 4096 x 768 float32, 101 MB: 17.2 us with part of the windows in L2,
// 21 to 25 out of a cold cache (4.0 to 4.8 TB/s). Bound by latency and sectors rather
// than HBM (a warp waits 7.4 cycles an instruction for memory, DRAM is at a third): a
// lane's windows start 48 bytes from its neighbour's, so that an access touches
// sectors that two others touch again.
#include <algorithm>

#include "packed.cuh"
#include "seqops.cuh"

namespace b2e {
namespace {

constexpr int kConvWarps = 4;

// VC channels of a token as they lie in memory, two values a register in 16 bits.
template <int T, int VC>
struct Raw {
  static constexpr int N = T == kF32 || VC == 1 ? VC : VC / 2;
  uint32_t u[N];
  __device__ __forceinline__ void load(const void* p) {
    if constexpr (VC == 1 && T != kF32) {
      u[0] = __ldg(reinterpret_cast<const uint16_t*>(p));
    } else if constexpr (N == 4) {
      const uint4 r = __ldg(reinterpret_cast<const uint4*>(p));
      u[0] = r.x; u[1] = r.y; u[2] = r.z; u[3] = r.w;
    } else if constexpr (N == 2) {
      const uint2 r = __ldg(reinterpret_cast<const uint2*>(p));
      u[0] = r.x; u[1] = r.y;
    } else {
      u[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    }
  }
  __device__ __forceinline__ F2 pair(int i) const {
    if constexpr (T == kF32) {
      return f2(u[VC == 1 ? 0 : 2 * i], u[VC == 1 ? 0 : 2 * i + 1]);
    } else if constexpr (T == kBF16) {
      return f2(bf_lo(u[i]), bf_hi(u[i]));
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      return f2(f.x, f.y);
    }
  }
};

template <int T, int VC>
__device__ __forceinline__ void store_pairs(void* p, const F2* y) {
  float v[VC == 1 ? 2 : VC];
#pragma unroll
  for (int i = 0; i < (VC == 1 ? 1 : VC / 2); ++i) split(y[i], v[2 * i], v[2 * i + 1]);
  if constexpr (VC == 1) {
    LowP<T>::store(p, 0, v[0]);
  } else if constexpr (T == kF32) {
    __stcs(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
  } else {
    uint32_t u[VC / 2];
#pragma unroll
    for (int j = 0; j < VC / 2; ++j) {
      if constexpr (T == kBF16) {
        u[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
      } else {
        const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
        u[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    if constexpr (VC == 8)
      __stcs(reinterpret_cast<uint4*>(p), make_uint4(u[0], u[1], u[2], u[3]));
    else
      __stcs(reinterpret_cast<uint2*>(p), make_uint2(u[0], u[1]));
  }
}

// VC * N contiguous floats, 16-byte aligned when VC > 1.
template <int VC, int N>
__device__ __forceinline__ void load_rows(const float* p, float (&v)[VC][N]) {
  if constexpr (VC > 1) {
    float flat[VC * N];
#pragma unroll
    for (int i = 0; i < VC * N / 4; ++i) {
      const float4 a = reinterpret_cast<const float4*>(p)[i];
      flat[4 * i] = a.x; flat[4 * i + 1] = a.y; flat[4 * i + 2] = a.z; flat[4 * i + 3] = a.w;
    }
#pragma unroll
    for (int i = 0; i < VC * N; ++i) v[i / N][i % N] = flat[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[0][i] = p[i];
  }
}
template <int VC, int N>
__device__ __forceinline__ void store_rows(float* p, const float (&v)[VC][N]) {
  if constexpr (VC > 1) {
#pragma unroll
    for (int i = 0; i < VC * N / 4; ++i)
      reinterpret_cast<float4*>(p)[i] =
          make_float4(v[4 * i / N][4 * i % N], v[(4 * i + 1) / N][(4 * i + 1) % N], v[(4 * i + 2) / N][(4 * i + 2) % N],
                      v[(4 * i + 3) / N][(4 * i + 3) % N]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = v[0][i];
  }
}

// Column j of a window (or of the weights) in pairs of channels.
template <int VC, int N>
__device__ __forceinline__ F2 pair_of(const float (&v)[VC][N], int i, int j) {
  return VC == 1 ? f2(v[0][j], v[0][j]) : f2(v[2 * i % VC][j], v[(2 * i + 1) % VC][j]);
}

template <int VC, int TAPS>
struct Weights {
  static constexpr int P = VC == 1 ? 1 : VC / 2, W = TAPS - 1;
  F2 w[TAPS][P], bias[P];
  __device__ __forceinline__ Weights(const float* weight, const float* b) {
    float v[VC][TAPS];
    load_rows<VC, TAPS>(weight, v);
#pragma unroll
    for (int i = 0; i < P; ++i) {
#pragma unroll
      for (int j = 0; j < TAPS; ++j) w[j][i] = pair_of(v, i, j);
      bias[i] = b ? f2(b[VC == 1 ? 0 : 2 * i], b[VC == 1 ? 0 : 2 * i + 1]) : f2(0.f, 0.f);
    }
  }
  // One token: `last` are the inputs before it, which move on by one.
  template <int T>
  __device__ __forceinline__ void token(F2 (&last)[W][P], const Raw<T, VC>& raw, int silu, F2 (&y)[P]) const {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const F2 in = raw.pair(i);
      y[i] = bias[i];
#pragma unroll
      for (int j = 0; j < W; ++j) y[i] = fma2(w[j][i], last[j][i], y[i]);
      y[i] = fma2(w[W][i], in, y[i]);
      if (silu) y[i] = silu2(y[i]);
#pragma unroll
      for (int j = 0; j + 1 < W; ++j) last[j][i] = last[j + 1][i];
      last[W - 1][i] = in;
    }
  }
};

template <int T, int VC, int TAPS>
__global__ void __launch_bounds__(32 * kConvWarps) k_conv(const ConvParams p, int len, int vblocks, long long warps) {
  constexpr int W = TAPS - 1, P = VC == 1 ? 1 : VC / 2, U = VC == 8 ? 4 : 8;  // U tokens in flight
  constexpr int ESZ = T == kF32 ? 4 : 2;
  const long long gw = (long long)blockIdx.x * kConvWarps + (threadIdx.x >> 5);
  if (gw >= warps) return;
  const int tile = int(gw / vblocks), lane = threadIdx.x & 31;
  const int c = (int(gw % vblocks) * 32 + lane) * VC;
  const SeqTile t = seq_tile(p.plan, tile, len);
  if (lane == 31 && gw % vblocks == 0) seq_report(p.plan, tile, false, p.err);
  if (!t.live || c >= p.channels) return;
  const int slot = p.plan.slots ? p.plan.slots[t.seq] : t.seq;
  if (slot < 0 || slot >= p.plan.state_rows) {
    *p.err = 1;
    return;
  }
  const int end = min(t.end, t.first + len);
  const bool head = t.first == t.start;
  const long long xs = p.ldx * ESZ, ys = p.ldy * ESZ;
  const char* xp = reinterpret_cast<const char*>(p.x) + t.first * xs + (long long)c * ESZ;
  char* yp = reinterpret_cast<char*>(p.y) + t.first * ys + (long long)c * ESZ;
  int left = end - t.first;
  Raw<T, VC> raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (u < left) raw[u].load(xp + u * xs);
  const Weights<VC, TAPS> k(p.w + (long long)c * TAPS, p.bias ? p.bias + c : nullptr);
  float* win = p.window + ((long long)slot * p.channels + c) * W;
  F2 last[W][P];  // last[j]: input of token first - W + j
  if (head) {
    float old[VC][W], neu[VC][W];
    load_rows<VC, W>(win, old);
#pragma unroll
    for (int j = 0; j < W; ++j)
#pragma unroll
      for (int i = 0; i < P; ++i) last[j][i] = pair_of(old, i, j);
    const int n = t.end - t.start;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const int at = n - W + j;  // token of the sequence, or at + W of the old window
      Raw<T, VC> in;
      if (at >= 0) in.load(xp + at * xs);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        float a = 0.f, b = 0.f;
        if (at >= 0) {
          split(in.pair(i), a, b);
        } else {
#pragma unroll
          for (int o = 0; o < W; ++o)
            if (o == at + W) split(pair_of(old, i, o), a, b);
        }
        neu[VC == 1 ? 0 : 2 * i][j] = a;
        if (VC > 1) neu[(2 * i + 1) % VC][j] = b;
      }
    }
    store_rows<VC, W>(win, neu);
  } else {  // a tile holds more than W tokens: the inputs before a later tile are the sequence's
#pragma unroll
    for (int j = 0; j < W; ++j) {
      Raw<T, VC> in;
      in.load(xp - (W - j) * xs);
#pragma unroll
      for (int i = 0; i < P; ++i) last[j][i] = in.pair(i);
    }
  }
  F2 y[P];
#pragma unroll 1
  for (; left >= U; left -= U) {
    xp += U * xs;
    Raw<T, VC> next[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u < left - U) next[u].load(xp + u * xs);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      k.token(last, raw[u], p.silu, y);
      store_pairs<T, VC>(yp, y);
      yp += ys;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = next[u];
  }
#pragma unroll
  for (int u = 0; u < U - 1; ++u)
    if (u < left) {
      k.token(last, raw[u], p.silu, y);
      store_pairs<T, VC>(yp, y);
      yp += ys;
    }
}

// One token a sequence: the windows' bytes count. A warp takes kStepSeqs
// sequences for its channels, so that the weights are read once for them and
// all their windows are in flight together.
constexpr int kStepSeqs = 4;

template <int T, int VC, int TAPS>
__global__ void __launch_bounds__(32 * kConvWarps) k_conv_step(const ConvParams p, int vblocks, long long warps) {
  constexpr int W = TAPS - 1, P = VC == 1 ? 1 : VC / 2, ESZ = T == kF32 ? 4 : 2;
  const long long gw = (long long)blockIdx.x * kConvWarps + (threadIdx.x >> 5);
  const int c = (int(gw % vblocks) * 32 + int(threadIdx.x & 31)) * VC, s0 = int(gw / vblocks) * kStepSeqs;
  if (gw >= warps || c >= p.channels) return;
  float old[kStepSeqs][VC][W];
  Raw<T, VC> in[kStepSeqs];
  long long at[kStepSeqs];
#pragma unroll
  for (int i = 0; i < kStepSeqs; ++i) {
    const int s = s0 + i;
    int slot = -1;
    if (s < p.plan.seqs) {
      slot = p.plan.slots ? p.plan.slots[s] : s;
      if (slot < 0 || slot >= p.plan.state_rows) {
        slot = -1;
        *p.err = 1;
      }
    }
    at[i] = slot < 0 ? -1 : ((long long)slot * p.channels + c) * W;
    if (slot >= 0) {
      load_rows<VC, W>(p.window + at[i], old[i]);
      in[i].load(reinterpret_cast<const char*>(p.x) + (s * p.ldx + c) * ESZ);
    }
  }
  const Weights<VC, TAPS> k(p.w + (long long)c * TAPS, p.bias ? p.bias + c : nullptr);
#pragma unroll
  for (int i = 0; i < kStepSeqs; ++i) {
    if (at[i] < 0) continue;
    F2 last[W][P], y[P];
#pragma unroll
    for (int j = 0; j < W; ++j)
#pragma unroll
      for (int n = 0; n < P; ++n) last[j][n] = pair_of(old[i], n, j);
    k.token(last, in[i], p.silu, y);
    store_pairs<T, VC>(reinterpret_cast<char*>(p.y) + ((s0 + i) * p.ldy + c) * ESZ, y);
#pragma unroll
    for (int j = 0; j < W; ++j)
#pragma unroll
      for (int n = 0; n < P; ++n) {
        float a, b;
        split(last[j][n], a, b);
        old[i][VC == 1 ? 0 : 2 * n][j] = a;
        if (VC > 1) old[i][(2 * n + 1) % VC][j] = b;
      }
    store_rows<VC, W>(p.window + at[i], old[i]);
  }
}

template <int T, int VC, int TAPS, bool step>
void launch(const ConvParams& p, cudaStream_t s) {
  const int vblocks = ceil_div(p.channels, 32 * VC);
  // Tiles of 32 tokens read 3 of them again, tiles of 8 as many; short tiles where
  // long ones would leave the SMs without enough loads in flight. bf16, tiles of 32
  // against 8: 500 x 1280 8.4 / 4.6 us, 2000 x 1280 8.4 / 6.7, 8000 x 1280 15.2 /
  // 15.4, 15000 x 1280 19.1 / 24.3, 10000 x 4352 42 / 55.
  const int len = (long long)p.plan.tokens * vblocks >= 32LL * 148 * 8 ? 32 : 8;
  const long long warps = (step ? ceil_div(p.plan.seqs, kStepSeqs) : seq_tiles(p.plan, len)) * vblocks;
  const long long grid = (warps + kConvWarps - 1) / kConvWarps;
  B2E_CHECK(grid <= 0x7fffffffLL, kErrInvalid, "causal_conv: too many tiles");
  if constexpr (step)
    k_conv_step<T, VC, TAPS><<<unsigned(grid), 32 * kConvWarps, 0, s>>>(p, vblocks, warps);
  else
    k_conv<T, VC, TAPS><<<unsigned(grid), 32 * kConvWarps, 0, s>>>(p, len, vblocks, warps);
  B2E_CUDA(cudaGetLastError());
}

template <int T, int VC, bool step>
void launch_taps(const ConvParams& p, cudaStream_t s) {
  if (p.taps == 2) return launch<T, VC, 2, step>(p, s);
  if (p.taps == 3) return launch<T, VC, 3, step>(p, s);
  launch<T, VC, 4, step>(p, s);
}

template <int T, bool step>
void launch_type(const ConvParams& p, cudaStream_t s) {
  constexpr int VC = T == kF32 || step ? 4 : 8;  // 16 bytes of x a lane; four channels of the windows, which bound a step
  const auto aligned = [](const void* v, size_t a) { return (reinterpret_cast<uintptr_t>(v) & (a - 1)) == 0; };
  const size_t xa = VC * (T == kF32 ? 4 : 2);
  const bool vec = p.channels % VC == 0 && p.ldx % VC == 0 && p.ldy % VC == 0 && aligned(p.x, xa) && aligned(p.y, xa) &&
                   aligned(p.w, 16) && aligned(p.window, 16);
  if (vec)
    launch_taps<T, VC, step>(p, s);
  else
    launch_taps<T, 1, step>(p, s);
}

}  // namespace

void causal_conv(const ConvParams& p, cudaStream_t s) {
  if (p.plan.seqs == 0 || p.plan.tokens == 0) return;
  const bool step = p.plan.starts == nullptr;
  if (p.type == kF32) return step ? launch_type<kF32, true>(p, s) : launch_type<kF32, false>(p, s);
  if (p.type == kBF16) return step ? launch_type<kBF16, true>(p, s) : launch_type<kBF16, false>(p, s);
  step ? launch_type<kF16, true>(p, s) : launch_type<kF16, false>(p, s);
}

}  // namespace b2e
