// Depthwise causal convolution over packed sequences with a window of the last
// taps - 1 inputs a state row (CausalConv1d, model/modules.py:37-41, applied to
// every token of a sequence instead of one).
//
//   v = window[slot] ++ x[sequence];  y[t] = act(bias + sum_j w[j] v[t + j]);  window[slot] <- last taps - 1 of v
//
// Bound by HBM: each x and y once, a window once each way. A warp takes 32
// vectors of four channels over a tile of tokens and keeps the
// last taps - 1 inputs in registers, so a token is read once and a tile reads
// only taps - 1 inputs of its neighbour's again. The tile that starts a
// sequence is the only one that reads the window, and it writes it too: no
// other tile can see the new one.
#include <algorithm>

#include "seqops.cuh"

namespace b2e {
namespace {

constexpr int kConvWarps = 4;

template <int T, int VC>
__device__ __forceinline__ void load_vec(const void* p, long long i, float (&v)[VC]) {
  if constexpr (VC == 1) {
    v[0] = LowP<T>::load(p, size_t(i));
  } else if constexpr (T == kF32) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i));
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  } else {
    const uint2 r = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + i));
    const uint32_t u[2] = {r.x, r.y};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if constexpr (T == kBF16) {
        v[2 * j] = __uint_as_float(u[j] << 16);
        v[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[j]));
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
      }
    }
  }
}

template <int T, int VC>
__device__ __forceinline__ void store_vec(void* p, long long i, const float (&v)[VC]) {
  if constexpr (VC == 1) {
    LowP<T>::store(p, size_t(i), v[0]);
  } else if constexpr (T == kF32) {
    __stcs(reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i), make_float4(v[0], v[1], v[2], v[3]));
  } else {
    uint32_t u[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if constexpr (T == kBF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        u[j] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
        u[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    __stcs(reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p) + i), make_uint2(u[0], u[1]));
  }
}

// VC * N contiguous floats, 16-byte aligned when VC > 1.
template <int VC, int N>
__device__ __forceinline__ void load_rows(const float* p, float (&v)[VC][N]) {
  if constexpr (VC * N % 4 == 0 && VC > 1) {
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
    for (int i = 0; i < VC * N; ++i) v[i / N][i % N] = p[i];
  }
}
template <int VC, int N>
__device__ __forceinline__ void store_rows(float* p, const float (&v)[VC][N]) {
  if constexpr (VC * N % 4 == 0 && VC > 1) {
#pragma unroll
    for (int i = 0; i < VC * N / 4; ++i)
      reinterpret_cast<float4*>(p)[i] =
          make_float4(v[4 * i / N][4 * i % N], v[(4 * i + 1) / N][(4 * i + 1) % N], v[(4 * i + 2) / N][(4 * i + 2) % N],
                      v[(4 * i + 3) / N][(4 * i + 3) % N]);
  } else {
#pragma unroll
    for (int i = 0; i < VC * N; ++i) p[i] = v[i / N][i % N];
  }
}

// silu with the hardware's exponential and reciprocal: a relative error of a few
// 2^-22 where the result matters, against ~40 instructions a value for the
// library's, which would bound the kernel ahead of HBM.
__device__ __forceinline__ float silu_fast(float v) { return __fdividef(v, 1.0f + __expf(-v)); }

template <int T, int VC, int TAPS>
__global__ void __launch_bounds__(32 * kConvWarps) k_conv(const ConvParams p, int len, int vblocks, long long warps) {
  constexpr int W = TAPS - 1, U = 8;  // tokens whose loads are in flight together
  const long long gw = (long long)blockIdx.x * kConvWarps + (threadIdx.x >> 5);
  if (gw >= warps) return;
  const int tile = int(gw / vblocks), lane = threadIdx.x & 31;
  const int c = (int(gw % vblocks) * 32 + lane) * VC;
  const SeqTile t = seq_tile(p.plan, tile, len);
  if (!t.live && p.err && t.start < t.end && (t.start < 0 || t.end > p.plan.tokens)) *p.err = 1;
  if (!t.live || c >= p.channels) return;
  const int slot = p.plan.slots ? p.plan.slots[t.seq] : t.seq;
  if (slot < 0 || slot >= p.plan.state_rows) {
    if (p.err) *p.err = 1;
    return;
  }
  float w[VC][TAPS], bias[VC];
  load_rows<VC, TAPS>(p.w + (long long)c * TAPS, w);
#pragma unroll
  for (int i = 0; i < VC; ++i) bias[i] = p.bias ? p.bias[c + i] : 0.f;
  float* win = p.window + ((long long)slot * p.channels + c) * W;
  const bool head = t.first == t.start;
  float last[W][VC], old[VC][W];  // last[j]: input of token first - W + j
  if (head) {
    load_rows<VC, W>(win, old);
#pragma unroll
    for (int j = 0; j < W; ++j)
#pragma unroll
      for (int i = 0; i < VC; ++i) last[j][i] = old[i][j];
  } else {  // a tile holds more than W tokens: the inputs before a later tile are the sequence's
#pragma unroll
    for (int j = 0; j < W; ++j) load_vec<T, VC>(p.x, (t.first - W + j) * p.ldx + c, last[j]);
  }
  const int end = min(t.end, t.first + len);
  for (int t0 = t.first; t0 < end; t0 += U) {
    float in[U][VC];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (t0 + u < end) load_vec<T, VC>(p.x, (t0 + u) * p.ldx + c, in[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (t0 + u < end) {
        float y[VC];
#pragma unroll
        for (int i = 0; i < VC; ++i) {
          float s = bias[i];
#pragma unroll
          for (int j = 0; j < W; ++j) s = fmaf(w[i][j], last[j][i], s);
          s = fmaf(w[i][W], in[u][i], s);
          y[i] = p.silu ? silu_fast(s) : s;
#pragma unroll
          for (int j = 0; j + 1 < W; ++j) last[j][i] = last[j + 1][i];
          last[W - 1][i] = in[u][i];
        }
        store_vec<T, VC>(p.y, (t0 + u) * p.ldy + c, y);
      }
    }
  }
  if (head) {
    const int n = t.end - t.start;
    float neu[VC][W];
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const int at = n - W + j;  // token of the sequence, or at + W of the old window
      if (at >= 0) {
        float in[VC];
        load_vec<T, VC>(p.x, (t.start + at) * p.ldx + c, in);
#pragma unroll
        for (int i = 0; i < VC; ++i) neu[i][j] = in[i];
      } else {
#pragma unroll
        for (int i = 0; i < VC; ++i) {
          neu[i][j] = 0.f;
#pragma unroll
          for (int k = 0; k < W; ++k)
            if (k == at + W) neu[i][j] = old[i][k];
        }
      }
    }
    store_rows<VC, W>(win, neu);
  }
}

// One token a sequence: the windows' bytes count. A warp takes kStepSeqs
// sequences for its channels, so that the weights are read once for them and
// all their windows are in flight together.
constexpr int kStepSeqs = 4;

template <int T, int VC, int TAPS>
__global__ void __launch_bounds__(32 * kConvWarps) k_conv_step(const ConvParams p, int vblocks, long long warps) {
  constexpr int W = TAPS - 1;
  const long long gw = (long long)blockIdx.x * kConvWarps + (threadIdx.x >> 5);
  const int c = (int(gw % vblocks) * 32 + int(threadIdx.x & 31)) * VC, s0 = int(gw / vblocks) * kStepSeqs;
  if (gw >= warps || c >= p.channels) return;
  float old[kStepSeqs][VC][W], in[kStepSeqs][VC];
  long long at[kStepSeqs];
#pragma unroll
  for (int i = 0; i < kStepSeqs; ++i) {
    const int s = s0 + i;
    int slot = -1;
    if (s < p.plan.seqs) {
      slot = p.plan.slots ? p.plan.slots[s] : s;
      if (slot < 0 || slot >= p.plan.state_rows) {
        slot = -1;
        if (p.err) *p.err = 1;
      }
    }
    at[i] = slot < 0 ? -1 : ((long long)slot * p.channels + c) * W;
    if (slot >= 0) {
      load_rows<VC, W>(p.window + at[i], old[i]);
      load_vec<T, VC>(p.x, s * p.ldx + c, in[i]);
    }
  }
  float w[VC][TAPS], bias[VC];
  load_rows<VC, TAPS>(p.w + (long long)c * TAPS, w);
#pragma unroll
  for (int i = 0; i < VC; ++i) bias[i] = p.bias ? p.bias[c + i] : 0.f;
#pragma unroll
  for (int i = 0; i < kStepSeqs; ++i) {
    if (at[i] < 0) continue;
    float y[VC];
#pragma unroll
    for (int k = 0; k < VC; ++k) {
      float s = bias[k];
#pragma unroll
      for (int j = 0; j < W; ++j) s = fmaf(w[k][j], old[i][k][j], s);
      s = fmaf(w[k][W], in[i][k], s);
      y[k] = p.silu ? silu_fast(s) : s;
#pragma unroll
      for (int j = 0; j + 1 < W; ++j) old[i][k][j] = old[i][k][j + 1];
      old[i][k][W - 1] = in[i][k];
    }
    store_vec<T, VC>(p.y, (s0 + i) * p.ldy + c, y);
    store_rows<VC, W>(p.window + at[i], old[i]);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <int T, int VC, int TAPS>
void launch(const ConvParams& p, cudaStream_t s) {
  const int vblocks = ceil_div(p.channels, 32 * VC);
  const bool step = p.plan.starts == nullptr;
  // Tiles of 32 tokens read 3 of them again; short tiles where long ones would
  // leave the SMs without enough loads in flight.
  const int len = (long long)p.plan.tokens * vblocks >= 32LL * 148 * 16 ? 32 : 8;
  const long long warps = (step ? ceil_div(p.plan.seqs, kStepSeqs) : seq_tiles(p.plan, len)) * vblocks;
  const long long grid = (warps + kConvWarps - 1) / kConvWarps;
  B2E_CHECK(grid <= 0x7fffffffLL, kErrInvalid, "causal_conv: too many tiles");
  if (step)
    k_conv_step<T, VC, TAPS><<<unsigned(grid), 32 * kConvWarps, 0, s>>>(p, vblocks, warps);
  else
    k_conv<T, VC, TAPS><<<unsigned(grid), 32 * kConvWarps, 0, s>>>(p, len, vblocks, warps);
  B2E_CUDA(cudaGetLastError());
}

template <int T, int VC>
void launch_taps(const ConvParams& p, cudaStream_t s) {
  if (p.taps == 2) return launch<T, VC, 2>(p, s);
  if (p.taps == 3) return launch<T, VC, 3>(p, s);
  launch<T, VC, 4>(p, s);
}

template <int T>
void launch_type(const ConvParams& p, cudaStream_t s) {
  constexpr int VC = 4;
  const auto aligned = [](const void* v) { return (reinterpret_cast<uintptr_t>(v) & (VC * (T == kF32 ? 4 : 2) - 1)) == 0; };
  const bool vec = p.channels % VC == 0 && p.ldx % VC == 0 && p.ldy % VC == 0 && aligned(p.x) && aligned(p.y) &&
                   aligned16(p.w) && aligned16(p.window);
  if (vec)
    launch_taps<T, VC>(p, s);
  else
    launch_taps<T, 1>(p, s);
}

}  // namespace

void causal_conv(const ConvParams& p, cudaStream_t s) {
  if (p.plan.seqs == 0 || p.plan.tokens == 0) return;
  if (p.type == kF32) return launch_type<kF32>(p, s);
  if (p.type == kBF16) return launch_type<kBF16>(p, s);
  launch_type<kF16>(p, s);
}

}  // namespace b2e
