// RMS norm with the residual's addition and an 8-bit output, and the plain
// 8-bit quantisers.
//
//   v = x + r;  n = v / sqrt(mean(v^2) + eps) * w
//   scale[g] = max(max over 128 columns of |n| / 448, 2^-100);  q = e4m3(n * (1 / scale))
//
// v, its square sum, n and the scales are float32 (a row whose squares leave
// float32's range is summed again, scaled); v is rounded once to the residual's type
// where it is returned, n once to e4m3. Multiplying by the
// reciprocal instead of dividing moves n by at most one float32 ulp ahead of a
// rounding to 4 bits.
//
// Bound by HBM: 1 byte of q and 2 or 4 bytes each of x, r and v a value. A row
// stays in registers between its sum and its output, so it is read once; a
// thread's vectors are eight columns, so a group of 128 is sixteen neighbouring
// lanes and its maximum four shuffles. A row is taken by 32, 128 or 256 threads.
// 16384 x 4096 bf16 with a residual: 83 us (5.7 TB/s), 88 out of a cold cache;
// 90 with 256 threads a row instead of 128. 1 x 2048: 2.5 us.
#include <algorithm>
#include <cuda_fp8.h>

#include "mbarrier.cuh"
#include "seqops.cuh"

namespace b2e {
namespace {

// The factor that brings a row's values where their squares are float32 numbers: 0,
// none needed, for a mean square (and eps) between 2^-100 and the largest float32, or
// NaN. Of 2^31 columns, squares that overflow together leave the largest between 2^-103
// and 2^56, so their sum below 2^87; a mean below 2^-100 leaves the sum below 2^111.
__device__ __forceinline__ float rescale(float ms) { return ms > 3.4028235e38f ? 0x1p-100f : ms < 0x1p-100f ? 0x1p90f : 0.f; }
__device__ __forceinline__ float root(float ss, int cols, float eps, float up) { return up / sqrtf(ss / float(cols) + eps * up * up); }

// max that keeps a NaN, so that a group holding one gets a NaN scale.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

template <int T>
__device__ __forceinline__ void load8(const void* p, long long i, float (&v)[8]) {
  if constexpr (T == kF32) {
    const float4* f = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
    const float4 a = __ldg(f), b = __ldg(f + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 r = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i));
    const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
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

template <int T>
__device__ __forceinline__ void store8(void* p, long long i, const float (&v)[8]) {
  if constexpr (T == kF32) {
    float4* f = reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i);
    __stcs(f, make_float4(v[0], v[1], v[2], v[3]));
    __stcs(f + 1, make_float4(v[4], v[5], v[6], v[7]));
  } else {
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (T == kBF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        u[j] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
        u[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    __stcs(reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p) + i), make_uint4(u[0], u[1], u[2], u[3]));
  }
}

// Rows of a multiple of eight columns, 16-byte aligned: TPR threads a row, NV
// vectors of eight columns a thread.
// The bounds on registers keep 16384 x 4096 at 83 us; without them the second sum took
// eight more, a CTA an SM less, and 95 us.
template <int X, int R, int TPR, int NV>
__global__ void __launch_bounds__(256, NV == 4 ? 4 : NV == 2 ? 5 : 8) k_rms_fp8(const RmsFp8Params p) {
  constexpr int RPB = 256 / TPR, WPR = TPR / 32;
  __shared__ float red[8];
  const int tid = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const int row = blockIdx.x * RPB + sub;
  const bool live = row < p.rows;
  const int nvec = p.cols / 8, groups = ceil_div(p.cols, kFp8Group);
  float v[NV][8], ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int u = tid + i * TPR;
    if (live && u < nvec) {
      load8<X>(p.x, row * p.ldx + u * 8, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    }
  }
  if (p.residual) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = tid + i * TPR;
      if (live && u < nvec) {
        float r[8];
        load8<R>(p.residual, row * p.ldr + u * 8, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] += r[j];
      }
    }
  }
  float rs = 1.f;
  if (p.norm) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(v[i][j], v[i][j], ss);
    ss = warp_sum(ss);
    if constexpr (WPR > 1) {
      const int w = threadIdx.x >> 5;
      if ((threadIdx.x & 31) == 0) red[w] = ss;
      __syncthreads();
      ss = 0.f;
#pragma unroll
      for (int k = 0; k < WPR; ++k) ss += red[sub * WPR + k];
    }
    const float ms = ss / float(p.cols) + p.eps, up = rescale(ms);
    rs = 1.0f / sqrtf(ms);
    if (up != 0.f) {  // of all the row's threads
      ss = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(v[i][j] * up, v[i][j] * up, ss);
      ss = warp_sum(ss);
      if constexpr (WPR > 1) {
        named_bar(1 + sub, TPR);
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
        named_bar(1 + sub, TPR);
        ss = 0.f;
#pragma unroll
        for (int k = 0; k < WPR; ++k) ss += red[sub * WPR + k];
      }
      rs = root(ss, p.cols, p.eps, up);
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int u = tid + i * TPR;
    const bool in = live && u < nvec;
    if (in && p.total) store8<R>(p.total, (long long)row * p.cols + u * 8, v[i]);
    float m = 0.f;
    if (in && p.norm) {
      float w[8];
      if (p.weight) {
        const float4 a = *reinterpret_cast<const float4*>(p.weight + u * 8), b = *reinterpret_cast<const float4*>(p.weight + u * 8 + 4);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[i][j] *= rs;
        if (p.weight) v[i][j] *= w[j];
      }
    }
    if (in && p.normed) store8<X>(p.normed, (long long)row * p.cols + u * 8, v[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max_nan(m, fabsf(v[i][j]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (in) {
      const float scale = max_nan(m / kFp8Max, kFp8MinScale), inv = 1.0f / scale;
      uint2 o;
      o.x = to_e4m3x4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
      o.y = to_e4m3x4(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv);
      __stcs(reinterpret_cast<uint2*>(p.q + row * p.ldq + u * 8), o);
      if (u % 16 == 0) p.scale[(long long)row * groups + u / 16] = scale;
    }
  }
}

// Any width, stride and alignment: one CTA a row, the row read twice (the
// second time from cache); a warp takes a group of 128 columns.
template <int X, int R>
__global__ void __launch_bounds__(256) k_rms_fp8_any(const RmsFp8Params p) {
  __shared__ float red[32];
  const long long row = blockIdx.x;
  const int groups = ceil_div(p.cols, kFp8Group), lane = threadIdx.x & 31;
  auto value = [&](int j) {
    float v = LowP<X>::load(p.x, row * p.ldx + j);
    if (p.residual) v += LowP<R>::load(p.residual, row * p.ldr + j);
    return v;
  };
  float rs = 1.f;
  if (p.norm || p.total) {
    float ss = 0.f;
    for (int j = threadIdx.x; j < p.cols; j += blockDim.x) {
      const float v = value(j);
      ss = fmaf(v, v, ss);
    }
    ss = block_sum(ss, red);
    const float ms = ss / float(p.cols) + p.eps, up = rescale(ms);
    rs = p.norm ? 1.0f / sqrtf(ms) : 1.f;
    if (p.norm && up != 0.f) {
      ss = 0.f;
      for (int j = threadIdx.x; j < p.cols; j += blockDim.x) {
        const float v = value(j) * up;
        ss = fmaf(v, v, ss);
      }
      __syncthreads();
      rs = root(block_sum(ss, red), p.cols, p.eps, up);
    }
  }
  for (int g = threadIdx.x >> 5; g < groups; g += blockDim.x >> 5) {
    float v[4], m = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = g * kFp8Group + i * 32 + lane;
      v[i] = 0.f;
      if (j < p.cols) {
        v[i] = value(j);
        if (p.total) LowP<R>::store(p.total, row * p.cols + j, v[i]);
        if (p.norm) {
          v[i] *= rs;
          if (p.weight) v[i] *= p.weight[j];
        }
        if (p.normed) LowP<X>::store(p.normed, row * p.cols + j, v[i]);
      }
      m = max_nan(m, fabsf(v[i]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float scale = max_nan(m / kFp8Max, kFp8MinScale), inv = 1.0f / scale;
    if (lane == 0) p.scale[row * groups + g] = scale;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = g * kFp8Group + i * 32 + lane;
      if (j < p.cols) p.q[row * p.ldq + j] = __nv_cvt_float_to_fp8(v[i] * inv, __NV_SATFINITE, __NV_E4M3);
    }
  }
}

// One CTA a 128 x 128 block of a weight.
__global__ void __launch_bounds__(256) k_quant_weight(const QuantWeightParams p) {
  __shared__ float red[8];
  const int r0 = blockIdx.y * kFp8Group, c0 = blockIdx.x * kFp8Group;
  const int c = c0 + (threadIdx.x & 127), rstep = threadIdx.x >> 7;
  float m = 0.f;
  if (c < p.cols)
    for (int r = r0 + rstep; r < min(r0 + kFp8Group, p.rows); r += 2) m = max_nan(m, fabsf(load_as(p.w_type, p.w, r * p.ldw + c)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  m = red[0];
#pragma unroll
  for (int k = 1; k < 8; ++k) m = max_nan(m, red[k]);
  const float scale = max_nan(m / kFp8Max, kFp8MinScale), inv = 1.0f / scale;
  if (threadIdx.x == 0) p.scale[(long long)blockIdx.y * gridDim.x + blockIdx.x] = scale;
  if (c < p.cols)
    for (int r = r0 + rstep; r < min(r0 + kFp8Group, p.rows); r += 2)
      p.q[r * p.ldq + c] = __nv_cvt_float_to_fp8(load_as(p.w_type, p.w, r * p.ldw + c) * inv, __NV_SATFINITE, __NV_E4M3);
}

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

template <int X, int R, int TPR>
void launch_tpr(const RmsFp8Params& p, cudaStream_t s) {
  const int nv = ceil_div(p.cols / 8, TPR), grid = ceil_div(p.rows, 256 / TPR);
  if (nv <= 1)
    k_rms_fp8<X, R, TPR, 1><<<grid, 256, 0, s>>>(p);
  else if (nv <= 2)
    k_rms_fp8<X, R, TPR, 2><<<grid, 256, 0, s>>>(p);
  else
    k_rms_fp8<X, R, TPR, 4><<<grid, 256, 0, s>>>(p);
}

template <int X, int R>
void launch_types(const RmsFp8Params& p, cudaStream_t s) {
  const bool vec = p.cols % 8 == 0 && p.cols <= 8192 && p.ldq % 8 == 0 && aligned(p.q, 8) && aligned(p.x, 16) &&
                   (p.ldx * dtype_size(X)) % 16 == 0 && (!p.residual || (aligned(p.residual, 16) && (p.ldr * dtype_size(R)) % 16 == 0)) &&
                   (!p.weight || aligned(p.weight, 16)) && (!p.total || aligned(p.total, 16)) && (!p.normed || aligned(p.normed, 16));
  // Few rows want many threads each, many rows few registers idle and no barrier.
  // bf16 with a residual: 600 x 1024 takes 4.1 us with 32 threads a row, 2.7 with
  // 128; 16384 x 1024 20.4 and 23.2 (34 with 256). 16384 x 1536 47.8 with 128, 43.0
  // with 256; 16384 x 2048 53 and 48; 16384 x 3584 78 and 84; 300 x 4096 4.6 and
  // 3.8, 16384 x 4096 83 and 90.
  if (!vec) {
    k_rms_fp8_any<X, R><<<p.rows, 256, 0, s>>>(p);
  } else if (p.cols <= 256 || (p.cols <= 1024 && p.rows >= 148 * 18)) {
    launch_tpr<X, R, 32>(p, s);
  } else if (p.cols <= 1024 || (p.cols > 2048 && p.cols <= 4096 && p.rows >= 148 * 5)) {
    launch_tpr<X, R, 128>(p, s);
  } else {
    launch_tpr<X, R, 256>(p, s);
  }
  B2E_CUDA(cudaGetLastError());
}

}  // namespace

void rms_fp8(const RmsFp8Params& p, cudaStream_t s) {
  if (p.rows == 0) return;
  const int r = p.residual ? p.r_type : p.x_type;
  if (p.x_type == kF32) return launch_types<kF32, kF32>(p, s);
  if (p.x_type == kBF16) return r == kF32 ? launch_types<kBF16, kF32>(p, s) : launch_types<kBF16, kBF16>(p, s);
  return r == kF32 ? launch_types<kF16, kF32>(p, s) : launch_types<kF16, kF16>(p, s);
}

void quantize_weight_fp8(const QuantWeightParams& p, cudaStream_t s) {
  k_quant_weight<<<dim3(ceil_div(p.cols, kFp8Group), ceil_div(p.rows, kFp8Group)), 256, 0, s>>>(p);
  B2E_CUDA(cudaGetLastError());
}

}  // namespace b2e
