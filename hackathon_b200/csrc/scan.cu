// Selective scan of the Mamba2 layer over packed sequences and over single
// tokens (the recurrence of model/mamba2.py:128-165, with its softplus, decay,
// skip and gate):
//
//   dt = softplus(dt);  h <- exp(a dt) h + (dt x) b^T;  y = (h c + d x) silu(z)
//
// h is [size, state] float32 a (sequence, head), x [size], b and c [state], dt, a
// and d scalars of the head. Everything is held in float32; y is rounded once.
//
// Here: the single-token kernels, the recurrence kernel that walks a sequence
// token by token with the state in registers (any type and size), the join of a
// sequence's segments, and the choice between these and the chunked tensor-core
// kernel (scan_tc.cu).
#include <algorithm>

#include "scan.cuh"

namespace b2e {
namespace {

// ------------------------------------------------------------ single tokens
//
// Bound by HBM: the state is read and written once (64 KB a head at 64 x 128)
// and everything else is small. A CTA of four warps takes a block of state rows:
// LPR lanes cover one row (Q vectors of four floats each), a thread holds R
// vectors, all in flight before their first use, and R row sums close together:
// each exchange also halves the sums a lane carries on. Short CTAs, eight or more
// on an SM, keep 128 KB in flight there.

// Sums of R values a lane over the LPR lanes of a row group: lane l of the group
// ends with the sum of value `which`, complete when its other index bits are zero.
template <int LPR, int R>
__device__ __forceinline__ float group_sums(float (&v)[R], int lane, int& which) {
  which = 0;
  int n = R;
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) {
    if (n > 1) {
      const bool up = lane & o;
      n >>= 1;
#pragma unroll
      for (int i = 0; i < R / 2; ++i)
        if (i < n) {
          const float send = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
      which = which * 2 + (up ? 1 : 0);
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    }
  }
  return v[0];
}

template <int T, int LPR, int Q, int R>
__global__ void __launch_bounds__(128) k_scan_step(const ScanParams p) {
  constexpr int RPW = 32 / LPR;  // rows a warp takes in one vector
  const int seq = blockIdx.x / p.heads, h = blockIdx.x % p.heads;
  const int slot = p.plan.slots ? p.plan.slots[seq] : seq;
  if (slot < 0 || slot >= p.plan.state_rows) {
    if (threadIdx.x == 0 && p.err) *p.err = 1;
    return;
  }
  const int lane = threadIdx.x & 31, c0 = lane % LPR, nv = p.state / 4;
  const int r0 = (blockIdx.y * 4 + (threadIdx.x >> 5)) * (R * RPW) + lane / LPR;  // rows r0 + RPW i
  float4* H = reinterpret_cast<float4*>(p.ssm + ((long long)slot * p.heads + h) * p.size * p.state);
  float4 cur[R][Q];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (r0 + RPW * i < p.size && c0 + LPR * q < nv) cur[i][q] = ld_stream(H + (long long)(r0 + RPW * i) * nv + c0 + LPR * q);
  const float dtr = p.dt[seq * p.lddt + h];
  float4 b[Q], c[Q];
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int n = (c0 + LPR * q) * 4;
    float t[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (n < p.state) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        t[j] = LowP<T>::load(p.b, size_t(seq * p.ldb + n + j));
        t[4 + j] = LowP<T>::load(p.c, size_t(seq * p.ldc + n + j));
      }
    }
    b[q] = make_float4(t[0], t[1], t[2], t[3]);
    c[q] = make_float4(t[4], t[5], t[6], t[7]);
  }
  const float dt = p.softplus ? softplusf_(dtr) : dtr, dc = expf(p.a[h] * dt);
  float dot[R], xs[R];
#pragma unroll
  for (int i = 0; i < R; ++i)
    xs[i] = r0 + RPW * i < p.size ? LowP<T>::load(p.x, size_t(seq * p.ldx + h * p.size + r0 + RPW * i)) : 0.f;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    dot[i] = 0.f;
    const float u = dt * xs[i];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      if (r0 + RPW * i >= p.size || c0 + LPR * q >= nv) continue;
      const float4 o = cur[i][q];
      const float4 n = make_float4(fmaf(dc, o.x, u * b[q].x), fmaf(dc, o.y, u * b[q].y), fmaf(dc, o.z, u * b[q].z),
                                   fmaf(dc, o.w, u * b[q].w));
      st_stream(H + (long long)(r0 + RPW * i) * nv + c0 + LPR * q, n);
      dot[i] += fmaf(c[q].w, n.w, fmaf(c[q].z, n.z, fmaf(c[q].y, n.y, c[q].x * n.x)));
    }
  }
  int which;
  const float sum = group_sums<LPR, R>(dot, lane, which);
  // every lane of a row group holds one of its rows' sums; the lanes that hold
  // the same one differ in the bits behind those that chose it
  constexpr int TAIL = LPR > R ? LPR / R : 1;
  const int r = r0 + RPW * which;
  if (r < p.size && c0 % TAIL == 0) {
    const float dv = p.d ? p.d[h] : 0.f;
    float y = fmaf(dv, LowP<T>::load(p.x, size_t(seq * p.ldx + h * p.size + r)), sum);
    if (p.z) y *= siluf_(LowP<T>::load(p.z, size_t(seq * p.ldz + h * p.size + r)));
    LowP<T>::store(p.y, size_t(seq * p.ldy + h * p.size + r), y);
  }
}

// States whose rows are not whole 16-byte vectors: a warp takes a state row.
template <int T>
__global__ void __launch_bounds__(256) k_scan_step_any(const ScanParams p) {
  const int seq = blockIdx.x / p.heads, h = blockIdx.x % p.heads, lane = threadIdx.x & 31;
  const int slot = p.plan.slots ? p.plan.slots[seq] : seq;
  if (slot < 0 || slot >= p.plan.state_rows) {
    if (threadIdx.x == 0 && p.err) *p.err = 1;
    return;
  }
  const float dtr = p.dt[seq * p.lddt + h];
  const float dt = p.softplus ? softplusf_(dtr) : dtr, dc = expf(p.a[h] * dt), dv = p.d ? p.d[h] : 0.f;
  for (int r = threadIdx.x >> 5; r < p.size; r += blockDim.x >> 5) {
    float* H = p.ssm + (((long long)slot * p.heads + h) * p.size + r) * p.state;
    const float xv = LowP<T>::load(p.x, size_t(seq * p.ldx + h * p.size + r)), u = dt * xv;
    float dot = 0.f;
    for (int n = lane; n < p.state; n += 32) {
      const float v = fmaf(dc, H[n], u * LowP<T>::load(p.b, size_t(seq * p.ldb + n)));
      H[n] = v;
      dot = fmaf(LowP<T>::load(p.c, size_t(seq * p.ldc + n)), v, dot);
    }
    dot = warp_sum(dot);
    if (lane == 0) {
      float y = fmaf(dv, xv, dot);
      if (p.z) y *= siluf_(LowP<T>::load(p.z, size_t(seq * p.ldz + h * p.size + r)));
      LowP<T>::store(p.y, size_t(seq * p.ldy + h * p.size + r), y);
    }
  }
}

// ------------------------------------------------------ the recurrence kernel
//
// A CTA of 128 threads walks one segment of a sequence for one head and 64 state
// rows. A thread holds two state rows (of the pair r, r + 32) by a quarter of
// the columns, interleaved by four, in registers: 2 x state / 4 floats. Bound by
// the FP32 pipe: three operations a state element and token (two packed), 16
// shared-memory vectors a thread and token.

constexpr int kTok = 16;  // tokens staged together

struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 pack2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

// J: vectors of four columns a thread (state <= 16 J). `seg` 0: whole
// sequences, states from and to ssm. Otherwise segments of `seg` tokens; `ends`:
// each but a sequence's last leaves its own contribution to the state (zero
// start) and its decay in the workspace; else each starts from the workspace.
template <int T, int J>
__global__ void __launch_bounds__(128) k_scan_seq(const ScanParams p, ScanWork wk, int seg, int ends) {
  constexpr int N = 16 * J;
  __shared__ float4 sb[kTok][N / 4], sc[kTok][N / 4];
  __shared__ float sx[kTok][64], sy[kTok][64], sdt[kTok], sdec[kTok];
  const int tile = blockIdx.x / p.heads, h = blockIdx.x % p.heads, p0 = blockIdx.y * 64;
  SeqTile t;
  if (seg > 0) {
    t = seq_tile(p.plan, tile, seg);
  } else {
    t.seq = tile;
    t.start = t.first = p.plan.starts ? p.plan.starts[tile] : tile;
    t.end = p.plan.starts ? p.plan.starts[tile + 1] : tile + 1;
    t.live = t.start >= 0 && t.end <= p.plan.tokens && t.start < t.end;
  }
  if (!t.live) return;
  const int slot = p.plan.slots ? p.plan.slots[t.seq] : t.seq;
  if (slot < 0 || slot >= p.plan.state_rows) {
    if (threadIdx.x == 0 && p.err) *p.err = 1;
    return;
  }
  const int end = seg > 0 ? min(t.end, t.first + seg) : t.end;
  if (ends && end == t.end) return;
  const int q = threadIdx.x & 3, r0 = threadIdx.x >> 2;
  const long long hp = (long long)p.size * p.state;
  float* own = p.ssm + ((long long)slot * p.heads + h) * hp;
  float* part = wk.state + ((long long)tile * p.heads + h) * hp;
  const float* from = seg > 0 ? part : own;
  float* to = ends ? part : own;
  F2 H[2][J][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int r = p0 + r0 + 32 * i, n = (j * 4 + q) * 4;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      if (!ends && r < p.size)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (n + k < p.state) v[k] = from[(long long)r * p.state + n + k];
      H[i][j][0] = pack2(v[0], v[1]);
      H[i][j][1] = pack2(v[2], v[3]);
    }
  const float av = p.a[h], dv = p.d ? p.d[h] : 0.f;
  float logsum = 0.f;  // of thread 0: log of the segment's decay
  for (int t0 = t.first; t0 < end; t0 += kTok) {
    const int n = min(kTok, end - t0);
    __syncthreads();
    for (int i = threadIdx.x; i < n * N; i += 128) {
      const int k = i / N, c = i % N;
      float bv = 0.f, cv = 0.f;
      if (c < p.state) {
        bv = LowP<T>::load(p.b, size_t((t0 + k) * p.ldb + c));
        cv = LowP<T>::load(p.c, size_t((t0 + k) * p.ldc + c));
      }
      reinterpret_cast<float*>(sb[k])[c] = bv;
      reinterpret_cast<float*>(sc[k])[c] = cv;
    }
    for (int i = threadIdx.x; i < n * 64; i += 128) {
      const int k = i / 64, r = p0 + i % 64;
      sx[k][i % 64] = r < p.size ? LowP<T>::load(p.x, size_t((t0 + k) * p.ldx + h * p.size + r)) : 0.f;
    }
    if (threadIdx.x < n) {
      const float dtr = p.dt[(t0 + threadIdx.x) * p.lddt + h];
      const float dt = p.softplus ? softplusf_(dtr) : dtr;
      sdt[threadIdx.x] = dt;
      sdec[threadIdx.x] = expf(av * dt);
    }
    __syncthreads();
    if (ends && threadIdx.x == 0)
      for (int k = 0; k < n; ++k) logsum += av * sdt[k];
    for (int k = 0; k < n; ++k) {
      const float dt = sdt[k], dc = sdec[k];
      const F2 dc2 = pack2(dc, dc);
      const float ua = dt * sx[k][r0], ub = dt * sx[k][r0 + 32];
      const F2 u[2] = {pack2(ua, ua), pack2(ub, ub)};
      F2 y[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const float4 b4 = sb[k][j * 4 + q], c4 = sc[k][j * 4 + q];
        const F2 b0 = pack2(b4.x, b4.y), b1 = pack2(b4.z, b4.w), c0 = pack2(c4.x, c4.y), c1 = pack2(c4.z, c4.w);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          H[i][j][0] = fma2(dc2, H[i][j][0], mul2(u[i], b0));
          H[i][j][1] = fma2(dc2, H[i][j][1], mul2(u[i], b1));
          y[i] = fma2(c0, H[i][j][0], y[i]);
          y[i] = fma2(c1, H[i][j][1], y[i]);
        }
      }
      if (!ends) {
        const float2 a0 = unpack2(y[0]), a1 = unpack2(y[1]);
        float s0 = a0.x + a0.y, s1 = a1.x + a1.y;
        s0 += __shfl_xor_sync(0xffffffffu, s0, 1);
        s1 += __shfl_xor_sync(0xffffffffu, s1, 1);
        s0 += __shfl_xor_sync(0xffffffffu, s0, 2);
        s1 += __shfl_xor_sync(0xffffffffu, s1, 2);
        if (q == 0) {
          sy[k][r0] = s0;
          sy[k][r0 + 32] = s1;
        }
      }
    }
    if (ends) continue;
    __syncthreads();
    for (int i = threadIdx.x; i < n * 64; i += 128) {
      const int k = i / 64, r = p0 + i % 64;
      if (r >= p.size) continue;
      const long long row = t0 + k;
      float y = fmaf(dv, sx[k][i % 64], sy[k][i % 64]);
      if (p.z) y *= siluf_(LowP<T>::load(p.z, size_t(row * p.ldz + h * p.size + r)));
      LowP<T>::store(p.y, size_t(row * p.ldy + h * p.size + r), y);
    }
  }
  if (ends && threadIdx.x == 0 && p0 == 0) wk.log_decay[(long long)tile * p.heads + h] = logsum;
  if (ends || end == t.end) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int r = p0 + r0 + 32 * i, n = (j * 4 + q) * 4;
        const float2 lo = unpack2(H[i][j][0]), hi = unpack2(H[i][j][1]);
        const float v[4] = {lo.x, lo.y, hi.x, hi.y};
        if (r < p.size)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (n + k < p.state) to[(long long)r * p.state + n + k] = v[k];
      }
  }
}

// The states that a sequence's segments start from, in order: start[0] = ssm,
// start[k + 1] = decay[k] start[k] + own contribution[k]. In place over the
// contributions. One thread an element of the state.
__global__ void __launch_bounds__(256) k_scan_join(const ScanParams p, ScanWork wk, int seg) {
  const int seq = blockIdx.x / p.heads, h = blockIdx.x % p.heads;
  const long long hp = (long long)p.size * p.state, e = (long long)blockIdx.y * blockDim.x + threadIdx.x;
  const int start = p.plan.starts[seq], end = p.plan.starts[seq + 1];
  const int slot = p.plan.slots ? p.plan.slots[seq] : seq;
  if (e >= hp || start < 0 || end > p.plan.tokens || start >= end || slot < 0 || slot >= p.plan.state_rows) return;
  const int segs = ceil_div(end - start, seg);
  const long long tile0 = start / seg + seq;
  float v = p.ssm[((long long)slot * p.heads + h) * hp + e];
  float* at = wk.state + (tile0 * p.heads + h) * hp + e;
  const float* ld = wk.log_decay + tile0 * p.heads + h;
  constexpr int U = 8;  // contributions in flight
  for (int k0 = 0; k0 < segs; k0 += U) {
    float c[U], g[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k0 + u + 1 < segs) {
        c[u] = at[(long long)(k0 + u) * p.heads * hp];
        g[u] = ld[(long long)(k0 + u) * p.heads];
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k0 + u < segs) {
        at[(long long)(k0 + u) * p.heads * hp] = v;
        if (k0 + u + 1 < segs) v = fmaf(expf(g[u]), v, c[u]);
      }
  }
}

template <int T>
void launch_step(const ScanParams& p, cudaStream_t s) {
  const long long items = (long long)p.plan.seqs * p.heads;
  B2E_CHECK(items <= 0x7fffffffLL, kErrInvalid, "mamba2_scan: too many (sequence, head) pairs");
  if (p.state % 4 != 0) {
    k_scan_step_any<T><<<unsigned(items), 256, 0, s>>>(p);
  } else {
    // lanes of a row by its width; rows a CTA takes: 4 warps x R vectors x 32 / LPR
    const auto grid = [&](int rows) { return dim3{unsigned(items), unsigned(ceil_div(p.size, rows)), 1}; };
    if (p.state <= 32)
      k_scan_step<T, 8, 1, 8><<<grid(128), 128, 0, s>>>(p);
    else if (p.state <= 64)
      k_scan_step<T, 16, 1, 8><<<grid(64), 128, 0, s>>>(p);
    else if (p.state <= 128)
      k_scan_step<T, 32, 1, 8><<<grid(32), 128, 0, s>>>(p);
    else
      k_scan_step<T, 32, 2, 4><<<grid(16), 128, 0, s>>>(p);
  }
  B2E_CUDA(cudaGetLastError());
}

template <int T>
void launch_seq(const ScanParams& p, const ScanWork& wk, int seg, int ends, cudaStream_t s) {
  const long long tiles = seg > 0 ? seq_tiles(p.plan, seg) : p.plan.seqs;
  B2E_CHECK(tiles * p.heads <= 0x7fffffffLL, kErrInvalid, "mamba2_scan: too many (segment, head) pairs");
  const dim3 grid{unsigned(tiles * p.heads), unsigned(ceil_div(p.size, 64)), 1};
  if (p.state <= 64)
    k_scan_seq<T, 4><<<grid, 128, 0, s>>>(p, wk, seg, ends);
  else if (p.state <= 128)
    k_scan_seq<T, 8><<<grid, 128, 0, s>>>(p, wk, seg, ends);
  else
    k_scan_seq<T, 16><<<grid, 128, 0, s>>>(p, wk, seg, ends);
  B2E_CUDA(cudaGetLastError());
}

bool single_tokens(const ScanParams& p) {
  return p.plan.starts == nullptr || (p.plan.longest == 1 && p.plan.tokens == p.plan.seqs);
}

template <int T>
void launch_type(const ScanParams& p, cudaStream_t s) {
  if (single_tokens(p)) return launch_step<T>(p, s);
  const int seg = scan_segment(p);
  if (scan_tc_eligible(p)) return scan_tc(p, seg, s);
  ScanWork wk{};
  if (seg > 0) {
    wk = scan_work(p, seg);
    launch_seq<T>(p, wk, seg, 1, s);
    scan_join(p, wk, seg, s);
  }
  launch_seq<T>(p, wk, seg, 0, s);
}

}  // namespace

void scan_join(const ScanParams& p, const ScanWork& wk, int seg, cudaStream_t s) {
  const long long hp = (long long)p.size * p.state;
  k_scan_join<<<dim3(unsigned(p.plan.seqs) * p.heads, unsigned((hp + 255) / 256)), 256, 0, s>>>(p, wk, seg);
  B2E_CUDA(cudaGetLastError());
}

ScanWork scan_work(const ScanParams& p, int seg) {
  const long long pairs = seq_tiles(p.plan, seg) * p.heads;
  ScanWork w;
  w.log_decay = static_cast<float*>(p.work);
  w.state = w.log_decay + (pairs + 63) / 64 * 64;
  return w;
}

// Splitting a sequence costs a second pass over its tokens (the contributions)
// and its segments' states in the workspace, so it is done only where whole
// sequences would leave SMs idle: segments of a multiple of 128 tokens, as many
// as give each SM four CTAs of the recurrence kernel, or one of the chunked one.
int scan_segment(const ScanParams& p) {
  if (single_tokens(p)) return 0;
  const bool tc = scan_tc_eligible(p);
  const long long per = tc ? (p.heads + 1) / 2 : (long long)p.heads * ceil_div(p.size, 64), want = tc ? 148 : 148 * 4;
  if (p.plan.seqs * per >= want || p.plan.longest <= 256) return 0;
  const long long segs = std::max<long long>(1, want / per);
  const long long len = (p.plan.tokens + segs - 1) / segs;
  const int seg = int(std::max<long long>(128, (len + 127) / 128 * 128));
  return p.plan.longest > seg ? seg : 0;
}

size_t scan_workspace(const ScanParams& p) {
  const int seg = scan_segment(p);
  if (seg == 0) return 0;
  const size_t pairs = size_t(seq_tiles(p.plan, seg)) * p.heads;
  return ((pairs + 63) / 64 * 64 + pairs * p.size * p.state) * 4;
}

void mamba2_scan(const ScanParams& p, cudaStream_t s) {
  if (p.plan.seqs == 0 || p.plan.tokens == 0) return;
  if (p.type == kF32) return launch_type<kF32>(p, s);
  if (p.type == kBF16) return launch_type<kBF16>(p, s);
  launch_type<kF16>(p, s);
}

}  // namespace b2e
