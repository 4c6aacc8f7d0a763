// Selective scan of the Mamba2 layer over packed sequences and over single
// tokens (the recurrence of model/mamba2.py:128-165, with its softplus, decay,
// skip and gate):
//
//   dt = softplus(dt);  h <- exp(a dt) h + (dt x) b^T;  y = (h c + d x) silu(z)
//
// h is [size, state] float32 a (sequence, head), x [size], b and c [state], dt, a
// and d scalars of the head. In this file's kernels everything is held in float32 and
// y is rounded once.
//
// Here: the single-token kernels, the recurrence kernel that walks a sequence
// token by token with the state in registers (any type and size), the join of a
// sequence's segments, and the choice between these and the chunked tensor-core
// kernel (scan_tc.cu).
#include <algorithm>
#include <type_traits>

#include "packed.cuh"
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
    if (threadIdx.x == 0) *p.err = 1;
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
    if (threadIdx.x == 0) *p.err = 1;
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
// A CTA of 128 threads walks one segment of a sequence for one head and 8 R state
// rows. Sixteen lanes cover a row, a thread holds R rows by J vectors of four
// columns (interleaved by lane) in registers. The decay of a token is one scalar
// for the whole head, so the registers hold H = h / P with P the product of the
// decays since it was last 1:
//
//   P <- decay P;  H <- H + (dt / P) x b^T;  y = P (H c)
//
// two operations a state element and token instead of three, and one instead of
// two where only the state is wanted. P is multiplied into H when it leaves
// [2^-12, 2^12] (P and the token's decay one after the other, as h would have
// been multiplied) and at the end, so dt x b has 2^12 of headroom less than
// float32's range. A decay is rounded into P as it would be into h, and 1 / P is the
// hardware's reciprocal (one ulp): the outputs are 2.1e-7 from 64 bits (relative
// 2-norm, 64 sequences of 10000 tokens in all).
//
// That batch, 8 heads of 64 x 128, float32: 187 us, of which the main pass is 139, the
// pass for the segments' contributions 44 and their join 13. Bound by latency and
// issue, with 13 warps on an SM: 57% of the issue slots are taken and the FP32 pipe is
// busy half of the time that an SM is; an SM is idle for a quarter of the main pass,
// behind its last segment. The layout keeps shared memory off that path: a token costs
// a thread 2 J + R / 4 vectors. With a join 8 us slower than now: 195 us as it is, 220 with three
// operations, 204 with four rows a thread, 294 with two rows and 32 columns, where
// shared memory bound it. Tokens are staged in blocks of 16, the next block by
// cp.async while one is computed where the operands are float32 vectors.

constexpr int kTok = 16;  // tokens staged together
constexpr float kLowP = 0x1p-12f;  // bounds of P

__device__ __forceinline__ void cp_async16(void* dst, const void* src, int bytes) {  // zeros behind `bytes`
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(uint32_t(__cvta_generic_to_shared(dst))), "l"(src), "r"(bytes)
               : "memory");
}

// `seg` 0: whole sequences, states from and to ssm. Otherwise segments of `seg`
// tokens; `ends`: each but a sequence's last leaves its own contribution to the
// state (zero start) and its decay in the workspace; else each starts from the
// workspace. ASYNC: float32 operands in whole aligned vectors.
template <int T, int J, int R, bool ends, bool ASYNC>
__global__ void __launch_bounds__(128) k_scan_seq(const ScanParams p, ScanWork wk, int seg) {
  constexpr int N = 64 * J, ROWS = 8 * R, B = ASYNC ? 2 : 1;
  __shared__ __align__(16) float sb[B][kTok][N], sc[B][ends ? 1 : kTok][N];
  __shared__ __align__(16) float sx[B][kTok][ROWS];
  __shared__ float sy[kTok][ROWS], sdt[B][kTok], sdec[B][kTok];
  const int tile = blockIdx.x / p.heads, h = blockIdx.x % p.heads, p0 = blockIdx.y * ROWS;
  SeqTile t;
  if (seg > 0) {
    t = seq_tile(p.plan, tile, seg);
  } else {
    t = seq_whole(p.plan, tile);
  }
  if (threadIdx.x == 127 && h == 0 && p0 == 0) seq_report(p.plan, tile, seg == 0, p.err);
  if (!t.live) return;
  const int slot = p.plan.slots ? p.plan.slots[t.seq] : t.seq;
  if (slot < 0 || slot >= p.plan.state_rows) {
    if (threadIdx.x == 0) *p.err = 1;
    return;
  }
  const int end = seg > 0 && t.end - t.first > seg ? t.first + seg : t.end;
  if (ends && end == t.end) return;
  const int lane = threadIdx.x & 31, c16 = lane & 15, rg = threadIdx.x >> 4;
  const long long hp = (long long)p.size * p.state;
  float* own = p.ssm + ((long long)slot * p.heads + h) * hp;
  const long long place = seg > 0 ? work_place(wk, p.plan, seg, t.seq, t.start, t.k) : 0;
  float* part = wk.state + (place * p.heads + h) * hp;
  const float* from = seg > 0 && t.end - t.start > seg ? part : own;
  float* to = ends ? part : own;
  const bool vec = p.state % 4 == 0;  // (the tables then start on 16 bytes)
  const float av = p.a[h], dv = p.d ? p.d[h] : 0.f;

  // a block of tokens into buffer `buf`
  const auto stage = [&](int t0, int buf) {
    const int n = min(kTok, end - t0);
    if constexpr (ASYNC) {
      const float* pb = static_cast<const float*>(p.b);
      const float* pc = static_cast<const float*>(p.c);
      const float* px = static_cast<const float*>(p.x) + h * p.size + p0;
      for (int i = threadIdx.x; i < n * (N / 4); i += 128) {
        const int k = i / (N / 4), c = i % (N / 4) * 4, in = c < p.state ? 16 : 0;
        cp_async16(&sb[buf][k][c], pb + (t0 + k) * p.ldb + (in ? c : 0), in);
        if (!ends) cp_async16(&sc[buf][k][c], pc + (t0 + k) * p.ldc + (in ? c : 0), in);
      }
      for (int i = threadIdx.x; i < n * (ROWS / 4); i += 128) {
        const int k = i / (ROWS / 4), r = i % (ROWS / 4) * 4, in = p0 + r < p.size ? 16 : 0;
        cp_async16(&sx[buf][k][r], px + (t0 + k) * p.ldx + (in ? r : 0), in);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    } else {
      for (int i = threadIdx.x; i < n * N; i += 128) {
        const int k = i / N, c = i % N;
        const bool in = c < p.state;
        sb[buf][k][c] = in ? LowP<T>::load(p.b, size_t((t0 + k) * p.ldb + c)) : 0.f;
        if (!ends) sc[buf][k][c] = in ? LowP<T>::load(p.c, size_t((t0 + k) * p.ldc + c)) : 0.f;
      }
      for (int i = threadIdx.x; i < n * ROWS; i += 128) {
        const int k = i / ROWS, r = p0 + i % ROWS;
        sx[buf][k][i % ROWS] = r < p.size ? LowP<T>::load(p.x, size_t((t0 + k) * p.ldx + h * p.size + r)) : 0.f;
      }
    }
  };
  const auto raw_dt = [&](int t0) { return int(threadIdx.x) < min(kTok, end - t0) ? p.dt[(t0 + int(threadIdx.x)) * p.lddt + h] : 0.f; };
  const auto decays = [&](float raw, int buf) {
    if (threadIdx.x < kTok) {
      const float dt = p.softplus ? softplusf_(raw) : raw;
      sdt[buf][threadIdx.x] = dt;
      sdec[buf][threadIdx.x] = expf(av * dt);
    }
  };
  if (ASYNC) {
    stage(t.first, 0);
    decays(raw_dt(t.first), 0);
  }

  F2 H[R][J][2];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int r = p0 + rg * R + i, n = (j * 16 + c16) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (!ends && r < p.size && n < p.state) {
        const float* f = from + (long long)r * p.state + n;
        if (vec) {
          v = *reinterpret_cast<const float4*>(f);
        } else {
          v.x = f[0];
          if (n + 1 < p.state) v.y = f[1];
          if (n + 2 < p.state) v.z = f[2];
          if (n + 3 < p.state) v.w = f[3];
        }
      }
      H[i][j][0] = f2(v.x, v.y);
      H[i][j][1] = f2(v.z, v.w);
    }
  float logsum = 0.f;  // of thread 0: log of the segment's decay
  float P = 1.f;       // the state is P H
  const auto scale_state = [&](float f) {
    const F2 f2x = f2(f, f);
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < J; ++j) {
        H[i][j][0] = mul2(H[i][j][0], f2x);
        H[i][j][1] = mul2(H[i][j][1], f2x);
      }
  };
  int buf = 0;
  for (int t0 = t.first; t0 < end; t0 += kTok) {
    const int n = min(kTok, end - t0);
    float next = 0.f;
    if constexpr (ASYNC) {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncthreads();
      if (t0 + kTok < end) {
        stage(t0 + kTok, buf ^ 1);
        next = raw_dt(t0 + kTok);
      }
    } else {
      __syncthreads();
      stage(t0, 0);
      decays(raw_dt(t0), 0);
      __syncthreads();
    }
    if (ends && threadIdx.x == 0)
      for (int k = 0; k < n; ++k) logsum += av * sdt[buf][k];
#pragma unroll 1
    for (int k = 0; k < n; ++k) {
      const float dc = sdec[buf][k], pn = P * dc;
      const bool keep = pn >= kLowP && pn <= 1.f / kLowP;  // not for a NaN
      if (!keep) {
        scale_state(P);
        scale_state(dc);
      }
      P = keep ? pn : 1.f;
      const float dt = sdt[buf][k] * rcp(P);
      F2 u[R], y[R];
#pragma unroll
      for (int i = 0; i < R; i += 4) {
        const float4 x = *reinterpret_cast<const float4*>(&sx[buf][k][rg * R + i]);
        const float v[4] = {dt * x.x, dt * x.y, dt * x.z, dt * x.w};
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          u[i + m] = f2(v[m], v[m]);
          y[i + m] = f2(0.f, 0.f);
        }
      }
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const float4 b4 = *reinterpret_cast<const float4*>(&sb[buf][k][(j * 16 + c16) * 4]);
        const float4 c4 = ends ? b4 : *reinterpret_cast<const float4*>(&sc[buf][ends ? 0 : k][(j * 16 + c16) * 4]);
        const F2 b0 = f2(b4.x, b4.y), b1 = f2(b4.z, b4.w), c0 = f2(c4.x, c4.y), c1 = f2(c4.z, c4.w);
#pragma unroll
        for (int i = 0; i < R; ++i) {
          H[i][j][0] = fma2(u[i], b0, H[i][j][0]);
          H[i][j][1] = fma2(u[i], b1, H[i][j][1]);
          if (!ends) {
            y[i] = fma2(c0, H[i][j][0], y[i]);
            y[i] = fma2(c1, H[i][j][1], y[i]);
          }
        }
      }
      if (!ends) {
        float sums[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
          float a, b;
          split(y[i], a, b);
          sums[i] = a + b;
        }
        int which;
        const float v = group_sums<16, R>(sums, lane, which);
        if (c16 % (16 / R) == 0) sy[k][rg * R + which] = P * v;
      }
    }
    if (ASYNC && t0 + kTok < end) decays(next, buf ^ 1);
    if (!ends) {
      __syncthreads();
      for (int i = threadIdx.x; i < n * ROWS; i += 128) {
        const int k = i / ROWS, r = p0 + i % ROWS;
        if (r >= p.size) continue;
        const long long row = t0 + k;
        float y = fmaf(dv, sx[buf][k][i % ROWS], sy[k][i % ROWS]);
        if (p.z) y *= siluf_(LowP<T>::load(p.z, size_t(row * p.ldz + h * p.size + r)));
        LowP<T>::store(p.y, size_t(row * p.ldy + h * p.size + r), y);
      }
    }
    if (ASYNC) buf ^= 1;
  }
  if (ends && threadIdx.x == 0 && p0 == 0) wk.log_decay[place * p.heads + h] = logsum;
  if (ends || end == t.end) {
    scale_state(P);
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int r = p0 + rg * R + i, n = (j * 16 + c16) * 4;
        float4 v;
        split(H[i][j][0], v.x, v.y);
        split(H[i][j][1], v.z, v.w);
        if (r < p.size && n < p.state) {
          float* f = to + (long long)r * p.state + n;
          if (vec) {
            *reinterpret_cast<float4*>(f) = v;
          } else {
            f[0] = v.x;
            if (n + 1 < p.state) f[1] = v.y;
            if (n + 2 < p.state) f[2] = v.z;
            if (n + 3 < p.state) f[3] = v.w;
          }
        }
      }
  }
}

// The states that a sequence's segments start from, in order: start[0] = ssm,
// start[k + 1] = decay[k] start[k] + own contribution[k]. In place over the
// contributions. One thread a vector of V elements of the state; a sequence of
// one segment starts from ssm itself.
template <int V>
__global__ void __launch_bounds__(256) k_scan_join(const ScanParams p, ScanWork wk, int seg) {
  const int seq = blockIdx.x / p.heads, h = blockIdx.x % p.heads;
  const long long hp = (long long)p.size * p.state, e = ((long long)blockIdx.y * blockDim.x + threadIdx.x) * V;
  const int start = p.plan.starts[seq], end = p.plan.starts[seq + 1];
  const int slot = p.plan.slots ? p.plan.slots[seq] : seq;
  if (e >= hp || start < 0 || end > p.plan.tokens || end < start || end - start <= seg || slot < 0 || slot >= p.plan.state_rows) return;
  const int segs = ceil_div(end - start, seg);
  const long long zeroth = work_place(wk, p.plan, seg, seq, start, 0) * p.heads + h, rest = work_place(wk, p.plan, seg, seq, start, 1) * p.heads + h;
  const auto place = [&](int k) { return k > 0 ? rest + (long long)(k - 1) * p.heads : zeroth; };
  const auto load = [](const float* at, float (&v)[V]) {
    if constexpr (V == 4) {
      const float4 a = *reinterpret_cast<const float4*>(at);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    } else {
      v[0] = at[0];
    }
  };
  float v[V];
  load(p.ssm + ((long long)slot * p.heads + h) * hp + e, v);
  float* at = wk.state + e;
  constexpr int U = 4;  // contributions in flight
  for (int k0 = 0; k0 < segs; k0 += U) {
    float c[U][V], g[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k0 + u + 1 < segs) {
        load(at + place(k0 + u) * hp, c[u]);
        g[u] = wk.log_decay[place(k0 + u)];
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k0 + u < segs) {
        if constexpr (V == 4)
          *reinterpret_cast<float4*>(at + place(k0 + u) * hp) = make_float4(v[0], v[1], v[2], v[3]);
        else
          at[place(k0 + u) * hp] = v[0];
        if (k0 + u + 1 < segs) {
          const float d = expf(g[u]);
#pragma unroll
          for (int i = 0; i < V; ++i) v[i] = fmaf(d, v[i], c[u][i]);
        }
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

template <int T, bool ends>
void launch_seq(const ScanParams& p, const ScanWork& wk, int seg, cudaStream_t s) {
  const long long tiles = seg > 0 ? seq_tiles(p.plan, seg) : p.plan.seqs;
  B2E_CHECK(tiles * p.heads <= 0x7fffffffLL, kErrInvalid, "mamba2_scan: too many (segment, head) pairs");
  const auto run = [&](auto j, auto r, auto async) {
    constexpr int J = decltype(j)::value, R = decltype(r)::value;
    const dim3 grid{unsigned(tiles * p.heads), unsigned(ceil_div(p.size, 8 * R)), 1};
    k_scan_seq<T, J, R, ends, decltype(async)::value><<<grid, 128, 0, s>>>(p, wk, seg);
  };
  const auto by_state = [&](auto async) {
    using std::integral_constant;
    if (p.state <= 64)
      run(integral_constant<int, 1>{}, integral_constant<int, 8>{}, async);
    else if (p.state <= 128)
      run(integral_constant<int, 2>{}, integral_constant<int, 8>{}, async);
    else
      run(integral_constant<int, 4>{}, integral_constant<int, 4>{}, std::false_type{});  // two blocks would not fit
  };
  if constexpr (T == kF32) {
    const auto rows16 = [](const void* v, long long ld) { return (reinterpret_cast<uintptr_t>(v) & 15) == 0 && ld % 4 == 0; };
    if (p.state % 4 == 0 && p.size % 4 == 0 && rows16(p.x, p.ldx) && rows16(p.b, p.ldb) && rows16(p.c, p.ldc))
      by_state(std::true_type{});
    else
      by_state(std::false_type{});
  } else {
    by_state(std::false_type{});
  }
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
    launch_seq<T, true>(p, wk, seg, s);
    scan_join(p, wk, seg, s);
  }
  launch_seq<T, false>(p, wk, seg, s);
}

}  // namespace

void scan_join(const ScanParams& p, const ScanWork& wk, int seg, cudaStream_t s) {
  const long long hp = (long long)p.size * p.state;
  const unsigned pairs = unsigned(p.plan.seqs) * p.heads;
  if (p.state % 4 == 0)
    k_scan_join<4><<<dim3(pairs, unsigned((hp / 4 + 255) / 256)), 256, 0, s>>>(p, wk, seg);
  else
    k_scan_join<1><<<dim3(pairs, unsigned((hp + 255) / 256)), 256, 0, s>>>(p, wk, seg);
  B2E_CUDA(cudaGetLastError());
}

ScanWork scan_work(const ScanParams& p, int seg) {
  const long long pairs = work_places(p.plan, seg) * p.heads;
  ScanWork w;
  w.firsts = std::min(p.plan.seqs, p.plan.tokens / seg);
  w.log_decay = static_cast<float*>(p.work);
  w.state = w.log_decay + (pairs + 63) / 64 * 64;
  return w;
}

// Splitting sequences costs a second pass over their tokens (the contributions)
// and the segments' states in the workspace, so it is done only where the longest
// sequence, walked by one CTA, would take more than twice what the tokens take
// spread evenly over the CTAs that run at once (four of the recurrence kernel on
// an SM, one of the chunked kernel). Segments then are that even share in blocks
// of 128 tokens: rounded down for the recurrence kernel, whose CTAs queue, up for
// the chunked one, where one CTA too many is a second wave. 64 sequences of 10000
// tokens in all (up to 700), 8 heads, float32: 288 us whole, 195 us split in 128
// tokens (187 with today's join), 254 us in 256.
int scan_segment(const ScanParams& p) {
  if (single_tokens(p)) return 0;
  const bool tc = scan_tc_eligible(p);
  const long long per = tc ? (p.heads + 1) / 2 : (long long)p.heads * ceil_div(p.size, 64), slots = tc ? 148 : 148 * 4;
  const long long share = ((long long)p.plan.tokens * per + slots - 1) / slots;
  if (p.plan.longest <= std::max<long long>(256, share * 2 + share / 4)) return 0;
  const long long seg = std::max<long long>(128, (share + (tc ? 127 : 0)) / 128 * 128);
  return p.plan.longest > seg ? int(seg) : 0;
}

size_t scan_workspace(const ScanParams& p) {
  const int seg = scan_segment(p);
  if (seg == 0) return 0;
  const size_t pairs = size_t(work_places(p.plan, seg)) * p.heads;
  return ((pairs + 63) / 64 * 64 + pairs * p.size * p.state) * 4;
}

void mamba2_scan(const ScanParams& p, cudaStream_t s) {
  if (p.plan.seqs == 0 || p.plan.tokens == 0) return;
  if (p.type == kF32) return launch_type<kF32>(p, s);
  if (p.type == kBF16) return launch_type<kBF16>(p, s);
  launch_type<kF16>(p, s);
}

}  // namespace b2e
