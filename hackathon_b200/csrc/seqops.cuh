// The prompt-side operators of the Mamba2 layer (include/b2e.h, the
// b2e_*_fp8 / b2e_causal_conv / b2e_mamba2_scan entry points): parameters and
// launchers of norm_fp8.cu, fp8_gemm.cu, conv.cu, scan.cu and scan_tc.cu.
#pragma once
#include "common.cuh"

namespace b2e {

// Rows, columns, tokens and channels of a call: indices are 32-bit (offsets are not),
// and a tile's or a block's last ones may lie behind the end.
constexpr int kMaxExtent = 0x7fffffff - 1023;
constexpr int kMaxSeqs = 1 << 30;
constexpr int kFp8Group = 128;        // values of a row (rows x columns of a weight block) that share a scale
constexpr float kFp8Max = 448.0f;     // largest finite e4m3 value
constexpr float kFp8MinScale = 7.888609052210118e-31f;  // 2^-100: an all-zero group keeps a finite reciprocal

// Error word of these operators on the current device (one int, zero when every
// bounded wait finished and every plan entry was in range).
int* seqops_error_word();

struct RmsFp8Params {
  const void* x;
  int x_type;
  long long ldx;
  const void* residual;  // or null
  int r_type;            // type of residual and total
  long long ldr;
  const float* weight;   // or null (ones)
  float eps;
  int norm;              // 0: quantise x as it is
  int rows, cols;
  uint8_t* q;            // e4m3, row stride ldq
  long long ldq;
  float* scale;          // [rows, ceil(cols / 128)]
  void* total;           // [rows, cols] of r_type, or null
  void* normed;          // [rows, cols] of x_type, or null
};
void rms_fp8(const RmsFp8Params& p, cudaStream_t s);

struct QuantWeightParams {
  const void* w;
  int w_type;
  long long ldw;
  int rows, cols;
  uint8_t* q;
  long long ldq;
  float* scale;  // [ceil(rows / 128), ceil(cols / 128)]
};
void quantize_weight_fp8(const QuantWeightParams& p, cudaStream_t s);

struct Fp8GemmParams {
  const uint8_t* x;
  long long ldx;
  const float* xs;  // [m, ceil(k / 128)]
  int m, k;
  const uint8_t* w;
  long long ldw;
  const float* ws;  // [ceil(n / 128), ceil(k / 128)]
  int n;
  const float* bias;  // or null
  int relu;
  void* y;
  int y_type;
  long long ldy;
  int* err;
};
void fp8_gemm(const Fp8GemmParams& p, cudaStream_t s);

// A packed batch of sequences: sequence i is rows [starts[i], starts[i + 1]) of
// the operands and row slots[i] of a state table of `state_rows` rows. Null
// starts: one token a sequence. Null slots: row i.
struct SeqPlan {
  const int* starts;
  const int* slots;
  const int* order;  // or null: the sequences in the order that their work starts in, longest first
  int seqs, tokens, state_rows;
  int longest;  // tokens of the longest sequence
};

struct ConvParams {
  SeqPlan plan;
  float* window;  // [state_rows, channels, taps - 1]
  const void* x;  // [tokens, channels], row stride ldx
  long long ldx;
  int type;
  const float* w;     // [channels, taps]
  const float* bias;  // or null
  int channels, taps, silu;
  void* y;  // [tokens, channels], row stride ldy
  long long ldy;
  int* err;
};
void causal_conv(const ConvParams& p, cudaStream_t s);

struct ScanParams {
  SeqPlan plan;
  float* ssm;  // [state_rows, heads, size, state]
  int type;    // of x, b, c, z, y
  const void* x;
  long long ldx;  // row stride; a row is heads * size contiguous values
  const void* b;
  long long ldb;
  const void* c;
  long long ldc;
  const float* dt;
  long long lddt;
  const float* a;  // [heads]
  const float* d;  // [heads] or null
  const void* z;   // or null
  long long ldz;
  void* y;  // [tokens, heads * size], row stride ldy
  long long ldy;
  int heads, size, state;
  int softplus;
  void* work;  // scan_workspace() bytes, 16-byte aligned
  size_t work_bytes;
  int* err;
};
constexpr int kScanMaxState = 256;
// Tokens of a segment (a multiple of 128, or 0: each sequence whole) that the
// scan splits sequences into, and the workspace that takes.
int scan_segment(const ScanParams& p);
size_t scan_workspace(const ScanParams& p);
void mamba2_scan(const ScanParams& p, cudaStream_t s);

// ---- device: the sequence of a virtual tile -------------------------------
// Tiles of `len` tokens over a packed batch without a table of tiles: sequence
// i owns the virtual tiles [starts[i] / len + i, starts[i + 1] / len + i], which
// are at least as many as it needs, so a launch of tokens / len + seqs tiles
// covers every sequence and a tile past its sequence's end does nothing.
__host__ __device__ inline long long seq_tiles(const SeqPlan& p, int len) {
  return (long long)(p.tokens / len) + p.seqs;
}

struct SeqTile {
  int seq, start, end, first;  // sequence, its rows [start, end), first row of the tile
  int k;                       // of the sequence's tiles
  bool live;
};

// One warp looks the tile's sequence up (32 probes a round); every lane returns
// the same answer. `starts` are bounds-checked here: a plan that the host did
// not make cannot lead a kernel outside its operands.
__device__ __forceinline__ SeqTile seq_tile(const SeqPlan& p, int tile, int len) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = p.seqs;  // the answer is the last i in [lo, hi) with starts[i] / len + i <= tile
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int i = lo + lane * step;
    const bool le = i < hi && p.starts[i] / len + i <= tile;
    const unsigned m = __ballot_sync(0xffffffffu, le);
    const int last = 31 - __clz(int(m | 1u));
    const int nlo = lo + last * step;
    hi = min(hi, nlo + step);
    lo = nlo;
  }
  SeqTile t;
  t.seq = lo;
  t.start = p.starts[lo];
  t.end = p.starts[lo + 1];
  t.k = tile - (t.start / len + lo);
  const long long first = t.start + (long long)t.k * len;
  t.first = int(first);
  t.live = t.start >= 0 && t.end <= p.tokens && t.k >= 0 && first < t.end;
  return t;
}

// Tile `i` of a launch with one tile a sequence.
__device__ __forceinline__ SeqTile seq_whole(const SeqPlan& p, int i) {
  SeqTile t;
  t.seq = p.order ? p.order[i] : i;
  t.k = 0;
  t.live = t.seq >= 0 && t.seq < p.seqs;
  t.start = t.first = t.live ? p.starts[t.seq] : 0;
  t.end = t.live ? p.starts[t.seq + 1] : 0;
  t.live = t.live && t.start >= 0 && t.end <= p.tokens && t.start < t.end;
  return t;
}

// Reports a plan whose entries leave its operands: tile i of a launch that covers
// every sequence (there are at least as many tiles) answers for sequence i, whatever
// tile i itself works on, because bad starts can hide a sequence from the search.
// `whole`: the launch goes by `order`. One thread a tile.
__device__ __forceinline__ void seq_report(const SeqPlan& p, int tile, bool whole, int* err) {
  if (tile >= p.seqs) return;
  const int s = p.starts[tile], e = p.starts[tile + 1], o = whole && p.order ? p.order[tile] : 0;
  if (s < 0 || e < s || e > p.tokens || o < 0 || o >= p.seqs) *err = 1;
}

}  // namespace b2e
