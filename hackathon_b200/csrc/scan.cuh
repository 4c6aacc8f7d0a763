// Shared by the scan kernels (scan.cu, scan_tc.cu).
#pragma once
#include "seqops.cuh"

namespace b2e {

// Workspace of a scan whose sequences are split into segments of `seg` tokens: for
// each (segment of a split sequence, head), first its contribution to the state, then
// the state it starts from. Sequences of one segment, however many, take none.
struct ScanWork {
  float* log_decay = nullptr;  // [places, heads]
  float* state = nullptr;      // [places, heads, size, state]
  int firsts = 0;              // places of first segments, ahead of the others': min(seqs, tokens / seg)
};
// Places of a batch, and the place of segment k of split sequence `seq`, whose rows
// start at `start`. No two meet, without a table: two split sequences start more than
// seg rows apart, so in different blocks of seg rows; a later segment k goes by block
// start / seg + k, and the next sequence's start at the earliest in the block of this
// one's last, which its own segments k >= 1 lie behind.
inline long long work_places(const SeqPlan& p, int seg) {
  const long long blocks = p.tokens / seg;
  return blocks + (p.seqs < blocks ? p.seqs : blocks);
}
__device__ __forceinline__ long long work_place(const ScanWork& w, const SeqPlan& p, int seg, int seq, int start, int k) {
  const int block = start / seg;
  return k > 0 ? (long long)w.firsts + block + k - 1 : p.seqs <= w.firsts ? seq : block;
}
ScanWork scan_work(const ScanParams& p, int seg);
// The chunked tensor-core kernel (scan_tc.cu): whether it takes these operands,
// and the scan itself.
bool scan_tc_eligible(const ScanParams& p);
void scan_tc(const ScanParams& p, int seg, cudaStream_t s);
void scan_join(const ScanParams& p, const ScanWork& wk, int seg, cudaStream_t s);

}  // namespace b2e
