// Shared by the scan kernels (scan.cu, scan_tc.cu).
#pragma once
#include "seqops.cuh"

namespace b2e {

// Workspace of a scan whose sequences are split: for each (virtual segment,
// head), first its contribution to the state, then the state it starts from.
struct ScanWork {
  float* log_decay = nullptr;  // [segments, heads]
  float* state = nullptr;      // [segments, heads, size, state]
};
ScanWork scan_work(const ScanParams& p, int seg);
// The chunked tensor-core kernel (scan_tc.cu): whether it takes these operands,
// and the scan itself.
bool scan_tc_eligible(const ScanParams& p);
void scan_tc(const ScanParams& p, int seg, cudaStream_t s);
void scan_join(const ScanParams& p, const ScanWork& wk, int seg, cudaStream_t s);

}  // namespace b2e
