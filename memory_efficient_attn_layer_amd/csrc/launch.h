// Kernel ids and the timed launch shared by the entry points' files.
#pragma once

#include <hip/hip_runtime.h>

namespace mea {

namespace kernel_ids {
enum KernelId {
  K_QKVG_PROJ, K_ATTN_FWD, K_GATE_OPROJ, K_PREP, K_DZ_GATE_BWD,
  K_ATTN_BWD_DQ, K_ATTN_BWD_DKDV, K_DW_PARTIAL, K_DW_REDUCE, K_DX,
  K_ATTN_DECODE, K_DECODE_COMBINE, K_SKINNY_GEMM, K_TABLE_GRAD, K_TABLE_ROWS,
  K_GROUPED_FWD, K_GROUPED_DQ, K_GROUPED_DKDV, K_GROUPED_JOIN, K_TREE_ATTN, K_TREE_COMBINE,
  K_APPEND_PLAN, K_APPEND_ROWS, K_ACCEPT_PLAN, K_ACCEPT_ROWS, K_TRUNCATE,
  K_FORK, K_FORK_READ, K_FORK_WRITE, K_COMPACT_PLAN, K_COMPACT_MOVE, K_COUNT
};
}  // namespace kernel_ids

// The events around one recorded launch (null: not recorded).
struct TimedLaunch {
  hipEvent_t begin = nullptr, end = nullptr;
};
hipError_t record_begin(int kernel, hipStream_t s, TimedLaunch* t);
void record_end(int kernel, hipStream_t s, const TimedLaunch& t);

// Runs `launch` (which returns a hipError_t); when profiling is on, brackets
// it with events on stream s.
template <class F>
hipError_t timed(int kernel, hipStream_t s, F launch) {
  TimedLaunch t;
  const hipError_t rc = record_begin(kernel, s, &t);
  if (rc != hipSuccess) return rc;
  const hipError_t e = launch();
  if (t.begin != nullptr) record_end(kernel, s, t);
  return e;
}

}  // namespace mea
