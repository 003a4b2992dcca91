// The accepted path of a tree of drafted tokens: from node 0, whose token is given, to the first child (by index)
// whose token is the one that the model picked after the current node, and so on.
//
// Children follow their parents, so one pass over the nodes finds the whole path: a warp a sequence holds 64 nodes at
// a time in registers (a lane two), and each step of the path is a vote over them.  Bound by the latency of the loads
// and of a vote a step: in a graph 4099 trees of up to 64 nodes (3 MB) take 3.2 us, 7 of up to 24 take 1.9.
#pragma once

#include "dk_common.cuh"

namespace dk {
namespace accept {

constexpr int kThreads = 128;

enum : int { kDetRows = 0x660 };   // row offsets that do not ascend inside the rows

struct Params {
  const int32_t* parents;   // index in the sequence, -1 for node 0
  const int64_t* tokens;
  const int64_t* picked;
  const int32_t* cu_rows;   // [n_seqs + 1]
  int32_t n_seqs, n_rows, max_keep;
  int32_t* keep;            // [n_seqs][max_keep], -1 behind the path
  int32_t* n_keep;
  int64_t* next;            // the pick after the path's last node; -1 without nodes
};

__global__ void __launch_bounds__(kThreads) accept_kernel(const Params p) {
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t b = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (b >= p.n_seqs) return;
  const int r0 = p.cu_rows[b], r1 = p.cu_rows[b + 1];
  int n = r1 - r0;
  if (r0 < 0 || r1 < r0 || r1 > p.n_rows) {
    if (lane == 0) report_error(DK_ERR_DEVICE_CHECK, kDetRows);
    n = 0;
  }
  int32_t* keep = p.keep + b * p.max_keep;
  int kept = n > 0 ? 1 : 0, cur = 0;
  int64_t pick = -1;
  if (n > 0 && lane == 0) keep[0] = 0;
  for (int c0 = 0; c0 < n; c0 += 64) {
    int par[2];
    int64_t tok[2], nxt[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = c0 + 32 * h + lane;
      const bool in = i < n;
      par[h] = in ? p.parents[r0 + i] : -1;
      tok[h] = in ? p.tokens[r0 + i] : 0;
      nxt[h] = in ? p.picked[r0 + i] : 0;
    }
    if (c0 == 0) pick = __shfl_sync(0xffffffffu, nxt[0], 0);
    if (kept == p.max_keep) break;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int first = c0 + 32 * h;
      while (kept < p.max_keep) {
        // later nodes of these 32 that agree with the pick after `cur`
        const uint32_t hit = __ballot_sync(0xffffffffu, par[h] == cur && first + lane > cur && tok[h] == pick);
        if (hit == 0) break;
        const int at = __ffs(hit) - 1;
        cur = first + at;
        pick = __shfl_sync(0xffffffffu, nxt[h], at);
        if (lane == 0) keep[kept] = cur;
        ++kept;
      }
    }
  }
  for (int i = kept + lane; i < p.max_keep; i += 32) keep[i] = -1;
  if (lane == 0) {
    p.n_keep[b] = kept;
    p.next[b] = pick;
  }
}

}  // namespace accept
}  // namespace dk
