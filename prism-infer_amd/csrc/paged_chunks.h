// What the kernel over chunks of a paged cache does beside its attention: the
// sequences' validity, reported to the host, and the rows outside every sequence.
// `Args` has the fields of the launch's arguments that are named here.
#pragma once

#include "common.h"

namespace prism {

template <typename Args>
__device__ __forceinline__ void flag_sequence(const Args& a, int i) {
  atomicMin(a.status, i);
  if (a.report != nullptr) a.report[0] = 1;  // (every writer stores the same)
}

// The outcome that a host waits for, from the first workgroup alone and long
// before the others are done: every sequence's lengths and block ids.  Threads
// are spread over the sequences first, then over a sequence's pages.  keys_of(i):
// the sequence's keys, or -1 where its lengths are invalid.
template <typename Args, typename F>
__device__ void check_metadata(const Args& a, int& first_bad, F keys_of) {  // (first_bad: in LDS)
  constexpr int kAtOnce = 8;
  const int tid = threadIdx.x, threads = blockDim.x;
  if (tid == 0) first_bad = INT32_MAX;
  __syncthreads();
  int across = 1;  // sequences at a time
  while (across < a.batch && across < threads) across *= 2;
  for (int i = tid & (across - 1); i < a.batch; i += across) {
    const int keys = keys_of(i);
    bool good = keys >= 0;
    const int pages = good ? (keys - 1) / a.page + 1 : 0;
    for (int p = tid / across; p < pages; p += kAtOnce * (threads / across)) {
      int id[kAtOnce];
#pragma unroll
      for (int x = 0; x < kAtOnce; ++x)
        id[x] = a.bt[static_cast<int64_t>(i) * a.bt_sb + static_cast<int64_t>(min(p + x * (threads / across), pages - 1)) * a.bt_sn];
#pragma unroll
      for (int x = 0; x < kAtOnce; ++x) good = good && id[x] >= 0 && id[x] < a.num_blocks;
    }
    if (!good) atomicMin(&first_bad, i);
  }
  __syncthreads();
  if (tid != 0) return;
  if (first_bad != INT32_MAX) flag_sequence(a, first_bad);
  a.report[1] = a.cu_q[0];
  a.report[2] = a.cu_q[a.batch];
  __hip_atomic_store(a.report + 3, 1, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_SYSTEM);
}

// Rows outside every sequence are 0: `workers` workgroups share them.
template <int D, typename Args>
__device__ void zero_padding(const Args& a, int64_t me, int64_t workers) {
  const int first = min(max(a.cu_q[0], 0), a.total_q), end = min(max(a.cu_q[a.batch], first), a.total_q);
  const int64_t per_row = static_cast<int64_t>(a.heads) * (D / 8);
  const int64_t chunks = (first + (a.total_q - end)) * per_row;
  for (int64_t x = me * blockDim.x + threadIdx.x; x < chunks; x += workers * blockDim.x) {
    int64_t row = x / per_row;
    const int rest = static_cast<int>(x - row * per_row);
    if (row >= first) row += end - first;
    *reinterpret_cast<u32x4*>(a.out + row * a.o_st + rest / (D / 8) * a.o_sh + rest % (D / 8) * 8) = u32x4{0, 0, 0, 0};
  }
}

}  // namespace prism
