// A step's attention metadata from the requests' lengths: offsets, lengths,
// block tables with the blocks that new tokens need, and the slot of every new
// token.
//
//   cu[i]       = sum_{j < i} new_j               ctx_i  = cached_i + new_i
//   held_i      = ceil(cached_i / P)              need_i = ceil(ctx_i / P)
//   base_i      = start + sum_{j < i} (need_j - held_j)
//   table[i][w] = held ids (w < held_i), free[base_i + w - held_i] (w < need_i), -1
//   slot(token) = table[i][pos / P] P + pos % P,  pos = cached_i + token - cu[i]
//
// One launch: every workgroup makes both sums over all requests itself (a scan
// in LDS), then writes its share of the tokens and of the tables, four entries
// a thread.  A second launch, or a grid that waits for one scan, would cost
// more than the repeated scans, whose loads hit the L2.
#include "common.h"

#include <algorithm>

namespace prism {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxBatch = 8192;  // three words of LDS each
constexpr int kMaxInt = 0x7FFFFFFF;

struct MetaArgs {
  const int32_t* tables;
  int64_t t_sb, t_sw;
  const int32_t* cached;
  const int32_t* fresh;
  const int32_t* free;
  const int32_t* free_start;
  int num_free, batch, width, page, num_tokens;
  int32_t* slots;
  int32_t* positions;
  int32_t* cu;
  int32_t* ctx;
  int32_t* tail;  // max context length, next free entry, lowest request that does not fit
  int32_t* out;
};

// Sums stay at INT32_MAX once they reach it.
__device__ __forceinline__ int add_sat(int x, int y) {
  const uint32_t s = static_cast<uint32_t>(x) + static_cast<uint32_t>(y);
  return static_cast<int>(min(s, static_cast<uint32_t>(kMaxInt)));
}

struct Request {
  int cached, fresh, held, need;
  bool bad;
};

// Lengths that cannot be are taken as the nearest that can, and reported.
__device__ __forceinline__ Request request(const MetaArgs& a, int i) {
  const int c = a.cached[i], n = a.fresh[i];
  const int64_t ctx = static_cast<int64_t>(max(c, 0)) + max(n, 0), room = static_cast<int64_t>(a.width) * a.page;
  Request r;
  r.cached = max(c, 0);
  r.fresh = max(n, 0);
  r.held = static_cast<int>(min((static_cast<int64_t>(r.cached) + a.page - 1) / a.page, static_cast<int64_t>(a.width)));
  r.need = static_cast<int>(min((ctx + a.page - 1) / a.page, static_cast<int64_t>(a.width)));
  r.bad = c < 0 || n < 0 || ctx > room;
  return r;
}

__global__ void __launch_bounds__(kThreads) step_metadata_kernel(const MetaArgs a) {
  extern __shared__ int lds[];
  int* cu = lds;                   // [batch + 1]
  int* base = cu + a.batch + 1;    // [batch + 1]
  int* cached = base + a.batch + 1;
  __shared__ int part[2][kThreads / 64];
  __shared__ int outcome[2];
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  const int per = (a.batch + kThreads - 1) / kThreads;
  const int i0 = min(tid * per, a.batch), i1 = min(i0 + per, a.batch);

  int sum_n = 0, sum_b = 0;
  for (int i = i0; i < i1; ++i) {
    const Request r = request(a, i);
    sum_n = add_sat(sum_n, r.fresh);
    sum_b = add_sat(sum_b, r.need - r.held);
  }
  int run_n = sum_n, run_b = sum_b;  // inclusive over the wave
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int n = __shfl_up(run_n, off), b = __shfl_up(run_b, off);
    if (lane >= off) run_n = add_sat(run_n, n), run_b = add_sat(run_b, b);
  }
  if (lane == 63) part[0][wave] = run_n, part[1][wave] = run_b;
  if (tid == 0) outcome[0] = 0, outcome[1] = kMaxInt;
  __syncthreads();
  const int start = a.free_start == nullptr ? 0 : *a.free_start;
  // exclusive: the sums in front of this thread's requests
  int at_n = __shfl_up(run_n, 1), at_b = __shfl_up(run_b, 1);
  if (lane == 0) at_n = at_b = 0;
  for (int w = 0; w < wave; ++w) at_n = add_sat(at_n, part[0][w]), at_b = add_sat(at_b, part[1][w]);
  at_b = add_sat(at_b, max(start, 0));
  int longest = 0, first_bad = kMaxInt;
  for (int i = i0; i < i1; ++i) {
    const Request r = request(a, i);
    cu[i] = at_n;
    base[i] = at_b;
    cached[i] = r.cached;
    at_n = add_sat(at_n, r.fresh);
    at_b = add_sat(at_b, r.need - r.held);
    const int ctx = add_sat(r.cached, r.fresh);
    longest = max(longest, ctx);
    if (r.bad || at_n > a.num_tokens || at_b > a.num_free || start < 0) first_bad = min(first_bad, i);
    if (blockIdx.x == 0) {
      a.cu[i + 1] = at_n;
      a.ctx[i] = ctx;
    }
    if (i == a.batch - 1) cu[a.batch] = at_n, base[a.batch] = at_b;
  }
  if (blockIdx.x == 0) {
    atomicMax(&outcome[0], longest);
    atomicMin(&outcome[1], first_bad);
  }
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) {
    a.cu[0] = 0;
    a.tail[0] = outcome[0];
    a.tail[1] = a.batch > 0 ? base[a.batch] : max(start, 0);
    a.tail[2] = outcome[1];
  }

  // the block of entry w of request i, which holds `held` blocks
  auto block_of = [&](int i, int w, int held) {
    if (w < held) return a.tables[static_cast<int64_t>(i) * a.t_sb + static_cast<int64_t>(w) * a.t_sw];
    const int64_t e = static_cast<int64_t>(base[i]) + (w - held);
    return e < a.num_free ? a.free[e] : -1;
  };
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  const int64_t me = static_cast<int64_t>(blockIdx.x) * kThreads + tid;
  const int64_t token_quads = (static_cast<int64_t>(a.num_tokens) + 3) / 4;
  const int total = a.batch > 0 ? cu[a.batch] : 0;
  for (int64_t x = me; x < token_quads; x += step) {
    const int t0 = static_cast<int>(4 * x);
    int i = 0;  // last request that starts at or before t0
    if (t0 < total) {
      int lo = 0, hi = a.batch;
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (cu[mid] <= t0) lo = mid;
        else hi = mid;
      }
      i = lo;
    }
    int slot[4], position[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      slot[j] = -1;
      position[j] = 0;
      const int t = t0 + j;
      if (t >= total || t < t0) continue;
      while (cu[i + 1] <= t) ++i;
      const int64_t pos = static_cast<int64_t>(cached[i]) + (t - cu[i]);
      position[j] = static_cast<int>(min(pos, static_cast<int64_t>(kMaxInt)));
      const int64_t w = pos / a.page;
      if (w >= a.width) continue;
      const int held = static_cast<int>(min((static_cast<int64_t>(cached[i]) + a.page - 1) / a.page, static_cast<int64_t>(a.width)));
      const int id = block_of(i, static_cast<int>(w), held);
      const int64_t s = static_cast<int64_t>(id) * a.page + (pos - w * a.page);
      if (id >= 0 && s <= kMaxInt) slot[j] = static_cast<int>(s);
    }
    typedef int i32x4 __attribute__((ext_vector_type(4)));  // (the rows are padded to four entries)
    *reinterpret_cast<i32x4*>(a.slots + t0) = i32x4{slot[0], slot[1], slot[2], slot[3]};
    *reinterpret_cast<i32x4*>(a.positions + t0) = i32x4{position[0], position[1], position[2], position[3]};
  }
  const int64_t entries = static_cast<int64_t>(a.batch) * a.width;
  for (int64_t x = me; x < entries; x += step) {
    const int i = static_cast<int>(x / a.width), w = static_cast<int>(x - static_cast<int64_t>(i) * a.width);
    const Request r = request(a, i);
    a.out[x] = w < r.need || w < r.held ? block_of(i, w, r.held) : -1;
  }
}

int64_t padded(int64_t n) { return align_up(n, 4); }

}  // namespace

int preload_step_metadata() {
  hipFuncAttributes attr;
  return check_hip(hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(&step_metadata_kernel)), "preload_step_metadata");
}

}  // namespace prism

extern "C" int64_t prism_step_metadata_words(int batch, int width, int num_tokens) {
  using namespace prism;
  if (batch < 0 || width < 0 || num_tokens < 0) return 0;
  return 2 * padded(num_tokens) + padded(2 * static_cast<int64_t>(batch) + 4) + static_cast<int64_t>(batch) * width;
}

extern "C" int prism_step_metadata(const int32_t* block_tables, const int64_t bt_strides[2], const int32_t* cached_lens,
                                   const int32_t* query_lens, const int32_t* free_blocks, int num_free,
                                   const int32_t* free_start, int batch, int width, int block_size, int num_tokens,
                                   int32_t* packed, void* stream) {
  using namespace prism;
  clear_error();
  if (batch < 0 || width < 0 || block_size <= 0 || num_tokens < 0 || num_free < 0) {
    set_error("prism_step_metadata: invalid geometry");
    return PRISM_ERR_INVALID;
  }
  if (batch > kMaxBatch) {
    set_error("prism_step_metadata: at most %d requests per step, got %d", kMaxBatch, batch);
    return PRISM_ERR_LAYOUT;
  }
  if (!packed || !bt_strides || (batch > 0 && (!cached_lens || !query_lens)) || (batch > 0 && width > 0 && !block_tables) ||
      (num_free > 0 && !free_blocks)) {
    set_error("prism_step_metadata: null argument");
    return PRISM_ERR_INVALID;
  }
  if (!aligned(packed, 16)) {
    set_error("prism_step_metadata: the output must be 16-byte aligned");
    return PRISM_ERR_LAYOUT;
  }
  MetaArgs a{};
  a.tables = block_tables;
  a.t_sb = bt_strides[0], a.t_sw = bt_strides[1];
  a.cached = cached_lens;
  a.fresh = query_lens;
  a.free = free_blocks;
  a.free_start = free_start;
  a.num_free = num_free, a.batch = batch, a.width = width, a.page = block_size, a.num_tokens = num_tokens;
  a.slots = packed;
  a.positions = packed + padded(num_tokens);
  a.cu = packed + 2 * padded(num_tokens);
  a.ctx = a.cu + batch + 1;
  a.tail = a.ctx + batch;
  a.out = a.cu + padded(2 * static_cast<int64_t>(batch) + 4);
  const int64_t work = std::max<int64_t>(ceil_div(num_tokens, 4), static_cast<int64_t>(batch) * width);
  const int64_t grid = std::min<int64_t>(std::max<int64_t>(ceil_div(work, kThreads), 1), 4 * device_cu_count());
  const size_t lds = (3 * static_cast<size_t>(batch) + 2) * sizeof(int);
  if (lds > 64 * 1024)
    if (int rc = check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(&step_metadata_kernel),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)),
                           "prism_step_metadata"))
      return rc;
  hipLaunchKernelGGL(step_metadata_kernel, dim3(static_cast<unsigned>(grid)), dim3(kThreads), lds, static_cast<hipStream_t>(stream), a);
  return check_launch("step_metadata_kernel launch");
}
