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
// in LDS), then writes its share of the tokens and of the tables.  A second
// launch, or a grid that waits for one scan, would cost more than the repeated
// scans, whose loads hit the L2.  The kernel is a chain of two loads (lengths,
// block ids) and what is between them: divisions by the block size are
// multiplications, and the scan goes by DPP.  64 requests of one token 3.5 us, 32
// prompts of 32k tokens 4.0, 1024 requests of 130k tokens and 524k table entries
// 5.9 (the scan alone 2.6, 2.8 and 3.6); with 64-bit divisions, scans through LDS
// and an atomic per lane 9.6, 9.8 and 14.8.
#include "common.h"
#include "divide.h"
#include "wave_ops.h"

#include <algorithm>

namespace prism {
namespace {

constexpr int kMaxThreads = 1024;
constexpr int kMaxBatch = 8192;  // three words of LDS each
constexpr int kMaxInt = 0x7FFFFFFF;
constexpr int kMostItems = kMaxInt - 64;  // tokens, table steps

typedef int i32x4 __attribute__((ext_vector_type(4)));

struct MetaArgs {
  const int32_t* tables;
  int64_t t_sb, t_sw;
  const int32_t* cached;
  const int32_t* fresh;
  const int32_t* free;
  const int32_t* free_start;
  int num_free, batch, width, page, num_tokens;
  Divisor by_page, by_row;  // by_row: entries of a table row, in steps of `wide`
  int wide;                 // table entries per thread: 4 where rows hold whole quads, else 1
  int quads;                // of the tables: a thread's four entries can be loaded at once, they start on 16 bytes
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

struct AddSat {
  __device__ int operator()(int x, int y) const { return add_sat(x, y); }
};

// Blocks of n tokens, at most a table row.
__device__ __forceinline__ int blocks_of(const MetaArgs& a, int n) {
  return n == 0 ? 0 : min(divide(n - 1, a.by_page) + 1, a.width);
}

struct Request {
  int cached, fresh, taken;  // taken: free blocks
  bool bad;
};

// Lengths that cannot be are taken as the nearest that can, and reported.
__device__ __forceinline__ Request request(const MetaArgs& a, int i) {
  const int c = a.cached[i], n = a.fresh[i];
  Request r;
  r.cached = max(c, 0);
  r.fresh = max(n, 0);
  r.taken = blocks_of(a, add_sat(r.cached, r.fresh)) - blocks_of(a, r.cached);
  const int64_t ctx = static_cast<int64_t>(r.cached) + r.fresh;
  r.bad = c < 0 || n < 0 || ctx > static_cast<int64_t>(a.width) * a.page || ctx > kMaxInt;
  return r;
}

__global__ void __launch_bounds__(kMaxThreads) step_metadata_kernel(const MetaArgs a) {
  extern __shared__ int lds[];
  int* cu = lds;                         // [batch + 1]
  int* base = cu + a.batch + 1;          // [batch + 1]: first free entry that the request takes
  int* cached = base + a.batch + 1;
  __shared__ int part[2][kMaxThreads / 64];
  __shared__ int outcome[2];
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, threads = blockDim.x;
  const int per = (a.batch + threads - 1) / threads;
  const int i0 = min(tid * per, a.batch), i1 = min(i0 + per, a.batch);
  const int start = a.free_start == nullptr ? 0 : *a.free_start;

  Request r{0, 0, 0, false};
  int sum_n = 0, sum_b = 0;
  for (int i = i0; i < i1; ++i) {
    r = request(a, i);
    sum_n = add_sat(sum_n, r.fresh);
    sum_b = add_sat(sum_b, r.taken);
  }
  const int run_n = wave_scan(sum_n, AddSat()), run_b = wave_scan(sum_b, AddSat());
  if (lane == 63) part[0][wave] = run_n, part[1][wave] = run_b;
  if (tid == 0) outcome[0] = 0, outcome[1] = kMaxInt;
  __syncthreads();
  // exclusive: the sums in front of this thread's requests
  int at_n = __builtin_amdgcn_update_dpp(0, run_n, 0x138, 0xF, 0xF, false);  // wave_shr:1
  int at_b = __builtin_amdgcn_update_dpp(0, run_b, 0x138, 0xF, 0xF, false);
  {  // (lane l holds wave l's sums)
    const bool front = lane < wave;
    at_n = add_sat(at_n, wave_reduce(front ? part[0][lane] : 0, AddSat()));
    at_b = add_sat(at_b, wave_reduce(front ? part[1][lane] : 0, AddSat()));
  }
  at_b = add_sat(at_b, max(start, 0));
  // (a first free entry behind the free blocks is none that a request took)
  const int last_free = min(max(a.num_free, start), kMaxInt - 1);
  int longest = 0, first_bad = kMaxInt;
  for (int i = i0; i < i1; ++i) {
    if (per > 1) r = request(a, i);
    cu[i] = at_n;
    base[i] = at_b;
    cached[i] = r.cached;
    at_n = add_sat(at_n, r.fresh);
    at_b = add_sat(at_b, r.taken);
    const int ctx = add_sat(r.cached, r.fresh);
    longest = max(longest, ctx);
    if (r.bad || at_n > a.num_tokens || at_b > last_free || start < 0) first_bad = min(first_bad, i);
    if (blockIdx.x == 0) {
      a.cu[i + 1] = at_n;
      a.ctx[i] = ctx;
    }
    if (i == a.batch - 1) cu[a.batch] = at_n, base[a.batch] = at_b;
  }
  if (blockIdx.x == 0) {  // (one atomic a wave: the lanes' would go one by one)
    longest = wave_reduce(longest, Max());
    first_bad = kMaxInt - wave_reduce(kMaxInt - first_bad, Max());
    if (lane == 0) atomicMax(&outcome[0], longest), atomicMin(&outcome[1], first_bad);
  }
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) {
    a.cu[0] = 0;
    a.tail[0] = outcome[0];
    a.tail[1] = a.batch > 0 ? base[a.batch] : max(start, 0);
    a.tail[2] = outcome[1];
  }

  // Entry w of request i, which holds `held` blocks: where it is, or null.
  auto entry = [&](int i, int w, int held) -> const int32_t* {
    const int64_t e = static_cast<int64_t>(base[i]) + (w - held);
    if (w < held) return a.tables + static_cast<int64_t>(i) * a.t_sb + static_cast<int64_t>(w) * a.t_sw;
    return e < a.num_free ? a.free + e : nullptr;
  };
  // Tokens first, then steps of the tables: an item per thread, so that the
  // loads of both are under way together.  (Whole waves of either kind: one that
  // held both would do them in turn.)
  const int per_row = a.width / a.wide, steps = a.batch * per_row, total = a.batch > 0 ? cu[a.batch] : 0;
  const int64_t table0 = (static_cast<int64_t>(a.num_tokens) + 63) / 64 * 64;
  const int64_t step = static_cast<int64_t>(gridDim.x) * threads;
  for (int64_t x = static_cast<int64_t>(blockIdx.x) * threads + tid; x < table0 + steps; x += step) {
    if (x < table0) {
      const int t = static_cast<int>(min(x, static_cast<int64_t>(kMaxInt)));
      if (t >= a.num_tokens) continue;
      int slot = -1, position = 0;
      if (t < total) {
        int i = 0, n = a.batch;  // the last request that starts at or before t is among n from i on
        while (n > 1) {
          const int q = (n + 3) / 4;
          const int c1 = cu[min(i + q, a.batch)], c2 = cu[min(i + 2 * q, a.batch)], c3 = cu[min(i + 3 * q, a.batch)];
          const int past = (c1 <= t) + (c2 <= t) + (c3 <= t);
          i += past * q;
          n = past < 3 ? q : n - 3 * q;
        }
        const int held = blocks_of(a, cached[i]);
        position = add_sat(cached[i], t - cu[i]);
        const int w = divide(position, a.by_page);
        const int32_t* at = w < a.width ? entry(i, w, held) : nullptr;
        const int id = at != nullptr ? *at : -1;
        const int64_t s = static_cast<int64_t>(id) * a.page + (position - w * a.page);
        if (id >= 0 && s <= kMaxInt) slot = static_cast<int>(s);
      }
      a.slots[t] = slot;
      a.positions[t] = position;
      continue;
    }
    const int y = static_cast<int>(x - table0), i = divide(y, a.by_row), w0 = (y - i * per_row) * a.wide;
    const int held = blocks_of(a, cached[i]), need = held + (base[i + 1] - base[i]);
    const int32_t* at[4] = {nullptr, nullptr, nullptr, nullptr};
    int32_t* dst = a.out + static_cast<int64_t>(i) * a.width + w0;
    i32x4 id = {-1, -1, -1, -1};
    if (a.quads && w0 + 4 <= held) {
      id = *reinterpret_cast<const i32x4*>(a.tables + static_cast<int64_t>(i) * a.t_sb + w0);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < a.wide && w0 + j < need) at[j] = entry(i, w0 + j, held);
#pragma unroll
      for (int j = 0; j < 4; ++j) id[j] = at[j] != nullptr ? *at[j] : -1;
    }
    if (a.wide == 4) *reinterpret_cast<i32x4*>(dst) = id;
    else *dst = id[0];
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
  const int64_t table_steps = static_cast<int64_t>(batch) * (width % 4 == 0 ? width / 4 : width);
  if (num_tokens > kMostItems || table_steps > kMostItems) {
    set_error("prism_step_metadata: too many tokens or table entries for one step");
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
  a.wide = width > 0 && width % 4 == 0 ? 4 : 1;
  a.quads = a.wide == 4 && a.t_sw == 1 && a.t_sb % 4 == 0 && aligned(block_tables, 16);
  a.by_page = divisor(block_size);
  a.by_row = divisor(std::max(width / a.wide, 1));
  a.slots = packed;
  a.positions = packed + padded(num_tokens);
  a.cu = packed + 2 * padded(num_tokens);
  a.ctx = a.cu + batch + 1;
  a.tail = a.ctx + batch;
  a.out = a.cu + padded(2 * static_cast<int64_t>(batch) + 4);
  // one request per thread where a workgroup can hold them; two workgroups of 1024 threads fill a CU
  const int threads = batch <= 256 ? 256 : batch <= 512 ? 512 : kMaxThreads;
  const int64_t work = align_up(num_tokens, 64) + table_steps;
  const int64_t most = static_cast<int64_t>(device_cu_count()) * 2048 / threads;
  const int64_t grid = std::min<int64_t>(std::max<int64_t>(ceil_div(work, threads), 1), most);
  const size_t lds = (3 * static_cast<size_t>(batch) + 2) * sizeof(int);
  if (lds > 64 * 1024)
    if (int rc = check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(&step_metadata_kernel),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)),
                           "prism_step_metadata"))
      return rc;
  hipLaunchKernelGGL(step_metadata_kernel, dim3(static_cast<unsigned>(grid)), dim3(threads), lds, static_cast<hipStream_t>(stream), a);
  return check_launch("step_metadata_kernel launch");
}
