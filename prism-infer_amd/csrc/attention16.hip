// Causal attention over 16-bit keys and values: whole prompts whose K/V are
// packed like their queries, and chunks of new tokens over a paged cache.
//
//   o[j, h] = sum_{t <= p} w_t v[t, h / G],  w = softmax_t(scale q[j, h] . k[t, h / G]),  p = klen - qlen + j
//
// for token j of a sequence of qlen queries and klen keys (its last qlen tokens
// are the queries'); a row that sees no key (p < 0) is 0, one whose visible
// scores are all -inf is 0 / 0, NaN.
//
// Work layout.  The G query heads of a kv head share its keys, so the rows of
// one kv head are (token, head in the group) pairs, token major: any group size
// and any chunk length fill the columns of the MFMAs.  A workgroup owns a block
// of kRows of these rows of one sequence and kv head, a wave 32 of them.  Tiles
// of 64 keys go through LDS, loaded there directly.
//
// Per tile a wave computes S^T = K Q^T with 32x32x16 MFMAs: a row is one lane
// column from the scores to the output, so its running max, its sum and the
// rescaling of its accumulators are lane-local.  P^T, rounded to the cache's
// type (weights of at most 2^8, in float16 2^15, against fp32 sums), is the B
// operand of O^T += V^T P^T as it stands, V^T comes from ds_read_b64_tr_b16.
//
// Bound by the MFMAs (busy 71% of the cycles) and the exponentials beside them: a
// wave's tile is 32 MFMAs of 32 cycles and about 112 VALU instructions, 32 of
// them exponentials of 16 cycles, and two waves share a SIMD.  With the three
// parts of a tile one after the other 2 x 8192 tokens (32 / 8 heads) took 1414
// us; with the next tile's scores and the last one's output beside the softmax
// 946 to 1004 (1095 to 1162 TFLOP/s, 0.9 of a large library product on the same
// card).  Prompts of one to three tiles are bound by what is around the loop:
// lookup, first loads and scores, last values, stores (80 prompts of 100 tokens,
// 64 / 8 heads: 133 us with loads and stores of parts of lines, dependent reads in
// the last product and a division per use, 74 now).
#include "common.h"
#include "divide.h"
#include "wave_ops.h"

#include <algorithm>

namespace prism {
namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int kKeys = 64;              // keys per tile
constexpr int kWaves = 4;              // per group of waves
constexpr int kMostKeys = 0x7FFFF000;  // of a sequence: positions a few tiles further fit in 32 bits
constexpr int kMostRows = 1 << 29;     // of a kv head: sums of blocks over 256 sequences fit in 32 bits
constexpr int kCols = 32;              // rows per wave: the columns of a 32x32 MFMA

// Where keys come from: packed like the queries, pages that hold whole tiles,
// or pages of a multiple of 16 keys.
enum Source { kPacked, kPages, kSmallPages };

struct AttnArgs {
  const uint16_t* q;
  int64_t q_st, q_sh;  // strides in elements (dim stride 1)
  const uint16_t* k;
  const uint16_t* v;
  int64_t k_sn, k_st, k_sh, v_sn, v_st, v_sh;  // page, token, head
  const int32_t* bt;
  int64_t bt_sb, bt_sn;
  const int32_t* ctx;   // paged: keys of each sequence
  const int32_t* cu_q;
  const int32_t* cu_k;  // packed; null over pages
  uint16_t* out;
  int64_t o_st, o_sh;
  int batch, heads, kv_heads, group, page, num_blocks, width, total_q, total_k;
  float scale_log2;
  int* status;
  int* report;  // pinned, or null: [0] set to 1 where a sequence is flagged, [1] and [2] the packed rows' extent, [3] set
                // to 1 once these are known
  Divisor by_group, by_kv_heads;
  int slots;      // workgroups that the chip holds at once
  int room;       // of one kv head
  uint8_t* work;  // scratch of split blocks (SplitScratch), or null: no block is split
};

// A block whose keys are split: its rows, and where its parts are.
struct SplitBlock {
  int qs, row0, rows, head, slot, parts;
};

// Scratch of split blocks: how many there are, their descriptions, then the
// parts by slot, kRows rows of fp32 outputs (unnormalised) and (max, sum).
constexpr int kBlockRows = kCols * kWaves;
struct SplitScratch {
  int* count;
  SplitBlock* blocks;
  float* out;
  float* ml;
  __host__ __device__ SplitScratch(uint8_t* p, int slots, int dim) {
    count = reinterpret_cast<int*>(p);
    blocks = reinterpret_cast<SplitBlock*>(p + 256);
    out = reinterpret_cast<float*>(p + blocks_end(slots));
    ml = out + static_cast<int64_t>(slots) * kBlockRows * dim;
  }
  static __host__ __device__ int64_t blocks_end(int slots) { return 256 + (static_cast<int64_t>(slots) * sizeof(SplitBlock) + 255) / 256 * 256; }
  static int64_t bytes(int slots, int dim) { return blocks_end(slots) + static_cast<int64_t>(slots) * kBlockRows * (dim + 2) * 4; }
};

template <bool F16>
struct Type;
// kShift: weights are 2^kShift times exp(score - max) (the running max is kept less by
// kShift, sums and outputs carry the same factor).  kSumLimit: largest sum of a
// lane's 32 weights that keeps the running max, 8 times what the max itself allows.
template <>
struct Type<false> {
  typedef bf16x8 vec;
  static constexpr uint32_t kInf = 0x7F80u;
  static constexpr float kShift = 0.f, kSumLimit = 256.f;
  static __device__ __forceinline__ floatx16 mfma(vec a, vec b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
// float16 ends at 2^-24 and at 65504: the factor takes weights that small down to
// 2^-31 of the max (40000 keys of 2^-24.6 beside one of 1 were off by half otherwise),
// and the limit keeps every weight finite.
template <>
struct Type<true> {
  typedef f16x8 vec;
  static constexpr uint32_t kInf = 0x7C00u;
  static constexpr float kShift = 7.f, kSumLimit = 32768.f;
  static __device__ __forceinline__ floatx16 mfma(vec a, vec b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*)p));
}

__device__ __forceinline__ const uint8_t* uniform_ptr(const void* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
  return reinterpret_cast<const uint8_t*>((static_cast<uint64_t>(hi) << 32) | lo);
}

struct Seq {
  int q0, qlen, k0, klen;
};

__device__ __forceinline__ void flag_sequence(const AttnArgs& a, int i) {
  atomicMin(a.status, i);
  if (a.report != nullptr) a.report[0] = 1;  // (every writer stores the same)
}

// Rows and keys of K sequences from i on; good: whether their lengths are valid
// (packed: offsets in order and inside the tensors).  Others are out of the work.
template <int SRC, int K>
__device__ __forceinline__ void sequences(const AttnArgs& a, int i, Seq (&s)[K], bool (&good)[K]) {
  int q[K + 1], k[K + 1];
#pragma unroll
  for (int j = 0; j <= K; ++j) {
    q[j] = a.cu_q[min(i + j, a.batch)];
    if (SRC == kPacked) k[j] = a.cu_k[min(i + j, a.batch)];
    else k[j] = a.ctx[min(i + j, a.batch - 1)];
  }
#pragma unroll
  for (int j = 0; j < K; ++j) {
    s[j] = SRC == kPacked ? Seq{q[j], q[j + 1] - q[j], k[j], k[j + 1] - k[j]} : Seq{q[j], q[j + 1] - q[j], 0, k[j]};
    good[j] = i + j < a.batch && q[j] >= 0 && q[j + 1] >= q[j] && q[j + 1] <= a.total_q && s[j].klen <= kMostKeys;
    if (SRC == kPacked) good[j] = good[j] && k[j] >= 0 && k[j + 1] >= k[j] && k[j + 1] <= a.total_k;
    else good[j] = good[j] && q[j + 1] > q[j] && s[j].klen >= s[j].qlen && s[j].klen <= static_cast<int64_t>(a.width) * a.page;
  }
}

constexpr int kMinPart = 4;  // tiles

// Time of a launch of `wgs` workgroups, in units of 64 ns, whose longest walks
// `tiles` tiles (1.1 us each, 1.9 where the CUs hold two workgroups); of split
// blocks, the parts' rows in fp32 and the second launch.  Not split and split, us:
// one token behind 700 keys 14.8 and 11.4, behind 12000 153 and 21, 200 tokens of
// two sequences behind 4000 63.9 and 46.3 (32 / 8 heads); behind 700 19.9 and 30.5.
__device__ inline int split_cost(const AttnArgs& a, int tiles, int wgs, bool split) {
  const int tile = 2 * wgs > a.slots ? 30 : 17;
  return tiles * tile + (split ? 90 + wgs / 3 : 0);
}

struct Work {
  int seq, block, head;
  int part, parts;     // of the block's keys
  int total;           // workgroups of one kv head
  int split;           // 0, or its blocks where some are split: then
  int index, slot;     // the block's number among them, and its first part's among all parts
  Seq s;
};

// Workgroup -> its work, heads fastest, so that with 8 kv heads each XCD reads
// one head's K/V.  K sequences per lane, all in registers, for batches of up to
// 64 K: one load of the offsets, then wave reductions.
//
// Up to 64 sequences with more blocks than the chip holds at once: blocks with
// most keys go first, so that the launch ends on short ones.  Block j of a
// sequence ends after about (level + j) ROWS / G keys, a binary search over levels
// finds the rank's level, a scan over the sequences with a block there its
// sequence.  Otherwise sequence by sequence, in reverse.  us by levels and in
// reverse (32 / 8 heads): 6 prompts of 61 to 1900 tokens 139.5 and 142, 20 of them
// 182.5 and 184.5; but 4 x 2048 tokens behind 8192 1089 and 1080, 40 prompts of 500
// to 3000 1359 and 1214, 64 of 100 to 1900 897 and 796: many sequences' blocks side by
// side share fewer keys in the L2.
//
// Where blocks are few and long their keys are split: into parts of the fewest
// tiles for which all parts fit the chip at once, if that pays.
// Returns false for a workgroup beyond the real blocks.
template <int SRC, int ROWS, int K>
__device__ __forceinline__ bool locate(const AttnArgs& a, int me, bool flag, Work& w) {
  const int lane = __lane_id();
  int rank = divide(me, a.by_kv_heads);
  w.head = me - rank * a.kv_heads;
  w.part = w.split = 0;
  w.parts = 1;
  Seq s[K];
  bool good[K];
  sequences<SRC, K>(a, lane * K, s, good);
  int n[K], l0[K], blocks = 0, top = 0, longest = 0;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    n[k] = good[k] ? (s[k].qlen * a.group + ROWS - 1) / ROWS : 0;
    l0[k] = 1 + static_cast<int>(min(static_cast<int64_t>(max(s[k].klen - s[k].qlen, 0)) * a.group / ROWS, static_cast<int64_t>(1 << 29)));
    if (SRC != kPacked && flag && !good[k] && lane * K + k < a.batch) flag_sequence(a, lane * K + k);
    blocks += n[k];
    top = max(top, n[k] == 0 ? 0 : l0[k] + n[k]);
    longest = max(longest, n[k] == 0 ? 0 : (s[k].klen - 1) / kKeys + 1);
  }
  w.total = wave_reduce(blocks, Add());
  int hit_k = 0, l = 0;
  // parts of a sequence's blocks (more than the chip holds: any number)
  auto parts_of = [&](int klen, int tiles) {
    const int part = (klen - 1) / kKeys / tiles + 1;
    return min(max(part, 1), 1 << 16);
  };
  auto total_parts = [&](int tiles) {
    int sum = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) sum += n[k] * parts_of(s[k].klen, tiles);
    return wave_reduce(sum, Add());
  };
  int tiles = 0;  // of a part
  if (a.work != nullptr && w.total > 0 && w.total < a.room) {
    longest = wave_reduce(longest, Max());
    int lo = kMinPart, hi = max(longest, kMinPart);
    while (lo < hi) {  // fewest tiles for which the parts fit
      const int mid = (lo + hi) / 2;
      if (total_parts(mid) <= a.room) hi = mid;
      else lo = mid + 1;
    }
    const int all = total_parts(lo);
    if (all > w.total && split_cost(a, lo, all * a.kv_heads, true) < split_cost(a, longest, w.total * a.kv_heads, false)) tiles = lo;
    if (tiles > 0) {
      w.split = w.total;
      w.total = all;
      if (rank >= all) return false;
      int mine = 0, before = 0;  // parts and blocks of the lane's sequences
#pragma unroll
      for (int k = 0; k < K; ++k) mine += n[k] * parts_of(s[k].klen, tiles);
      const int incl = wave_scan(mine, Add()), incl_blocks = wave_scan(blocks, Add());
      l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(incl > rank));
      rank -= uniform_int(__builtin_amdgcn_readlane(incl - mine, l));
      int slot = __builtin_amdgcn_readlane(incl - mine, l);
      before = __builtin_amdgcn_readlane(incl_blocks - blocks, l);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int nk = __builtin_amdgcn_readlane(n[k], l);
        const int parts = parts_of(__builtin_amdgcn_readlane(s[k].klen, l), tiles);
        if (rank >= 0 && rank < nk * parts) {
          hit_k = k;
          w.block = rank / parts;
          w.part = rank - w.block * parts;
          w.parts = parts;
          w.slot = slot + w.block * parts;
          w.index = before + w.block;
        }
        rank -= nk * parts;  // (below 0 once found)
        slot += nk * parts;
        before += nk;
      }
    }
  }
  if (tiles == 0) {
    if (rank >= w.total) return false;
    if (K > 1 || w.total <= a.room) {  // all start at once, or many are short: sequence by sequence, in reverse
      const int left = w.total - 1 - rank, incl = wave_scan(blocks, Add());
      l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(incl > left));
      w.block = left - __builtin_amdgcn_readlane(incl - blocks, l);
#pragma unroll
      for (int k = 0; k + 1 < K; ++k) {
        const int nk = __builtin_amdgcn_readlane(n[k], l);
        if (hit_k == k && w.block >= nk) {
          w.block -= nk;
          hit_k = k + 1;
        }
      }
    } else {
      auto above = [&](int u) { return wave_reduce(min(max(l0[0] + n[0] - 1 - max(u, l0[0] - 1), 0), n[0]), Add()); };
      int lo = 0, hi = wave_reduce(top, Max());
      while (lo < hi) {  // smallest level with at most `rank` blocks above it
        const int mid = (lo + hi) / 2;
        if (above(mid) <= rank) hi = mid;
        else lo = mid + 1;
      }
      const int at = n[0] > 0 && lo >= l0[0] && lo < l0[0] + n[0] ? 1 : 0;
      const int left = rank - above(lo), incl = wave_scan(at, Add());
      l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(incl > left));
      w.block = lo - __builtin_amdgcn_readlane(l0[0], l);
    }
  }
  w.seq = l * K + hit_k;
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (k == hit_k)
      w.s = Seq{__builtin_amdgcn_readlane(s[k].q0, l), __builtin_amdgcn_readlane(s[k].qlen, l),
                __builtin_amdgcn_readlane(s[k].k0, l), __builtin_amdgcn_readlane(s[k].klen, l)};
  return true;
}

// Larger batches: sequence by sequence, in reverse, nothing split.
template <int SRC, int ROWS>
__device__ __forceinline__ bool locate_many(const AttnArgs& a, int me, bool flag, Work& w) {
  const int lane = __lane_id();
  const int rank = divide(me, a.by_kv_heads);
  w.head = me - rank * a.kv_heads;
  w.part = w.split = 0;
  w.parts = 1;
  auto blocks_of = [&](int i, Seq& s, bool report) {
    Seq one[1];
    bool good[1];
    sequences<SRC, 1>(a, i, one, good);
    s = one[0];
    if (SRC != kPacked && report && !good[0] && i < a.batch) flag_sequence(a, i);
    return good[0] ? (s.qlen * a.group + ROWS - 1) / ROWS : 0;
  };
  w.total = 0;
  Seq s;
  // (sequences that overlap could make any number of blocks)
  for (int base = 0; base < a.batch; base += 64) w.total = min(w.total + wave_reduce(blocks_of(base + lane, s, flag), Add()), 1 << 30);
  const int target = w.total - 1 - rank;
  if (target < 0) return false;
  int before = 0;
  for (int base = 0; base < a.batch; base += 64) {
    const int n = blocks_of(base + lane, s, false);
    const int incl = wave_scan(n, Add()) + before;  // (at most 2^28 beyond the total's limit)
    const uint64_t hit = __builtin_amdgcn_ballot_w64(target < incl && target >= incl - n);
    if (hit != 0) {
      const int l = __builtin_ctzll(hit);
      w.seq = base + l;
      w.block = target - __builtin_amdgcn_readlane(incl - n, l);
      w.s = Seq{__builtin_amdgcn_readlane(s.q0, l), __builtin_amdgcn_readlane(s.qlen, l), __builtin_amdgcn_readlane(s.k0, l),
                __builtin_amdgcn_readlane(s.klen, l)};
      return true;
    }
    before = __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

// The outcome that a host waits for, from the first workgroup alone and long
// before the others are done: every sequence's lengths and block ids.  Threads
// are spread over the sequences first, then over a sequence's pages.
template <int SRC>
__device__ void check_metadata(const AttnArgs& a, int& first_bad) {  // (in LDS)
  constexpr int kAtOnce = 8;
  const int tid = threadIdx.x, threads = blockDim.x;
  if (tid == 0) first_bad = INT32_MAX;
  __syncthreads();
  int across = 1;  // sequences at a time
  while (across < a.batch && across < threads) across *= 2;
  for (int i = tid & (across - 1); i < a.batch; i += across) {
    Seq s[1];
    bool good[1];
    sequences<SRC, 1>(a, i, s, good);
    const int pages = good[0] ? (s[0].klen - 1) / a.page + 1 : 0;
    for (int p = tid / across; p < pages; p += kAtOnce * (threads / across)) {
      int id[kAtOnce];
#pragma unroll
      for (int x = 0; x < kAtOnce; ++x)
        id[x] = a.bt[static_cast<int64_t>(i) * a.bt_sb + static_cast<int64_t>(min(p + x * (threads / across), pages - 1)) * a.bt_sn];
#pragma unroll
      for (int x = 0; x < kAtOnce; ++x) good[0] = good[0] && id[x] >= 0 && id[x] < a.num_blocks;
    }
    if (!good[0]) atomicMin(&first_bad, i);
  }
  __syncthreads();
  if (tid != 0) return;
  if (first_bad != INT32_MAX) flag_sequence(a, first_bad);
  a.report[1] = a.cu_q[0];
  a.report[2] = a.cu_q[a.batch];
  __hip_atomic_store(a.report + 3, 1, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_SYSTEM);
}

// Rows outside every sequence are 0: the workgroups beyond the real blocks
// (one per kv head at least) share them.
template <int D>
__device__ void zero_padding(const AttnArgs& a, int checks, int real_blocks) {
  const int first = min(max(a.cu_q[0], 0), a.total_q), end = min(max(a.cu_q[a.batch], first), a.total_q);
  const int64_t others = checks + static_cast<int64_t>(real_blocks) * a.kv_heads;
  const int64_t me = blockIdx.x - others, workers = gridDim.x - others;
  const int64_t per_row = static_cast<int64_t>(a.heads) * (D / 8);
  const int64_t chunks = (first + (a.total_q - end)) * per_row;
  for (int64_t x = me * blockDim.x + threadIdx.x; x < chunks; x += workers * blockDim.x) {
    int64_t row = x / per_row;
    const int rest = static_cast<int>(x - row * per_row);
    if (row >= first) row += end - first;
    *reinterpret_cast<u32x4*>(a.out + row * a.o_st + rest / (D / 8) * a.o_sh + rest % (D / 8) * 8) = u32x4{0, 0, 0, 0};
  }
}

// 16-byte chunk swizzle of key t's row in LDS: chunk x holds the row's chunk
// x ^ swz(t).  64 banks of 4 bytes; ds_read_b128 serves 16 lanes at a time,
// ds_read_b64 (and _tr_b16) 32.  K reads (row c, chunk 2 x + g) then meet 16
// distinct chunks of a 256-byte span, V reads (4 rows, 4 chunks of each) all of
// it.  Rows of 64 dims are half a span: their parity is a chunk bit already.
template <int D>
__device__ __forceinline__ int swz(int t) {
  const int t0 = t & 1, t1 = (t >> 1) & 1, t2 = (t >> 2) & 1, t3 = (t >> 3) & 1;
  return D == 128 ? (t0 << 2) | (t1 << 3) | t2 | (t3 << 1) : (t1 << 2) | t2 | (t3 << 1);
}

// Two fp32 values -> two 16-bit ones, to nearest even.
template <bool F16>
__device__ __forceinline__ uint32_t pack(float lo, float up) {
  if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{lo, up}, f16x2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{lo, up}, bf16x2));
}

template <bool F16, int D, int SRC, int GROUPS>
__global__ void __launch_bounds__(64 * kWaves * GROUPS) __attribute__((amdgpu_waves_per_eu(2)))
attention16_kernel(const AttnArgs a) {
  using T = Type<F16>;
  typedef typename T::vec vec;
  constexpr int kRows = kBlockRows;
  constexpr int kRow = D * 2;                 // bytes of a key's row in LDS
  constexpr int kPayload = kKeys * kRow;      // a tile's K or V
  constexpr int kSteps = D / 16;              // MFMAs per 32 x 32 scores
  constexpr int kDims = D / 32;               // 32-dim tiles of the output
  constexpr int kPairs = D / 8;               // K operands of a tile, and V operands
  constexpr int kLoadRows = 1024 / kRow;      // rows per load of a wave
  constexpr int kLoads = kKeys / kLoadRows / kWaves;
  constexpr int kV = 2 * kPayload;            // two stages of K, then two of V
  constexpr int kShare = 4 * kPayload + 2 * kCols * kRow;  // of a group, with the last two waves' queries
  __shared__ __attribute__((aligned(256))) uint8_t lds[GROUPS * kShare];

  // With a report the first workgroups (one per kv head, which keeps the others'
  // XCDs) are the check's.
  const int checks = SRC != kPacked && a.report != nullptr ? a.kv_heads : 0;
  const int me = static_cast<int>(blockIdx.x) - checks;
  if (me < 0) {
    if (blockIdx.x == 0) check_metadata<SRC>(a, *reinterpret_cast<int*>(lds));
    return;
  }
  Work work;
  const bool first_wave = me == 0 && checks == 0 && threadIdx.x < 64;  // flags sequences
  const bool found = a.batch <= 64 ? locate<SRC, kRows, 1>(a, me, first_wave, work)
                     : a.batch <= 256 ? locate<SRC, kRows, 4>(a, me, first_wave, work) : locate_many<SRC, kRows>(a, me, first_wave, work);
  if (me == 0 && threadIdx.x == 0 && a.work != nullptr) *SplitScratch(a.work, a.slots, D).count = work.split * a.kv_heads;
  if (!found) {
    // (Its arguments are loaded anew: shared with the loop, they take scalar registers
    // there and pages' places spill; 2 chunks behind 12000 104 us, 106 with them shared.)
    auto* args = __builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(args));
    zero_padding<D>(*(const AttnArgs*)args, checks, work.total);
    return;
  }
  const int seq = uniform_int(work.seq), block = uniform_int(work.block), h = uniform_int(work.head);
  const int tid = threadIdx.x % (64 * kWaves);  // in the group
  const int wave = uniform_int(tid / 64);
  const int group = GROUPS == 1 ? 0 : uniform_int(threadIdx.x / (64 * kWaves));
  const int lane = tid % 64;
  const int c = lane % 32;
  const int g = lane / 32;

  const Seq s = work.s;
  const int qs = uniform_int(s.q0), qlen = uniform_int(s.qlen), klen = uniform_int(s.klen);
  const int prefix = klen - qlen;
  const int rows = qlen * a.group;
  const int row0 = block * kRows + wave * kCols;                               // the wave's first row
  const int kend = min(klen, prefix + divide(min((block + 1) * kRows, rows) - 1, a.by_group) + 1);  // keys [0, kend) are needed
  const int wpos0 = prefix + divide(row0, a.by_group);                      // position of the wave's first row
  const int wlast = row0 < rows ? prefix + divide(min(row0 + kCols, rows) - 1, a.by_group) : -1;  // and of its last
  // the group's tiles, and the wave's end
  const int part = uniform_int(work.part), parts = uniform_int(work.parts);
  const int all_tiles = kend > 0 ? (kend - 1) / kKeys + 1 : 0;
  int t0 = 0, t1 = all_tiles;
  if (parts > 1) {
    const int per_part = uniform_int((all_tiles + parts - 1) / parts);
    t0 = min(part * per_part, all_tiles);
    t1 = min(t0 + per_part, all_tiles);
  }
  const int steps = (t1 - t0 + GROUPS - 1) / GROUPS;  // tiles of a group, the same for the barriers of all
  if (GROUPS > 1) {
    t0 = min(t0 + group * steps, t1);
    t1 = min(t0 + steps, t1);
  }
  const int tw = wlast >= 0 ? min(t1, wlast / kKeys + 1) : 0;

  // ---- tile loads, straight into LDS.  A load of a wave covers kLoadRows rows;
  // row and swizzled chunk of a lane do not change from load to load.  Asm so
  // that the compiler's wait-count pass does not drain these loads before each
  // LDS read of another stage.
  const int lrow = wave * kLoadRows + lane / (64 / kLoadRows);
  const int lchunk = (lane % (64 / kLoadRows)) ^ swz<D>(lrow);
  const int k_st = static_cast<int>(a.k_st) * 2, v_st = static_cast<int>(a.v_st) * 2;  // bytes
  const uint8_t* k_head = reinterpret_cast<const uint8_t*>(a.k + static_cast<int64_t>(s.k0) * a.k_st + h * a.k_sh);
  const uint8_t* v_head = reinterpret_cast<const uint8_t*>(a.v + static_cast<int64_t>(s.k0) * a.v_st + h * a.v_sh);
  const int32_t* bt_row = SRC == kPacked ? nullptr : a.bt + static_cast<int64_t>(seq) * a.bt_sb;
  auto load_ids = [&](int base) { return bt_row[static_cast<int64_t>(min(base + lane, a.width - 1)) * a.bt_sn]; };
  // The table is walked tile by tile; 64 consecutive entries sit in one register.
  constexpr int kGroups = SRC == kSmallPages ? kKeys / 16 : 1;  // entries per tile
  struct Place {
    int blk[kGroups];  // pages, per 16 keys where a tile may lie in several (-1: not needed)
    int row;           // of the first key in its page
    bool ok;
  };
  int page = 0, page_row = 0, ids_base = 0, ids = 0;
  auto start_walk = [&]() {
    if constexpr (SRC != kPacked) {
      page = t0 == 0 ? 0 : uniform_int(t0 * kKeys / a.page);
      page_row = t0 * kKeys - page * a.page;
      ids_base = page;
      ids = load_ids(page);
    }
  };
  auto look_up = [&](int t) {
    Place p;
    p.ok = true;
    if constexpr (SRC != kPacked) {
      p.row = page_row;
#pragma unroll
      for (int x = 0; x < kGroups; ++x) {
        p.blk[x] = -1;
        if (SRC == kPages || t * kKeys + x * 16 < kend) {  // groups past the keys needed are not looked up
          if (page >= ids_base + 64) {
            ids_base = page;
            ids = load_ids(page);
          }
          p.blk[x] = __builtin_amdgcn_readlane(ids, page - ids_base);
          p.ok = p.ok && p.blk[x] >= 0 && p.blk[x] < a.num_blocks;
          page_row += kKeys / kGroups;
          if (page_row == a.page) {
            page_row = 0;
            ++page;
          }
        }
      }
      if (!p.ok && tid == 0) flag_sequence(a, seq);
    }
    return p;
  };
  auto load_chunks = [&](const uint8_t* base, uint32_t off, uint32_t dst) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 : : "v"(off), "s"(uniform_ptr(base)), "s"(dst) : "memory", "m0");
  };
  uint8_t* const share = lds + group * kShare;
  const uint32_t lds0 = lds_address(share);
  // Starts the loads of K or V of tile t into LDS offset `stage`.  (A tile that
  // cannot be loaded leaves the stage as it was: its sequence is flagged.)
  auto issue = [&](int t, const Place& place, bool isv, uint32_t stage) {
    if (!place.ok) return;
    const int st_bytes = isv ? v_st : k_st;
    const uint8_t* head_base = isv ? v_head : k_head;
    const int64_t page_bytes = (isv ? a.v_sn : a.k_sn) * 2;
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
      const int tr = l * kWaves * kLoadRows;  // first row of the waves' loads
      const uint8_t* base;
      int r;  // the lane's row from there
      if constexpr (SRC == kPacked) {
        base = head_base + static_cast<int64_t>(t * kKeys) * st_bytes;
        r = min(lrow + tr, klen - 1 - t * kKeys);  // (rows past the last key repeat it)
      } else {
        const int x = SRC == kPages ? 0 : uniform_int((tr + wave * kLoadRows) / 16);
        int b = place.blk[0], p = place.row + 16 * x;
#pragma unroll
        for (int y = 1; y < kGroups; ++y) {
          if (x == y) b = place.blk[y];
          if (p >= a.page) p -= a.page;
        }
        if (SRC == kSmallPages && b < 0) continue;
        p += tr - 16 * x;
        base = head_base + b * page_bytes + static_cast<int64_t>(p) * st_bytes;
        r = lrow;
      }
      load_chunks(base, static_cast<uint32_t>(r * st_bytes + lchunk * 16),
                  uniform_int(lds0 + stage + static_cast<uint32_t>(wave) * 1024 + static_cast<uint32_t>(tr) * kRow));
    }
  };

  // the first tiles' loads, then the queries'
  Place place[3] = {};  // of tiles t, t + 1 and t + 2
  if (t0 < t1) {
    start_walk();
    place[0] = look_up(t0);
    issue(t0, place[0], false, 0);
    issue(t0, place[0], true, kV + kPayload);
    if (t0 + 1 < t1) {
      place[1] = look_up(t0 + 1);
      issue(t0 + 1, place[1], false, kPayload);
    }
  }

  // The queries: whole rows through LDS (where V of the second tile goes, and
  // behind the stages), swizzled as K's.  (16 bytes a lane of 32 rows at a time, as
  // the MFMA wants them, take four loads per line: 80 prompts of 100 tokens 94 us, 87 now.)
  const int pos = row0 + c < rows ? prefix + divide(row0 + c, a.by_group) : -1;  // of the lane's row; below 0: it sees no key, or is none
  const uint32_t q_lds = wave < 2 ? kV + wave * kCols * kRow : 4 * kPayload + (wave - 2) * kCols * kRow;
#pragma unroll
  for (int l = 0; l < kCols / kLoadRows; ++l) {
    const int r = l * kLoadRows + lane / (64 / kLoadRows), row = min(row0 + r, rows - 1);
    const int tok = divide(row, a.by_group), head = h * a.group + (row - tok * a.group);
    const uint16_t* src = a.q + static_cast<int64_t>(qs + tok) * a.q_st + static_cast<int64_t>(head) * a.q_sh +
                          8 * ((lane % (64 / kLoadRows)) ^ swz<D>(r));
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
                 : : "v"(src), "s"(uniform_int(lds0 + q_lds + l * 1024)) : "memory", "m0");
  }

  vec qop[kSteps];
  const float scale = a.scale_log2 == 0.f ? 1.f : fabsf(a.scale_log2);

  // per-lane LDS offsets inside a stage; other chunks differ by an exclusive or
  const uint32_t k_rd = c * kRow + ((g ^ swz<D>(c)) << 4);
  uint32_t v_rd;
  {
    const int l16 = lane % 16, t = 4 * g + (l16 >> 2);
    v_rd = t * kRow + (((2 * ((lane / 16) % 2) + ((l16 & 3) >> 1)) ^ swz<D>(t)) << 4) + (l16 & 1) * 8;
  }
  auto read_k = [&](uint32_t stage, int pair) {  // pair: 32-key half, MFMA step
    const int b = pair / kSteps, x = pair % kSteps;
    return *reinterpret_cast<const u32x4*>(share + b * 32 * kRow + ((stage + k_rd) ^ (x << 5)));
  };
  // V^T operand: k-slots 8 g + 0..3 of 16-key group m are keys 16 m + 4 g + 0..3,
  // slots 8 g + 4..7 the keys 8 further, the order of the score rows
  auto read_v = [&](uint32_t stage, int pair) {  // pair: 16-key group m, 32-dim tile n
    const int m = pair / kDims, n = pair % kDims;
    union {
      s16x4 half[2];
      u32x4 w;
    } u;
#pragma unroll
    for (int x = 0; x < 2; ++x)
      u.half[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          reinterpret_cast<lds_s16x4*>(lds0 + ((stage + v_rd) ^ (n << 6) ^ (x << 5)) + (16 * m + 8 * x) * kRow));
    return u.w;
  };
  // keys that nobody sees, which may hold anything, as 0
  auto drop_unseen = [&](u32x4& w, int pair, int key0) {
    const int left = kend - key0 - 16 * (pair / kDims) - 4 * g;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const int j = 8 * (d / 2) + 2 * (d % 2);
      w[d] &= (j < left ? 0xFFFFu : 0u) | (j + 1 < left ? 0xFFFF0000u : 0u);
    }
  };

  floatx16 acc[kDims];  // O^T: dims 32 n + 8 (r / 4) + 4 g + r % 4 of the lane's row
  float m_run, l_run;
  auto reset = [&]() {
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
    m_run = pos >= 0 ? -INFINITY : 0.f;  // 0 of a row without a key, to the end: it does not count as rising, and is told by it
    l_run = 0.f;
  };
  auto scores_step = [&](int x, const u32x4& k, floatx16& sc) {
    if (x == 0)
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[r] = 0.f;
    sc = T::mfma(__builtin_bit_cast(vec, k), qop[x], sc);
  };
  auto output_step = [&](int pair, const u32x4& v, const u32x4 (&p)[4]) {
    acc[pair % kDims] = T::mfma(__builtin_bit_cast(vec, v), __builtin_bit_cast(vec, p[pair / kDims]), acc[pair % kDims]);
  };
  // Scores of keys that the lane's row does not see.
  auto mask = [&](int key0, floatx16 (&sc)[2]) {
    const int last = pos - key0 - 4 * g;  // last visible key, as a row offset of the lane
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[b][r] = 32 * b + 8 * (r / 4) + r % 4 <= last ? sc[b][r] : -INFINITY;
  };
  // Weights of a tile against its maxima, which the accumulators are rescaled to.
  auto settle = [&](const floatx16 (&sc)[2], u32x4 (&pa)[4], float& ps) {
    float tmax = fmaxf(sc[0][0], sc[1][0]);
#pragma unroll
    for (int r = 1; r < 16; ++r) tmax = fmaxf(tmax, fmaxf(sc[0][r], sc[1][r]));
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(tmax), __float_as_uint(tmax), false, false);
    tmax = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * scale - T::kShift;
    const float m_new = tmax > m_run ? tmax : m_run;
    // (no key seen: keep the accumulators, all zero, from (-inf) - (-inf))
    const float alpha = m_new > m_run ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.f;
    m_run = m_new;
    l_run *= alpha;
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[d][r] *= alpha;
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    ps = 0.f;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[b][r], scale, -m_use));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[b][r + 1], scale, -m_use));
        pa[2 * b + r / 8][r % 8 / 2] = pack<F16>(p0, p1);
        ps += p0 + p1;
      }
  };
  // (a wave meets the others' barriers by their number, wherever in its code it stands)
  auto barrier = [&]() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  };
  auto landed = [&]() { __builtin_amdgcn_s_waitcnt(0xF70); };  // vmcnt(0)

  // ---- the loop.  Iteration t takes the scores of tile t + 1 (MFMAs), the
  // softmax of tile t (VALU) and the product of tile t - 1's weights with its
  // values (MFMAs), which do not depend on each other.  An MFMA holds its wave
  // until the one before it is through, so they are laid out by hand, in slots
  // of one MFMA and the VALU work that fits beside it.
  reset();
  {
    uint32_t k_next = kPayload, v_prev = kV;  // stages of K of tile t + 1 and V of tile t - 1
    landed();
    barrier();
#pragma unroll
    for (int x = 0; x < kSteps; ++x) qop[x] = __builtin_bit_cast(vec, *reinterpret_cast<const u32x4*>(share + ((q_lds + k_rd) ^ (x << 5))));
    // The exponent's scale is positive, so that a masked score is -inf: a negative
    // one is the queries' sign, and with 0 all queries are 0, as they are without a row.
    if (a.scale_log2 <= 0.f || row0 + kCols > rows) {
      const uint32_t keep = a.scale_log2 == 0.f || row0 + c >= rows ? 0u : ~0u;
      const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u & keep : 0u;
#pragma unroll
      for (int x = 0; x < kSteps; ++x) {
        u32x4 w = __builtin_bit_cast(u32x4, qop[x]);
#pragma unroll
        for (int d = 0; d < 4; ++d) w[d] = (w[d] & keep) ^ flip;
        qop[x] = __builtin_bit_cast(vec, w);
      }
    }
    floatx16 sa[2], sb[2];
    u32x4 pa[4], pb[4];
    if (t0 < tw) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) scores_step(i % kSteps, read_k(0, i), sa[i / kSteps]);
    }
    // A wave's first tile: its weights, and the next scores where there is a next tile.
    auto first_tile = [&](floatx16 (&sc)[2], floatx16 (&sn)[2], u32x4 (&pn)[4]) {
      if (t0 + 1 < tw) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) scores_step(i % kSteps, read_k(k_next, i), sn[i / kSteps]);
      }
      if (t0 * kKeys + kKeys - 1 > wpos0) mask(t0 * kKeys, sc);
      // (Behind a condition that the compiler cannot see through, as on the other
      // tiles: without one the loop's registers spill, 80 of them.)
      int always = 1;
      asm volatile("" : "+s"(always));
      float ps = 0.f;
#pragma unroll
      for (int m = 0; m < 4; ++m) pn[m] = u32x4{0, 0, 0, 0};
      if (always) settle(sc, pn, ps);
      l_run += ps;
    };
    // Its tile t: weights pn from scores sc, next scores sn, output of tile t - 1
    // with weights pp.  Past the last tile the scores are taken from stale bytes,
    // for nothing.
    auto tile = [&](int t, floatx16 (&sc)[2], floatx16 (&sn)[2], u32x4 (&pp)[4], u32x4 (&pn)[4]) {
      constexpr int kPerSlot = 16 / kPairs;  // halves of a pair of weights beside an MFMA
      constexpr int kAhead = 1;              // operands are read this many pairs ahead
      uint32_t v_tile = v_prev;
      if constexpr (SRC != kPacked && D == 128) asm volatile("" : "+v"(v_tile));  // (hoisted, V's eight addresses spill)
      u32x4 kq[kAhead + 1], vq[kAhead + 1];
      float ps = 0.f, x1 = 0.f, e0 = 0.f;
      auto half = [&](int i) {
        const int m = i / 8, b = m / 2, r = m % 2 * 8 + i % 8 / 2 * 2;
        if (i % 2 == 0) {
          e0 = __builtin_amdgcn_exp2f(fmaf(sc[b][r], scale, -m_run));
          x1 = fmaf(sc[b][r + 1], scale, -m_run);
        } else {
          const float e1 = __builtin_amdgcn_exp2f(x1);
          pn[m][r % 8 / 2] = pack<F16>(e0, e1);
          ps += e0 + e1;
        }
      };
      if (t * kKeys + kKeys - 1 > wpos0) mask(t * kKeys, sc);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        kq[i] = read_k(k_next, i);
        vq[i] = read_v(v_tile, i);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        if (i + kAhead < kPairs) {
          kq[(i + kAhead) % (kAhead + 1)] = read_k(k_next, i + kAhead);
          vq[(i + kAhead) % (kAhead + 1)] = read_v(v_tile, i + kAhead);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (j == 0) scores_step(i % kSteps, kq[i % (kAhead + 1)], sn[i / kSteps]);
          else output_step(i, vq[i % (kAhead + 1)], pp);
#pragma unroll
          for (int y = 0; y < kPerSlot; ++y) half((2 * i + j) * kPerSlot + y);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      // The weights were formed against the running max as it stood; their sum tells
      // whether that was low enough, or is no number.  Only otherwise are maxima
      // taken.  (The pins keep the weights in front of the branch.)
      asm volatile("" : "+v"(ps), "+v"(pn[0]), "+v"(pn[1]), "+v"(pn[2]), "+v"(pn[3]));
      if (__builtin_amdgcn_ballot_w64(!(ps <= T::kSumLimit)) != 0) settle(sc, pn, ps);
      l_run += ps;
    };
    // The step that begins iteration t of every wave: K of tile t + 1 and V of
    // tile t - 1 have landed for all; K of tile t + 2 and V of tile t go where K
    // of tile t and V of tile t - 2 were, which every wave is done with.
    auto begin = [&](int t) {
      landed();
      barrier();
      if (t + 2 < t1) {
        place[2] = look_up(t + 2);
        issue(t + 2, place[2], false, k_next ^ kPayload);
      }
      if (t > t0 && t < t1) issue(t, place[0], true, v_prev ^ kPayload);  // (the first is under way)
      place[0] = place[1];
      place[1] = place[2];
    };
    auto next = [&]() {
      k_next ^= kPayload;
      v_prev ^= kPayload;
    };
    // Waves part ways at the end of their rows' keys, but meet at as many barriers.
    int t = t0;
    if (t0 < tw) {
      begin(t);
      first_tile(sa, sb, pa);
      next();
      bool odd = false;
      for (++t; t < tw; ++t) {
        begin(t);
        tile(t, sb, sa, pa, pb);
        next();
        odd = ++t == tw;
        if (odd) break;
        begin(t);
        tile(t, sa, sb, pb, pa);
        next();
      }
      if (odd)
#pragma unroll
        for (int m = 0; m < 4; ++m) pa[m] = pb[m];
      begin(t);
      const int key0 = (t - 1) * kKeys;
      const bool cut = key0 + kKeys > kend;
      u32x4 v[kPairs];  // (the scores' registers are free)
#pragma unroll
      for (int i = 0; i < kPairs; ++i) v[i] = read_v(v_prev, i);
      if (cut)
#pragma unroll
        for (int i = 0; i < kPairs; ++i) drop_unseen(v[i], i, key0);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) output_step(i, v[i], pa);
      next();
      ++t;
    }
    for (; t <= t0 + steps; ++t) {
      begin(t);
      next();
    }
  }

  // A value that is no finite number multiplied by a masked weight's 0 is no
  // 0.  A wave with an output that is not finite walks its tiles once more, one
  // thing after the other and straight from memory (the others may be done):
  // such values are taken out of the product and added to the rows that see
  // their key.
  float check = 0.f;  // no finite number if one of them is none
#pragma unroll
  for (int d = 0; d < kDims; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) check = fmaf(acc[d][r], 0.f, check);
  if (__builtin_amdgcn_ballot_w64(check != 0.f) != 0 && (SRC == kPacked || a.num_blocks > 0)) {
    reset();
    auto key_row = [&](const uint8_t* head, int64_t page_bytes, int st_bytes, int key) {
      key = min(key, kend - 1);
      if constexpr (SRC == kPacked) return head + static_cast<int64_t>(key) * st_bytes;
      const int page = key / a.page, blk = bt_row[static_cast<int64_t>(page) * a.bt_sn];
      return head + min(max(blk, 0), a.num_blocks - 1) * page_bytes + static_cast<int64_t>(key - page * a.page) * st_bytes;
    };
#pragma unroll 1
    for (int t = t0; t < tw; ++t) {
      const int key0 = t * kKeys;
      floatx16 sc[2];
      u32x4 pa[4];
      float ps;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const uint8_t* row = key_row(k_head, a.k_sn * 2, k_st, key0 + 32 * b + c) + 16 * g;
#pragma unroll
        for (int x = 0; x < kSteps; ++x) scores_step(x, *reinterpret_cast<const u32x4*>(row + 32 * x), sc[b]);
      }
      mask(key0, sc);
      settle(sc, pa, ps);
      l_run += ps;
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const uint8_t* row[8];
        u32x4 seen;  // 1 where the lane's row sees the key of the slot
        constexpr uint32_t kOne = F16 ? 0x3C00u : 0x3F80u;
        const int first = key0 + 16 * m + 4 * g;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = first + 8 * (j / 4) + j % 4;
          row[j] = key_row(v_head, a.v_sn * 2, v_st, key) + 2 * c;
          const uint32_t bit = key <= pos ? kOne : 0u;
          seen[j / 2] = j % 2 ? seen[j / 2] | (bit << 16) : bit;
        }
#pragma unroll
        for (int n = 0; n < kDims; ++n) {
          u32x4 clean;
          uint32_t value[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            value[j] = *reinterpret_cast<const uint16_t*>(row[j] + 64 * n);
            const uint32_t finite = (value[j] & T::kInf) == T::kInf ? 0u : value[j];
            clean[j / 2] = j % 2 ? clean[j / 2] | (finite << 16) : finite;
          }
          output_step(m * kDims + n, clean, pa);
#pragma unroll 1
          for (int kind = 0; kind < 3; ++kind) {  // infinities of either sign, NaN: how many of them a row sees
            u32x4 is;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const bool hit = kind == 2 ? (value[j] & 0x7FFFu) > T::kInf : value[j] == (T::kInf | (kind == 1 ? 0x8000u : 0u));
              const uint32_t bit = hit ? kOne : 0u;
              is[j / 2] = j % 2 ? is[j / 2] | (bit << 16) : bit;
            }
            const float what = kind == 2 ? __uint_as_float(0x7FC00000u) : kind == 1 ? -INFINITY : INFINITY;
            floatx16 count;
#pragma unroll
            for (int r = 0; r < 16; ++r) count[r] = 0.f;
            count = T::mfma(__builtin_bit_cast(vec, is), __builtin_bit_cast(vec, seen), count);
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[n][r] = count[r] > 0.f ? acc[n][r] + what : acc[n][r];
          }
        }
      }
    }
  }

  // ---- epilogue
  const auto lsw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l_run), __float_as_uint(l_run), false, false);
  float l_tot = __uint_as_float(lsw[0]) + __uint_as_float(lsw[1]);
  uint8_t* const mine = lds + wave * kCols * kRow;  // K's stages of the first group: every wave is past the last scores
  if constexpr (GROUPS > 1) {
    // The second group's waves leave their outputs in its stages, lane by lane, for
    // the first one's to join.
    static_assert(GROUPS == 2 && kWaves * kDims * 4 * 1024 == 4 * kPayload, "an output fills a group's stages");
    barrier();  // (every wave is past its last values)
    uint8_t* const theirs = lds + kShare + wave * kDims * 4 * 1024 + lane * 16;
    if (group == 1) {
#pragma unroll
      for (int d = 0; d < kDims; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<floatx4*>(theirs + (4 * d + i) * 1024) =
              floatx4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
      *reinterpret_cast<floatx2*>(mine + lane * 8) = floatx2{m_run, l_tot};
    }
    barrier();
    if (group == 1) return;
    // a group without a visible key holds zeros and weighs nothing; a NaN sum goes through
    const floatx2 other = *reinterpret_cast<const floatx2*>(mine + lane * 8);
    const bool live0 = l_tot != 0.f, live1 = other[1] != 0.f;
    const float m = fmaxf(live0 ? m_run : -INFINITY, live1 ? other[0] : -INFINITY);
    const float w0 = live0 ? __builtin_amdgcn_exp2f(m_run - m) : 0.f, w1 = live1 ? __builtin_amdgcn_exp2f(other[0] - m) : 0.f;
    if (live0 || live1) m_run = m;
    l_tot = l_tot * w0 + other[1] * w1;
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const floatx4 x = *reinterpret_cast<const floatx4*>(theirs + (4 * d + i) * 1024);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[d][4 * i + j] = acc[d][4 * i + j] * w0 + x[j] * w1;
      }
  }
  if (work.split > 0 && part == 0 && tid == 0)  // (a block of one part: no rows to join)
    SplitScratch(a.work, a.slots, D).blocks[work.index * a.kv_heads + h] =
        SplitBlock{qs, block * kRows, parts > 1 ? rows : 0, h, work.slot * a.kv_heads + h, parts};
  if (parts > 1) {
    const SplitScratch scratch(a.work, a.slots, D);
    if (row0 + c >= rows) return;
    const int64_t cell = (static_cast<int64_t>(work.slot + part) * a.kv_heads + h) * kRows + wave * kCols + c;
    float* dst = scratch.out + cell * D + 4 * g;
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<floatx4*>(dst + 32 * d + 8 * i) =
            floatx4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
    if (g == 0) *reinterpret_cast<floatx2*>(scratch.ml + 2 * cell) = floatx2{m_run, l_tot};
    return;
  }
  // Rows leave through LDS, so that a store covers whole rows, and past the L2,
  // which keeps K and V (80 prompts of 100 tokens 87 us, 74 so).  Chunks are
  // swizzled by row.
  const float inv = pos < 0 ? 0.f : 1.f / l_tot;  // (a sum of 0, all scores -inf, or a NaN one makes the row NaN)
  constexpr int kChunks = kRow / 16;  // of an output row
#pragma unroll
  for (int d = 0; d < kDims; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<u32x2*>(mine + c * kRow + (((4 * d + i) ^ (c % kChunks)) << 4) + 8 * g) =
          u32x2{pack<F16>(acc[d][4 * i] * inv, acc[d][4 * i + 1] * inv), pack<F16>(acc[d][4 * i + 2] * inv, acc[d][4 * i + 3] * inv)};
#pragma unroll
  for (int j = 0; j < kCols * kChunks / 64; ++j) {
    const int r = j * (64 / kChunks) + lane / kChunks, chunk = lane % kChunks, row = row0 + r;
    const u32x4 x = *reinterpret_cast<const u32x4*>(mine + r * kRow + ((chunk ^ (r % kChunks)) << 4));
    const int at = divide(row, a.by_group), in_group = row - at * a.group;
    if (row < rows)
      __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(a.out + static_cast<int64_t>(qs + at) * a.o_st +
                                                              static_cast<int64_t>(h * a.group + in_group) * a.o_sh + 8 * chunk));
  }
}

// Joins the parts of split blocks: half a wave per row, each lane D / 32 dims.
// Eight parts' sums and rows are loaded at once.
template <bool F16, int D>
__global__ void __launch_bounds__(256) attention16_join_kernel(const AttnArgs a) {
  constexpr int kPer = D / 32, kBatch = 8;
  typedef float vals __attribute__((ext_vector_type(kPer)));
  const SplitScratch scratch(a.work, a.slots, D);
  const int lane = threadIdx.x % 32;
  const int index = static_cast<int>(blockIdx.x) / (kBlockRows / 8);
  const int r = static_cast<int>(blockIdx.x) % (kBlockRows / 8) * 8 + threadIdx.x / 32;
  const SplitBlock b = scratch.blocks[index];  // (anything where there is none)
  const int row = b.row0 + r;
  if (index >= *scratch.count || row >= b.rows) return;
  const int64_t step = static_cast<int64_t>(a.kv_heads) * kBlockRows;  // from part to part
  const int64_t cell = static_cast<int64_t>(b.slot) * kBlockRows + r;
  const floatx2* ml = reinterpret_cast<const floatx2*>(scratch.ml) + cell;
  const float* src = scratch.out + cell * D + lane * kPer;
  float m = -INFINITY, l = 0.f;
  vals o = {};
  const bool none = ml->x == 0.f && ml->y == 0.f;  // the row sees no key: in every part a max of 0 and no sum
  for (int p0 = 0; p0 < b.parts; p0 += kBatch) {
    floatx2 x[kBatch];
    vals v[kBatch];
#pragma unroll
    for (int p = 0; p < kBatch; ++p) {
      const int64_t at = min(p0 + p, b.parts - 1) * step;  // (the last again where there is none: it weighs nothing)
      x[p] = ml[at];
      v[p] = *reinterpret_cast<const vals*>(src + at * D);
    }
    // Parts without a visible key hold zeros and weigh nothing; a NaN sum goes
    // through whatever its part's weight is.
    float top = m;
#pragma unroll
    for (int p = 0; p < kBatch; ++p) top = x[p][1] != 0.f ? fmaxf(top, x[p][0]) : top;
    const float old = top > m ? __builtin_amdgcn_exp2f(m - top) : 1.f;
    m = top;
    l *= old;
    o *= old;
#pragma unroll
    for (int p = 0; p < kBatch; ++p) {
      const bool live = p0 + p < b.parts && x[p][1] != 0.f;
      const float w = live ? __builtin_amdgcn_exp2f(x[p][0] - m) : 0.f;
      l = live ? fmaf(w, x[p][1], l) : l;
#pragma unroll
      for (int j = 0; j < kPer; ++j) o[j] = live ? fmaf(w, v[p][j], o[j]) : o[j];
    }
  }
  const float inv = none ? 0.f : 1.f / l;
  const int tok = divide(row, a.by_group), head = b.head * a.group + (row - tok * a.group);
  uint32_t* dst = reinterpret_cast<uint32_t*>(a.out + static_cast<int64_t>(b.qs + tok) * a.o_st +
                                              static_cast<int64_t>(head) * a.o_sh + lane * kPer);
#pragma unroll
  for (int j = 0; j < kPer; j += 2) dst[j / 2] = pack<F16>(o[j] * inv, o[j + 1] * inv);
}

// The chip holds eight waves per CU (registers, LDS).
int chip_slots(int groups) { return 2 / groups * device_cu_count(); }

int64_t block_bound(int batch, int64_t total_q, int heads, int kv_heads) {
  return (ceil_div(total_q * (heads / kv_heads), kBlockRows) + batch) * kv_heads;
}

// Groups of waves per workgroup: two, each with half of a block's keys, where
// there are about as many blocks as CUs and they are long.  One group per
// workgroup and two workgroups per CU hide each other's first loads and last
// stores, which more blocks need; fewer blocks are split over the chip.  us with
// one group and with two: one prompt of 1000 tokens (32 / 8 heads) 25.5 and 22.9,
// of 2048 (16 heads of 64 dims) 30.4 and 22.4, four of 200 to 3500 (8 / 2 heads)
// 65.3 and 54.2; 32 of 100 (32 / 8 heads) 23.8 and 37.6, one of 4096 143 and 168
// (1032 blocks), one of 4096 over 4 / 1 heads 42.9 and 55.1 (129).
int wave_groups(int batch, int64_t total_q, int heads, int kv_heads, int64_t average_keys) {
  const int64_t cus = device_cu_count(), blocks = block_bound(batch, total_q, heads, kv_heads);
  return 2 * blocks > cus + 2 * kv_heads && 4 * blocks <= 7 * cus && total_q * (heads / kv_heads) >= int64_t{4} * kBlockRows * batch &&
                 average_keys >= 12 * kKeys ? 2 : 1;
}

// Whether blocks may be split: the fewest blocks that the rows make leave room for
// parts, and the longest context could be more than one of them.
bool may_split(int batch, int64_t total_q, int heads, int kv_heads, int64_t most_keys, int groups) {
  const int64_t least = std::max<int64_t>(ceil_div(total_q * (heads / kv_heads), kBlockRows), 1) * kv_heads;
  return batch <= 256 && 2 * least <= chip_slots(groups) && most_keys > 2 * kMinPart * groups * kKeys;
}

template <bool F16, int D, int SRC, int GROUPS>
int launch(const AttnArgs& a, hipStream_t stream) {
  const int64_t rows = static_cast<int64_t>(a.total_q) * a.group;
  // every sequence may end in a partial block; one more for rows outside them
  const int64_t blocks = (ceil_div(rows, kCols * kWaves) + a.batch + 1) * a.kv_heads;
  const int64_t checks = SRC != kPacked && a.report != nullptr ? a.kv_heads : 0;
  const int64_t grid = checks + (a.work == nullptr ? blocks : std::max<int64_t>(blocks, a.slots + a.kv_heads));  // (parts never outnumber the slots)
  if (rows > kMostRows || grid * 64 * kWaves * GROUPS > UINT32_MAX) {
    set_error("attention over 16-bit keys: too many query rows for one launch");
    return PRISM_ERR_INVALID;
  }
  hipLaunchKernelGGL((attention16_kernel<F16, D, SRC, GROUPS>), dim3(static_cast<unsigned>(grid)), dim3(64 * kWaves * GROUPS), 0,
                     stream, a);
  if (int rc = check_launch("attention16_kernel launch")) return rc;
  if (a.work == nullptr) return PRISM_OK;
  const int64_t split = std::min<int64_t>(blocks, a.slots) * (kBlockRows / 8);
  hipLaunchKernelGGL((attention16_join_kernel<F16, D>), dim3(static_cast<unsigned>(split)), dim3(256), 0, stream, a);
  return check_launch("attention16_join_kernel launch");
}

template <bool F16, int D, int GROUPS>
int by_source(const AttnArgs& a, hipStream_t stream) {
  if (a.cu_k != nullptr) return launch<F16, D, kPacked, GROUPS>(a, stream);  // (a table without columns has no address)
  return a.page % kKeys == 0 ? launch<F16, D, kPages, GROUPS>(a, stream) : launch<F16, D, kSmallPages, GROUPS>(a, stream);
}

template <bool F16, int D>
int by_groups(const AttnArgs& a, int groups, hipStream_t stream) {
  return groups == 2 ? by_source<F16, D, 2>(a, stream) : by_source<F16, D, 1>(a, stream);
}

// How a launch is laid out, from static sizes; most_keys and average_keys: of a sequence.
struct Layout {
  int groups, slots;
  bool split;
  Layout(int batch, int64_t total_q, int heads, int kv_heads, int64_t most_keys, int64_t average_keys)
      : groups(wave_groups(batch, total_q, heads, kv_heads, average_keys)), slots(chip_slots(groups)),
        split(may_split(batch, total_q, heads, kv_heads, most_keys, groups)) {}
  int64_t scratch(int head_dim) const { return split ? SplitScratch::bytes(slots, head_dim) : 0; }
};

Layout packed_layout(int batch, int total_q, int total_k, int heads, int kv_heads) {
  return Layout(batch, total_q, heads, kv_heads, total_k, total_k / std::max(batch, 1));
}

Layout paged_layout(int batch, int total_q, int heads, int kv_heads, int page, int width) {
  const int64_t capacity = static_cast<int64_t>(width) * page;
  return Layout(batch, total_q, heads, kv_heads, capacity, capacity);
}

// Without scratch for the parts no block is split.
int dispatch(AttnArgs a, int dtype, int head_dim, const Layout& layout, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  a.slots = layout.slots;
  const int groups = layout.groups;
  const int64_t need = layout.scratch(head_dim);
  a.work = need > 0 && workspace != nullptr && aligned(workspace, 256) && workspace_bytes >= need ? static_cast<uint8_t*>(workspace) : nullptr;
  a.room = a.slots / a.kv_heads;
  a.by_group = divisor(a.group);
  a.by_kv_heads = divisor(a.kv_heads);
  if (dtype == PRISM_DTYPE_F16)
    return head_dim == 128 ? by_groups<true, 128>(a, groups, stream) : by_groups<true, 64>(a, groups, stream);
  return head_dim == 128 ? by_groups<false, 128>(a, groups, stream) : by_groups<false, 64>(a, groups, stream);
}

// What both entries ask of q, K, V and out: types, heads, dims and layout.
// Tile loads address the rows of a tile (or a page) by a 32-bit offset.
int check_layout(const char* what, int dtype, int heads, int kv_heads, int head_dim, const void* q, const int64_t* qs,
                 const void* k, const int64_t* ks, const void* v, const int64_t* vs, int rank, const void* out,
                 const int64_t* os) {
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0) {
    set_error("%s: num_heads=%d must be a multiple of num_kv_heads=%d", what, heads, kv_heads);
    return PRISM_ERR_INVALID;
  }
  if (dtype != PRISM_DTYPE_BF16 && dtype != PRISM_DTYPE_F16) {
    set_error("%s: q, K and V must be bf16 or float16 (dtype code %d)", what, dtype);
    return PRISM_ERR_LAYOUT;
  }
  if (head_dim != 64 && head_dim != 128) {
    set_error("%s: head_dim must be 64 or 128, got %d", what, head_dim);
    return PRISM_ERR_LAYOUT;
  }
  bool good = aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(out, 16);
  for (int i = 0; i < 3; ++i) good = good && (i == 2 ? qs[i] == 1 && os[i] == 1 : qs[i] % 8 == 0 && os[i] % 8 == 0);
  for (int i = 0; i < rank; ++i)
    good = good && (i == rank - 1 ? ks[i] == 1 && vs[i] == 1 : ks[i] % 8 == 0 && vs[i] % 8 == 0);
  if (!good) {
    set_error("%s: q, K/V and out need unit-stride head dims and 16-byte aligned rows", what);
    return PRISM_ERR_LAYOUT;
  }
  for (const int64_t* s : {ks, vs})
    if (s[rank - 3] < 0 || s[rank - 3] > INT32_MAX / (4 * kKeys)) {
      set_error("%s: 64 key rows must span less than 1 GiB", what);
      return PRISM_ERR_LAYOUT;
    }
  return PRISM_OK;
}

}  // namespace

int preload_attention16() {
  hipFuncAttributes attr;
  return check_hip(hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(&attention16_kernel<false, 128, kPacked, 1>)), "preload_attention16");
}

// prism_paged_prefill_ws over 16-bit caches; its geometry, strides and status are checked there.
int paged_prefill16(const void* q, const int64_t* qs, const void* k, const void* v, int dtype, const int64_t* ks,
                    const int64_t* vs, const int32_t* bt, const int64_t* bts, const int32_t* ctx, const int32_t* cu_q,
                    void* out, const int64_t* os, int batch, int total_q, int heads, int kv_heads, int head_dim, int page,
                    int num_blocks, int width, float scale, int32_t* status, void* workspace, int64_t workspace_bytes,
                    int32_t* report, hipStream_t stream) {
  if (int rc = check_layout("prism_paged_prefill", dtype, heads, kv_heads, head_dim, q, qs, k, ks, v, vs, 4, out, os)) return rc;
  if (page % 16 != 0) {
    set_error("prism_paged_prefill: page size must be a multiple of 16, got %d", page);
    return PRISM_ERR_LAYOUT;
  }
  if (batch == 0 || total_q == 0) return PRISM_OK;
  // (without columns, or without pages, every sequence is flagged before a table, or a cache, is read)
  if (!q || !out || !ctx || !cu_q || (width > 0 && !bt) || (num_blocks > 0 && (!k || !v))) {
    set_error("prism_paged_prefill: null argument");
    return PRISM_ERR_INVALID;
  }
  AttnArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_st = qs[0], a.q_sh = qs[1];
  a.k = static_cast<const uint16_t*>(k), a.v = static_cast<const uint16_t*>(v);
  a.k_sn = ks[0], a.k_st = ks[1], a.k_sh = ks[2];
  a.v_sn = vs[0], a.v_st = vs[1], a.v_sh = vs[2];
  a.bt = bt;
  a.bt_sb = bts[0], a.bt_sn = bts[1];
  a.ctx = ctx;
  a.cu_q = cu_q;
  a.out = static_cast<uint16_t*>(out);
  a.o_st = os[0], a.o_sh = os[1];
  a.batch = batch, a.heads = heads, a.kv_heads = kv_heads, a.group = heads / kv_heads;
  a.page = page, a.num_blocks = num_blocks, a.width = width, a.total_q = total_q;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.status = status;
  a.report = report;
  return dispatch(a, dtype, head_dim, paged_layout(batch, total_q, heads, kv_heads, page, width), workspace, workspace_bytes, stream);
}

}  // namespace prism

extern "C" int64_t prism_prompt_attention_workspace_bytes(int batch, int total_q, int total_k, int num_heads,
                                                          int num_kv_heads, int head_dim) {
  if (batch <= 0 || total_q <= 0 || total_k <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 ||
      head_dim <= 0)
    return 0;
  return prism::packed_layout(batch, total_q, total_k, num_heads, num_kv_heads).scratch(head_dim);
}

extern "C" int64_t prism_paged_prefill_16bit_workspace_bytes(int batch, int total_q, int num_heads, int num_kv_heads,
                                                             int head_dim, int page_size, int width) {
  if (batch <= 0 || total_q <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || head_dim <= 0 ||
      page_size <= 0 || width <= 0)
    return 0;
  return prism::paged_layout(batch, total_q, num_heads, num_kv_heads, page_size, width).scratch(head_dim);
}

extern "C" int prism_prompt_attention(const void* q, const int64_t q_strides[3], const void* k, const int64_t k_strides[3],
                                      const void* v, const int64_t v_strides[3], int dtype, const int32_t* cu_seqlens_q,
                                      const int32_t* cu_seqlens_k, void* out, const int64_t out_strides[3], int batch,
                                      int total_q, int total_k, int num_heads, int num_kv_heads, int head_dim, float scale,
                                      void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace prism;
  clear_error();
  if (batch < 0 || total_q < 0 || total_k < 0) {
    set_error("prism_prompt_attention: invalid geometry");
    return PRISM_ERR_INVALID;
  }
  if (total_q == 0) return PRISM_OK;
  if (!q || !q_strides || !k_strides || !v_strides || !out || !out_strides || !cu_seqlens_q || !cu_seqlens_k ||
      (total_k > 0 && (!k || !v))) {
    set_error("prism_prompt_attention: null argument");
    return PRISM_ERR_INVALID;
  }
  if (total_k > kMostKeys) {
    set_error("prism_prompt_attention: too many keys, %d", total_k);
    return PRISM_ERR_INVALID;
  }
  if (int rc = check_layout("prism_prompt_attention", dtype, num_heads, num_kv_heads, head_dim, q, q_strides, k, k_strides,
                            v, v_strides, 3, out, out_strides))
    return rc;
  AttnArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_st = q_strides[0], a.q_sh = q_strides[1];
  a.k = static_cast<const uint16_t*>(k), a.v = static_cast<const uint16_t*>(v);
  a.k_st = k_strides[0], a.k_sh = k_strides[1];
  a.v_st = v_strides[0], a.v_sh = v_strides[1];
  a.cu_q = cu_seqlens_q;
  a.cu_k = cu_seqlens_k;
  a.out = static_cast<uint16_t*>(out);
  a.o_st = out_strides[0], a.o_sh = out_strides[1];
  a.batch = batch, a.heads = num_heads, a.kv_heads = num_kv_heads, a.group = num_heads / num_kv_heads;
  a.total_q = total_q, a.total_k = total_k;
  a.scale_log2 = scale * 1.4426950408889634f;
  return dispatch(a, dtype, head_dim, packed_layout(batch, total_q, total_k, num_heads, num_kv_heads), workspace, workspace_bytes,
                  static_cast<hipStream_t>(stream));
}
