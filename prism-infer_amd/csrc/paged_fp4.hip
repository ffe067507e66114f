// Attention over a paged cache of 4-bit keys and values: one query token a
// sequence, and short chunks of a sequence's last tokens.
//
//   o[j, h] = sum_t w_t v[t, h / G],  w = softmax_t(scale q[j, h] . k[t, h / G]),
//   k[t] = 2^ek[t, d / 32] E2M1(k4[t, d]), v likewise,
//
// over the keys that token j sees.
//
// Per 64 keys of a kv head a wave takes S^T = K Q^T with 16x16x32 bf16 MFMAs.  The
// order of the contraction is free: lane group g of the operand has the 16 bytes of
// a key that it loads, in a product for each eight dims, so that a lane's values
// have one exponent and become bf16 with it, exactly.  (The block-scaled MFMA takes
// the bytes as they are, but aligns products to the largest with few bits: sums were
// off by up to 2^-11 of the largest product.)  Queries are bf16; float16 ones, of 11
// bits, are the sum of two.  A row of scores is one lane column.  P^T is
// the B operand of O^T += V^T P^T as it stands; V^T comes from
// ds_read_b64_tr_b4, 16 keys of a dim at a time, and becomes bf16 exactly.  Values'
// exponents are by key and 32 dims: they go into the weights.  With R rows a 16-row
// operand has room for 16 / R of these: column group x holds the weights for the
// x-th block of dims, and the output of other blocks' columns is dropped.  Weights
// are rounded to bf16 against fp32 sums.
//
// Bound by HBM: 2 (D / 2 + D / 32) bytes of a key and head.
//
// Work layout.  A workgroup's waves are kv heads, and parts of the keys where there
// are fewer heads, so that the rows of a token are read together.  A step is 64 keys
// of each wave.  All sequences' steps are one list, of which a workgroup has an equal
// share: parts of a sequence that lies in several shares are joined by a second
// kernel.
#include "common.h"
#include "divide.h"
#include "fp4.h"
#include "fp8_mfma.h"
#include "paged_chunks.h"
#include "wave_ops.h"

#include <algorithm>

namespace prism {

// Chunks in blocks of 128 rows (attention16.hip).
int64_t paged_prefill4_workspace_bytes(int batch, int total_q, int heads, int kv_heads, int head_dim, int page, int width);
int paged_prefill4(const void* q, const int64_t* qs, const void* k, const void* v, int dtype, const int64_t* ks, const int64_t* vs,
                   const void* ke, const void* ve, const int64_t* kes, const int64_t* ves, const int32_t* bt, const int64_t* bts,
                   const int32_t* ctx, const int32_t* cu_q, void* out, const int64_t* os, int batch, int total_q, int heads,
                   int kv_heads, int head_dim, int page, int num_blocks, int width, float scale, int32_t* status, void* workspace,
                   int64_t workspace_bytes, int32_t* report, hipStream_t stream);

namespace {

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;

constexpr int kWaves = 8;
constexpr int kTile = 64;        // keys of a wave's step
constexpr int kPadding = 64;     // workgroups for rows outside the sequences
constexpr int kMinSteps = 1;     // of a share
constexpr int kMostKeys = 0x7FFFF000;  // of a sequence: positions a few steps further fit in 32 bits

struct Fp4Args {
  const uint16_t* q;
  int64_t q_st, q_sh;  // elements
  const uint8_t* k;
  const uint8_t* v;
  const uint8_t* ks;
  const uint8_t* vs;
  int64_t k_sn, v_sn, ks_sn, vs_sn;  // bytes: block, token, head
  int64_t k_sh, v_sh, ks_sh, vs_sh;
  int k_st, v_st, ks_st, vs_st;
  const int32_t* bt;
  int64_t bt_sb, bt_sn;
  const int32_t* ctx;
  const int32_t* max_ctx;  // one token a sequence
  const int32_t* cu_q;     // chunks
  uint16_t* out;
  int64_t o_st, o_sh;
  int batch, heads, kv_heads, group, page, num_blocks, width, total_q;
  float scale_log2;
  int* status;
  int* report;
  int heads_log2;  // of the kv heads of a workgroup
  int shares;      // workgroups
  uint8_t* work;
  Divisor by_group, by_page;
};

// A sequence's part of the list that begins in share w and ends in a later one:
// description w.  Parts: slot 2 w + 1, then slots 2 (w + 1), 2 (w + 2), ...
struct Split {
  int parts, seq, head, row0, rows, q0;
};

template <int D, int R>
struct Scratch {
  static constexpr int kPart = R * D + 2 * R;  // floats of a head: rows, then (max, sum)
  Split* splits;
  float* parts;
  __host__ __device__ Scratch(uint8_t* p, int shares) : splits(reinterpret_cast<Split*>(p)), parts(reinterpret_cast<float*>(p + head(shares))) {}
  static __host__ __device__ int64_t head(int shares) { return (static_cast<int64_t>(shares) * sizeof(Split) + 255) / 256 * 256; }
};

__device__ __forceinline__ int64_t uniform_int64(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(static_cast<uint64_t>(v) >> 32));
  return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}

// LDS writes of a wave are read by its other lanes: program order is enough for the
// hardware, the compiler has to be told.
__device__ __forceinline__ void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A sequence: its queries, keys, blocks of rows, and steps of a block.
struct Seq {
  int q0, qlen, klen, blocks, steps;
};

template <int R, bool CHUNK>
__device__ __forceinline__ Seq sequence(const Fp4Args& a, int i, int step_log2) {
  Seq s{i, 1, a.ctx[i], 0, 0};
  const int64_t room = min(static_cast<int64_t>(a.width) * a.page, static_cast<int64_t>(kMostKeys));
  bool good = true;
  if (CHUNK) {
    s.q0 = a.cu_q[i];
    const int end = a.cu_q[i + 1];
    good = s.q0 >= 0 && end > s.q0 && end <= a.total_q && s.klen >= end - s.q0 && s.klen <= room;
    s.qlen = end - s.q0;
  } else {
    s.klen = static_cast<int>(min(static_cast<int64_t>(max(min(s.klen, *a.max_ctx), 0)), room));
  }
  if (good) {
    s.blocks = (s.qlen * a.group + R - 1) / R * (a.kv_heads >> a.heads_log2);
    s.steps = max((s.klen + (1 << step_log2) - 1) >> step_log2, 1);
  }
  return s;
}

// Two fp32 values -> two bf16 ones, to nearest even.
__device__ __forceinline__ uint32_t pack_bf16(float lo, float up) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{lo, up}, bf16x2));
}

template <bool F16>
__device__ __forceinline__ uint32_t pack_out(float lo, float up) {
  if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{lo, up}, f16x2));
  else return pack_bf16(lo, up);
}

// Eight E2M1 codes times a power of two -> bf16, exact.
__device__ __forceinline__ bf16x8 fp4x8_to_bf16x8(uint32_t w, float scale = 1.0f) {
  const u32x4 r = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3))};
  return __builtin_bit_cast(bf16x8, r);
}

__device__ __forceinline__ float sum_across_groups(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}

// What a lane holds of R rows of D dims: vector x covers dims 32 (x / 2 * kPer +
// group of the lane's column) + 16 (x % 2) + 4 (lane / 16) + 0..3 of row lane % R.
template <int D, int R>
struct Shape {
  static constexpr int kPer = 16 / R;         // blocks of 32 dims beside each other
  static constexpr int kSets = D / 32 / kPer;
  static constexpr int kVecs = 2 * kSets;
  static __device__ __forceinline__ int dim(int x, int lane) {
    return 32 * (x / 2 * kPer + lane % 16 / R) + 16 * (x % 2) + 4 * (lane / 16);
  }
};

template <bool F16, int D, int R>
__device__ __forceinline__ void write_row(const Fp4Args& a, const floatx4 (&o)[Shape<D, R>::kVecs], float l, int q0, int head, int row, int lane) {
  const float inv = l == 0.f ? 0.f : 1.f / l;  // (no visible key: zeros; a NaN sum goes through)
  const int tok = divide(row, a.by_group);
  uint16_t* dst = a.out + static_cast<int64_t>(q0 + tok) * a.o_st + static_cast<int64_t>(head * a.group + row - tok * a.group) * a.o_sh;
#pragma unroll
  for (int x = 0; x < Shape<D, R>::kVecs; ++x)
    *reinterpret_cast<u32x2*>(dst + Shape<D, R>::dim(x, lane)) =
        u32x2{pack_out<F16>(o[x][0] * inv, o[x][1] * inv), pack_out<F16>(o[x][2] * inv, o[x][3] * inv)};
}

template <bool F16, int D, int R, bool CHUNK>
__global__ void __launch_bounds__(64 * kWaves) paged_fp4_kernel(const Fp4Args a) {
  constexpr int kRow = D / 2;             // bytes of a key
  constexpr int kChunks = kRow / 16;
  constexpr int kVLoads = kTile * kRow / 1024;
  constexpr int kVKeys = 64 / kChunks;    // keys of a load of values
  constexpr int kPer = Shape<D, R>::kPer, kSets = Shape<D, R>::kSets, kVecs = Shape<D, R>::kVecs;
  constexpr int kTerms = F16 ? 2 : 1;     // bf16 terms of a query
  constexpr int kWords = kRow / 16;       // of a key in a lane: products of the scores
  constexpr int kStage = kTile * kRow + 2 * kTile * 4;
  constexpr int kJoin = kVecs * 1024 + 512;
  constexpr int kShare = (kStage > kJoin ? kStage : kJoin);
  __shared__ __attribute__((aligned(256))) uint8_t lds[kWaves * kShare];

  const int lane = threadIdx.x % 64, wave = uniform_int(threadIdx.x / 64);
  const int n = lane % 16, g = lane / 16;
  const int wg_heads = 1 << a.heads_log2, subs_log2 = 3 - a.heads_log2;
  const int my_head = wave & (wg_heads - 1), sub = wave >> a.heads_log2;
  const int step_log2 = 6 + subs_log2;
  int me = static_cast<int>(blockIdx.x);
  const Scratch<D, R> scratch(a.work, a.shares);
  if constexpr (CHUNK) {  // the first workgroup may be the check's, the last ones are the padding's
    if (a.report != nullptr && me == 0) {
      check_metadata(a, *reinterpret_cast<int*>(lds), [&](int i) {
        const Seq s = sequence<R, CHUNK>(a, i, step_log2);
        return s.steps > 0 ? s.klen : -1;
      });
      return;
    }
    me -= a.report != nullptr ? 1 : 0;
    if (me >= a.shares) {
      zero_padding<D>(a, me - a.shares, kPadding);
      return;
    }
  }

  // ---- this workgroup's share of the list.  A lane has `each` sequences.
  const int each = (a.batch + 63) / 64;
  int64_t mine = 0;
  for (int j = 0; j < each; ++j) {
    const int i = lane * each + j;
    if (i < a.batch) {
      const Seq s = sequence<R, CHUNK>(a, i, step_log2);
      mine += static_cast<int64_t>(s.blocks) * s.steps;
      if (CHUNK && s.steps == 0 && me == 0 && threadIdx.x < 64) flag_sequence(a, i);
    }
  }
  int64_t incl = mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int64_t x = __shfl_up(incl, d);
    incl += lane >= d ? x : 0;
  }
  const int64_t total = uniform_int64(__shfl(incl, 63));
  const int64_t share = max((total + a.shares - 1) / a.shares, static_cast<int64_t>(kMinSteps));
  int64_t left_from = me * share;
  const int64_t left_to = min(left_from + share, total);
  if (threadIdx.x == 0) scratch.splits[me].parts = 0;
  if (left_from >= left_to) return;
  int seq;
  int64_t offset;  // in the sequence
  {
    const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(incl > left_from));
    offset = left_from - uniform_int64(__shfl(incl - mine, l));
    seq = l * each;
  }
  int64_t left = left_to - left_from;

  uint8_t* const stage = lds + wave * kShare;
  uint8_t* const v_stage = stage;
  uint32_t* const ks_stage = reinterpret_cast<uint32_t*>(stage + kTile * kRow);
  uint32_t* const vs_stage = ks_stage + kTile;
  const float scale = a.scale_log2 == 0.f ? 1.f : fabsf(a.scale_log2);

  while (left > 0) {
    Seq s = sequence<R, CHUNK>(a, seq, step_log2);
    const int64_t all = static_cast<int64_t>(s.blocks) * s.steps;
    if (offset >= all) {
      offset -= all;
      ++seq;
      continue;
    }
    s.q0 = uniform_int(s.q0), s.qlen = uniform_int(s.qlen), s.klen = uniform_int(s.klen), s.steps = uniform_int(s.steps);
    const int at = uniform_int(static_cast<int>(offset / s.steps));
    const int step0 = uniform_int(static_cast<int>(offset - static_cast<int64_t>(at) * s.steps));
    const int steps = uniform_int(static_cast<int>(min(static_cast<int64_t>(s.steps - step0), left)));
    const int head_groups = a.kv_heads >> a.heads_log2;
    const int row_block = at / head_groups;
    const int h = ((at - row_block * head_groups) << a.heads_log2) + my_head;
    const int row0 = row_block * R, rows = s.qlen * a.group;

    // ---- the queries
    const int my_row = row0 + n % R;
    const bool real = my_row < rows;
    const int tok = CHUNK ? divide(min(my_row, rows - 1), a.by_group) : 0;
    const int first_seen = CHUNK ? s.klen - s.qlen + divide(row0, a.by_group) + 1 : s.klen;  // keys that every row sees
    const int kend = CHUNK ? s.klen - s.qlen + divide(min(row0 + R, rows) - 1, a.by_group) + 1 : s.klen;
    const int seen = CHUNK ? s.klen - s.qlen + tok + 1 : s.klen;
    bf16x8 qop[kTerms][kWords];
    {
      const uint16_t* src = a.q + static_cast<int64_t>(s.q0 + tok) * a.q_st +
                            static_cast<int64_t>(h * a.group + min(my_row, rows - 1) - tok * a.group) * a.q_sh;
      const uint32_t keep = !real || a.scale_log2 == 0.f ? 0u : ~0u, flip = a.scale_log2 < 0.f ? 0x80008000u & keep : 0u;
#pragma unroll
      for (int x = 0; x < kWords; ++x) {
        u32x4 w = *reinterpret_cast<const u32x4*>(src + (g * kWords + x) * 8);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          w[j] = (w[j] & keep) ^ flip;
          if constexpr (F16) {
            const float lo = f16_bits_to_f32(w[j] & 0xFFFFu), hi = f16_bits_to_f32(w[j] >> 16);
            const uint32_t first = pack_bf16(lo, hi);
            w[j] = first;
            u32x4 rest = __builtin_bit_cast(u32x4, qop[kTerms - 1][x]);
            rest[j] = pack_bf16(lo - __uint_as_float(first << 16), hi - __uint_as_float(first & 0xFFFF0000u));
            qop[kTerms - 1][x] = __builtin_bit_cast(bf16x8, rest);
          }
        }
        qop[0][x] = __builtin_bit_cast(bf16x8, w);
      }
    }

    // ---- the wave's tiles: t0, t0 + subs, ... below t1
    const int subs = 1 << subs_log2;
    const int need = (kend + kTile - 1) / kTile;
    int t = (step0 << subs_log2) + sub;
    const int t1 = min((step0 + steps) << subs_log2, need);
    const uint8_t* const k_head = a.k + h * a.k_sh;
    const uint8_t* const v_head = a.v + h * a.v_sh;
    const uint8_t* const ks_head = a.ks + h * a.ks_sh;
    const uint8_t* const vs_head = a.vs + h * a.vs_sh;
    const int32_t* bt_row = a.bt + static_cast<int64_t>(seq) * a.bt_sb;
    int ids_base = 0, ids = 0;
    auto load_ids = [&](int base) {
      ids_base = base;
      ids = bt_row[static_cast<int64_t>(min(base + lane, a.width - 1)) * a.bt_sn];
    };

    typedef uint32_t k_words __attribute__((ext_vector_type(kWords)));
    k_words kw[4];
    u32x4 vw[kVLoads];
    uint32_t ksw = 0, vsw = 0;
    int missing = 0;  // bit x: the x-th 16 keys of the tile are not there
    auto issue = [&](int tile) {
      missing = 0;
      int blk[4], row[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int key = tile * kTile + 16 * x;
        blk[x] = row[x] = 0;
        if (key >= kend) {
          missing |= 1 << x;
          continue;
        }
        const int p = divide(key, a.by_page);
        row[x] = key - p * a.page;
        if (p >= ids_base + 64) load_ids(p);
        blk[x] = __builtin_amdgcn_readlane(ids, p - ids_base);
        if (blk[x] < 0 || blk[x] >= a.num_blocks) {
          if (CHUNK && lane == 0) flag_sequence(a, seq);
          missing |= 1 << x;
          blk[x] = row[x] = 0;
        }
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint8_t* base = k_head + blk[x] * a.k_sn + static_cast<int64_t>(row[x]) * a.k_st;
        kw[x] = *reinterpret_cast<const k_words*>(base + (n * a.k_st + g * 4 * kWords));
      }
      {
        const int x = lane / 16;
        const int b = x == 0 ? blk[0] : x == 1 ? blk[1] : x == 2 ? blk[2] : blk[3];
        const int r = (x == 0 ? row[0] : x == 1 ? row[1] : x == 2 ? row[2] : row[3]) + n;
        const uint8_t* kp = ks_head + b * a.ks_sn + static_cast<int64_t>(r) * a.ks_st;
        const uint8_t* vp = vs_head + b * a.vs_sn + static_cast<int64_t>(r) * a.vs_st;
        if constexpr (D == 128) {
          ksw = *reinterpret_cast<const uint32_t*>(kp);
          vsw = *reinterpret_cast<const uint32_t*>(vp);
        } else {
          ksw = *reinterpret_cast<const uint16_t*>(kp);
          vsw = *reinterpret_cast<const uint16_t*>(vp);
        }
      }
#pragma unroll
      for (int x = 0; x < kVLoads; ++x) {
        int b = blk[x * kVKeys / 16], r = row[x * kVKeys / 16];
        if (kVKeys == 32 && lane >= 32) b = blk[2 * x + 1], r = row[2 * x + 1];
        const uint8_t* base = v_head + b * a.v_sn + static_cast<int64_t>(r) * a.v_st;
        vw[x] = *reinterpret_cast<const u32x4*>(base + (lane / kChunks % 16 * a.v_st + lane % kChunks * 16));
      }
    };

    floatx4 acc[D / 16];
#pragma unroll
    for (int x = 0; x < D / 16; ++x) acc[x] = floatx4{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_run = 0.f;

    if (t < t1) {
      load_ids(uniform_int(divide(t * kTile, a.by_page)));
      issue(t);
    }
    for (; t < t1; t += subs) {
      const int key0 = t * kTile, gone = missing;
      // ---- values and exponents to LDS, scores
#pragma unroll
      for (int x = 0; x < kVLoads; ++x) {
        const int key = x * kVKeys + lane / kChunks;
        *reinterpret_cast<u32x4*>(v_stage + key * kRow + ((lane % kChunks ^ (key / 16 % kChunks)) << 4)) = vw[x];
      }
      ks_stage[lane] = ksw;
      vs_stage[lane] = vsw;
      const bool nan_block = (((vsw & 0x7F7F7F7Fu) + 0x01010101u) & vsw & 0x80808080u) != 0;
      const bool special = __builtin_amdgcn_ballot_w64(nan_block) != 0 || gone != 0 || key0 + kTile > first_seen;
      wave_lds_order();
      floatx4 sc[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint32_t e = reinterpret_cast<const uint8_t*>(ks_stage)[(16 * x + n) * 4 + (D == 128 ? g : g / 2)];
        const float ke = e == 255u ? __uint_as_float(0x7FC00000u) : __uint_as_float(e << 23);
        sc[x] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int y = 0; y < kWords; ++y) {
          const bf16x8 key = fp4x8_to_bf16x8(kw[x][y], ke);
#pragma unroll
          for (int term = kTerms - 1; term >= 0; --term) sc[x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(key, qop[term][y], sc[x], 0, 0, 0);
        }
      }
      u32x4 ve[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) ve[x] = *reinterpret_cast<const u32x4*>(vs_stage + 16 * x + 4 * g);
      if (t + subs < t1) issue(t + subs);

      // ---- softmax
      if (special) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            sc[x][i] = key0 + 16 * x + 4 * g + i < seen && !(gone >> x & 1) ? sc[x][i] : -INFINITY;
      }
      float top = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3]));
#pragma unroll
      for (int x = 1; x < 4; ++x) top = fmaxf(top, fmaxf(fmaxf(sc[x][0], sc[x][1]), fmaxf(sc[x][2], sc[x][3])));
      top = wave_max_across_groups(top) * scale;
      const float m_new = fmaxf(m_run, top);
      if (__builtin_amdgcn_ballot_w64(m_new > m_run) != 0) {
        const float alpha = m_new > m_run ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.f;
        l_run *= alpha;
#pragma unroll
        for (int x = 0; x < D / 16; ++x) acc[x] *= alpha;
        m_run = m_new;
      }
      const float m_use = m_run == -INFINITY ? 0.f : m_run;
      float p[4][4];
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[x][i] = __builtin_amdgcn_exp2f(fmaf(sc[x][i], scale, -m_use));
          l_run += p[x][i];
        }

      // ---- output
#pragma unroll
      for (int set = 0; set < kSets; ++set) {
        const int shift = 8 * (set * kPer + n / R);
        u32x4 pw[2];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          float w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t e = (ve[x][i] >> shift) & 0xFFu;
            w[i] = p[x][i] * __uint_as_float(e << 23);
            if (special) {
              const bool sees = key0 + 16 * x + 4 * g + i < seen && !(gone >> x & 1);
              w[i] = !sees ? 0.f : e == 255u ? __uint_as_float(0x7FC00000u) : w[i];
            }
          }
          pw[x / 2][x % 2 * 2] = pack_bf16(w[0], w[1]);
          pw[x / 2][x % 2 * 2 + 1] = pack_bf16(w[2], w[3]);
        }
#pragma unroll
        for (int y = 0; y < 2 * kPer; ++y) {
          const int m = set * 2 * kPer + y;  // 16 dims
          const int key = 16 * (n / 4) + 4 * g + n % 4;
          const uint8_t* src = v_stage + key * kRow + (((m / 2) ^ (n / 4 % kChunks)) << 4) + m % 2 * 8;
          const i32x2 w = __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_i32x2*)(src));
          acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp4x8_to_bf16x8(w[0]), __builtin_bit_cast(bf16x8, pw[0]), acc[m], 0, 0, 0);
          acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp4x8_to_bf16x8(w[1]), __builtin_bit_cast(bf16x8, pw[1]), acc[m], 0, 0, 0);
        }
      }
      wave_lds_order();
    }

    // ---- the columns' own blocks
    float l_tot = sum_across_groups(l_run);
    floatx4 o[kVecs];
#pragma unroll
    for (int x = 0; x < kVecs; ++x) {
      o[x] = acc[x / 2 * 2 * kPer + x % 2];
#pragma unroll
      for (int y = 1; y < kPer; ++y)
        if (n / R == y) o[x] = acc[(x / 2 * kPer + y) * 2 + x % 2];
    }
    if (subs > 1) {  // parts of the keys in other waves
      floatx4* own = reinterpret_cast<floatx4*>(stage);
      floatx2* own_ml = reinterpret_cast<floatx2*>(stage + kVecs * 1024);
      if (sub > 0) {
#pragma unroll
        for (int x = 0; x < kVecs; ++x) own[x * 64 + lane] = o[x];
        own_ml[lane] = floatx2{m_run, l_tot};
      }
      __syncthreads();
      if (sub == 0) {
        for (int y = 1; y < subs; ++y) {
          const uint8_t* theirs = lds + (my_head + (y << a.heads_log2)) * kShare;
          const floatx2 ml = reinterpret_cast<const floatx2*>(theirs + kVecs * 1024)[lane];
          const float m = fmaxf(m_run, ml[0]);
          const float w0 = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - m), w1 = ml[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[0] - m);
          // (a part without keys has max -inf and zeros; one whose scores are all NaN has max -inf and a NaN sum)
          l_tot = l_tot != l_tot || ml[1] != ml[1] ? __uint_as_float(0x7FC00000u) : l_tot * w0 + ml[1] * w1;
#pragma unroll
          for (int x = 0; x < kVecs; ++x) o[x] = o[x] * w0 + reinterpret_cast<const floatx4*>(theirs)[x * 64 + lane] * w1;
          m_run = m;
        }
      }
      __syncthreads();
    }
    const bool begins = step0 == 0, ends = step0 + steps == s.steps;
    if (begins && ends) {
      if (sub == 0 && real) write_row<F16, D, R>(a, o, l_tot, s.q0, h, my_row, lane);
    } else if (sub == 0) {
      float* part = scratch.parts + (((static_cast<int64_t>(me) * 2 + (begins ? 1 : 0)) << a.heads_log2) + my_head) * Scratch<D, R>::kPart;
#pragma unroll
      for (int x = 0; x < kVecs; ++x) reinterpret_cast<floatx4*>(part)[x * 64 + lane] = o[x];
      if (lane < R) reinterpret_cast<floatx2*>(part + R * D)[lane] = floatx2{m_run, l_tot};
      if (begins && threadIdx.x == 0) {
        const int64_t more = (s.steps - steps + share - 1) / share;
        scratch.splits[me] = Split{1 + static_cast<int>(more), seq, h, row0, rows, s.q0};
      }
    }
    left -= steps;
    offset += steps;
  }
}

// Joins the parts of a split sequence: a workgroup per share that one begins in
// and head, its waves taking parts in turn.
constexpr int kJoinWaves = 4;

template <bool F16, int D, int R>
__global__ void __launch_bounds__(64 * kJoinWaves) paged_fp4_join_kernel(const Fp4Args a) {
  constexpr int kVecs = Shape<D, R>::kVecs, kPart = Scratch<D, R>::kPart;
  __shared__ floatx4 rows[kJoinWaves][kVecs * 64];
  __shared__ floatx2 stats[kJoinWaves][64];
  const Scratch<D, R> scratch(a.work, a.shares);
  const int me = static_cast<int>(blockIdx.x) >> a.heads_log2, my_head = static_cast<int>(blockIdx.x) & ((1 << a.heads_log2) - 1);
  const Split s = scratch.splits[me];
  if (s.parts == 0) return;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  float m_run = -INFINITY, l_run = 0.f;
  floatx4 o[kVecs];
#pragma unroll
  for (int x = 0; x < kVecs; ++x) o[x] = floatx4{0.f, 0.f, 0.f, 0.f};
  auto join = [&](float m1, float l1, const floatx4 (&v)[kVecs]) {
    const float m = fmaxf(m_run, m1);
    const float w0 = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - m), w1 = m1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m1 - m);
    l_run = l_run != l_run || l1 != l1 ? __uint_as_float(0x7FC00000u) : l_run * w0 + l1 * w1;
#pragma unroll
    for (int x = 0; x < kVecs; ++x) o[x] = o[x] * w0 + v[x] * w1;
    m_run = m;
  };
  constexpr int kAtOnce = kVecs <= 2 ? 4 : 2;
  for (int p0 = wave * kAtOnce; p0 < s.parts; p0 += kJoinWaves * kAtOnce) {
    floatx4 v[kAtOnce][kVecs];
    floatx2 ml[kAtOnce];
#pragma unroll
    for (int y = 0; y < kAtOnce; ++y) {
      const int p = min(p0 + y, s.parts - 1);
      const int64_t slot = p == 0 ? 2 * static_cast<int64_t>(me) + 1 : 2 * (static_cast<int64_t>(me) + p);
      const float* part = scratch.parts + ((slot << a.heads_log2) + my_head) * kPart;
#pragma unroll
      for (int x = 0; x < kVecs; ++x) v[y][x] = reinterpret_cast<const floatx4*>(part)[x * 64 + lane];
      ml[y] = reinterpret_cast<const floatx2*>(part + R * D)[lane % R];
    }
#pragma unroll
    for (int y = 0; y < kAtOnce; ++y)
      if (p0 + y < s.parts) join(ml[y][0], ml[y][1], v[y]);
  }
#pragma unroll
  for (int x = 0; x < kVecs; ++x) rows[wave][x * 64 + lane] = o[x];
  stats[wave][lane] = floatx2{m_run, l_run};
  __syncthreads();
  if (wave != 0) return;
  for (int y = 1; y < kJoinWaves; ++y) {
    floatx4 v[kVecs];
#pragma unroll
    for (int x = 0; x < kVecs; ++x) v[x] = rows[y][x * 64 + lane];
    join(stats[y][lane][0], stats[y][lane][1], v);
  }
  const int row = s.row0 + lane % R;
  if (row < s.rows) write_row<F16, D, R>(a, o, l_run, s.q0, s.head + my_head, row, lane);
}

int heads_log2(int kv_heads) { return kv_heads % 8 == 0 ? 3 : kv_heads % 4 == 0 ? 2 : kv_heads % 2 == 0 ? 1 : 0; }

int row_block(bool chunks, int group, int head_dim) {
  if (chunks || group > 8) return 16;
  return group > 4 || head_dim == 64 ? 8 : 4;
}

int share_count() { return 2 * device_cu_count(); }

int64_t scratch_bytes(bool chunks, int group, int kv_heads, int head_dim) {
  const int r = row_block(chunks, group, head_dim), shares = share_count();
  return Scratch<128, 16>::head(shares) + ((static_cast<int64_t>(2 * shares) << heads_log2(kv_heads)) * (r * head_dim + 2 * r)) * 4;
}

// Chunks of more than this many rows of a kv head go to blocks of 128 rows.
#ifndef WIDE_ROWS
#define WIDE_ROWS 16
#endif
bool wide_chunks(int batch, int total_q, int group) { return static_cast<int64_t>(total_q) * group > static_cast<int64_t>(WIDE_ROWS) * batch; }

template <bool F16, int D, int R, bool CHUNK>
int launch(const Fp4Args& a, hipStream_t stream) {
  const int others = CHUNK ? kPadding + (a.report != nullptr ? 1 : 0) : 0;
  hipLaunchKernelGGL((paged_fp4_kernel<F16, D, R, CHUNK>), dim3(a.shares + others), dim3(64 * kWaves), 0, stream, a);
  if (int rc = check_launch("paged_fp4_kernel launch")) return rc;
  hipLaunchKernelGGL((paged_fp4_join_kernel<F16, D, R>), dim3(a.shares << a.heads_log2), dim3(64 * kJoinWaves), 0, stream, a);
  return check_launch("paged_fp4_join_kernel launch");
}

template <bool F16>
int dispatch(const Fp4Args& a, int head_dim, hipStream_t stream) {
  const bool chunks = a.cu_q != nullptr;
  const int r = row_block(chunks, a.group, head_dim);
  if (head_dim == 128) {
    if (chunks) return launch<F16, 128, 16, true>(a, stream);
    return r == 4 ? launch<F16, 128, 4, false>(a, stream) : r == 8 ? launch<F16, 128, 8, false>(a, stream) : launch<F16, 128, 16, false>(a, stream);
  }
  if (chunks) return launch<F16, 64, 16, true>(a, stream);
  return r == 8 ? launch<F16, 64, 8, false>(a, stream) : launch<F16, 64, 16, false>(a, stream);
}

}  // namespace

int preload_paged_fp4() {
  hipFuncAttributes attr;
  return check_hip(hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(&paged_fp4_kernel<false, 128, 4, false>)), "preload_paged_fp4");
}

}  // namespace prism

extern "C" int64_t prism_paged_fp4_workspace_bytes(int chunks, int batch, int total_q, int num_heads, int num_kv_heads, int head_dim,
                                                   int page_size, int width) {
  if (batch <= 0 || total_q <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || head_dim <= 0 ||
      page_size <= 0 || width < 0)
    return 0;
  if (chunks != 0 && prism::wide_chunks(batch, total_q, num_heads / num_kv_heads))
    return prism::paged_prefill4_workspace_bytes(batch, total_q, num_heads, num_kv_heads, head_dim, page_size, width);
  return prism::scratch_bytes(chunks != 0, num_heads / num_kv_heads, num_kv_heads, head_dim);
}

extern "C" int prism_paged_fp4(const void* q, int q_dtype, const int64_t q_strides[3], const void* k_cache, const void* v_cache,
                               const int64_t k_strides[4], const int64_t v_strides[4], const void* k_scale, const void* v_scale,
                               const int64_t ks_strides[4], const int64_t vs_strides[4], const int32_t* block_tables,
                               const int64_t bt_strides[2], const int32_t* context_lens, const int32_t* max_context_len,
                               const int32_t* cu_seqlens_q, void* out, const int64_t out_strides[3], int batch, int total_q,
                               int num_heads, int num_kv_heads, int head_dim, int page_size, int num_blocks, int width,
                               float scale, int32_t* status, int32_t* report, void* workspace, int64_t workspace_bytes,
                               void* stream_ptr) {
  using namespace prism;
  clear_error();
  const char* what = "prism_paged_fp4";
  if (batch < 0 || total_q < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || page_size <= 0 ||
      num_blocks < 0 || width < 0) {
    set_error("%s: invalid geometry batch=%d rows=%d heads=%d kv_heads=%d page=%d blocks=%d width=%d", what, batch, total_q, num_heads,
              num_kv_heads, page_size, num_blocks, width);
    return PRISM_ERR_INVALID;
  }
  if (q_dtype != PRISM_DTYPE_BF16 && q_dtype != PRISM_DTYPE_F16) {
    set_error("%s: queries must be bf16 or float16 (dtype code %d)", what, q_dtype);
    return PRISM_ERR_LAYOUT;
  }
  if (head_dim != 64 && head_dim != 128) {
    set_error("%s: head_dim must be 64 or 128, got %d", what, head_dim);
    return PRISM_ERR_LAYOUT;
  }
  if (page_size % 16 != 0) {
    set_error("%s: page size must be a multiple of 16, got %d", what, page_size);
    return PRISM_ERR_LAYOUT;
  }
  if (batch == 0 || total_q == 0) return PRISM_OK;
  const bool chunks = cu_seqlens_q != nullptr;
  if (!q || !out || !q_strides || !out_strides || !k_strides || !v_strides || !ks_strides || !vs_strides || !bt_strides || !context_lens ||
      (width > 0 && !block_tables) || (num_blocks > 0 && (!k_cache || !v_cache || !k_scale || !v_scale)) || (chunks ? !status : !max_context_len)) {
    set_error("%s: null argument", what);
    return PRISM_ERR_INVALID;
  }
  if (!chunks && total_q < batch) {
    set_error("%s: %d query rows for %d sequences", what, total_q, batch);
    return PRISM_ERR_INVALID;
  }
  const int exponents = head_dim / 32;
  bool good = aligned(q, 16) && aligned(out, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(k_scale, exponents) &&
              aligned(v_scale, exponents);
  for (int i = 0; i < 3; ++i) good = good && (i == 2 ? q_strides[i] == 1 && out_strides[i] == 1 : q_strides[i] % 8 == 0 && out_strides[i] % 8 == 0);
  for (int i = 0; i < 4; ++i) {
    good = good && (i == 3 ? k_strides[i] == 1 && v_strides[i] == 1 && ks_strides[i] == 1 && vs_strides[i] == 1
                           : k_strides[i] % 16 == 0 && v_strides[i] % 16 == 0 && ks_strides[i] % exponents == 0 && vs_strides[i] % exponents == 0);
  }
  if (!good) {
    set_error("%s: q, out and caches need unit-stride head dims and aligned rows", what);
    return PRISM_ERR_LAYOUT;
  }
  for (const int64_t* s : {k_strides, v_strides, ks_strides, vs_strides})
    if (s[1] < 0 || s[1] > INT32_MAX / page_size) {
      set_error("%s: a page must span less than 2 GiB", what);
      return PRISM_ERR_LAYOUT;
    }
  const int64_t need = prism_paged_fp4_workspace_bytes(chunks, batch, total_q, num_heads, num_kv_heads, head_dim, page_size, width);
  if (workspace_bytes < need || (need > 0 && (!workspace || !aligned(workspace, 256)))) {
    set_error("%s: the workspace needs %lld bytes, 256-byte aligned", what, static_cast<long long>(need));
    return PRISM_ERR_INVALID;
  }
  if (chunks && wide_chunks(batch, total_q, num_heads / num_kv_heads))
    return paged_prefill4(q, q_strides, k_cache, v_cache, q_dtype, k_strides, v_strides, k_scale, v_scale, ks_strides, vs_strides,
                          block_tables, bt_strides, context_lens, cu_seqlens_q, out, out_strides, batch, total_q, num_heads,
                          num_kv_heads, head_dim, page_size, num_blocks, width, scale, status, workspace, need, report,
                          static_cast<hipStream_t>(stream_ptr));
  Fp4Args a{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_st = q_strides[0], a.q_sh = q_strides[1];
  a.k = static_cast<const uint8_t*>(k_cache), a.v = static_cast<const uint8_t*>(v_cache);
  a.ks = static_cast<const uint8_t*>(k_scale), a.vs = static_cast<const uint8_t*>(v_scale);
  a.k_sn = k_strides[0], a.k_st = static_cast<int>(k_strides[1]), a.k_sh = k_strides[2];
  a.v_sn = v_strides[0], a.v_st = static_cast<int>(v_strides[1]), a.v_sh = v_strides[2];
  a.ks_sn = ks_strides[0], a.ks_st = static_cast<int>(ks_strides[1]), a.ks_sh = ks_strides[2];
  a.vs_sn = vs_strides[0], a.vs_st = static_cast<int>(vs_strides[1]), a.vs_sh = vs_strides[2];
  a.bt = block_tables;
  a.bt_sb = bt_strides[0], a.bt_sn = bt_strides[1];
  a.ctx = context_lens;
  a.max_ctx = max_context_len;
  a.cu_q = cu_seqlens_q;
  a.out = static_cast<uint16_t*>(out);
  a.o_st = out_strides[0], a.o_sh = out_strides[1];
  a.batch = batch, a.heads = num_heads, a.kv_heads = num_kv_heads, a.group = num_heads / num_kv_heads;
  a.page = page_size, a.num_blocks = num_blocks, a.total_q = total_q;
  a.width = num_blocks > 0 ? width : 0;  // (without pages nothing is read)
  a.scale_log2 = scale * 1.4426950408889634f;
  a.status = status;
  a.report = report;
  a.heads_log2 = heads_log2(num_kv_heads);
  a.shares = share_count();
  a.work = static_cast<uint8_t*>(workspace);
  a.by_group = divisor(a.group);
  a.by_page = divisor(page_size);
  hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
  return q_dtype == PRISM_DTYPE_F16 ? dispatch<true>(a, head_dim, stream) : dispatch<false>(a, head_dim, stream);
}
