// Attention over a paged cache of 4-bit keys and values, one query token a sequence
// (chunks of tokens: attention16.hip).
//
//   o[h] = sum_t w_t v[t, h / G],  w = softmax_t(scale q[h] . k[t, h / G]),
//   k[t, d] = 2^ek[t, d / 32] E2M1(k4[t, d]), v likewise.
//
// Per 64 keys of a kv head a wave takes S^T = K Q^T with 16x16x32 bf16 MFMAs.  The
// order of the contraction is free: lane group g of the operand has the 16 bytes of
// a key that it loads, in a product for each eight dims, so that a lane's values
// have one exponent and become bf16 with it, exactly.  (The block-scaled MFMA takes
// the bytes as they are, but aligns products to the largest with few bits: sums were
// off by up to 2^-11 of the largest product.)  Float16 queries meet float16 keys,
// 2^-4 of them, where all of a step's keys are such numbers; else bf16 keys, which are
// exact at every exponent, meet the queries as the sum of two bf16 numbers, exact too, in
// twice the products.  A row of scores is one lane column.  P^T is
// the B operand of O^T += V^T P^T as it stands; V^T comes from
// ds_read_b64_tr_b4, 16 keys of a dim at a time, and becomes bf16 exactly.  Values'
// exponents are by key and 32 dims: they go into the weights.  With R rows a 16-row
// operand has room for 16 / R of these: column group x holds the weights for the
// x-th block of dims, and the output of other blocks' columns is dropped.  Weights
// are rounded to bf16 against fp32 sums; for float16 queries they are the sum of two
// bf16 numbers, whose 16 bits leave the output's 11.
//
// Bound by HBM: 2 (D / 2 + D / 32) bytes of a key and head.  16 x 32768 keys (32 / 8
// heads of 128 dims) 106 us, 5.4 TB/s, of which 5 the join; loads alone 100.  Bound by
// the chain of dependent loads where there is little: one conversation of 1800 keys 10.
//
// Work layout.  A workgroup's four waves are kv heads, and parts of the keys where
// there are fewer heads.  A step is 64 keys of each wave, which they load together,
// 16 keys of all their heads each (with a wave's loads its own head's alone, 64 bytes
// of a key, half lines, the same work stayed at 4.6 TB/s whatever else it did).  All
// sequences' steps are one list, of which a workgroup has an equal
// share: parts of a sequence that lies in several shares are joined by a second
// kernel.
#include "common.h"
#include "divide.h"
#include "fp4.h"
#include "fp8_mfma.h"
#include "wave_ops.h"

#include <algorithm>
#include <type_traits>

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

constexpr int kWavesLog2 = 2, kWaves = 1 << kWavesLog2;
constexpr int kTile = 64;        // keys of a wave's step
constexpr int kWholeSteps = 2;   // up to which a sequence is not split
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
  const int32_t* max_ctx;
  uint16_t* out;
  int64_t o_st, o_sh;
  int batch, heads, kv_heads, group, page, num_blocks, width;
  int room;  // keys that a block table holds
  float scale_log2;
  int heads_log2;  // of the kv heads of a workgroup
  int shares;      // workgroups
  int splits;      // descriptions
  bool by_number;
  bool whole;      // sequences are not split: they have few steps each
  int numbers;     // blocks of rows times groups of kv heads, of all sequences
  uint8_t* work;
  Divisor by_page, by_shares, by_cus;
};

// A sequence's part of the list (of a block of rows and a group of kv heads): how many
// shares it lies in, from share w on.  Parts: slot 2 w + 1, then 2 (w + 1), 2 (w + 2),
// ...  Described by its number where there are as many shares, else by w.
struct Split {
  int parts, share, seq, head, row0;
};

template <int D, int R>
struct Scratch {
  static constexpr int kPart = R * D + 2 * R;  // floats of a head: rows, then (max, sum)
  Split* splits;
  float* parts;
  __host__ __device__ Scratch(uint8_t* p, int shares) : splits(reinterpret_cast<Split*>(p)), parts(reinterpret_cast<float*>(p + head(shares))) {}
  static __host__ __device__ int64_t head(int shares) { return (static_cast<int64_t>(shares) * sizeof(Split) + 255) / 256 * 256; }
};

// The lane, as a value that is not known to be the same one: what is computed from it
// is computed where it stands, and does not take registers over the whole kernel.
__device__ __forceinline__ uint32_t fresh(uint32_t lane) {
  asm volatile("" : "+v"(lane));
  return lane;
}

// LDS writes of a wave are read by its other lanes: program order is enough for the
// hardware, the compiler has to be told.
__device__ __forceinline__ void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A sequence's keys.
__device__ __forceinline__ int keys_of(const Fp4Args& a, int i) { return min(max(min(a.ctx[i], *a.max_ctx), 0), a.room); }

template <bool F16>
__device__ __forceinline__ uint32_t pack_out(float lo, float up) {
  if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{lo, up}, f16x2));
  else return pack_bf16(lo, up);
}

// Eight E2M1 codes times a power of two -> bf16, exact.
constexpr uint32_t kKeyShift = 4;  // float16 keys are 2^-4 of themselves: 65504 is held as 65536, no float16 number
__device__ __forceinline__ bf16x8 fp4x8_to_bf16x8(uint32_t w, float scale = 1.0f) {
  const u32x4 r = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3))};
  return __builtin_bit_cast(bf16x8, r);
}

// Exponent bytes of keys, four a word, that 2^-4 of a float16 number does not hold all
// codes of: 0.5 * 2^(108 - 127 - 4) is its smallest, 6 * 2^(144 - 127 - 4) ends below its
// largest.  Of 0 and 1, nobody's keys and blocks of zeros, it makes 0, which such keys'
// scores are to 2^-100.
__device__ __forceinline__ uint32_t off_float16(uint32_t w) {
  const uint32_t low = w & 0x7F7F7F7Fu;
  const uint32_t above = (low + 0x6F6F6F6Fu) & w;                                // 145 to 255
  const uint32_t below = (low + 0x7E7E7E7Eu) & ~(low + 0x14141414u) & ~w;        // 2 to 107
  return (above | below) & 0x80808080u;
}

// ... times 2^(e - 127) of an exponent byte, as the scores' operand.
template <bool F16>
__device__ __forceinline__ u32x4 widen_key(uint32_t w, uint32_t e) {
  if constexpr (!F16) return __builtin_bit_cast(u32x4, fp4x8_to_bf16x8(w, __uint_as_float(e << 23)));
  const float scale = __uint_as_float((max(e, kKeyShift + 1u) - kKeyShift) << 23);
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3))};
}

template <bool F16>
__device__ __forceinline__ floatx4 score_product(const u32x4& k, const u32x4& q, floatx4 c) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, k), __builtin_bit_cast(f16x8, q), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k), __builtin_bit_cast(bf16x8, q), c, 0, 0, 0);
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
  static constexpr int kJoined = 2;  // vectors of a workgroup that joins parts
  static __device__ __forceinline__ int dim(int x, int lane) {
    return 32 * (x / 2 * kPer + lane % 16 / R) + 16 * (x % 2) + 4 * (lane / 16);
  }
};

// N vectors from x0 on
template <bool F16, int D, int R, int N>
__device__ __forceinline__ void write_row(const Fp4Args& a, const floatx4 (&o)[N], float l, int seq, int head, int row, int x0, int lane) {
  const float inv = l == 0.f ? 0.f : 1.f / l;  // (no visible key: zeros; a NaN sum goes through)
  uint16_t* dst = a.out + static_cast<int64_t>(seq) * a.o_st + static_cast<int64_t>(head * a.group + row) * a.o_sh;
#pragma unroll
  for (int x = 0; x < N; ++x)
    *reinterpret_cast<u32x2*>(dst + Shape<D, R>::dim(x0 + x, lane)) =
        u32x2{pack_out<F16>(o[x][0] * inv, o[x][1] * inv), pack_out<F16>(o[x][2] * inv, o[x][3] * inv)};
}

// Partial results of the same rows together: a part without keys has max -inf and
// zeros, one whose scores are all NaN max -inf and a NaN sum.
template <int N>
__device__ __forceinline__ void join(float& m, float& l, floatx4 (&o)[N], float m1, float l1, const floatx4 (&o1)[N]) {
  const float top = fmaxf(m, m1);
  const float w0 = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top), w1 = m1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m1 - top);
  l = l != l || l1 != l1 ? __uint_as_float(0x7FC00000u) : l * w0 + l1 * w1;
#pragma unroll
  for (int x = 0; x < N; ++x) o[x] = o[x] * w0 + o1[x] * w1;
  m = top;
}

// How a workgroup's waves meet kv heads and pages: a head each; fewer heads, and the
// 16 subs keys of a wave's loads in one page; fewer heads, any pages.  (Keys in one
// page have one base and 32-bit offsets: 64 x 16000 keys of 2 heads, pages of 256,
// 67.5 us with the last, 57.8 with the second.)
enum Heads { kFour, kOnePage, kAnyPages };

template <bool F16, int D, int R, Heads HEADS>
__global__ void __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(3))) paged_fp4_kernel(const Fp4Args a) {
  constexpr int kRow = D / 2;             // bytes of a key
  constexpr int kChunks = kRow / 16, kChunksLog2 = D == 128 ? 2 : 1;
  constexpr int kLoads = kTile * kRow / 1024;  // of a wave, of K and of V
  constexpr int kPer = Shape<D, R>::kPer, kSets = Shape<D, R>::kSets, kVecs = Shape<D, R>::kVecs;
  constexpr int kTerms = F16 ? 2 : 1;     // bf16 terms of a weight
  constexpr int kWords = kRow / 16;       // of a key in a lane: products of the scores
  // a wave's share of LDS: K, V, their exponents, V's as numbers, by 32 dims; then joined parts
  constexpr int kKeyExps = 2 * kTile * kRow, kValueExps = kKeyExps + kTile * 4, kNumbers = kValueExps + kTile * 4;
  constexpr int kStage = kNumbers + kTile * D / 8, kJoin = kVecs * 1024 + 512;
  constexpr int kShare = (kStage > kJoin ? kStage : kJoin) + 64;  // (heads' rows a quarter of the banks apart)
  static_assert(kShare % 256 == 64, "rows of four heads meet different banks");
  __shared__ __attribute__((aligned(256))) uint8_t lds[kWaves * kShare];
  __shared__ __attribute__((aligned(16))) int absent[kWaves * 4];  // by 16 keys of a step: 1 where they have no block (read four at a time)

  const uint32_t lane = threadIdx.x % 64, n = lane % 16, g = lane / 16;
  const int wave = uniform_int(threadIdx.x / 64);
  const int heads_log2 = HEADS == kFour ? kWavesLog2 : a.heads_log2;
  const int subs_log2 = kWavesLog2 - heads_log2;
  const int my_head = wave & ((1 << heads_log2) - 1), sub = wave >> heads_log2;
  const int step_log2 = 6 + subs_log2;
  const int me = static_cast<int>(blockIdx.x);
  const Scratch<D, R> scratch(a.work, a.shares);
  // a sequence's blocks: of R rows, for each group of kv heads
  const int head_groups = a.kv_heads >> heads_log2, blocks = head_groups * ((a.group + R - 1) / R);
  auto steps_of = [&](int keys) { return max((keys + (1 << step_log2) - 1) >> step_log2, 1); };
  auto listed = [&](int keys) { return a.whole ? 1 : steps_of(keys); };  // entries of the list

  // ---- this workgroup's share of the list.  A lane has `each` sequences.
  const int each = (a.batch + 63) / 64;
  int mine = 0;
  for (int j = 0; j < each; ++j) {
    const int i = static_cast<int>(lane) * each + j;
    if (i < a.batch) mine += listed(keys_of(a, i));
  }
  mine *= blocks;
  const int incl = wave_scan(mine, Add());
  const int total = __builtin_amdgcn_readlane(incl, 63);
  // Its steps: as many as spread the list over the chip's places, but up to three where
  // it is shorter and sequences have several, for fewer parts (one conversation of 16000
  // keys 22 -> 17 us, eight of 2600 18.7 -> 18; of up to a step a CU one: 1800 keys 10.7,
  // with two 14; 300 sequences of a step or two, one after the other 26.5, else 20).
  const int least = !a.whole && total / 4 >= a.numbers ? min(divide(total - 1, a.by_cus), 2) : 0;
  const int share = max(divide(total - 1, a.by_shares), least) + 1;
  const int from = me * share;
  int left = min(share, total - from);
  if (!a.by_number && threadIdx.x == 0) scratch.splits[me].parts = 0;
  if (left <= 0) return;
  int seq, offset;  // in the sequence
  {
    const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(incl > from));
    offset = from - __builtin_amdgcn_readlane(incl - mine, l);
    seq = l * each;
  }

  uint8_t* const stage = lds + wave * kShare;
  uint8_t* const v_stage = stage + kTile * kRow;
  uint32_t* const ks_stage = reinterpret_cast<uint32_t*>(stage + kKeyExps);
  uint32_t* const vs_stage = reinterpret_cast<uint32_t*>(stage + kValueExps);
  float* const numbers = reinterpret_cast<float*>(stage + kNumbers);
  const float scale = (a.scale_log2 == 0.f ? 1.f : fabsf(a.scale_log2)) * (F16 ? static_cast<float>(1u << kKeyShift) : 1.f);

  while (left > 0) {
    const int klen = uniform_int(keys_of(a, seq)), seq_steps = uniform_int(listed(klen));
    const int all = blocks * seq_steps;
    if (offset >= all) {
      offset -= all;
      ++seq;
      continue;
    }
    const int at = uniform_int(static_cast<uint32_t>(offset) / static_cast<uint32_t>(seq_steps));
    const int step0 = uniform_int(offset - at * seq_steps), steps = uniform_int(min(seq_steps - step0, left));
    const int row_block = at / head_groups;
    const int h0 = (at - row_block * head_groups) << heads_log2, h = h0 + my_head;
    const int my_row = row_block * R + n % R;
    const bool real = my_row < a.group;

    // ---- the queries
    u32x4 qop[kWords];
    {
      const uint16_t* src = a.q + static_cast<int64_t>(seq) * a.q_st + static_cast<int64_t>(h * a.group + min(my_row, a.group - 1)) * a.q_sh;
      const uint32_t keep = !real || a.scale_log2 == 0.f ? 0u : ~0u, flip = a.scale_log2 < 0.f ? 0x80008000u & keep : 0u;
#pragma unroll
      for (int x = 0; x < kWords; ++x) {
        qop[x] = *reinterpret_cast<const u32x4*>(src + (g * kWords + x) * 8);
#pragma unroll
        for (int j = 0; j < 4; ++j) qop[x][j] = (qop[x][j] & keep) ^ flip;
      }
    }

    // ---- loads of a step: 16 subs keys of all heads.  Keys and values past the L2
    // (16 x 32768 keys: 120 us, 99 so); exponents of other heads share lines.
    const int subs = 1 << subs_log2;
    const uint8_t* const k_head = a.k + h0 * a.k_sh;
    const uint8_t* const v_head = a.v + h0 * a.v_sh;
    const uint8_t* const ks_head = a.ks + h0 * a.ks_sh;
    const uint8_t* const vs_head = a.vs + h0 * a.vs_sh;
    const int32_t* bt_row = a.bt + static_cast<int64_t>(seq) * a.bt_sb;
    int ids_base = 0, ids = 0;
    auto load_ids = [&](int base) {
      ids_base = base;
      ids = bt_row[static_cast<int64_t>(min(base + static_cast<int>(lane), a.width - 1)) * a.bt_sn];
    };
    auto first_key = [&](int step) { return (step << step_log2) + (wave << (4 + subs_log2)); };

    u32x4 kw[kLoads], vw[kLoads];
    uint32_t ksw = 0, vsw = 0;
    int missing = 0;  // bit x: the x-th 16 keys of the wave's loads are not there
    typedef typename std::conditional<D == 128, uint32_t, uint16_t>::type exponents;
    auto issue = [&](int step) {
      constexpr int kGroups = HEADS == kAnyPages ? 4 : 1;
      const int all = HEADS == kOnePage ? (1 << subs) - 1 : 1;
      missing = 0;
      int blk[kGroups], row[kGroups];
#pragma unroll
      for (int x = 0; x < kGroups; ++x) {
        const int key = first_key(step) + 16 * x;
        blk[x] = row[x] = 0;
        if (x >= subs || key >= klen) {  // (nobody's keys: any bytes of the cache)
          missing |= all << x;
          continue;
        }
        const int p = divide(key, a.by_page);
        row[x] = key - p * a.page;
        if (p >= ids_base + 64) load_ids(p);
        blk[x] = uniform_int(__builtin_amdgcn_readlane(ids, p - ids_base));
        if (blk[x] < 0 || blk[x] >= a.num_blocks) {
          missing |= all << x;
          blk[x] = row[x] = 0;
        }
      }
      // a lane's rows: `key` of the wave's, in the page of its 16
      auto at = [&](const uint8_t* head, int64_t sn, int st, uint32_t key, uint32_t offset) {
        if constexpr (HEADS != kAnyPages) {  // a uniform base, 32-bit offsets of the lanes
          return head + blk[0] * sn + static_cast<int64_t>(row[0]) * st + (key * st + offset);
        } else {
          int b = blk[0], r = row[0];
#pragma unroll
          for (int x = 1; x < kGroups; ++x) {
            const int bx = uniform_int(blk[x]), rx = uniform_int(row[x]);  // (as an element by number the table goes to memory)
            if (key / 16 == x) b = bx, r = rx;
          }
          return head + b * sn + (static_cast<int64_t>(r) + key % 16) * st + offset;
        }
      };
      const uint32_t l = fresh(lane), heads = 1u << heads_log2;
      {
        const uint32_t key = l >> heads_log2, head = l & (heads - 1);
        ksw = *reinterpret_cast<const exponents*>(at(ks_head, a.ks_sn, a.ks_st, key, head * static_cast<uint32_t>(a.ks_sh)));
        vsw = *reinterpret_cast<const exponents*>(at(vs_head, a.vs_sn, a.vs_st, key, head * static_cast<uint32_t>(a.vs_sh)));
      }
      const int per = heads_log2 + kChunksLog2;  // lanes of a key
      const uint32_t head = l / kChunks & (heads - 1), chunk = l % kChunks;
#pragma unroll
      for (int x = 0; x < kLoads; ++x) {
        const uint32_t key = (x << (6 - per)) + (l >> per);
        kw[x] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at(k_head, a.k_sn, a.k_st, key, head * static_cast<uint32_t>(a.k_sh) + chunk * 16)));
        vw[x] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at(v_head, a.v_sn, a.v_st, key, head * static_cast<uint32_t>(a.v_sh) + chunk * 16)));
      }
    };
    // ... to the shares of the waves that compute with them
    auto deliver = [&]() {
      const uint32_t l = fresh(lane), heads = 1u << heads_log2;
      const uint32_t before = (wave & (kWaves - 1)) << (4 + subs_log2);  // keys of the step
      const int per = heads_log2 + kChunksLog2;
      const uint32_t head = l / kChunks & (heads - 1), chunk = l % kChunks;
#pragma unroll
      for (int x = 0; x < kLoads; ++x) {
        const uint32_t all = before | x << (6 - per) | l >> per, key = all % kTile;
        uint8_t* to = lds + (head + (all / kTile << heads_log2)) * kShare + key * kRow;
        *reinterpret_cast<u32x4*>(to + ((chunk ^ (key / 4 % kChunks)) << 4)) = kw[x];
        *reinterpret_cast<u32x4*>(to + kTile * kRow + ((chunk ^ (key / 16 % kChunks)) << 4)) = vw[x];
      }
      const uint32_t all = before | l >> heads_log2, key = all % kTile;
      uint32_t* to = reinterpret_cast<uint32_t*>(lds + ((l & (heads - 1)) + (all / kTile << heads_log2)) * kShare + kKeyExps) + key;
      to[0] = ksw;
      to[kTile] = vsw;
      if (l < subs) absent[(wave << subs_log2) + l] = missing >> l & 1;
    };
    // (what is in flight to registers stays so)
    auto meet = [&]() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory"); };

    typedef uint32_t k_words __attribute__((ext_vector_type(kWords)));
    floatx4 acc[D / 16];
#pragma unroll
    for (int x = 0; x < D / 16; ++x) acc[x] = floatx4{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_run = 0.f;
    float above = 0.f, most = 256.f;  // of the running max over the scores' own, and of a lane's sum of weights
    int nan_blocks = 0;  // bit x: a key has a NaN exponent for values' 32 dims x; the last one: for its own

    const int end = klen > 0 ? step0 + (a.whole ? steps_of(klen) : steps) : step0;  // (without keys there may be no cache)
    if (step0 < end) {
      if (first_key(step0) < klen) load_ids(uniform_int(divide(first_key(step0), a.by_page)));
      issue(step0);
    }
    for (int step = step0; step < end; ++step) {
      deliver();
      meet();
      if (step + 1 < end) issue(step + 1);
      const int key0 = (step << step_log2) + sub * kTile;
      if (key0 >= klen) {
        meet();
        continue;
      }
      const uint32_t lw = fresh(lane);
      const u32x4 none = *reinterpret_cast<const u32x4*>(absent + 4 * sub);
      const int gone = uniform_int(static_cast<int>(none[0] | none[1] << 1 | none[2] << 2 | none[3] << 3));
      const bool partial = gone != 0 || key0 + kTile > klen;
      uint32_t kx = ks_stage[lw], vx = vs_stage[lw];
      if (partial && (static_cast<int>(key0 + lw) >= klen || (gone >> (lw / 16) & 1))) kx = vx = 0;  // nobody's: 0 times anything finite
      auto has_nan = [](uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & w & 0x80808080u; };
      auto has_large = [](uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x30303030u) & w & 0x80808080u; };  // 208 and more
      if (__builtin_amdgcn_ballot_w64((has_nan(kx) | has_large(vx)) != 0) != 0) {
        if (has_nan(kx) != 0) nan_blocks |= 1 << (D / 32);
#pragma unroll
        for (int x = 0; x < D / 32; ++x)
          if ((vx >> (8 * x) & 0xFFu) == 0xFFu) vx &= ~(0xFFu << (8 * x)), nan_blocks |= 1 << x;
        // Values of up to 2^128: weights of at most 2^-24 leave 2^22 keys' sum of them finite.
        if (__builtin_amdgcn_ballot_w64(has_large(vx) != 0) != 0) above = 32.f, most = 0x1p-24f;
      }
      if (partial) ks_stage[lw] = kx;
#pragma unroll
      for (int x = 0; x < D / 32; ++x) numbers[x * kTile + lw] = __uint_as_float((vx >> (8 * x) & 0xFFu) << 23);
      wave_lds_order();
      const bool wide = F16 && __builtin_amdgcn_ballot_w64(off_float16(kx) != 0) != 0;
      floatx4 sc[4];
      auto scores = [&]() __attribute__((always_inline)) {
        const uint32_t k_rd = n * kRow + (((D == 128 ? g : g / 2) ^ (n / 4 % kChunks)) << 4) + (D == 128 ? 0 : g % 2 * 8);
        auto read_k = [&](int x) { return *reinterpret_cast<const k_words*>(stage + k_rd + 16 * x * kRow); };
        auto read_ke = [&](int x) { return static_cast<uint32_t>(reinterpret_cast<const uint8_t*>(ks_stage)[(16 * x + n) * 4 + (D == 128 ? g : g / 2)]); };
        uint32_t ke[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          ke[x] = read_ke(x);
          sc[x] = floatx4{0.f, 0.f, 0.f, 0.f};
        }
        if (F16 && __builtin_expect(wide, false)) {
#pragma unroll
          for (int y = 0; y < kWords; ++y) {
            uint32_t w[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) w[x] = *reinterpret_cast<const uint32_t*>(stage + k_rd + 16 * x * kRow + 4 * y);
            u32x4 whole = qop[y], q[2];
            asm volatile("" : "+v"(whole));  // (split where it is used: kept, the terms spill)
            split_float16(whole, 1.0f / (1u << kKeyShift), q[0], q[1]);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const u32x4 k = widen_key<false>(w[x], ke[x]);
#pragma unroll
              for (int term = 0; term < 2; ++term) sc[x] = score_product<false>(k, q[term], sc[x]);
              __builtin_amdgcn_sched_barrier(0);
            }
          }
        } else {
          k_words w[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) w[x] = read_k(x);
          // (four products that do not wait for each other)
#pragma unroll
          for (int y = 0; y < kWords; ++y)
#pragma unroll
            for (int x = 0; x < 4; ++x) sc[x] = score_product<F16>(widen_key<F16>(w[x][y], ke[x]), qop[y], sc[x]);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (partial) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int left_keys = gone >> x & 1 ? 0 : klen - key0 - 16 * x - 4 * static_cast<int>(g);
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[x][i] = i < left_keys ? sc[x][i] : -INFINITY;
          }
        }
      };
      scores();

      // ---- softmax.  Weights against the running max as it stands; their sum tells
      // whether that is high enough (2^8, beside large values 2^-24), or is no number, as
      // before the first: only then the scores are taken once more, and their max.
      auto weights = [&](float m) __attribute__((always_inline)) {
        float sum = 0.f;
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sc[x][i] = __builtin_amdgcn_exp2f(fmaf(sc[x][i], scale, -m));
            sum += sc[x][i];
          }
        return sum;
      };
      float sum = weights(m_run);
      if (__builtin_amdgcn_ballot_w64(!(sum <= most)) != 0) {
        scores();
        float top = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3]));
#pragma unroll
        for (int x = 1; x < 4; ++x) top = fmaxf(top, fmaxf(fmaxf(sc[x][0], sc[x][1]), fmaxf(sc[x][2], sc[x][3])));
        top = wave_max_across_groups(top) * scale;
        const float m_new = fmaxf(m_run, top + above);
        const float alpha = m_new > m_run ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.f;
        l_run *= alpha;
#pragma unroll
        for (int x = 0; x < D / 16; ++x) acc[x] *= alpha;
        m_run = m_new;
        sum = weights(m_run == -INFINITY ? 0.f : m_run);
      }
      l_run += sum;
      __builtin_amdgcn_sched_barrier(0);

      // ---- output.  (The lane's place anew: kept, its eight forms take registers.)
      const uint32_t l = fresh(lane);
      const uint32_t v_rd = (16 * (l / 4 % 4) + 4 * (l / 16) + l % 4) * kRow + ((l / 4 % 4 % kChunks) << 4);
#pragma unroll
      for (int set = 0; set < kSets; ++set) {
        u32x4 pw[kTerms][2];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          floatx4 w = sc[x] * *reinterpret_cast<const floatx4*>(numbers + (set * kPer + n / R) * kTile + 16 * x + 4 * g);
#pragma unroll
          for (int term = 0; term < kTerms; ++term)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t two = pack_bf16(w[2 * i], w[2 * i + 1]);
              pw[term][x / 2][x % 2 * 2 + i] = two;
              w[2 * i] -= __uint_as_float(two << 16);
              w[2 * i + 1] -= __uint_as_float(two & 0xFFFF0000u);
            }
        }
        auto read_v = [&](int m) {  // 16 dims of 64 keys
          return __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_i32x2*)(v_stage + ((v_rd ^ (m / 2 << 4)) + m % 2 * 8)));
        };
        i32x2 next[2] = {read_v(set * 2 * kPer), read_v(set * 2 * kPer + 1)};
#pragma unroll
        for (int y = 0; y < 2 * kPer; y += 2) {
          const int m = set * 2 * kPer + y;
          const i32x2 w0 = next[0], w1 = next[1];
          if (y + 2 < 2 * kPer) next[0] = read_v(m + 2), next[1] = read_v(m + 3);
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const bf16x8 v0 = fp4x8_to_bf16x8(w0[z]), v1 = fp4x8_to_bf16x8(w1[z]);
#pragma unroll
            for (int term = 0; term < kTerms; ++term) {
              acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, __builtin_bit_cast(bf16x8, pw[term][z]), acc[m], 0, 0, 0);
              acc[m + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, __builtin_bit_cast(bf16x8, pw[term][z]), acc[m + 1], 0, 0, 0);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      meet();
    }

    // ---- the columns' own blocks
    float l_tot = sum_across_groups(l_run);
    if (__builtin_amdgcn_ballot_w64(nan_blocks != 0) != 0) {
#pragma unroll
      for (int x = 0; x < D / 32; ++x)
        if (__builtin_amdgcn_ballot_w64(nan_blocks >> x & 1) != 0)
#pragma unroll
          for (int y = 0; y < 4; ++y) acc[2 * x][y] = acc[2 * x + 1][y] = __uint_as_float(0x7FC00000u);
      if (__builtin_amdgcn_ballot_w64(nan_blocks >> (D / 32)) != 0) l_tot = __uint_as_float(0x7FC00000u);
    }
    floatx4 o[kVecs];
    const uint32_t le = fresh(lane);
#pragma unroll
    for (int x = 0; x < kVecs; ++x) {
      o[x] = acc[x / 2 * 2 * kPer + x % 2];
#pragma unroll
      for (int y = 1; y < kPer; ++y)
        if (le % 16 / R == y) o[x] = acc[(x / 2 * kPer + y) * 2 + x % 2];
    }
    if (subs > 1) {  // parts of the keys in other waves
      floatx4* own = reinterpret_cast<floatx4*>(stage);
      floatx2* own_ml = reinterpret_cast<floatx2*>(stage + kVecs * 1024);
      if (sub > 0) {
#pragma unroll
        for (int x = 0; x < kVecs; ++x) own[x * 64 + le] = o[x];
        own_ml[le] = floatx2{m_run, l_tot};
      }
      __syncthreads();
      if (sub == 0) {
        for (int y = 1; y < subs; ++y) {
          const uint8_t* theirs = lds + (my_head + (y << heads_log2)) * kShare;
          const floatx2 ml = reinterpret_cast<const floatx2*>(theirs + kVecs * 1024)[le];
          floatx4 o1[kVecs];
#pragma unroll
          for (int x = 0; x < kVecs; ++x) o1[x] = reinterpret_cast<const floatx4*>(theirs)[x * 64 + le];
          join(m_run, l_tot, o, ml[0], ml[1], o1);
        }
      }
      __syncthreads();
    }
    const bool begins = step0 == 0, ends = step0 + steps == seq_steps;
    if (begins && ends) {
      if (sub == 0 && real) write_row<F16, D, R>(a, o, l_tot, seq, h, row_block * R + le % R, 0, le);
    } else if (sub == 0) {
      float* part = scratch.parts + (((static_cast<int64_t>(me) * 2 + (begins ? 1 : 0)) << heads_log2) + my_head) * Scratch<D, R>::kPart;
#pragma unroll
      for (int x = 0; x < kVecs; ++x) reinterpret_cast<floatx4*>(part)[x * 64 + le] = o[x];
      if (le < R) reinterpret_cast<floatx2*>(part + R * D)[le] = floatx2{m_run, l_tot};
    }
    if (begins && threadIdx.x == 0 && (a.by_number || !ends)) {
      scratch.splits[a.by_number ? seq * blocks + at : me] =
          Split{ends ? 0 : 1 + (seq_steps - steps + share - 1) / share, me, seq, h, row_block * R};
    }
    left -= steps;
    offset += steps;
  }
}

// Joins the parts of split sequences: a workgroup per description, head and two
// vectors, its waves taking parts in turn.
constexpr int kJoinWaves = 8;

template <bool F16, int D, int R>
__global__ void __launch_bounds__(64 * kJoinWaves) paged_fp4_join_kernel(const Fp4Args a) {
  constexpr int kVecs = Shape<D, R>::kJoined, kPart = Scratch<D, R>::kPart;
  __shared__ floatx4 rows[kJoinWaves][kVecs * 64];
  __shared__ floatx2 stats[kJoinWaves][64];
  const Scratch<D, R> scratch(a.work, a.shares);
  const int my_head = static_cast<int>(blockIdx.x) & ((1 << a.heads_log2) - 1);
  const Split s = scratch.splits[blockIdx.x >> a.heads_log2];
  if (s.parts == 0) return;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, x0 = static_cast<int>(blockIdx.y) * kVecs;
  float m_run = -INFINITY, l_run = 0.f;
  floatx4 o[kVecs];
#pragma unroll
  for (int x = 0; x < kVecs; ++x) o[x] = floatx4{0.f, 0.f, 0.f, 0.f};
  constexpr int kAtOnce = 4;
  for (int p0 = wave * kAtOnce; p0 < s.parts; p0 += kJoinWaves * kAtOnce) {
    floatx4 v[kAtOnce][kVecs];
    floatx2 ml[kAtOnce];
#pragma unroll
    for (int y = 0; y < kAtOnce; ++y) {
      const int p = min(p0 + y, s.parts - 1);
      const int64_t slot = p == 0 ? 2 * static_cast<int64_t>(s.share) + 1 : 2 * (static_cast<int64_t>(s.share) + p);
      const float* part = scratch.parts + ((slot << a.heads_log2) + my_head) * kPart;
#pragma unroll
      for (int x = 0; x < kVecs; ++x) v[y][x] = reinterpret_cast<const floatx4*>(part)[(x0 + x) * 64 + lane];
      ml[y] = reinterpret_cast<const floatx2*>(part + R * D)[lane % R];
    }
#pragma unroll
    for (int y = 0; y < kAtOnce; ++y)
      if (p0 + y < s.parts) join(m_run, l_run, o, ml[y][0], ml[y][1], v[y]);
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
    join(m_run, l_run, o, stats[y][lane][0], stats[y][lane][1], v);
  }
  const int row = s.row0 + lane % R;
  if (row < a.group) write_row<F16, D, R>(a, o, l_run, s.seq, s.head + my_head, row, x0, lane);
}

int heads_log2(int kv_heads) { return kv_heads % 4 == 0 ? 2 : kv_heads % 2 == 0 ? 1 : 0; }

// Rows of an operand: a kv head's group, rounded up.
int row_block(int group, int head_dim) { return group > 8 ? 16 : group > 4 || head_dim == 64 ? 8 : 4; }

int share_count() { return 3 * device_cu_count(); }

int64_t scratch_bytes(int group, int kv_heads, int head_dim) {
  const int r = row_block(group, head_dim), shares = share_count();
  return Scratch<128, 16>::head(shares) + ((static_cast<int64_t>(2 * shares) << heads_log2(kv_heads)) * (r * head_dim + 2 * r)) * 4;
}

template <bool F16, int D, int R>
int launch(const Fp4Args& a, hipStream_t stream) {
  const dim3 grid(a.shares), threads(64 * kWaves);
  if (a.heads_log2 == kWavesLog2) hipLaunchKernelGGL((paged_fp4_kernel<F16, D, R, kFour>), grid, threads, 0, stream, a);
  else if (a.page % (16 << (kWavesLog2 - a.heads_log2)) == 0) hipLaunchKernelGGL((paged_fp4_kernel<F16, D, R, kOnePage>), grid, threads, 0, stream, a);
  else hipLaunchKernelGGL((paged_fp4_kernel<F16, D, R, kAnyPages>), grid, threads, 0, stream, a);
  if (int rc = check_launch("paged_fp4_kernel launch")) return rc;
  if (a.whole) return PRISM_OK;
  hipLaunchKernelGGL((paged_fp4_join_kernel<F16, D, R>), dim3(a.splits << a.heads_log2, Shape<D, R>::kVecs / Shape<D, R>::kJoined), dim3(64 * kJoinWaves), 0, stream, a);
  return check_launch("paged_fp4_join_kernel launch");
}

template <bool F16>
int dispatch(const Fp4Args& a, int head_dim, hipStream_t stream) {
  const int r = row_block(a.group, head_dim);
  if (head_dim == 128)
    return r == 4 ? launch<F16, 128, 4>(a, stream) : r == 8 ? launch<F16, 128, 8>(a, stream) : launch<F16, 128, 16>(a, stream);
  return r == 8 ? launch<F16, 64, 8>(a, stream) : launch<F16, 64, 16>(a, stream);
}

}  // namespace

int preload_paged_fp4() {
  hipFuncAttributes attr;
  return check_hip(hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(&paged_fp4_kernel<false, 128, 4, kFour>)), "preload_paged_fp4");
}

}  // namespace prism

extern "C" int64_t prism_paged_fp4_workspace_bytes(int chunks, int batch, int total_q, int num_heads, int num_kv_heads, int head_dim,
                                                   int page_size, int width) {
  if (batch <= 0 || total_q <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || head_dim <= 0 ||
      page_size <= 0 || width < 0)
    return 0;
  if (chunks != 0)
    return prism::paged_prefill4_workspace_bytes(batch, total_q, num_heads, num_kv_heads, head_dim, page_size, width);
  return prism::scratch_bytes(num_heads / num_kv_heads, num_kv_heads, head_dim);
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
    if (s[1] < 0 || s[1] > INT32_MAX / 2 / page_size || s[2] < 0 || s[2] > INT32_MAX / 8) {
      set_error("%s: a page must span less than 1 GiB, and eight heads less than 2", what);
      return PRISM_ERR_LAYOUT;
    }
  const int64_t need = prism_paged_fp4_workspace_bytes(chunks, batch, total_q, num_heads, num_kv_heads, head_dim, page_size, width);
  if (workspace_bytes < need || (need > 0 && (!workspace || !aligned(workspace, 256)))) {
    set_error("%s: the workspace needs %lld bytes, 256-byte aligned", what, static_cast<long long>(need));
    return PRISM_ERR_INVALID;
  }
  if (chunks)
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
  a.out = static_cast<uint16_t*>(out);
  a.o_st = out_strides[0], a.o_sh = out_strides[1];
  a.batch = batch, a.heads = num_heads, a.kv_heads = num_kv_heads, a.group = num_heads / num_kv_heads;
  a.page = page_size, a.num_blocks = num_blocks;
  a.width = num_blocks > 0 ? width : 0;  // (without pages nothing is read)
  a.room = static_cast<int>(std::min<int64_t>(static_cast<int64_t>(a.width) * page_size, kMostKeys));
  a.scale_log2 = scale * 1.4426950408889634f;
  a.heads_log2 = heads_log2(num_kv_heads);
  a.shares = share_count();
  const int64_t numbers = static_cast<int64_t>(batch) * (num_kv_heads >> a.heads_log2) * ceil_div(a.group, row_block(a.group, head_dim));
  // (the steps of the list, and a share beyond it, in 32 bits)
  if (numbers * (static_cast<int64_t>(a.room) / kTile + 1) > (1 << 30)) {
    set_error("%s: %lld blocks of rows of up to %d keys are too many steps for one launch", what, static_cast<long long>(numbers), a.room);
    return PRISM_ERR_INVALID;
  }
  a.by_shares = divisor(a.shares);
  a.by_cus = divisor(device_cu_count());
  a.by_number = numbers <= a.shares;
  a.numbers = static_cast<int>(numbers);
  // Tables of few steps: parts and their join cost more than a second step in turn (8
  // heads, pages of 64: 64 sequences of 128 keys 11.1 us split, 9.2 whole; of four steps
  // 13.8 and 13.9, one sequence 10.1 and 12.4).
  a.whole = a.room <= kWholeSteps * kTile << (kWavesLog2 - a.heads_log2);
  a.splits = a.by_number ? static_cast<int>(numbers) : a.shares;
  a.work = static_cast<uint8_t*>(workspace);
  a.by_page = divisor(page_size);
  hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
  return q_dtype == PRISM_DTYPE_F16 ? dispatch<true>(a, head_dim, stream) : dispatch<false>(a, head_dim, stream);
}
