// Position rotation of a step's queries and keys, with the keys and values
// appended to a paged cache on the way; and rows of a cache read back.
//
//   a' = a c - b s,  b' = b c + a s,  (c, s) = (cos, sin)(position * rate_i)
//
// for each pair (a, b) = (x[i], x[i + n / 2]) of a head's first n dims, or
// (x[2 i], x[2 i + 1]) where pairs are neighbours; the other dims stay.  Products
// and sums are rounded one by one in fp32 and the results to the input's type, as
// an op of its own would leave them; then keys and values are stored as the store
// stores them (kv_quant.h, fp4.h), bit for bit what the two ops give in turn.
//
// Work layout.  A token's rows are its query, key and value heads in that order.
// D / 8 lanes hold a row, eight dims each, and a wave a pass of 64 / (D / 8) rows;
// a lane has the same dims in each of its wave's passes, so that the token's cosines
// and sines are loaded once.  The other half of a pair is another lane's.
// Bound by HBM (prompts) and by one launch with two dependent loads (single steps).
#include "common.h"
#include "divide.h"
#include "fp4.h"
#include "kv_quant.h"
#include "wave_ops.h"

#include <algorithm>

namespace prism {
namespace {

constexpr int kCachePlain = 0, kCacheFp8 = 1, kCacheFp8Scaled = 2, kCacheFp4 = 3;

struct RotateArgs {
  const char* q;
  const char* k;
  const char* v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;  // bytes
  const float* table;      // [max_positions, rotary]: cosines, then sines
  const int32_t* positions;
  int64_t axis_stride;
  const int32_t* axes;     // [rotary / 2], or null: all 0
  int num_axes, rotary, pairs;
  int64_t max_positions;
  char* q_out;             // dense
  char* k_out;             // dense, or null
  char* k_cache;
  char* v_cache;
  void* k_scale;
  void* v_scale;
  const int32_t* slots;
  int64_t tokens, num_slots;
  int q_heads, heads, dim, cache_dtype, kind;
  int waves_per_token;
  Divisor by_waves;
};

template <int IN>
struct Raw8 {  // eight values of the input's type, as loaded
  static constexpr int kWords = IN == PRISM_DTYPE_F32 ? 8 : 4;
  uint32_t w[kWords];
};

template <int IN>
__device__ __forceinline__ void to_float(const Raw8<IN>& r, float (&x)[8]) {
  if constexpr (IN == PRISM_DTYPE_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(r.w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (IN == PRISM_DTYPE_BF16) {
        x[2 * i] = __uint_as_float(r.w[i] << 16);
        x[2 * i + 1] = __uint_as_float(r.w[i] & 0xFFFF0000u);
      } else {
        x[2 * i] = f16_bits_to_f32(r.w[i] & 0xFFFFu);
        x[2 * i + 1] = f16_bits_to_f32(r.w[i] >> 16);
      }
    }
  }
}

__device__ __forceinline__ uint32_t pack16(int dtype, float lo, float hi) {
  return dtype == PRISM_DTYPE_BF16 ? f32_to_bf16_bits(lo) | (static_cast<uint32_t>(f32_to_bf16_bits(hi)) << 16)
                                   : f32_to_f16_bits(lo) | (static_cast<uint32_t>(f32_to_f16_bits(hi)) << 16);
}

template <int IN>
__device__ __forceinline__ void from_float(const float (&x)[8], Raw8<IN>& r) {
  if constexpr (IN == PRISM_DTYPE_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i] = __float_as_uint(x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = pack16(IN, x[2 * i], x[2 * i + 1]);
  }
}

template <int IN>
__device__ __forceinline__ Raw8<IN> load8(const char* p) {
  Raw8<IN> r;
#pragma unroll
  for (int i = 0; i < Raw8<IN>::kWords; i += 4) {
    const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p) + i / 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) r.w[i + j] = x[j];
  }
  return r;
}

template <int IN>
__device__ __forceinline__ void store8(char* p, const Raw8<IN>& r) {
#pragma unroll
  for (int i = 0; i < Raw8<IN>::kWords; i += 4)
    __builtin_nontemporal_store(u32x4{r.w[i], r.w[i + 1], r.w[i + 2], r.w[i + 3]}, reinterpret_cast<u32x4*>(p) + i / 4);
}

// Products and their sum, each rounded (no fused step, which would round once).
__device__ __forceinline__ float turned(float x, float c, float y, float s) {
#pragma clang fp contract(off)
  const float p = x * c, q = y * s;
  return p + q;
}

// The cosines and sines of `count` angles from index i on, for one token; NaN where
// a position, or an axis, is outside its range.
template <int N>
__device__ __forceinline__ void load_angles(const RotateArgs& a, int64_t token, int i, float (&c)[N], float (&s)[N]) {
  int axis[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    c[j] = s[j] = __uint_as_float(0x7FC00000u);
    axis[j] = a.axes == nullptr ? 0 : a.axes[i + j];
  }
  for (int x = 0; x < a.num_axes; ++x) {
    const int64_t at = a.positions[x * a.axis_stride + token];
    if (at < 0 || at >= a.max_positions) continue;
    const float* row = a.table + at * a.rotary + i;
    float cx[N], sx[N];
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const floatx4 u = *reinterpret_cast<const floatx4*>(row + j), v = *reinterpret_cast<const floatx4*>(row + a.rotary / 2 + j);
#pragma unroll
      for (int y = 0; y < 4; ++y) cx[j + y] = u[y], sx[j + y] = v[y];
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      c[j] = axis[j] == x ? cx[j] : c[j];
      s[j] = axis[j] == x ? sx[j] : s[j];
    }
  }
}

// A row's eight values of this lane -> the cache, at row `at` of its rows.
template <int IN, int LANES>
__device__ __forceinline__ void append8(const RotateArgs& a, const Raw8<IN>& r, char* cache, void* scales, int64_t at, int sub,
                                        bool live) {
  float x[8];
  if (a.kind == kCachePlain) {
    if (!live) return;
    if (a.cache_dtype == IN) {
      store8<IN>(cache + (at * LANES + sub) * (IN == PRISM_DTYPE_F32 ? 32 : 16), r);
      return;
    }
    to_float<IN>(r, x);
    if (a.cache_dtype == PRISM_DTYPE_F32) {
      Raw8<PRISM_DTYPE_F32> out;
      from_float<PRISM_DTYPE_F32>(x, out);
      store8<PRISM_DTYPE_F32>(cache + (at * LANES + sub) * 32, out);
    } else {
      u32x4 out;
#pragma unroll
      for (int i = 0; i < 4; ++i) out[i] = pack16(a.cache_dtype, x[2 * i], x[2 * i + 1]);
      *(reinterpret_cast<u32x4*>(cache) + at * LANES + sub) = out;
    }
    return;
  }
  to_float<IN>(r, x);
  if (a.kind == kCacheFp4) {
    uint32_t exponent;
    const uint32_t codes = fp4_quantize8(x, exponent);
    if (!live) return;
    reinterpret_cast<uint32_t*>(cache)[at * LANES + sub] = codes;
    if (sub % 4 == 0) static_cast<uint8_t*>(scales)[at * (LANES / 4) + sub / 4] = static_cast<uint8_t>(exponent);
    return;
  }
  u32x2 packed;
  float s = 0.f;
  if (a.kind == kCacheFp8Scaled) packed = quantize_row<LANES>(x, s);
  else packed = u32x2{fp8_encode4(x[0], x[1], x[2], x[3]), fp8_encode4(x[4], x[5], x[6], x[7])};
  if (!live) return;
  reinterpret_cast<u32x2*>(cache)[at * LANES + sub] = packed;
  if (a.kind == kCacheFp8Scaled && sub == 0) static_cast<float*>(scales)[at] = s;
}

template <int IN, int LANES, int PASSES>
__global__ void __launch_bounds__(256) rotate_store_kernel(const RotateArgs a) {
  constexpr int kRows = 64 / LANES;  // of a pass
  constexpr int kBytes = IN == PRISM_DTYPE_F32 ? 32 : 16;
  const int wave = uniform_int(static_cast<int>(blockIdx.x) * (blockDim.x / 64) + threadIdx.x / 64);
  const int token = divide(wave, a.by_waves), part = wave - token * a.waves_per_token;
  if (token >= a.tokens) return;
  const int lane = threadIdx.x % 64, sub = lane % LANES;
  const int rows = a.q_heads + 2 * a.heads;

  int row[PASSES];
  Raw8<IN> raw[PASSES];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    row[p] = (part * PASSES + p) * kRows + lane / LANES;
    const char* src = a.q + token * a.q_st + row[p] * a.q_sh;
    if (row[p] >= a.q_heads) src = a.k + token * a.k_st + (row[p] - a.q_heads) * a.k_sh;
    if (row[p] >= a.q_heads + a.heads) src = a.v + token * a.v_st + (row[p] - a.q_heads - a.heads) * a.v_sh;
    if (row[p] < rows) raw[p] = load8<IN>(src + sub * kBytes);
    else raw[p] = Raw8<IN>{};
  }
  const int32_t slot = a.slots[token];
  const bool stored = slot >= 0 && slot < a.num_slots;

  // The lane's angles.  Halves: eight, the same for the two lanes of the pairs;
  // neighbours: four.
  const int d = 8 * sub;
  const bool turns = d < a.rotary;
  float c[8], s[8];
  int other = lane;
  if (turns && !a.pairs) {
    const int half = a.rotary / 2;
    const bool first = d < half;
    load_angles<8>(a, token, first ? d : d - half, c, s);
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = first ? -s[j] : s[j];
    other = first ? lane + half / 8 : lane - half / 8;
  } else if (turns) {
    float c4[4], s4[4];
    load_angles<4>(a, token, d / 2, c4, s4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c[2 * j] = c[2 * j + 1] = c4[j];
      s[2 * j] = -s4[j];
      s[2 * j + 1] = s4[j];
    }
  }

#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int r = row[p];
    const bool is_v = r >= a.q_heads + a.heads;
    if (a.rotary > 0 && __builtin_amdgcn_ballot_w64(!is_v) != 0) {
      Raw8<IN> pair;
      if (!a.pairs) {
#pragma unroll
        for (int i = 0; i < Raw8<IN>::kWords; ++i) pair.w[i] = __shfl(raw[p].w[i], other);
      }
      if (turns && !is_v) {
        float x[8], y[8];
        to_float<IN>(raw[p], x);
        if (a.pairs) {
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = x[j ^ 1];
        } else {
          to_float<IN>(pair, y);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = turned(x[j], c[j], y[j], s[j]);
        from_float<IN>(x, raw[p]);
      }
    }
    if (r < a.q_heads) store8<IN>(a.q_out + ((static_cast<int64_t>(token) * a.q_heads + r) * LANES + sub) * kBytes, raw[p]);
    const bool appended = r >= a.q_heads && r < rows;
    if (__builtin_amdgcn_ballot_w64(appended) == 0) continue;
    const int h = r - a.q_heads - (is_v ? a.heads : 0);
    if (a.k_out != nullptr && appended && !is_v)
      store8<IN>(a.k_out + ((static_cast<int64_t>(token) * a.heads + h) * LANES + sub) * kBytes, raw[p]);
    append8<IN, LANES>(a, raw[p], is_v ? a.v_cache : a.k_cache, is_v ? a.v_scale : a.k_scale,
                       static_cast<int64_t>(slot) * a.heads + h, sub, appended && stored);
  }
}

// Any even number of rotated dims, any head_dim, alignment and stride: a thread per
// row (quantised in 32-dim blocks, or as a whole).
__device__ __forceinline__ float load_one(const char* p, int dtype, int64_t i) {
  if (dtype == PRISM_DTYPE_F32) return reinterpret_cast<const float*>(p)[i];
  const uint32_t bits = reinterpret_cast<const uint16_t*>(p)[i];
  return dtype == PRISM_DTYPE_BF16 ? bf16_bits_to_f32(bits) : f16_bits_to_f32(bits);
}

__device__ __forceinline__ float rounded(int dtype, float x) {
  if (dtype == PRISM_DTYPE_BF16) return bf16_bits_to_f32(f32_to_bf16_bits(x));
  if (dtype == PRISM_DTYPE_F16) return f16_bits_to_f32(f32_to_f16_bits(x));
  return x;
}

__device__ __forceinline__ void store_one(char* p, int dtype, int64_t i, float x) {
  if (dtype == PRISM_DTYPE_F32) reinterpret_cast<float*>(p)[i] = x;
  else if (dtype == PRISM_DTYPE_BF16) reinterpret_cast<uint16_t*>(p)[i] = f32_to_bf16_bits(x);
  else reinterpret_cast<uint16_t*>(p)[i] = f32_to_f16_bits(x);
}

__global__ void __launch_bounds__(256) rotate_store_rows_kernel(const RotateArgs a, int in) {
  const int rows = a.q_heads + 2 * a.heads;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (unit >= a.tokens * rows) return;
  const int64_t token = unit / rows;
  const int r = static_cast<int>(unit - token * rows);
  const bool is_q = r < a.q_heads, is_v = r >= a.q_heads + a.heads;
  const int h = is_q ? r : r - a.q_heads - (is_v ? a.heads : 0);
  const char* src = is_q ? a.q + token * a.q_st + h * a.q_sh : is_v ? a.v + token * a.v_st + h * a.v_sh : a.k + token * a.k_st + h * a.k_sh;
  const int half = a.rotary / 2;
  // value d of the row, turned and rounded to the input's type
  auto value = [&](int d) {
    const float x = load_one(src, in, d);
    if (is_v || d >= a.rotary) return x;
    const int i = a.pairs ? d / 2 : d < half ? d : d - half;
    const bool first = a.pairs ? d % 2 == 0 : d < half;
    const int axis = a.axes == nullptr ? 0 : a.axes[i];
    float c = __uint_as_float(0x7FC00000u), s = c;
    if (axis >= 0 && axis < a.num_axes) {
      const int64_t at = a.positions[axis * a.axis_stride + token];
      if (at >= 0 && at < a.max_positions) {
        c = a.table[at * a.rotary + i];
        s = a.table[at * a.rotary + half + i];
      }
    }
    const float y = load_one(src, in, a.pairs ? d ^ 1 : first ? d + half : d - half);
    return rounded(in, turned(x, c, y, first ? -s : s));
  };
  if (is_q) {
    for (int d = 0; d < a.dim; ++d) store_one(a.q_out, in, (token * a.q_heads + h) * a.dim + d, value(d));
    return;
  }
  if (a.k_out != nullptr && !is_v)
    for (int d = 0; d < a.dim; ++d) store_one(a.k_out, in, (token * a.heads + h) * a.dim + d, value(d));
  const int32_t slot = a.slots[token];
  if (slot < 0 || slot >= a.num_slots) return;
  char* cache = is_v ? a.v_cache : a.k_cache;
  const int64_t at = static_cast<int64_t>(slot) * a.heads + h;
  if (a.kind == kCachePlain) {
    for (int d = 0; d < a.dim; ++d) store_one(cache, a.cache_dtype, at * a.dim + d, value(d));
    return;
  }
  if (a.kind == kCacheFp4) {
    uint8_t* exponents = static_cast<uint8_t*>(is_v ? a.v_scale : a.k_scale) + at * (a.dim / kFp4Block);
    for (int b = 0; b < a.dim / kFp4Block; ++b) {
      float amax = 0.f;
      for (int d = 0; d < kFp4Block; ++d) amax = nan_max(amax, fabsf(value(b * kFp4Block + d)));
      const uint32_t exponent = fp4_exponent(amax);
      exponents[b] = static_cast<uint8_t>(exponent);
      for (int d = 0; d < kFp4Block; d += 8) {
        float x[8];
        for (int j = 0; j < 8; ++j) x[j] = value(b * kFp4Block + d + j);
        const uint32_t codes = fp4_encode8(x, exponent);
        for (int j = 0; j < 4; ++j) cache[(at * a.dim + b * kFp4Block + d) / 2 + j] = static_cast<char>(codes >> (8 * j));
      }
    }
    return;
  }
  float s = 1.f;
  if (a.kind == kCacheFp8Scaled) {
    float amax = 0.f;
    for (int d = 0; d < a.dim; ++d) amax = nan_max(amax, fabsf(value(d)));
    s = amax / kFp8Max;
    s = (s < kScaleFloor) ? kScaleFloor : s;
    static_cast<float*>(is_v ? a.v_scale : a.k_scale)[at] = s;
  }
  for (int d = 0; d < a.dim; ++d) {
    float x = value(d);
    if (a.kind == kCacheFp8Scaled) x = nan_min(nan_max(x / s, -kFp8Max), kFp8Max);
    cache[at * a.dim + d] = static_cast<char>(fp8_encode4(x, 0.f, 0.f, 0.f) & 0xFFu);
  }
}

template <int IN, int LANES, int PASSES>
int launch_passes(RotateArgs& a, hipStream_t stream) {
  const int passes = static_cast<int>(ceil_div(a.q_heads + 2 * a.heads, 64 / LANES));
  a.waves_per_token = static_cast<int>(ceil_div(passes, PASSES));
  a.by_waves = divisor(a.waves_per_token);
  // A launch holds 2^32 threads; beyond that the tokens are of several.
  const int64_t most = (UINT32_MAX - 255) / 64 / a.waves_per_token, row = LANES * (IN == PRISM_DTYPE_F32 ? 32 : 16);
  if (most == 0) {
    set_error("prism_kv_rotate_store: too many heads for one launch");
    return PRISM_ERR_INVALID;
  }
  for (int64_t left = a.tokens; left > 0;) {
    a.tokens = std::min(left, most);
    const int64_t waves = a.tokens * a.waves_per_token;
    hipLaunchKernelGGL((rotate_store_kernel<IN, LANES, PASSES>), dim3(static_cast<unsigned>(ceil_div(waves, 4))), dim3(256), 0, stream, a);
    if (int rc = check_launch("rotate_store_kernel launch")) return rc;
    left -= a.tokens;
    if (left == 0) break;
    a.q += a.tokens * a.q_st, a.k += a.tokens * a.k_st, a.v += a.tokens * a.v_st;
    if (a.positions != nullptr) a.positions += a.tokens;
    if (a.q_out != nullptr) a.q_out += a.tokens * a.q_heads * row;
    if (a.k_out != nullptr) a.k_out += a.tokens * a.heads * row;
    a.slots += a.tokens;
  }
  return PRISM_OK;
}

// A wave's passes share a token's cosines and sines: as many as leave the chip 16
// waves a CU.  One, two, four, six and twelve passes, us: 8192 tokens of three axes
// (32 / 8 heads of 128 dims, with the rows read back from a 4-bit cache) -, 66, 55,
// 49 and 48; 777 tokens (16 / 4 heads of 64) -, 6.2, 6.8, 7.2 and 8.5.
template <int IN, int LANES>
int launch_lanes(RotateArgs& a, hipStream_t stream) {
  const int64_t passes = ceil_div(a.q_heads + 2 * a.heads, 64 / LANES), enough = 16 * device_cu_count();
  if (a.tokens * ceil_div(passes, 6) >= enough) return launch_passes<IN, LANES, 6>(a, stream);
  return a.tokens * ceil_div(passes, 2) >= enough ? launch_passes<IN, LANES, 2>(a, stream) : launch_passes<IN, LANES, 1>(a, stream);
}

template <int IN>
int launch_rotate(RotateArgs& a, hipStream_t stream) {
  switch (a.dim) {
    case 64: return launch_lanes<IN, 8>(a, stream);
    case 128: return launch_lanes<IN, 16>(a, stream);
    default: return launch_lanes<IN, 32>(a, stream);
  }
}

// Rows of a cache at `slots` -> 16- or 32-bit rows; zeros for slots outside it.
// Eight values a thread.
struct LoadArgs {
  const uint8_t* cache[2];
  const uint8_t* scale[2];
  char* out[2];
  const int32_t* slots;
  int64_t num_slots;
  int units;  // of eight values, of K and of V
  int per_row, heads, kind, cache_dtype, out_dtype;
  Divisor by_token, by_row;
};

__global__ void __launch_bounds__(256) kv_load_kernel(const LoadArgs a) {
  const int which = blockIdx.y;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= a.units) return;
  const int per_token = a.heads * a.per_row;
  const int token = divide(static_cast<int>(i), a.by_token);
  const int rest = static_cast<int>(i) - token * per_token;
  const int32_t slot = a.slots[token];
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (slot >= 0 && slot < a.num_slots) {
    const int64_t at = static_cast<int64_t>(slot) * per_token + rest;  // in eights
    const int64_t row = static_cast<int64_t>(slot) * a.heads + divide(rest, a.by_row);
    if (a.kind == kCacheFp4) {
      fp4_decode8(reinterpret_cast<const uint32_t*>(a.cache[which])[at], e8m0_value(a.scale[which][at / 4]), x);
    } else if (a.kind == kCachePlain) {
      if (a.cache_dtype == PRISM_DTYPE_F32) {
        to_float<PRISM_DTYPE_F32>(load8<PRISM_DTYPE_F32>(reinterpret_cast<const char*>(a.cache[which]) + at * 32), x);
      } else {
        const char* p = reinterpret_cast<const char*>(a.cache[which]) + at * 16;
        if (a.cache_dtype == PRISM_DTYPE_BF16) to_float<PRISM_DTYPE_BF16>(load8<PRISM_DTYPE_BF16>(p), x);
        else to_float<PRISM_DTYPE_F16>(load8<PRISM_DTYPE_F16>(p), x);
      }
    } else {
      const u32x2 w = reinterpret_cast<const u32x2*>(a.cache[which])[at];
      const float s = a.kind == kCacheFp8Scaled ? reinterpret_cast<const float*>(a.scale[which])[row] : 1.f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const floatx2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[j], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[j], true);
        x[4 * j] = lo[0] * s, x[4 * j + 1] = lo[1] * s, x[4 * j + 2] = hi[0] * s, x[4 * j + 3] = hi[1] * s;
      }
    }
  }
  if (a.out_dtype == PRISM_DTYPE_F32) {
    Raw8<PRISM_DTYPE_F32> r;
    from_float<PRISM_DTYPE_F32>(x, r);
    store8<PRISM_DTYPE_F32>(a.out[which] + i * 32, r);
  } else {
    u32x4 r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = pack16(a.out_dtype, x[2 * j], x[2 * j + 1]);
    __builtin_nontemporal_store(r, reinterpret_cast<u32x4*>(a.out[which]) + i);
  }
}

int cache_kind(const char* what, int cache_dtype, const void* ks, const void* vs, int head_dim, int& kind) {
  if ((ks == nullptr) != (vs == nullptr)) {
    set_error("%s: K/V scale caches must be provided together", what);
    return PRISM_ERR_INVALID;
  }
  switch (cache_dtype) {
    case PRISM_DTYPE_FP4_E2M1:
      if (ks == nullptr) {
        set_error("%s: 4-bit caches need their exponents", what);
        return PRISM_ERR_INVALID;
      }
      if (head_dim % kFp4Block != 0) {
        set_error("%s: 4-bit caches need a head_dim that is a multiple of %d, got %d", what, kFp4Block, head_dim);
        return PRISM_ERR_INVALID;
      }
      kind = kCacheFp4;
      return PRISM_OK;
    case PRISM_DTYPE_FP8_E4M3FN: kind = ks != nullptr ? kCacheFp8Scaled : kCacheFp8; return PRISM_OK;
    case PRISM_DTYPE_F32:
    case PRISM_DTYPE_BF16:
    case PRISM_DTYPE_F16:
      if (ks != nullptr) {
        set_error("%s: token-head scales require FP8 K/V payload caches", what);
        return PRISM_ERR_INVALID;
      }
      kind = kCachePlain;
      return PRISM_OK;
    default: set_error("%s: unsupported cache dtype code %d", what, cache_dtype); return PRISM_ERR_INVALID;
  }
}

bool input_dtype(int d) { return d == PRISM_DTYPE_F32 || d == PRISM_DTYPE_BF16 || d == PRISM_DTYPE_F16; }

}  // namespace

int preload_rotary_store() {
  hipFuncAttributes attr;
  return check_hip(hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(&kv_load_kernel)), "preload_rotary_store");
}

}  // namespace prism

extern "C" int prism_kv_rotate_store(const void* q, const int64_t q_strides[3], const void* key, const int64_t key_strides[3],
                                     const void* value, const int64_t value_strides[3], int in_dtype, const float* cos_sin,
                                     int64_t max_positions, int rotary_dim, int interleaved, const int32_t* positions,
                                     int64_t axis_stride, int num_axes, const int32_t* axes, void* q_out, void* key_out,
                                     void* k_cache, void* v_cache, int cache_dtype, void* k_scale, void* v_scale,
                                     const int32_t* slot_mapping, int64_t num_tokens, int num_heads, int num_kv_heads,
                                     int head_dim, int64_t num_slots, void* stream_ptr) {
  using namespace prism;
  clear_error();
  const char* what = "prism_kv_rotate_store";
  if (num_tokens < 0 || num_heads < 0 || num_kv_heads <= 0 || head_dim <= 0 || num_slots < 0 || num_tokens > INT32_MAX) {
    set_error("%s: invalid geometry tokens=%lld heads=%d kv_heads=%d head_dim=%d slots=%lld", what,
              static_cast<long long>(num_tokens), num_heads, num_kv_heads, head_dim, static_cast<long long>(num_slots));
    return PRISM_ERR_INVALID;
  }
  if (!input_dtype(in_dtype)) {
    set_error("%s: unsupported input dtype code %d", what, in_dtype);
    return PRISM_ERR_INVALID;
  }
  if (rotary_dim < 0 || rotary_dim % 2 != 0 || rotary_dim > head_dim || max_positions < 0 || num_axes < 0 ||
      (rotary_dim > 0 && num_axes == 0)) {
    set_error("%s: rotary_dim=%d must be even and at most head_dim=%d, with positions", what, rotary_dim, head_dim);
    return PRISM_ERR_INVALID;
  }
  int kind;
  if (int rc = cache_kind(what, cache_dtype, k_scale, v_scale, head_dim, kind)) return rc;
  if (num_tokens == 0) return PRISM_OK;
  if (!key || !value || !k_cache || !v_cache || !slot_mapping || !key_strides || !value_strides ||
      (num_heads > 0 && (!q || !q_out || !q_strides)) || (rotary_dim > 0 && (!positions || (max_positions > 0 && !cos_sin)))) {
    set_error("%s: null pointer argument", what);
    return PRISM_ERR_INVALID;
  }
  const int64_t none[3] = {0, 0, 1};
  const int64_t* qs = num_heads > 0 ? q_strides : none;
  if (qs[2] != 1 || key_strides[2] != 1 || value_strides[2] != 1) {
    set_error("%s: q, key and value need unit-stride head dims", what);
    return PRISM_ERR_LAYOUT;
  }
  const int64_t rows = static_cast<int64_t>(num_heads) + 2 * static_cast<int64_t>(num_kv_heads);
  if (rows > INT32_MAX || num_tokens * rows > INT32_MAX) {
    set_error("%s: too many rows for one launch: %lld tokens of %lld heads", what, static_cast<long long>(num_tokens),
              static_cast<long long>(rows));
    return PRISM_ERR_INVALID;
  }
  const int64_t size = dtype_size(in_dtype);
  RotateArgs a{};
  a.q = static_cast<const char*>(q), a.k = static_cast<const char*>(key), a.v = static_cast<const char*>(value);
  a.q_st = qs[0] * size, a.q_sh = qs[1] * size;
  a.k_st = key_strides[0] * size, a.k_sh = key_strides[1] * size;
  a.v_st = value_strides[0] * size, a.v_sh = value_strides[1] * size;
  a.table = cos_sin;
  a.positions = positions;
  a.axis_stride = axis_stride;
  a.axes = axes;
  a.num_axes = rotary_dim > 0 ? num_axes : 0;
  a.rotary = rotary_dim, a.pairs = interleaved != 0;
  a.max_positions = max_positions;
  a.q_out = static_cast<char*>(q_out), a.k_out = static_cast<char*>(key_out);
  a.k_cache = static_cast<char*>(k_cache), a.v_cache = static_cast<char*>(v_cache);
  a.k_scale = k_scale, a.v_scale = v_scale;
  a.slots = slot_mapping;
  a.tokens = num_tokens, a.num_slots = num_slots;
  a.q_heads = num_heads, a.heads = num_kv_heads, a.dim = head_dim;
  a.cache_dtype = cache_dtype, a.kind = kind;
  hipStream_t stream = static_cast<hipStream_t>(stream_ptr);

  // Whole 16-byte chunks on both sides, pairs that are whole lanes apart.
  bool vector = (head_dim == 64 || head_dim == 128 || head_dim == 256) && rotary_dim % (interleaved ? 8 : 16) == 0 &&
                aligned(cos_sin, 16) && aligned(q_out, 16) && aligned(key_out, 16) && aligned(k_cache, 16) && aligned(v_cache, 16);
  for (const char* p : {a.q, a.k, a.v}) vector = vector && aligned(p, 16);
  for (int64_t s : {a.q_st, a.q_sh, a.k_st, a.k_sh, a.v_st, a.v_sh}) vector = vector && s % 16 == 0;
  if (vector) {
    switch (in_dtype) {
      case PRISM_DTYPE_BF16: return launch_rotate<PRISM_DTYPE_BF16>(a, stream);
      case PRISM_DTYPE_F16: return launch_rotate<PRISM_DTYPE_F16>(a, stream);
      default: return launch_rotate<PRISM_DTYPE_F32>(a, stream);
    }
  }
  hipLaunchKernelGGL(rotate_store_rows_kernel, dim3(static_cast<unsigned>(ceil_div(num_tokens * rows, 256))), dim3(256), 0, stream,
                     a, in_dtype);
  return check_launch("rotate_store_rows_kernel launch");
}

extern "C" int prism_kv_load(const void* k_cache, const void* v_cache, int cache_dtype, const void* k_scale, const void* v_scale,
                             const int32_t* slot_mapping, void* key_out, void* value_out, int out_dtype, int64_t num_tokens,
                             int num_heads, int head_dim, int64_t num_slots, void* stream) {
  using namespace prism;
  clear_error();
  const char* what = "prism_kv_load";
  if (num_tokens < 0 || num_heads <= 0 || head_dim <= 0 || num_slots < 0) {
    set_error("%s: invalid geometry tokens=%lld heads=%d head_dim=%d slots=%lld", what, static_cast<long long>(num_tokens),
              num_heads, head_dim, static_cast<long long>(num_slots));
    return PRISM_ERR_INVALID;
  }
  if (!input_dtype(out_dtype)) {
    set_error("%s: unsupported output dtype code %d", what, out_dtype);
    return PRISM_ERR_INVALID;
  }
  int kind;
  if (int rc = cache_kind(what, cache_dtype, k_scale, v_scale, head_dim, kind)) return rc;
  if (num_tokens == 0) return PRISM_OK;
  if (!slot_mapping || !key_out || !value_out || (num_slots > 0 && (!k_cache || !v_cache))) {
    set_error("%s: null pointer argument", what);
    return PRISM_ERR_INVALID;
  }
  if (head_dim % 8 != 0 || !aligned(k_cache, 16) || !aligned(v_cache, 16) || !aligned(key_out, 16) || !aligned(value_out, 16)) {
    set_error("%s: head_dim must be a multiple of 8 and the buffers 16-byte aligned", what);
    return PRISM_ERR_LAYOUT;
  }
  LoadArgs a{};
  a.cache[0] = static_cast<const uint8_t*>(k_cache), a.cache[1] = static_cast<const uint8_t*>(v_cache);
  a.scale[0] = static_cast<const uint8_t*>(k_scale), a.scale[1] = static_cast<const uint8_t*>(v_scale);
  a.out[0] = static_cast<char*>(key_out), a.out[1] = static_cast<char*>(value_out);
  a.slots = slot_mapping;
  a.per_row = head_dim / 8;
  a.heads = num_heads;
  a.num_slots = num_slots;
  const int64_t per_token = static_cast<int64_t>(num_heads) * a.per_row;
  if (per_token > INT32_MAX || num_tokens > INT32_MAX / per_token) {
    set_error("%s: too many rows for one launch", what);
    return PRISM_ERR_INVALID;
  }
  a.units = static_cast<int>(num_tokens * per_token);
  a.by_token = divisor(static_cast<int>(per_token));
  a.by_row = divisor(a.per_row);
  a.kind = kind, a.cache_dtype = cache_dtype, a.out_dtype = out_dtype;
  hipLaunchKernelGGL(kv_load_kernel, dim3(static_cast<unsigned>(ceil_div(a.units, 256)), 2), dim3(256), 0, static_cast<hipStream_t>(stream), a);
  return check_launch("kv_load_kernel launch");
}
