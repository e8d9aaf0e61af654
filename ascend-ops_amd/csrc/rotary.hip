// Rotary positions beyond the reference's neox operator: pairs either half a rotated part apart or next to each
// other, the rotated part any even number of leading elements of the head, q and k read in place from a fused
// projection, and the tables themselves built on the device for contexts stretched beyond what a model was
// trained on.
//
//   pair j of the rotated part (R elements): (x1, x2) = (x[j], x[j + R/2])  or  (x[2j], x[2j + 1])
//   out1 = x1 cos(p f_j) - x2 sin(p f_j),  out2 = x2 cos(p f_j) + x1 sin(p f_j);  elements R.. are copied
//
// Embedding: bound by HBM (4 bytes per element, the tables stay in the caches).  A thread moves 128-bit vectors:
// one vector of a head's row, or, with halves that are whole vectors, the two vectors that hold 8 pairs, so every
// element is loaded once.  16384 tokens, 32 + 8 heads of 128, fp32 tables: 53-57 us on an MI355X, 5.9-6.3 TB/s of the
// 336 MB of q and k; 64 tokens: 3.3 us, of which an empty launch takes 1.8.
//
// Tables: f_j = base^(-2j/R) and the angle p f_j are formed in 64 bits, as turns: the whole turns drop out by
// subtraction, exactly, and what is left (at most half a turn) loses nothing in 32 bits, so far positions are as
// exact as near ones.  A thread keeps its pair and walks kTableRows positions, which shares the power among them:
// 9.5 us for 32768 positions of 64 pairs in fp32 (16.8 MB).
#include <math.h>

#include "aops_common.h"

namespace aops {

enum RotaryScaling : int {
  kScaleNone = 0,
  kScaleLinear = 1,
  kScaleNtk = 2,
  kScaleDynamic = 3,
  kScaleYarn = 4,
  kScaleWaveLength = 5,
  kScalePairs = 6,
};

struct RotaryFreq {
  double log2_base, factor, low, high, original;
  float amplitude;
  int kind;  // what is left to do per pair: none, linear, yarn, by wave length or pairs
};

constexpr int kTableRows = 16;

template <typename T>
__global__ __launch_bounds__(256) void rotary_tables_kernel(T* __restrict__ cos_out, T* __restrict__ sin_out,
                                                            const float* __restrict__ pair_factors, int64_t positions,
                                                            uint32_t half, RotaryFreq fq) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t group = i / half;
  const uint32_t j = (uint32_t)(i - group * half);
  const int64_t first = group * kTableRows;
  if (first >= positions) return;
  double f = exp2(-fq.log2_base * ((double)j / (double)half));
  switch (fq.kind) {
    case kScaleLinear:
      f /= fq.factor;
      break;
    case kScaleYarn: {  // low .. high: from kept to divided
      const double ramp = fmin(fmax(((double)j - fq.low) / (fq.high - fq.low), 0.0), 1.0);
      f = f / fq.factor * ramp + f * (1.0 - ramp);
      break;
    }
    case kScaleWaveLength: {
      const double turns = fq.original * f * 0.15915494309189535;  // within the original context
      if (turns < fq.low) {
        f /= fq.factor;
      } else if (turns <= fq.high) {
        const double keep = (turns - fq.low) / (fq.high - fq.low);
        f = (1.0 - keep) * f / fq.factor + keep * f;
      }
      break;
    }
    case kScalePairs:
      f /= (double)pair_factors[j];
      break;
    default:
      break;
  }
  const double step = f * 0.15915494309189535;  // turns per position
  const int64_t last = min(first + kTableRows, positions);
  for (int64_t p = first; p < last; ++p) {
    const double t = (double)p * step;
    const float rest = (float)(t - rint(t));
    float s, c;
    sincospif(2.0f * rest, &s, &c);
    cos_out[p * half + j] = (T)(c * fq.amplitude);
    sin_out[p * half + j] = (T)(s * fq.amplitude);
  }
}

enum RotaryLayout : int { kHalfVectors = 0, kHalfElements = 1, kInterleaved = 2 };

struct RotaryArgs {
  const f16 *q, *k;
  f16 *out_q, *out_k;
  const int32_t* position_ids;
  const void *cos, *sin;
  int64_t q_token, q_head, k_token, k_head;  // strides in elements
  uint32_t total, units_per_head, heads_total, num_heads, num_kv_heads, head_dim, rotary_dim;
  int32_t max_position;
};

template <int N, typename T>
__device__ __forceinline__ void table_load(const T* p, float (&v)[N]) {
  // entries of a vector are N * sizeof(T) bytes apart from the next one's: aligned whenever a row holds whole vectors
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = (float)p[j];
}

template <>
__device__ __forceinline__ void table_load<8, f16>(const f16* p, float (&v)[8]) {
  const f16x8 t = ld128(p);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (float)t[j];
}

template <>
__device__ __forceinline__ void table_load<8, float>(const float* p, float (&v)[8]) {
  const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
}

template <int LAYOUT, typename T>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= a.total) return;
  const uint32_t unit = i % a.units_per_head;
  const uint32_t th = i / a.units_per_head;
  const uint32_t head = th % a.heads_total;  // q heads first, then k heads
  const uint32_t token = th / a.heads_total;
  const f16* src;
  f16* dst;
  if (head < a.num_heads) {
    src = a.q + token * a.q_token + head * a.q_head;
    dst = a.out_q + ((int64_t)token * a.num_heads + head) * a.head_dim;
  } else {
    src = a.k + token * a.k_token + (head - a.num_heads) * a.k_head;
    dst = a.out_k + ((int64_t)token * a.num_kv_heads + (head - a.num_heads)) * a.head_dim;
  }
  const uint32_t half = a.rotary_dim / 2;
  const int64_t pos = min(max(a.position_ids[token], 0), a.max_position - 1);
  const T* cos = static_cast<const T*>(a.cos) + pos * half;
  const T* sin = static_cast<const T*>(a.sin) + pos * half;
  if constexpr (LAYOUT == kHalfVectors) {
    const uint32_t rotated = half / 8;
    if (unit >= rotated) {  // behind the rotated part
      const uint32_t at = a.rotary_dim + (unit - rotated) * 8;
      st128_stream(dst + at, ld128_stream(src + at));
      return;
    }
    const f16x8 x1 = ld128_stream(src + unit * 8), x2 = ld128_stream(src + half + unit * 8);
    float c[8], s[8];
    table_load<8, T>(cos + unit * 8, c);
    table_load<8, T>(sin + unit * 8, s);
    f16x8 o1, o2;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float u = (float)x1[j], v = (float)x2[j];
      o1[j] = (f16)__builtin_fmaf(u, c[j], -(v * s[j]));
      o2[j] = (f16)__builtin_fmaf(v, c[j], u * s[j]);
    }
    st128_stream(dst + unit * 8, o1);
    st128_stream(dst + half + unit * 8, o2);
  } else {
    const f16x8 x = ld128_stream(src + unit * 8);
    f16x8 o = x;
    if constexpr (LAYOUT == kInterleaved) {
      if (unit * 8 < a.rotary_dim) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t pair = unit * 4 + j;
          if (pair >= half) break;
          const float u = (float)x[2 * j], v = (float)x[2 * j + 1], c = (float)cos[pair], s = (float)sin[pair];
          o[2 * j] = (f16)__builtin_fmaf(u, c, -(v * s));
          o[2 * j + 1] = (f16)__builtin_fmaf(v, c, u * s);
        }
      }
    } else {
      // halves that are no whole vectors: the partners of a vector's elements lie at odd places and are read singly
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t e = unit * 8 + j;
        if (e < half) {
          const float u = (float)x[j], v = (float)src[e + half], c = (float)cos[e], s = (float)sin[e];
          o[j] = (f16)__builtin_fmaf(u, c, -(v * s));
        } else if (e < a.rotary_dim) {
          const float u = (float)src[e - half], v = (float)x[j], c = (float)cos[e - half], s = (float)sin[e - half];
          o[j] = (f16)__builtin_fmaf(v, c, u * s);
        }
      }
    }
    st128_stream(dst + unit * 8, o);
  }
}

}  // namespace aops

extern "C" int aops_rotary_tables(void* cos_out, void* sin_out, int table_fp32, int64_t max_position,
                                  int64_t rotary_dim, double base, int scaling, double factor,
                                  double original_max_position, double low, double high, double attention_factor,
                                  const float* pair_factors, void* stream) {
  using namespace aops;
  constexpr double kTwoPi = 6.283185307179586;
  if (max_position < 0 || max_position > 0x7fffffff || rotary_dim < 2 || rotary_dim % 2 != 0 || rotary_dim > 65536)
    return AOPS_ERR_INVALID_ARGUMENT;
  if (!(base > 0.0) || !isfinite(base) || !(factor > 0.0) || !isfinite(factor) || !(attention_factor >= 0.0) ||
      !isfinite(attention_factor))
    return AOPS_ERR_INVALID_ARGUMENT;
  const bool needs_original = scaling == kScaleDynamic || scaling == kScaleYarn || scaling == kScaleWaveLength ||
                              (scaling == kScalePairs && attention_factor == 0.0 && factor > 1.0);
  if (needs_original && (!(original_max_position >= 1.0) || !isfinite(original_max_position)))
    return AOPS_ERR_INVALID_ARGUMENT;
  RotaryFreq fq = {log2(base), factor, 0.0, 1.0, original_max_position, 1.0f, scaling};
  double amplitude = attention_factor > 0.0 ? attention_factor : 1.0;
  const double r = (double)rotary_dim;
  switch (scaling) {
    case kScaleNone:
    case kScaleLinear:
      break;
    case kScaleNtk:
    case kScaleDynamic: {
      // a larger base instead of smaller positions: the last pair slows down by `factor`, the first not at all
      if (rotary_dim == 2) return AOPS_ERR_INVALID_ARGUMENT;
      double by = factor;
      if (scaling == kScaleDynamic) {
        const double length = (double)max_position;
        by = length > original_max_position ? factor * length / original_max_position - (factor - 1.0) : 1.0;
      }
      if (!(by > 0.0)) return AOPS_ERR_INVALID_ARGUMENT;
      fq.log2_base = log2(base) + log2(by) * r / (r - 2.0);
      fq.kind = kScaleNone;
      break;
    }
    case kScaleYarn: {
      // low: turns of the slowest pair that keeps its frequency (beta_fast); high: of the first that is fully divided
      if (!(high > 0.0) || !(low >= high) || !isfinite(low) || !(base > 1.0))
        return AOPS_ERR_INVALID_ARGUMENT;
      auto pair_of = [&](double turns) {
        return r * log(original_max_position / (turns * kTwoPi)) / (2.0 * log(base));
      };
      fq.low = fmax(floor(pair_of(low)), 0.0);
      fq.high = fmin(ceil(pair_of(high)), r - 1.0);
      if (fq.high <= fq.low) fq.high = fq.low + 0.001;
      if (attention_factor == 0.0 && factor > 1.0) amplitude = 0.1 * log(factor) + 1.0;
      break;
    }
    case kScaleWaveLength:
      if (!(low > 0.0) || !(high > low) || !isfinite(high)) return AOPS_ERR_INVALID_ARGUMENT;
      fq.low = low;
      fq.high = high;
      break;
    case kScalePairs:
      if (max_position > 0 && !pair_factors) return AOPS_ERR_INVALID_ARGUMENT;
      if (attention_factor == 0.0 && factor > 1.0) {
        if (original_max_position <= 1.0) return AOPS_ERR_INVALID_ARGUMENT;
        amplitude = sqrt(1.0 + log(factor) / log(original_max_position));
      }
      break;
    default:
      return AOPS_ERR_INVALID_ARGUMENT;
  }
  fq.amplitude = (float)amplitude;
  if (max_position == 0) return AOPS_OK;
  if (!cos_out || !sin_out) return AOPS_ERR_INVALID_ARGUMENT;
  const int64_t half = rotary_dim / 2;
  const int64_t threads = (max_position + kTableRows - 1) / kTableRows * half;
  const int64_t grid = (threads + 255) / 256;
  if (!grid_fits(grid, 256)) return AOPS_ERR_INVALID_ARGUMENT;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (table_fp32)
    rotary_tables_kernel<float><<<(unsigned)grid, 256, 0, st>>>(static_cast<float*>(cos_out),
                                                                static_cast<float*>(sin_out), pair_factors,
                                                                max_position, (uint32_t)half, fq);
  else
    rotary_tables_kernel<f16><<<(unsigned)grid, 256, 0, st>>>(static_cast<f16*>(cos_out), static_cast<f16*>(sin_out),
                                                              pair_factors, max_position, (uint32_t)half, fq);
  return record_launch_status(hipGetLastError());
}

extern "C" int aops_rotary_f16(const void* q, const void* k, const int32_t* position_ids, const void* cos_table,
                               const void* sin_table, int table_fp32, void* out_q, void* out_k, int64_t tokens,
                               int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, int64_t rotary_dim,
                               int64_t max_position, int interleaved, int64_t q_token_stride, int64_t q_head_stride,
                               int64_t k_token_stride, int64_t k_head_stride, void* stream) {
  using namespace aops;
  if (tokens < 0 || num_heads < 0 || num_heads > 0x7fffffff || num_kv_heads < 0 || num_kv_heads > 0x7fffffff || head_dim <= 0 || head_dim % 8 != 0 || rotary_dim < 2 ||
      rotary_dim % 2 != 0 || rotary_dim > head_dim || max_position < 0 || max_position > 0x7fffffff)
    return AOPS_ERR_INVALID_ARGUMENT;
  if (q_token_stride < 0 || q_head_stride < 0 || k_token_stride < 0 || k_head_stride < 0 || q_token_stride % 8 != 0 ||
      q_head_stride % 8 != 0 || k_token_stride % 8 != 0 || k_head_stride % 8 != 0)
    return AOPS_ERR_INVALID_ARGUMENT;
  const int64_t half = rotary_dim / 2;
  // halves of whole vectors (fp16: 8 elements; the table rows are then whole vectors too) go two vectors a thread
  const int layout = interleaved ? kInterleaved : half % 8 == 0 ? kHalfVectors : kHalfElements;
  const int64_t units = layout == kHalfVectors ? half / 8 + (head_dim - rotary_dim) / 8 : head_dim / 8;
  const int64_t heads = num_heads + num_kv_heads;
  if (tokens == 0 || heads == 0) return AOPS_OK;
  if (tokens > 0x7fffffff || heads > 0x7fffffff || head_dim > 0x7fffffff) return AOPS_ERR_INVALID_ARGUMENT;
  if (tokens > (((int64_t)1 << 32) - 256) / heads / units) return AOPS_ERR_INVALID_ARGUMENT;
  const int64_t total = tokens * heads * units;
  if (max_position == 0 || !position_ids || !cos_table || !sin_table) return AOPS_ERR_INVALID_ARGUMENT;
  if ((num_heads > 0 && (!q || !out_q)) || (num_kv_heads > 0 && (!k || !out_k))) return AOPS_ERR_INVALID_ARGUMENT;
  const RotaryArgs a = {static_cast<const f16*>(q), static_cast<const f16*>(k), static_cast<f16*>(out_q),
                        static_cast<f16*>(out_k), position_ids, cos_table, sin_table, q_token_stride, q_head_stride,
                        k_token_stride, k_head_stride, (uint32_t)total, (uint32_t)units, (uint32_t)heads,
                        (uint32_t)num_heads, (uint32_t)num_kv_heads, (uint32_t)head_dim, (uint32_t)rotary_dim,
                        (int32_t)max_position};
  auto kernel = layout == kInterleaved   ? (table_fp32 ? rotary_kernel<kInterleaved, float> : rotary_kernel<kInterleaved, f16>)
                : layout == kHalfVectors ? (table_fp32 ? rotary_kernel<kHalfVectors, float> : rotary_kernel<kHalfVectors, f16>)
                                         : (table_fp32 ? rotary_kernel<kHalfElements, float> : rotary_kernel<kHalfElements, f16>);
  kernel<<<(unsigned)((total + 255) / 256), 256, 0, static_cast<hipStream_t>(stream)>>>(a);
  return record_launch_status(hipGetLastError());
}
