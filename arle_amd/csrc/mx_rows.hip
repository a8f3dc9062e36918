// Rows to microscaled rows and back: quantisation, the numbers that elements stand for, and the residual's addition with
// the root-mean-square norm whose rows go straight into blocks.
//
// `threads` is the block's width as an argument: a kernel that asks the runtime for it takes 256 bytes of hidden arguments along, and a launch
// with more than about 100 bytes takes the host 0.7 us more (3.5 instead of 2.8).
//
// A microscaled row is padded with zeros to a multiple of 512 numbers (`padded`), so that the products behind it walk whole
// steps; every byte of it is written here.
#include "mx.h"

#include <type_traits>

namespace arle {

// Rows of one launch: a grid of 2^32 threads or more along an axis is refused, or taken modulo 2^32 without a word.
constexpr int kMxLaunchRows = 1 << 21;
template <typename Launch>
int mx_by_launches(int rows, Launch launch) {      // launch(first row, how many)
  for (int64_t at = 0; at < rows; at += kMxLaunchRows)
    if (const int e = launch(at, rows - at < kMxLaunchRows ? static_cast<int>(rows - at) : kMxLaunchRows)) return e;
  return 0;
}

// ---- quantisation: a thread owns eight columns of kRows rows, four lanes a block.  Bound by memory: 19,456 x 2,560 of bfloat16 to e2m1 24.3 us, 5.2
// TB/s, the rate of a copy.  Two rows a thread from 1,025 rows on (us, one / two / four / eight rows: 27.8 / 24.3 / 24.6 / 25.6; 2,048 x 4,096 to e4m3
// 7.0 / 6.6 / 7.2 / 7.4); with fewer, one, for as many workgroups as there can be.
template <typename T, int BITS, bool ALIGNED, int kRows>
__global__ __launch_bounds__(512) void mx_quantize_kernel(const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ elements,
                                                           uint8_t* __restrict__ scales, int rows, int width, int padded, int threads) {
  const int unit = blockIdx.y * threads + threadIdx.x;   // of eight columns
  const int col = 8 * unit;
  if (col >= padded) return;                                 // whole blocks: padded is a multiple of 32
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kRows;
  float4 v[kRows][2];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const T* p = x + min(row0 + r, static_cast<int64_t>(rows) - 1) * ldx;
    if constexpr (ALIGNED) {                                 // the width is a multiple of eight
      const int at = col < width ? col : width - 8;
      v[r][0] = ld4<T>(p + at);
      v[r][1] = ld4<T>(p + at + 4);
    } else {
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = to_float(p[min(col + i, width - 1)]);
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = col + i < width ? e[i] : 0.f;
      v[r][0] = float4{e[0], e[1], e[2], e[3]};
      v[r][1] = float4{e[4], e[5], e[6], e[7]};
    }
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    if (ALIGNED && col >= width) v[r][0] = v[r][1] = float4{0.f, 0.f, 0.f, 0.f};
    const uint32_t code = mx_code<BITS>(mx_lanes_max<4>(max(mx_max4(v[r][0]), mx_max4(v[r][1]))));
    const uint32_t lo = mx_pack4<BITS>(v[r][0], code), hi = mx_pack4<BITS>(v[r][1], code);
    const int64_t row = row0 + r;
    if (row < rows) {
      if constexpr (BITS == kMx8)
        *reinterpret_cast<uint2*>(elements + row * padded + col) = uint2{lo, hi};
      else
        *reinterpret_cast<uint32_t*>(elements + row * (padded / 2) + col / 2) = lo | hi << 16;
      if ((unit & 3) == 0) scales[row * (padded / kMxBlock) + col / kMxBlock] = static_cast<uint8_t>(code);
    }
  }
}

// ---- the numbers that the elements stand for: a thread owns eight columns of one row
template <typename TOut, int BITS>
__global__ __launch_bounds__(512) void mx_values_kernel(const uint8_t* __restrict__ elements, int64_t ld, const uint8_t* __restrict__ scales,
                                                         int64_t ld_scales, TOut* __restrict__ out, int width, int threads) {
  const int col = 8 * (blockIdx.y * threads + threadIdx.x);
  if (col >= width) return;
  const int64_t row = blockIdx.x;
  const float s = mx_scale(scales[row * ld_scales + col / kMxBlock]);
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  f32x2 p[4];
  if constexpr (BITS == kMx8) {
    const uint2 raw = *reinterpret_cast<const uint2*>(elements + row * ld + col);
    p[0] = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(raw.x), false);
    p[1] = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(raw.x), true);
    p[2] = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(raw.y), false);
    p[3] = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(raw.y), true);
  } else {
    const uint32_t raw = *reinterpret_cast<const uint32_t*>(elements + row * ld + col / 2);
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(raw, 1.0f, 0);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(raw, 1.0f, 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(raw, 1.0f, 2);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(raw, 1.0f, 3);
  }
  const float4 lo = {p[0][0] * s, p[0][1] * s, p[1][0] * s, p[1][1] * s}, hi = {p[2][0] * s, p[2][1] * s, p[3][0] * s, p[3][1] * s};
  TOut* o = out + row * width + col;
  if ((width & 7) == 0) {
    st4<TOut>(o, lo);
    st4<TOut>(o + 4, hi);
  } else {
    const float e[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < width) o[i] = from_float<TOut>(e[i]);
  }
}

// ---- residual[src] += delta 0 + delta 1 + ... (in place unless `rows` picks rows); row r = residual[src] / sqrt(mean of squares + eps) * w
//
// A workgroup owns a row and keeps it in registers: VPT groups of four columns a thread, eight lanes a block.  Sum of squares,
// root and products are 32 bits wide, and the blocks are made from the 32-bit products: no rounding between.
template <typename T, bool ALIGNED>
__device__ __forceinline__ float4 mx_ld4(const T* p, int col, int width) {   // zeros past the width
  if constexpr (ALIGNED) {
    const float4 v = ld4<T>(p + min(col, width - 4));
    return col < width ? v : float4{0.f, 0.f, 0.f, 0.f};
  } else {
    const uint32_t at = col, last = width - 1;      // (offsets that are known to be no less than zero take a register each, others two)
    const float a = to_float(p[min(at, last)]), b = to_float(p[min(at + 1, last)]), c = to_float(p[min(at + 2, last)]),
                d = to_float(p[min(at + 3, last)]);
    return float4{col < width ? a : 0.f, col + 1 < width ? b : 0.f, col + 2 < width ? c : 0.f, col + 3 < width ? d : 0.f};
  }
}

template <typename TD, typename TW, int BITS, bool ALIGNED, int THREADS, int VPT>
__global__ __launch_bounds__(THREADS) void mx_norm_kernel(float* __restrict__ residual, const TD* __restrict__ delta, int n_delta,
                                                           int64_t delta_stride, const TW* __restrict__ w, uint8_t* __restrict__ elements,
                                                           uint8_t* __restrict__ scales, const int* __restrict__ rows, int width, int padded,
                                                           float eps) {
  constexpr int kWaves = THREADS / kWave;
  __shared__ float lds[kWaves];
  const int64_t r = blockIdx.x;
  const int64_t src = rows ? rows[r] : r;
  float* res = residual + src * width;
  const TD* d = delta + src * width;
  // Up to two groups a thread the weight is on its way beside the row, and as many parts as there is room for.  Four groups of sixteen waves, which
  // have 128 registers, hold the row, its sum and one part more; the weight, which other rows have left in the caches, comes behind the sum.
  constexpr bool kWeightFirst = VPT < 4;
  float4 v[VPT], wv[VPT];
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int col = 4 * (threadIdx.x + j * THREADS);
    v[j] = mx_ld4<float, ALIGNED>(res, col, width);
    if constexpr (kWeightFirst) wv[j] = mx_ld4<TW, ALIGNED>(w, col, width);
  }
  if (n_delta > 0) {
    float4 sum[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) sum[j] = mx_ld4<TD, ALIGNED>(d, 4 * (threadIdx.x + j * THREADS), width);
    constexpr int kAhead = VPT == 1 ? 7 : VPT == 2 ? 3 : 1;      // parts on their way; past the last one nothing is fetched
    for (int p = 1; p < n_delta; p += kAhead) {
      float4 e[kAhead][VPT];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (p + u < n_delta)
#pragma unroll
          for (int j = 0; j < VPT; ++j) e[u][j] = mx_ld4<TD, ALIGNED>(d + (p + u) * delta_stride, 4 * (threadIdx.x + j * THREADS), width);
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (p + u < n_delta)
#pragma unroll
          for (int j = 0; j < VPT; ++j) {
            sum[j].x += e[u][j].x;
            sum[j].y += e[u][j].y;
            sum[j].z += e[u][j].z;
            sum[j].w += e[u][j].w;
          }
    }
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int col = 4 * (threadIdx.x + j * THREADS);
      v[j].x += sum[j].x;
      v[j].y += sum[j].y;
      v[j].z += sum[j].z;
      v[j].w += sum[j].w;
      if (!rows) {
        if constexpr (ALIGNED) {
          if (col < width) st4<float>(res + col, v[j]);
        } else {
          if (col < width) res[col] = v[j].x;
          if (col + 1 < width) res[col + 1] = v[j].y;
          if (col + 2 < width) res[col + 2] = v[j].z;
          if (col + 3 < width) res[col + 3] = v[j].w;
        }
      }
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < VPT; ++j) ss += v[j].x * v[j].x + v[j].y * v[j].y + v[j].z * v[j].z + v[j].w * v[j].w;
  const float inv = 1.0f / sqrtf(block_sum_once<kWaves>(ss, lds) / static_cast<float>(width) + eps);
  uint8_t* o = elements + r * (BITS == kMx8 ? padded : padded / 2);
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int col = 4 * (threadIdx.x + j * THREADS);
    if constexpr (!kWeightFirst) wv[j] = mx_ld4<TW, ALIGNED>(w, col, width);
    const float4 y = {v[j].x * inv * wv[j].x, v[j].y * inv * wv[j].y, v[j].z * inv * wv[j].z, v[j].w * inv * wv[j].w};
    // (a NaN factor on a column past the width would make its zero a NaN)
    const float4 z = {col < width ? y.x : 0.f, col + 1 < width ? y.y : 0.f, col + 2 < width ? y.z : 0.f, col + 3 < width ? y.w : 0.f};
    const uint32_t code = mx_code<BITS>(mx_lanes_max<8>(mx_max4(z)));
    if (col < padded) {
      mx_store4<BITS>(o, col, mx_pack4<BITS>(z, code));
      if ((threadIdx.x & 7) == 0) scales[r * (padded / kMxBlock) + col / kMxBlock] = static_cast<uint8_t>(code);
    }
  }
}

template <typename TD, typename TW, int BITS, bool ALIGNED>
int mx_norm_launch(float* residual, const void* delta, int n_delta, int64_t delta_stride, const void* w, uint8_t* elements, uint8_t* scales,
                   const int* rows, int n_rows, int width, int padded, float eps, bool many, hipStream_t s) {
#define ARLE_MX_NORM(THREADS, VPT)                                                                                       \
  mx_norm_kernel<TD, TW, BITS, ALIGNED, THREADS, VPT><<<n_rows, THREADS, 0, s>>>(                                        \
      residual, static_cast<const TD*>(delta), n_delta, delta_stride, static_cast<const TW*>(w), elements, scales, rows, width, padded, eps)
  // few rows: a group of columns a thread, so that a row's loads are one trip; many (more than 512 in all), which hide each other's trips: fewer waves
  // that wait for each other's sums (us, one group a thread / two: 1,024 x 2,560 8.4 / 7.8, 2,048 x 2,560 13.5 / 12.8, 4,096 x 4,096 37.3 / 35.0, 600 x
  // 4,096 8.3 / 7.8; level at 512 rows, and at 2,048 x 5,120 with four groups instead of two 26.1 / 26.8).  Past 8,192 columns four groups a thread:
  // 2,048 x 12,288 42.7 us, 6.5 TB/s (52.3 where three parts ahead and the weight beside the row spill registers), 2,048 x 12,290, whose columns are
  // loaded one by one, 76, one row of 12,288 with four parts 6.2
  if (padded <= 1024)
    ARLE_MX_NORM(256, 1);
  else if (padded <= 2048)
    if (many)
      ARLE_MX_NORM(256, 2);
    else
      ARLE_MX_NORM(512, 1);
  else if (padded <= 4096)
    if (many)
      ARLE_MX_NORM(512, 2);
    else
      ARLE_MX_NORM(1024, 1);
  else if (padded <= 8192)
    ARLE_MX_NORM(1024, 2);
  else
    ARLE_MX_NORM(1024, 4);
#undef ARLE_MX_NORM
  return launch_status();
}

}  // namespace arle

using namespace arle;

extern "C" int arle_mx_quantize(const void* x, int code, long long ldx, void* elements, void* scales, int bits, int rows, int width, int padded,
                                int aligned, void* stream) {
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int units = padded / 8, parts = (units + 511) / 512, threads = ((units + parts - 1) / parts + kWave - 1) / kWave * kWave;
  uint8_t* e = static_cast<uint8_t*>(elements);
  uint8_t* c = static_cast<uint8_t*>(scales);
#define ARLE_MX_Q(T, BITS, ALIGNED, ROWS)                                                                                                        \
  return mx_by_launches(rows, [&](int64_t at, int n) {                                                                                           \
    mx_quantize_kernel<T, BITS, ALIGNED, ROWS><<<dim3((n + ROWS - 1) / ROWS, parts), threads, 0, s>>>(                                           \
        static_cast<const T*>(x) + at * ldx, ldx, e + at * (padded * BITS / 8), c + at * (padded / kMxBlock), n, width, padded, threads);        \
    return launch_status();                                                                                                                      \
  })
#define ARLE_MX_QR(T, BITS, ALIGNED)          \
  do {                                        \
    if (rows <= 1024)                         \
      ARLE_MX_Q(T, BITS, ALIGNED, 1);         \
    else                                      \
      ARLE_MX_Q(T, BITS, ALIGNED, 2);         \
  } while (0)
#define ARLE_MX_QA(T, BITS)        \
  do {                             \
    if (aligned)                   \
      ARLE_MX_QR(T, BITS, true);   \
    else                           \
      ARLE_MX_QR(T, BITS, false);  \
  } while (0)
  if (code == kF32) {
    if (bits == kMx8)
      ARLE_MX_QA(float, kMx8);
    else
      ARLE_MX_QA(float, kMx4);
  } else {
    if (bits == kMx8)
      ARLE_MX_QA(bf16, kMx8);
    else
      ARLE_MX_QA(bf16, kMx4);
  }
#undef ARLE_MX_QA
#undef ARLE_MX_QR
#undef ARLE_MX_Q
}

extern "C" int arle_mx_values(const void* elements, long long ld, const void* scales, long long ld_scales, int bits, void* out, int out_code,
                              int rows, int width, void* stream) {
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int units = (width + 7) / 8, parts = (units + 511) / 512, threads = ((units + parts - 1) / parts + kWave - 1) / kWave * kWave;
  const uint8_t* e = static_cast<const uint8_t*>(elements);
  const uint8_t* c = static_cast<const uint8_t*>(scales);
  const auto go = [&](auto t, auto b) {
    using T = decltype(t);
    return mx_by_launches(rows, [&](int64_t at, int n) {
      mx_values_kernel<T, decltype(b)::value><<<dim3(n, parts), threads, 0, s>>>(e + at * ld, ld, c + at * ld_scales, ld_scales, static_cast<T*>(out) + at * width,
                                                                                width, threads);
      return launch_status();
    });
  };
  const auto with_bits = [&](auto t) { return bits == kMx8 ? go(t, std::integral_constant<int, kMx8>{}) : go(t, std::integral_constant<int, kMx4>{}); };
  return out_code == kF32 ? with_bits(float{}) : with_bits(bf16{});
}

extern "C" int arle_mx_add_rmsnorm(void* residual, const void* delta, int n_delta, long long delta_stride, int delta_code, const void* w,
                                   int w_code, void* elements, void* scales, int bits, const void* rows, int n_rows, int width, int padded,
                                   int aligned, float eps, void* stream) {
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto go = [&](auto td, auto tw, auto b, auto al) {
    using TD = decltype(td);
    constexpr int kBits = decltype(b)::value;
    return mx_by_launches(n_rows, [&](int64_t at, int n) {
      const int64_t src = rows == nullptr ? at * width : 0;      // picked rows are anywhere in the residual
      return mx_norm_launch<TD, decltype(tw), kBits, decltype(al)::value>(
          static_cast<float*>(residual) + src, static_cast<const TD*>(delta) + src, n_delta, delta_stride, w,
          static_cast<uint8_t*>(elements) + at * (padded * kBits / 8), static_cast<uint8_t*>(scales) + at * (padded / kMxBlock),
          rows == nullptr ? nullptr : static_cast<const int*>(rows) + at, n, width, padded, eps, n_rows > 512, s);
    });
  };
  auto with_align = [&](auto td, auto tw, auto b) { return aligned ? go(td, tw, b, std::true_type{}) : go(td, tw, b, std::false_type{}); };
  auto with_bits = [&](auto td, auto tw) {
    return bits == kMx8 ? with_align(td, tw, std::integral_constant<int, kMx8>{}) : with_align(td, tw, std::integral_constant<int, kMx4>{});
  };
  if (delta_code == kF32) return w_code == kF32 ? with_bits(float{}, float{}) : with_bits(float{}, bf16{});
  return w_code == kF32 ? with_bits(bf16{}, float{}) : with_bits(bf16{}, bf16{});
}
