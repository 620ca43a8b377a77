// RMS norm of rows with the residual's addition, and rows rounded to 8 bits with a scale for each 128 values
// (include/mlxr_fp8.h).
//
//   s = x + residual,   y = s * w / sqrt(mean(s^2) + eps),   q = e4m3(y / c),   c = max |y| of a block / 448
//
// in one pass: a row's s stays in fp32 registers between its sum of squares and its outputs, so each input is read once
// and each output written once.  A lane holds eight neighbouring elements (16 bytes of a 16-bit type) of every CHUNK, so a
// block of 128 is 16 neighbouring lanes of one chunk and its maximum four exchanges within a row of the SIMD.
//
// Bound by memory for many rows (2048 of 8192, bf16 with the residual, to 8 bits: 118 MB in 24 us, 4.9 TB/s), by the launch and one
// round trip for few (one row of 4096 2.7 us).
#include <algorithm>
#include <type_traits>
#include <cfloat>

#include "../../include/mlxr_fp8.h"
#include "e4m3.h"
#include "mfma16.h"
#include "qgemm_internal.h"

namespace mlxr {
namespace {

constexpr int kBlock = MLXR_FP8_BLOCK;

struct NormArgs {
  const void *x, *res, *weight;
  int64_t x_stride, res_stride;
  void *sum, *out;
  float* scales;
  int rows, K, blocks, weight_dtype, out_dtype;  // out_dtype: MLXR_E4M3 for 8 bits
  float eps;
  int norm;  // or only the rounding
};

template <int XT>
struct Row8 {  // eight elements as they lie in memory
  uint4 w[XT == DT_F32 ? 2 : 1];
  // ANY: at any element's address (the loads are as wide all the same), the row's last n where that is less than eight, then zeros.
  template <bool ANY>
  __device__ __forceinline__ void load(const void* p, int64_t at, int n) {
    typedef std::conditional_t<XT == DT_F32, uint32_t, uint16_t> Element;
    if constexpr (!ANY) {
      const uint4* q = (const uint4*)((const uint8_t*)p + at * (XT == DT_F32 ? 4 : 2));
#pragma unroll
      for (int i = 0; i < (XT == DT_F32 ? 2 : 1); ++i) w[i] = q[i];
    } else if (const Element* q = (const Element*)p + at; n >= 8) {
      __builtin_memcpy(w, q, sizeof w);
    } else {
      Element t[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] = e < n ? q[e] : (Element)0;
      __builtin_memcpy(w, t, sizeof w);
    }
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t u[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[XT == DT_F32].x, w[XT == DT_F32].y, w[XT == DT_F32].z, w[XT == DT_F32].w};
#pragma unroll
    for (int k = 0; k < 8; ++k)
      v[k] = XT == DT_F32 ? __builtin_bit_cast(float, u[k]) : unpack<XT == DT_F16>(u[k / 2], k & 1);
  }
};
template <bool ANY>
__device__ __forceinline__ void store8(void* p, int dtype, int64_t at, const float (&v)[8], int n) {
  if (ANY && n < 8) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) store_scalar(p, dtype, at + e, v[e]);
  } else if (ANY && dtype == DT_F32) {
    __builtin_memcpy((float*)p + at, v, sizeof v);
  } else if (dtype == DT_F32) {
    f32x4_t* o = (f32x4_t*)((float*)p + at);
    o[0] = f32x4_t{v[0], v[1], v[2], v[3]};
    o[1] = f32x4_t{v[4], v[5], v[6], v[7]};
  } else {
    u32x4_t o;
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = dtype == DT_F16 ? pack2<true>(v[2 * k], v[2 * k + 1]) : pack2<false>(v[2 * k], v[2 * k + 1]);
    if constexpr (ANY) __builtin_memcpy((uint16_t*)p + at, &o, sizeof o);
    else *(u32x4_t*)((uint16_t*)p + at) = o;
  }
}

__device__ __forceinline__ float scale_of(float top) { return top == 0.f ? 1.f : fmaxf(top / kE4m3Top, FLT_MIN); }

// Eight values of a block that 16 neighbouring lanes hold, to 8 bits; its scale.
__device__ __forceinline__ float eight_bits(float (&v)[8], uint2* out) {
  float top = largest(v);
#pragma unroll
  for (int d = 1; d < 16; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
  const float c = scale_of(top);
  divide(v, c);
  *out = make_uint2(e4m3x4(v), e4m3x4(v + 4));
  return c;
}

// LANES of a row (16 .. 1024, within a wavefront up to 64), CH chunks of eight elements a lane.  A workgroup is one row, or
// 256 / LANES rows.  ANY: rows of any length, stride and address.
template <int XT, int LANES, int CH, bool EIGHT, bool ANY>
__global__ __launch_bounds__(LANES > 256 ? LANES : 256) void norm_kernel(NormArgs a) {
  constexpr int THREADS = LANES > 256 ? LANES : 256, ROWS = THREADS / LANES, WAVES = LANES / 64;
  __shared__ float part[LANES > 64 ? THREADS / 64 : 1];
  const int tid = threadIdx.x, x = tid & (LANES - 1);
  const int row = blockIdx.x * ROWS + tid / LANES;
  const bool mine = row < a.rows;
  const int64_t r = mine ? row : 0;
  float v[CH][8];
  Row8<XT> raw[CH], res[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int k = 8 * (c * LANES + x);
    if (k < a.K) {
      raw[c].template load<ANY>(a.x, r * a.x_stride + k, a.K - k);
      if (a.res) res[c].template load<ANY>(a.res, r * a.res_stride + k, a.K - k);
    }
  }
  float sq = 0.f;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int k = 8 * (c * LANES + x);
    if (k < a.K) {
      raw[c].get(v[c]);
      if (a.res) {
        float u[8];
        res[c].get(u);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[c][e] += u[e];
      }
      if (a.sum && mine) store8<ANY>(a.sum, XT, r * a.K + k, v[c], a.K - k);
#pragma unroll
      for (int e = 0; e < 8; ++e) sq = __builtin_fmaf(v[c][e], v[c][e], sq);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = 0.f;
    }
  }
  if (a.norm) {
#pragma unroll
    for (int d = 1; d < (LANES < 64 ? LANES : 64); d *= 2) sq += __shfl_xor(sq, d);
    if constexpr (LANES > 64) {
      if ((tid & 63) == 0) part[tid >> 6] = sq;
      __syncthreads();
      const int w0 = (tid / LANES) * WAVES;
      sq = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) sq += part[w0 + w];
    }
    const float f = 1.f / __builtin_sqrtf(sq / (float)a.K + a.eps);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int k = 8 * (c * LANES + x);
      if (k >= a.K) continue;
      float w[8];
      if (!a.weight) {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = 1.f;
      } else if (a.weight_dtype == DT_F32) {
        Row8<DT_F32> q;
        q.template load<ANY>(a.weight, k, a.K - k);
        q.get(w);
      } else if (a.weight_dtype == DT_F16) {
        Row8<DT_F16> q;
        q.template load<ANY>(a.weight, k, a.K - k);
        q.get(w);
      } else {
        Row8<DT_BF16> q;
        q.template load<ANY>(a.weight, k, a.K - k);
        q.get(w);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = v[c][e] * f * w[e];
    }
  }
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int k = 8 * (c * LANES + x);
    if constexpr (EIGHT) {
      uint2 q;
      const float scale = eight_bits(v[c], &q);  // all lanes: those past K hold zeros
      if (mine && k < a.K) {
        uint8_t* o = (uint8_t*)a.out + r * a.K + k;
        if (!ANY) {
          *(uint2*)o = q;
        } else if (a.K - k >= 8) {
          __builtin_memcpy(o, &q, sizeof q);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e < a.K - k) o[e] = (uint8_t)((e < 4 ? q.x : q.y) >> (8 * (e & 3)));
        }
        if ((x & 15) == 0) a.scales[r * a.blocks + (k >> 7)] = scale;
      }
    } else if (mine && k < a.K) {
      store8<ANY>(a.out, a.out_dtype, r * a.K + k, v[c], a.K - k);
    }
  }
}

// Rows that registers do not hold, of any length, stride and address: a workgroup a row, element by element, read twice (a wavefront takes blocks of 128
// by turns in the second pass).  s is formed again there, from x and the residual: sum_dev may be either of them, so it is
// written in that pass, each element by the lane that has just read it.
template <int XT>
__global__ __launch_bounds__(256) void norm_any_kernel(NormArgs a) {
  __shared__ float part[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    auto value = [&](int k) {
      const float v = load_scalar(a.x, XT, r * a.x_stride + k);
      return a.res ? v + load_scalar(a.res, XT, r * a.res_stride + k) : v;
    };
    float f = 1.f;
    if (a.norm) {
      float sq = 0.f;
      for (int k = tid; k < a.K; k += 256) {
        const float v = value(k);
        sq = __builtin_fmaf(v, v, sq);
      }
#pragma unroll
      for (int d = 1; d < 64; d *= 2) sq += __shfl_xor(sq, d);
      __syncthreads();  // the row before has read its parts
      if (lane == 0) part[wave] = sq;
      __syncthreads();
      f = 1.f / __builtin_sqrtf((part[0] + part[1] + part[2] + part[3]) / (float)a.K + a.eps);
    }
    for (int b = wave; b < a.blocks; b += 4) {
      float v[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int k = b * kBlock + 64 * e + lane;
        if (k >= a.K) continue;
        v[e] = value(k);
        if (a.sum) store_scalar(a.sum, XT, r * a.K + k, v[e]);
        if (a.norm) v[e] = v[e] * f * (a.weight ? load_scalar(a.weight, a.weight_dtype, k) : 1.f);
        if (a.out_dtype != MLXR_E4M3) store_scalar(a.out, a.out_dtype, r * a.K + k, v[e]);
      }
      if (a.out_dtype != MLXR_E4M3) continue;
      float top = largest(v);
#pragma unroll
      for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
      const float c = scale_of(top);
      divide(v, c);
      const uint32_t q = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int k = b * kBlock + 64 * e + lane;
        if (k < a.K) ((uint8_t*)a.out)[r * a.K + k] = (uint8_t)(q >> (8 * e));
      }
      if (lane == 0) a.scales[r * a.blocks + b] = c;
    }
  }
}

// Weights: a workgroup a block of 128 x 128, 64 elements a thread.  Once for each weight of a model: 28672 x 8192 in bf16 644 us, 1.1 TB/s
// (two-byte loads).
template <int XT>
__global__ __launch_bounds__(256) void weight_kernel(const void* w, int N, int K, int blocks, uint8_t* out, float* scales) {
  __shared__ float part[4];
  const int tid = threadIdx.x, nb = blockIdx.x / blocks, kb = blockIdx.x - nb * blocks;
  const int k = kb * kBlock + (tid & 127);
  float v[64], top = 0.f;
#pragma unroll
  for (int i = 0; i < 64; ++i) {
    const int n = nb * kBlock + 2 * i + (tid >> 7);
    v[i] = n < N && k < K ? load_scalar(w, XT, (int64_t)n * K + k) : 0.f;
    top = fmaxf(top, fabsf(v[i]));
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
  if ((tid & 63) == 0) part[tid >> 6] = top;
  __syncthreads();
  const float c = scale_of(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
  if (tid == 0) scales[blockIdx.x] = c;
#pragma unroll
  for (int i = 0; i < 64; ++i) {
    const int n = nb * kBlock + 2 * i + (tid >> 7);
    if (n < N && k < K) out[(int64_t)n * K + k] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[i] / c, 0.f, 0, false);
  }
}

template <int XT, int LANES, int CH, bool ANY = false>
void launch_rows(const NormArgs& a, hipStream_t s) {
  constexpr int THREADS = LANES > 256 ? LANES : 256, ROWS = THREADS / LANES;
  constexpr int MOST = (1 << 20) * ROWS;  // rows of a launch, which has fewer than 2^32 threads
  const int64_t xs = XT == DT_F32 ? 4 : 2, os = a.out_dtype == MLXR_E4M3 ? 1 : a.out_dtype == DT_F32 ? 4 : 2;
  for (int64_t r0 = 0; r0 < a.rows; r0 += MOST) {
    NormArgs b = a;
    b.rows = (int)std::min<int64_t>(MOST, a.rows - r0);
    b.x = (const uint8_t*)a.x + r0 * a.x_stride * xs;
    if (a.res) b.res = (const uint8_t*)a.res + r0 * a.res_stride * xs;
    if (a.sum) b.sum = (uint8_t*)a.sum + r0 * a.K * xs;
    b.out = (uint8_t*)a.out + r0 * a.K * os;
    if (a.scales) b.scales = a.scales + r0 * a.blocks;
    const unsigned grid = (unsigned)((b.rows + ROWS - 1) / ROWS);
    if (a.out_dtype == MLXR_E4M3) norm_kernel<XT, LANES, CH, true, ANY><<<grid, THREADS, 0, s>>>(b);
    else norm_kernel<XT, LANES, CH, false, ANY><<<grid, THREADS, 0, s>>>(b);
  }
}

// Lanes of a row: as many as take it with one load each, up to 1024, so that all its loads are on their way at once: half as
// many take 3.3 us for one row of 4096 (2.7), 5.6 for one of 8192 (3.7), 25 for 2048 of 8192 (24).  Many short rows are enough by
// themselves, and fewer wavefronts meet at a row's sum: 2048 rows of 4096 11.9 and 12.9.
// Rows that do not lie at multiples of 16 bytes take the same way with a last lane of fewer elements, in four lengths: 2048 rows of
// 4097 18 us, of 8190 26 (element by element 47 and 88).
template <int XT>
void launch_norm(const NormArgs& a, bool wide, hipStream_t s) {
  const int K = a.K;
  if (K > 8 * 1024 * 4) {
    norm_any_kernel<XT><<<(unsigned)std::min(a.rows, 1 << 20), 256, 0, s>>>(a);
    return;
  }
  if (!wide) {
    if (K <= 512) return launch_rows<XT, 64, 1, true>(a, s);
    if (K <= 2048) return launch_rows<XT, 256, 1, true>(a, s);
    if (K <= 8192) return launch_rows<XT, 1024, 1, true>(a, s);
    return launch_rows<XT, 1024, 4, true>(a, s);
  }
  if (K <= 128) return launch_rows<XT, 16, 1>(a, s);
  if (K <= 256) return launch_rows<XT, 32, 1>(a, s);
  if (K <= 512) return launch_rows<XT, 64, 1>(a, s);
  if (K <= 1024) return launch_rows<XT, 128, 1>(a, s);
  if (K <= 2048) return launch_rows<XT, 256, 1>(a, s);
  if (K <= 4096) return a.rows >= 4 * device_cu_count() ? launch_rows<XT, 256, 2>(a, s) : launch_rows<XT, 512, 1>(a, s);
  if (K <= 8192) return launch_rows<XT, 1024, 1>(a, s);
  if (K <= 16384) return launch_rows<XT, 1024, 2>(a, s);
  launch_rows<XT, 1024, 4>(a, s);
}

bool float_type(int t) { return t == MLXR_F32 || t == MLXR_F16 || t == MLXR_BF16; }

int run_norm(NormArgs& a, int x_dtype, const char* what, hipStream_t s) {
  const int es = x_dtype == MLXR_F32 ? 4 : 2;
  auto even = [](const void* p, int64_t stride, int size) { return ((uintptr_t)p & 15) == 0 && stride * size % 16 == 0; };
  const int os = a.out_dtype == MLXR_E4M3 ? 1 : a.out_dtype == MLXR_F32 ? 4 : 2;
  const bool wide = a.K % 8 == 0 && even(a.x, a.x_stride, es) && (!a.res || even(a.res, a.res_stride, es)) &&
                    ((uintptr_t)a.sum & 15) == 0 && ((uintptr_t)a.weight & 15) == 0 && ((uintptr_t)a.out & (os == 1 ? 7 : 15)) == 0;
  a.blocks = (a.K + kBlock - 1) / kBlock;
  if (x_dtype == MLXR_F32) launch_norm<DT_F32>(a, wide, s);
  else if (x_dtype == MLXR_F16) launch_norm<DT_F16>(a, wide, s);
  else launch_norm<DT_BF16>(a, wide, s);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(MLXR_E_HIP, "%s launch: %s", what, hipGetErrorString(e));
  return MLXR_OK;
}

int check_rows(const char* what, int rows, int K, int64_t stride) {
  if (rows < 0 || K <= 0) return set_error(MLXR_E_INVALID, "%s: bad sizes", what);
  if (K > MLXR_FP8_MAX_SIZE || (int64_t)rows * K > (1ll << 40)) return set_error(MLXR_E_SHAPE, "%s: too many elements", what);
  if (rows > 1 && stride < 0) return set_error(MLXR_E_SHAPE, "%s: rows must not lie backwards", what);
  return MLXR_OK;
}

}  // namespace
}  // namespace mlxr

using namespace mlxr;

extern "C" int mlxr_rms_norm(int rows, int K, const void* x_dev, int x_dtype, int64_t x_stride, const void* residual_dev,
                             int64_t residual_stride, const void* weight_dev, int weight_dtype, float eps, void* sum_dev,
                             void* out_dev, int out_dtype, float* scales_dev, void* stream) {
  if (const int rc = check_rows("rms_norm", rows, K, x_stride)) return rc;
  if (residual_dev && rows > 1 && residual_stride < 0) return set_error(MLXR_E_SHAPE, "rms_norm: rows must not lie backwards");
  if (!float_type(x_dtype) || (weight_dev && !float_type(weight_dtype)) || (!float_type(out_dtype) && out_dtype != MLXR_E4M3))
    return set_error(MLXR_E_INVALID, "rms_norm: invalid dtype");
  if (rows == 0) return MLXR_OK;
  if (!x_dev || !out_dev || (out_dtype == MLXR_E4M3) != (scales_dev != nullptr))
    return set_error(MLXR_E_INVALID, scales_dev && out_dtype != MLXR_E4M3 ? "rms_norm: scales belong to 8 bits" : "null buffer");
  if (!(eps >= 0.f)) return set_error(MLXR_E_INVALID, "rms_norm: eps must not be negative");
  NormArgs a{x_dev, residual_dev, weight_dev, rows > 1 ? x_stride : 0, rows > 1 ? residual_stride : 0, sum_dev, out_dev, scales_dev,
             rows, K, 0, weight_dtype, out_dtype, eps, 1};
  return run_norm(a, x_dtype, "rms_norm", (hipStream_t)stream);
}

extern "C" int mlxr_quantize_fp8(int rows, int K, const void* x_dev, int x_dtype, int64_t x_stride, void* out_dev,
                                 float* scales_dev, void* stream) {
  if (const int rc = check_rows("quantize_fp8", rows, K, x_stride)) return rc;
  if (!float_type(x_dtype)) return set_error(MLXR_E_INVALID, "quantize_fp8: invalid dtype %d", x_dtype);
  if (rows == 0) return MLXR_OK;
  if (!x_dev || !out_dev || !scales_dev) return set_error(MLXR_E_INVALID, "null buffer");
  NormArgs a{x_dev, nullptr, nullptr, rows > 1 ? x_stride : 0, 0, nullptr, out_dev, scales_dev, rows, K, 0, 0, MLXR_E4M3, 0.f, 0};
  return run_norm(a, x_dtype, "quantize_fp8", (hipStream_t)stream);
}

extern "C" int mlxr_quantize_fp8_weight(int N, int K, const void* w_dev, int w_dtype, void* out_dev, float* scales_dev,
                                        void* stream) {
  if (N <= 0 || K <= 0) return set_error(MLXR_E_INVALID, "quantize_fp8_weight: bad sizes");
  if (!float_type(w_dtype)) return set_error(MLXR_E_INVALID, "quantize_fp8_weight: invalid dtype %d", w_dtype);
  if (!w_dev || !out_dev || !scales_dev) return set_error(MLXR_E_INVALID, "null buffer");
  const int nb = (N - 1) / kBlock + 1, kb = (K - 1) / kBlock + 1;
  if (N > MLXR_FP8_MAX_SIZE || K > MLXR_FP8_MAX_SIZE || (int64_t)nb * kb >= 1 << 24)
    return set_error(MLXR_E_SHAPE, "quantize_fp8_weight: too many elements");
  const hipStream_t s = (hipStream_t)stream;
  const unsigned grid = (unsigned)(nb * kb);
  if (w_dtype == MLXR_F32) weight_kernel<DT_F32><<<grid, 256, 0, s>>>(w_dev, N, K, kb, (uint8_t*)out_dev, scales_dev);
  else if (w_dtype == MLXR_F16) weight_kernel<DT_F16><<<grid, 256, 0, s>>>(w_dev, N, K, kb, (uint8_t*)out_dev, scales_dev);
  else weight_kernel<DT_BF16><<<grid, 256, 0, s>>>(w_dev, N, K, kb, (uint8_t*)out_dev, scales_dev);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(MLXR_E_HIP, "quantize_fp8_weight launch: %s", hipGetErrorString(e));
  return MLXR_OK;
}
