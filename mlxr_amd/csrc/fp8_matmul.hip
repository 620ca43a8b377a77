// Product of 8-bit floats with a scale for each block of 128 (include/mlxr_fp8.h).
//
//   y[m][n] = sum_b xs[m][b] ws[n / 128][b] P_b[m][n],   P_b = sum over the block's 128 k of x[m][k] w[n][k]
//
// One 16 x 16 x 128 matrix instruction is one block of K: it gives P_b of 16 x 16 outputs from zero, and the vector unit adds
// it, times the block's scale, to the fp32 total.  Weights are the first operand, activations the second, so a lane holds
// four neighbouring n of one m, whose scale is one value a lane; w's is one value a wavefront.  At the instruction's 32
// clocks four multiply-adds take 16 of the vector unit, beside it.
//
// The 8-bit instruction adds eight neighbouring products at a time and drops what each has below 2^-13 of the largest
// of them (measured; the sums of eight are then added in fp32; the instruction of 32 of K, half as fast, is off by the same): of
// random values 1.5e-5 of the result, a hundredth of half a step of bf16 and a sixteenth of f16's.  That is taken for 16-bit outputs of many rows, where the instruction bounds the
// kernel.  WIDE: both operands to bf16, which holds them exactly, and four 16 x 16 x 32 instructions, twice the clocks,
// whose sums keep fp32 (1e-7): fp32 outputs, and the kernels of few rows, which memory bounds.
//
// Both operands lie in memory as rows of K bytes, 128 of them (a line) a block.  They go to LDS by DMA, whole lines at a time,
// with the 16-byte piece c of row r at place c ^ (r / 2 % 8), so that the 16 rows of an operand's read lie in different banks;
// rows and pieces past the ends arrive as zeros.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "../../include/mlxr_fp8.h"
#include "qgemm_internal.h"
#include "qgemm_vmem.h"

namespace mlxr {
namespace fp8 {
namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8_t;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;
constexpr int kK = MLXR_FP8_BLOCK;
// A tile's rows lie within 32 bits of each other; a launch has fewer than 2^32 threads.
constexpr int kMaxK = 1 << 22, kMaxMN = 1 << 26;
constexpr int64_t kMaxOut = 1ll << 37;

struct Args {
  const uint8_t *x, *w;
  const float *xs, *ws;
  const void* bias;
  void* y;
  float* part;        // split K: fp32 partial sums [splits, M, N], or null
  int M, N, K, blocks;
  int bias_dtype, y_dtype;
  int tiles_m, tiles_n, per_split;  // per_split: blocks of K
};

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  return f32_to_f16_bits(lo) | ((uint32_t)f32_to_f16_bits(hi) << 16);
}

// An operand's 32 values of a lane: as they are, or as 16 pairs of bf16.
template <bool WIDE>
struct Operand {
  i32x8_t v;
  Operand() = default;
  __device__ __forceinline__ explicit Operand(const i32x8_t& raw) : v(raw) {}
};
template <>
struct Operand<true> {
  bf16x8_t v[4];
  Operand() = default;
  __device__ __forceinline__ explicit Operand(const i32x8_t& raw) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      typedef __attribute__((ext_vector_type(4))) uint32_t W;
      auto pair = [](int w, auto hi) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)w, 1.0f, decltype(hi)::value));
      };
      const W w = {pair(raw[2 * k], std::false_type()), pair(raw[2 * k], std::true_type()), pair(raw[2 * k + 1], std::false_type()),
                   pair(raw[2 * k + 1], std::true_type())};
      v[k] = __builtin_bit_cast(bf16x8_t, w);
    }
  }
};
__device__ __forceinline__ f32x4_t mfma128(const Operand<false>& a, const Operand<false>& b) {
  // scales of 2^0 (127): the blocks' own are not powers of two
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, f32x4_t{0, 0, 0, 0}, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
}
__device__ __forceinline__ f32x4_t mfma128(const Operand<true>& a, const Operand<true>& b) {
  f32x4_t c = {0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < 4; ++k) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[k], b.v[k], c, 0, 0, 0);
  return c;
}

// One DMA of 1 KiB (16 bytes a lane) or 256 bytes (4) to LDS at `dst`: lane l's piece lands at dst + 16 l (4 l).
template <int BYTES>
__device__ __forceinline__ void dma(i32x4_t rsrc, uint32_t voff, uint32_t soff, uint32_t dst) {
  const uint32_t m0v = (uint32_t)__builtin_amdgcn_readfirstlane((int)dst);
  soff = (uint32_t)__builtin_amdgcn_readfirstlane((int)soff);
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  if constexpr (BYTES == 16)
    asm volatile("s_mov_b32 m0, %3\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" : : "v"(voff), "s"(rsrc), "s"(soff), "s"(m0v) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %3\n\tbuffer_load_dword %0, %1, %2 offen lds" : : "v"(voff), "s"(rsrc), "s"(soff), "s"(m0v) : "memory", "m0");
#pragma clang diagnostic pop
}

// w's scales through the scalar cache: a vector load would be waited for together with the DMA behind it.
typedef const __attribute__((address_space(4))) float* scalar_p;
__device__ __forceinline__ scalar_p scalar_pointer(const float* p) { return (scalar_p)(uintptr_t)p; }

__device__ __forceinline__ int place(int r, int c) { return r * 128 + ((c ^ (r >> 1)) & 7) * 16; }

// Operand of rows r0 .. r0 + 15 of a tile in LDS: lane (r, g) takes pieces g and g + 4 of row r, in either operand.
__device__ __forceinline__ i32x8_t operand(const uint8_t* tile, int r0, int lane) {
  const int r = r0 + (lane & 15), g = lane >> 4;
  union {
    u32x4_t q[2];
    i32x8_t v;
  } u;
  u.q[0] = *(const u32x4_t*)(tile + place(r, g));
  u.q[1] = *(const u32x4_t*)(tile + place(r, g + 4));
  return u.v;
}

// Loads of R rows of a tile: R / 8 instructions of 8 rows, `first`, first + step, ...; lane l brings piece (l % 8) ^ swizzle of
// row l / 8.  K's last block may be short: pieces past it read nothing.
template <int N>
struct Rows {
  uint32_t voff[N];
  bool tail[N];  // past K in the last block
  __device__ __forceinline__ void init(int first, int step, int lane, int rows, int K) {
    const int left = K % kK;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = 8 * (first + i * step) + (lane >> 3), c = ((lane & 7) ^ (r >> 1)) & 7;
      voff[i] = r < rows ? (uint32_t)r * (uint32_t)K + 16u * c : OOB;
      tail[i] = left && 16 * c >= left;
    }
  }
};

// Tile order: workgroup id % 8 is the XCD; each takes a contiguous run of (split, group of 8 tile rows, tile column, row),
// so that the lines that neighbours share lie in its L2.
__device__ __forceinline__ void tile_of(const Args& a, int* split, int* tm, int* tn) {
  const int nb = (int)gridDim.x, tiles = a.tiles_m * a.tiles_n;
  // ids 8 i + x, i < (nb - x + 7) / 8, are the run of XCD x
  const int x = (int)blockIdx.x & 7, i = (int)blockIdx.x >> 3, each = nb >> 3, more = nb & 7;
  const int f = x * each + min(x, more) + i;
  *split = f / tiles;
  const int t = f - *split * tiles;
  const int per = 8 * a.tiles_n, grp = t / per, in = t - grp * per, height = min(8, a.tiles_m - 8 * grp);
  *tn = in / height;
  *tm = 8 * grp + in - *tn * height;
}

// BM x BN outputs a workgroup of WM x WN wavefronts, STAGES tiles of both operands in LDS.
template <int BM, int BN, int WM, int WN, int STAGES>
struct Tile {
  static constexpr int WAVES = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
  static constexpr int XR = BM / 8 / WAVES, WR = BN / 8 / WAVES;  // DMAs of a wavefront and block
  static constexpr int SCALES = BM < 64 ? 64 : BM;
  static constexpr int STAGE = (BM + BN) * kK + SCALES * 4;
  static constexpr int SR = (SCALES / 64 + WAVES - 1) / WAVES;
  static constexpr int DMAS = XR + WR + SR;
  static constexpr int EP_LD = 16 * TN + 4;                       // floats of a parked row
  static constexpr int PARK = 16 * EP_LD * 4;                     // bytes of a wavefront's 16 rows of m
  static constexpr int LDS = STAGES * STAGE > WAVES * PARK ? STAGES * STAGE : WAVES * PARK;
};

template <int BM, int BN, int WM, int WN, int STAGES, bool WIDE>
__global__ __launch_bounds__(64 * WM * WN, 1) void tile_kernel(Args a) {
  using T = Tile<BM, BN, WM, WN, STAGES>;
  constexpr int WAVES = T::WAVES, TM = T::TM, TN = T::TN;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave - wm * WN;
  int split, tm, tn;
  tile_of(a, &split, &tm, &tn);
  const int m0 = tm * BM, n0 = tn * BN, K = a.K;
  const int b0 = split * a.per_split, b1 = min(a.blocks, b0 + a.per_split);
  const int rows_x = min(BM, a.M - m0), rows_w = min(BN, a.N - n0);
  const i32x4_t rx = make_srsrc(a.x + (int64_t)m0 * K, (uint32_t)rows_x * (uint32_t)K);
  const i32x4_t rw = make_srsrc(a.w + (int64_t)n0 * K, (uint32_t)rows_w * (uint32_t)K);
  const i32x4_t rs = make_srsrc(a.xs + (int64_t)m0 * a.blocks, (uint32_t)rows_x * (uint32_t)a.blocks * 4u);
  Rows<T::XR> lx;
  Rows<T::WR> lw;
  lx.init(wave, WAVES, lane, rows_x, K);
  lw.init(wave, WAVES, lane, rows_w, K);
  uint32_t ls[T::SR];
  int sat[T::SR];
#pragma unroll
  for (int i = 0; i < T::SR; ++i) {
    sat[i] = (wave + i * WAVES) % (T::SCALES / 64);  // more wavefronts than parts: some bring the same
    const int m = 64 * sat[i] + lane;
    ls[i] = m < rows_x ? (uint32_t)m * (uint32_t)a.blocks * 4u : OOB;
  }
  const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
  // Always DMAS instructions, so that the waits are exact: blocks past the end read zeros into a stage that nobody reads.
  auto issue = [&](int b, int stage) {
    const bool live = b < b1, last = b == a.blocks - 1;
    const uint32_t at = base + (uint32_t)(stage * T::STAGE), soff = (uint32_t)b * kK;
#pragma unroll
    for (int i = 0; i < T::WR; ++i) dma<16>(rw, live && !(last && lw.tail[i]) ? lw.voff[i] : OOB, soff, at + (wave + i * WAVES) * 1024);
#pragma unroll
    for (int i = 0; i < T::XR; ++i)
      dma<16>(rx, live && !(last && lx.tail[i]) ? lx.voff[i] : OOB, soff, at + BN * kK + (wave + i * WAVES) * 1024);
#pragma unroll
    for (int i = 0; i < T::SR; ++i) dma<4>(rs, live ? ls[i] : OOB, (uint32_t)b * 4u, at + (BN + BM) * kK + sat[i] * 256);
  };

  f32x4_t acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[i][j] = f32x4_t{0, 0, 0, 0};

#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) issue(b0 + s, s);
  // the block of w's scales that this wavefront's columns lie in
  static_assert(kK % (BN / WN) == 0, "a wavefront's columns lie in one block of 128");
  const int nb = __builtin_amdgcn_readfirstlane(min((n0 + wn * (BN / WN)) / kK, (a.N - 1) / kK));
  const scalar_p ws = scalar_pointer(a.ws + (int64_t)nb * a.blocks);
  int stage = 0;
  for (int b = b0; b < b1; ++b) {
    vm_wait<(STAGES - 2) * T::DMAS>();
    __syncthreads();  // every wavefront's part of this stage is there, and the stage before it has been read
    issue(b + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
    const uint8_t* tw = lds + stage * T::STAGE;
    const uint8_t* tx = tw + BN * kK;
    const float* ts = (const float*)(tx + BM * kK);
    const float wsc = ws[b];
    float f[TM];
#pragma unroll
    for (int j = 0; j < TM; ++j) f[j] = ts[(wm * TM + j) * 16 + (lane & 15)] * wsc;
    Operand<WIDE> fx[TM], fw[2];
    f32x4_t p[2][TM];
#pragma unroll
    for (int j = 0; j < TM; ++j) fx[j] = Operand<WIDE>(operand(tx, (wm * TM + j) * 16, lane));
    fw[0] = Operand<WIDE>(operand(tw, wn * TN * 16, lane));
    // While the matrix unit works on 16 rows of w, the vector unit adds up the 16 before them and the next are read.
#pragma unroll
    for (int i = 0; i < TN; ++i) {
      if (i + 1 < TN) fw[(i + 1) & 1] = Operand<WIDE>(operand(tw, (wn * TN + i + 1) * 16, lane));
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        p[i & 1][j] = mfma128(fw[i & 1], fx[j]);
        if (i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i - 1][j][e] = __builtin_fmaf(p[(i - 1) & 1][j][e], f[j], acc[i - 1][j][e]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int j = 0; j < TM; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[TN - 1][j][e] = __builtin_fmaf(p[(TN - 1) & 1][j][e], f[j], acc[TN - 1][j][e]);
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
  vm_wait<0>();  // no DMA may still land in LDS
  __syncthreads();

  // Lane (m, g) holds columns 4 g .. 4 g + 3 of each tile: 16 rows of m at a time through LDS, stored as row segments.
  float* ep = (float*)lds + wave * (T::PARK / 4);
  const int cols = 16 * TN, nw = n0 + wn * cols;
  constexpr int PER = 4 * TN;          // lanes of a row
  constexpr int AT_ONCE = 64 / PER;    // rows
  const int c = 4 * (lane % PER), n = nw + c;
  float bias[4] = {0, 0, 0, 0};
  if (!a.part && a.bias) {
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[e] = n + e < a.N ? load_scalar(a.bias, a.bias_dtype, n + e) : 0.f;
  }
  void* out = a.part ? (void*)(a.part + (int64_t)split * a.M * a.N) : a.y;
  const int yt = a.part ? (int)DT_F32 : a.y_dtype;
  const bool vec = n + 3 < a.N;  // one store at any element's address
#pragma unroll
  for (int j = 0; j < TM; ++j) {
#pragma unroll
    for (int i = 0; i < TN; ++i) *(f32x4_t*)(ep + (lane & 15) * T::EP_LD + 16 * i + 4 * (lane >> 4)) = acc[i][j];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    f32x4_t v[16 / AT_ONCE];
#pragma unroll
    for (int r = 0; r < 16 / AT_ONCE; ++r) v[r] = *(const f32x4_t*)(ep + (r * AT_ONCE + lane / PER) * T::EP_LD + c);
#pragma unroll
    for (int r = 0; r < 16 / AT_ONCE; ++r) {
      const int m = m0 + (wm * TM + j) * 16 + r * AT_ONCE + lane / PER;
      if (m >= a.M) continue;
      const int64_t at = (int64_t)m * a.N + n;
      const float o[4] = {v[r][0] + bias[0], v[r][1] + bias[1], v[r][2] + bias[2], v[r][3] + bias[3]};
      if (vec) {
        if (yt == DT_F32) {
          __builtin_memcpy((float*)out + at, o, 16);
        } else {
          const uint2 h = yt == DT_BF16 ? make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])) : make_uint2(pack_f16x2(o[0], o[1]), pack_f16x2(o[2], o[3]));
          __builtin_memcpy((uint16_t*)out + at, &h, 8);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < a.N) store_scalar(out, yt, at + e, o[e]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

// Few rows of x: the weights are read once, and what bounds the kernel is how many of them are on their way.  A workgroup is
// 16 NT columns of y; its wavefronts take blocks of K by turns, each with a ring of its own in LDS that only it
// waits for, and meet once at the end.  Up to 16 rows, four wavefronts with three blocks on their way and two workgroups a CU, so that one
// starts while another ends: 4096 x 4096 at M = 1 5.7 us, 28672 x 8192 42 (5.6 TB/s), at M = 16 50; eight wavefronts and one
// workgroup 5.6, 48 and 57.
template <int NT, int MB, int STAGES, int WAVES>
struct Skinny {
  static constexpr int STAGE = (NT + MB) * 2048 + 256;
  static constexpr int DMAS = 2 * (NT + MB) + 1;
  static constexpr int RING = STAGES * STAGE;
  static constexpr int PARK = NT * MB * 1024;
  static constexpr int LDS = WAVES * (RING > PARK ? RING : PARK);
};

template <int NT, int MB, int STAGES, int WAVES, bool WIDE>
__global__ __launch_bounds__(64 * WAVES, 1) void skinny_kernel(Args a) {
  using S = Skinny<NT, MB, STAGES, WAVES>;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MB, K = a.K;
  const int rows_x = min(16 * MB, a.M - m0), rows_w = min(16 * NT, a.N - n0);
  const i32x4_t rx = make_srsrc(a.x + (int64_t)m0 * K, (uint32_t)rows_x * (uint32_t)K);
  const i32x4_t rw = make_srsrc(a.w + (int64_t)n0 * K, (uint32_t)rows_w * (uint32_t)K);
  const i32x4_t rs = make_srsrc(a.xs + (int64_t)m0 * a.blocks, (uint32_t)rows_x * (uint32_t)a.blocks * 4u);
  Rows<2 * MB> lx;
  Rows<2 * NT> lw;
  lx.init(0, 1, lane, rows_x, K);
  lw.init(0, 1, lane, rows_w, K);
  const uint32_t ls = lane < rows_x ? (uint32_t)lane * (uint32_t)a.blocks * 4u : OOB;
  uint8_t* ring = lds + wave * S::RING;
  const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)ring;
  auto issue = [&](int b, int stage) {
    const bool live = b < a.blocks, last = b == a.blocks - 1;
    const uint32_t at = base + (uint32_t)(stage * S::STAGE), soff = (uint32_t)b * kK;
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) dma<16>(rw, live && !(last && lw.tail[i]) ? lw.voff[i] : OOB, soff, at + i * 1024);
#pragma unroll
    for (int i = 0; i < 2 * MB; ++i) dma<16>(rx, live && !(last && lx.tail[i]) ? lx.voff[i] : OOB, soff, at + (2 * NT + i) * 1024);
    dma<4>(rs, live ? ls : OOB, (uint32_t)b * 4u, at + 2 * (NT + MB) * 1024);
  };
  f32x4_t acc[NT][MB];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j) acc[i][j] = f32x4_t{0, 0, 0, 0};
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) issue(wave + WAVES * s, s);
  const scalar_p ws = scalar_pointer(a.ws + (int64_t)(n0 / kK) * a.blocks);  // 16 NT divides 128
  int stage = 0;
  for (int b = wave; b < a.blocks; b += WAVES) {
    const float wsc = ws[b];
    issue(b + WAVES * (STAGES - 1), stage == 0 ? STAGES - 1 : stage - 1);
    vm_wait<(STAGES - 1) * S::DMAS>();
    const uint8_t* tw = ring + stage * S::STAGE;
    const uint8_t* tx = tw + NT * 2048;
    const float* ts = (const float*)(tx + MB * 2048);
#pragma unroll
    for (int j = 0; j < MB; ++j) {
      const Operand<WIDE> fx(operand(tx, 16 * j, lane));
      const float f = ts[16 * j + (lane & 15)] * wsc;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const f32x4_t p = mfma128(Operand<WIDE>(operand(tw, 16 * i, lane)), fx);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(p[e], f, acc[i][j][e]);
      }
    }
    // the operands are in registers before a DMA may replace them
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
  vm_wait<0>();
  __syncthreads();
  // [wave][m][n] with 16 NT columns
  float* all = (float*)lds;
  constexpr int COLS = 16 * NT, OUT = COLS * 16 * MB;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j)
      *(f32x4_t*)(all + wave * OUT + (16 * j + (lane & 15)) * COLS + 16 * i + 4 * (lane >> 4)) = acc[i][j];
  __syncthreads();
  for (int o = tid; o < OUT; o += 64 * WAVES) {
    const int m = m0 + o / COLS, n = n0 + o % COLS;
    if (m >= a.M || n >= a.N) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) v += all[w * OUT + o];
    if (a.bias) v += load_scalar(a.bias, a.bias_dtype, n);
    store_scalar(a.y, a.y_dtype, (int64_t)m * a.N + n, v);
  }
}

// The kernels: of few rows, and tiles of rows x columns of y.
enum Kind { AUTO = 0, SKINNY16, SKINNY32, TILE32x64, TILE64x128, TILE128x128, TILE128x256, TILE256x256, KINDS };
std::atomic<int> g_kind{AUTO}, g_splits{0};  // what tests force

// How a call runs.
struct Plan {
  Kind kind;
  int splits;  // of K, over workgroups
  size_t bytes;
};
constexpr int kMaxSplits = 16;
// Up to 16 rows the weights are streamed, above the kernel and split with the shortest time by a model: rounds of
// workgroups times blocks of K times the time of a block's step, no less than the weights at the rate at which a kernel
// streams them (TB/s), and the reduce (3 us and its fp32 partial sums at 4.5 TB/s).  The kernels of few rows split K over their
// wavefronts, need no reduce and start quickly: they serve small products of more rows too.
// us of a step measured where a workgroup is alone on its CU (two of 64 x 128 fit, which then take 1.5).  us, the best
// of all kernels and splits and the model's choice: 64 x 1024 x 4096 5.1 and 5.2 (of the tiles 8.3); 48 x 4096 x 1024 4.9 and 4.9
// (6.0); 128 x 1024 x 4096 7.1 and 7.1 (9.5); 32 x 14336 x 4096 16 and 16; 61 x 28672 x 8192 57 and 57; 64 x 8192 x 8192 21 and 21;
// 128 x 28672 x 8192 76 and 76; 256 x 8192 x 8192 41 and 41; 300 x 1024 x 4096 12.7 and 13.7; 512 x 14336 x 4096 51 and 51;
// 1024 x 4096 x 4096 29 and 29; 2048 x 14336 x 4096 137 and 137; 2048 x 4096 x 4096 44 and 44.  256 x 256
// and 128 x 256 have no WIDE form (registers).
Plan plan_of(int M, int N, int K, bool wide) {
  const int blocks = (K + kK - 1) / kK, cus = device_cu_count();
  Plan p{SKINNY16, 1, 0};
  struct Tiles {
    Kind kind;
    int bm, bn;
    double step, rate;
  };
  static const Tiles tiles[] = {{TILE32x64, 32, 64, 0.48, 4.5}, {TILE64x128, 64, 128, 0.8, 4.4}, {TILE128x128, 128, 128, 1.1, 2.9},
                                {TILE128x256, 128, 256, 1.5, 4}, {TILE256x256, 256, 256, 2.1, 4}};
  const int forced = g_kind.load(std::memory_order_relaxed), splits = g_splits.load(std::memory_order_relaxed);
  if (forced != AUTO) {
    p.kind = (Kind)forced;
    if (wide && p.kind > TILE128x128) p.kind = TILE128x128;
    p.splits = p.kind >= TILE32x64 ? std::max(1, std::min(splits, blocks)) : 1;
  } else if (M > 16) {
    double best = 1e30;
    if (M <= 1024) {
      const int m16 = (M + 15) / 16, m32 = (M + 31) / 32;  // each reads the weights
      const int64_t n16 = (int64_t)((N + 15) / 16) * m16, n32 = (int64_t)((N + 31) / 32) * m32;
      const double step16 = n16 <= cus ? 0.4 + 0.075 * blocks : (double)((n16 + 2 * cus - 1) / (2 * cus)) * (1 + 0.137 * blocks);
      const double us16 = 1.9 + std::max(step16, 1e-6 / 7 * m16 * N * K);
      const double us32 = 1.2 + std::max((double)((n32 + cus - 1) / cus) * (2.3 + 0.13 * blocks), 1e-6 / 3.3 * m32 * N * K);
      p.kind = us16 < us32 ? SKINNY16 : SKINNY32, best = std::min(us16, us32);
    }
    for (const Tiles& t : tiles) {
      if (wide && t.kind > TILE128x128) break;
      const int64_t n = (int64_t)((M + t.bm - 1) / t.bm) * ((N + t.bn - 1) / t.bn);
      for (int S = 1; S <= std::min(kMaxSplits, blocks); ++S) {
        if (S > 1 && n * (S - 1) >= 2 * cus) break;
        const int per = (blocks + S - 1) / S;
        if ((blocks + per - 1) / per != S) continue;
        const bool two = t.kind == TILE64x128 && n * S > cus;
        const double rounds = (double)((n * S + (two ? 2 : 1) * cus - 1) / ((two ? 2 : 1) * cus));
        const double us = 2 + std::max(rounds * per * (two ? 1.5 : t.step), 1e-6 / t.rate * N * K) + (S > 1 ? 3 + 8e-6 / 4.5 * S * M * N : 0);
        if (us < best) best = us, p.kind = t.kind, p.splits = S;
      }
    }
  }
  const int per = (blocks + p.splits - 1) / p.splits;
  p.splits = (blocks + per - 1) / per;
  if (p.splits > 1) p.bytes = (size_t)p.splits * M * N * sizeof(float);
  return p;
}

// Raises a kernel's LDS limit, once on each device.
hipError_t allow_lds(const void* fn, int bytes, std::atomic<uint64_t>* done) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (e != hipSuccess || (done->load(std::memory_order_acquire) & bit)) return e;
  e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == hipSuccess) done->fetch_or(bit, std::memory_order_release);
  return e;
}

template <int BM, int BN, int WM, int WN, int STAGES, bool WIDE>
hipError_t launch_tiles(Args& a, int splits, hipStream_t s) {
  using T = Tile<BM, BN, WM, WN, STAGES>;
  static std::atomic<uint64_t> done{0};
  const auto fn = tile_kernel<BM, BN, WM, WN, STAGES, WIDE>;
  if (const hipError_t e = allow_lds((const void*)fn, T::LDS, &done); e != hipSuccess) return e;
  a.tiles_m = (a.M + BM - 1) / BM, a.tiles_n = (a.N + BN - 1) / BN;
  a.per_split = (a.blocks + splits - 1) / splits;
  fn<<<dim3((unsigned)(a.tiles_m * a.tiles_n * splits)), dim3(64 * T::WAVES), T::LDS, s>>>(a);
  return hipGetLastError();
}
template <int NT, int MB, int STAGES, int WAVES, bool WIDE>
hipError_t launch_skinny(const Args& a, hipStream_t s) {
  using S = Skinny<NT, MB, STAGES, WAVES>;
  static std::atomic<uint64_t> done{0};
  const auto fn = skinny_kernel<NT, MB, STAGES, WAVES, WIDE>;
  if (const hipError_t e = allow_lds((const void*)fn, S::LDS, &done); e != hipSuccess) return e;
  fn<<<dim3((unsigned)((a.N + 16 * NT - 1) / (16 * NT)), (unsigned)((a.M + 16 * MB - 1) / (16 * MB))), dim3(64 * WAVES), S::LDS, s>>>(a);
  return hipGetLastError();
}

bool float_type(int t) { return t == MLXR_F32 || t == MLXR_F16 || t == MLXR_BF16; }
int check(int M, int N, int K) {
  if (M < 0 || N <= 0 || K <= 0) return set_error(MLXR_E_INVALID, "fp8_matmul: bad sizes");
  if (K % 16) return set_error(MLXR_E_SHAPE, "fp8_matmul: K must be a multiple of 16 (got %d)", K);
  if (M > kMaxMN || N > kMaxMN || K > kMaxK || (int64_t)M * N > kMaxOut)
    return set_error(MLXR_E_SHAPE, "fp8_matmul: too many elements");
  return MLXR_OK;
}

}  // namespace
}  // namespace fp8
}  // namespace mlxr

using namespace mlxr;
using namespace mlxr::fp8;

extern "C" int mlxr_fp8_test_force(int kind, int splits) {
  if (kind < 0 || kind >= KINDS || splits < 0) return set_error(MLXR_E_INVALID, "fp8_test_force: no such kernel");
  g_kind.store(kind), g_splits.store(splits);
  return MLXR_OK;
}

extern "C" int mlxr_fp8_matmul_workspace_size(int M, int N, int K, int y_dtype, size_t* bytes) {
  if (!bytes) return set_error(MLXR_E_INVALID, "null bytes");
  if (const int rc = check(M, N, K)) return rc;
  if (!float_type(y_dtype)) return set_error(MLXR_E_INVALID, "fp8_matmul: invalid dtype");
  *bytes = M ? plan_of(M, N, K, y_dtype == MLXR_F32).bytes : 0;
  return MLXR_OK;
}

extern "C" int mlxr_fp8_matmul(int M, int N, int K, const void* x_dev, const float* x_scale_dev, const void* w_dev,
                               const float* w_scale_dev, const void* bias_dev, int bias_dtype, void* y_dev, int y_dtype,
                               void* workspace_dev, size_t workspace_bytes, void* stream) {
  if (const int rc = check(M, N, K)) return rc;
  if (!float_type(y_dtype) || (bias_dev && !float_type(bias_dtype))) return set_error(MLXR_E_INVALID, "fp8_matmul: invalid dtype");
  if (M == 0) return MLXR_OK;
  if (!x_dev || !x_scale_dev || !w_dev || !w_scale_dev || !y_dev) return set_error(MLXR_E_INVALID, "null buffer");
  if (((uintptr_t)x_dev | (uintptr_t)w_dev | (uintptr_t)y_dev | (uintptr_t)workspace_dev) & 15)
    return set_error(MLXR_E_SHAPE, "fp8_matmul: x, w, y and workspace must lie at multiples of 16 bytes");
  const bool wide = y_dtype == MLXR_F32;
  const Plan p = plan_of(M, N, K, wide);
  if (workspace_bytes < p.bytes || (p.bytes && !workspace_dev))
    return set_error(MLXR_E_INVALID, "fp8_matmul: the workspace is smaller than mlxr_fp8_matmul_workspace_size");
  Args a{};
  a.x = (const uint8_t*)x_dev, a.w = (const uint8_t*)w_dev, a.xs = x_scale_dev, a.ws = w_scale_dev;
  a.bias = bias_dev, a.bias_dtype = bias_dtype, a.y = y_dev, a.y_dtype = y_dtype;
  a.M = M, a.N = N, a.K = K, a.blocks = (K + kK - 1) / kK;
  if (p.splits > 1) a.part = (float*)workspace_dev;
  const hipStream_t s = (hipStream_t)stream;
  hipError_t e;
  switch (p.kind) {
    case SKINNY16: e = launch_skinny<1, 1, 4, 4, true>(a, s); break;
    case SKINNY32: e = launch_skinny<2, 2, 2, 8, true>(a, s); break;
    case TILE32x64: e = wide ? launch_tiles<32, 64, 1, 4, 8, true>(a, p.splits, s) : launch_tiles<32, 64, 1, 4, 8, false>(a, p.splits, s); break;
    case TILE64x128: e = wide ? launch_tiles<64, 128, 1, 4, 3, true>(a, p.splits, s) : launch_tiles<64, 128, 1, 4, 3, false>(a, p.splits, s); break;
    case TILE128x256: e = launch_tiles<128, 256, 2, 4, 3, false>(a, p.splits, s); break;
    case TILE256x256: e = launch_tiles<256, 256, 4, 2, 2, false>(a, p.splits, s); break;
    default: e = wide ? launch_tiles<128, 128, 2, 2, 2, true>(a, p.splits, s) : launch_tiles<128, 128, 2, 4, 4, false>(a, p.splits, s); break;
  }
  if (e == hipSuccess && p.splits > 1)
    e = launch_splitk_reduce(a.part, (size_t)M * N, p.splits, bias_dev, bias_dtype, y_dev, y_dtype, M, N, s);
  if (e != hipSuccess) return set_error(MLXR_E_HIP, "fp8_matmul launch: %s", hipGetErrorString(e));
  return MLXR_OK;
}

namespace {
// Rows in 8 bits, their scales, the product's own workspace, each at a multiple of 256 bytes.
size_t padded(size_t bytes) { return (bytes + 255) & ~(size_t)255; }
size_t row_bytes(int M, int K) { return padded((size_t)M * K); }
size_t scale_bytes(int M, int K) { return padded((size_t)M * ((K + kK - 1) / kK) * sizeof(float)); }
}  // namespace

extern "C" int mlxr_fp8_linear_workspace_size(int M, int N, int K, int y_dtype, size_t* bytes) {
  if (const int rc = mlxr_fp8_matmul_workspace_size(M, N, K, y_dtype, bytes)) return rc;
  if (M) *bytes += row_bytes(M, K) + scale_bytes(M, K);
  return MLXR_OK;
}

extern "C" int mlxr_fp8_linear(int M, int N, int K, const void* x_dev, int x_dtype, int64_t x_stride, const void* w_dev,
                               const float* w_scale_dev, const void* bias_dev, int bias_dtype, void* y_dev, int y_dtype,
                               void* workspace_dev, size_t workspace_bytes, void* stream) {
  size_t need;
  if (const int rc = mlxr_fp8_linear_workspace_size(M, N, K, y_dtype, &need)) return rc;
  if (bias_dev && !float_type(bias_dtype)) return set_error(MLXR_E_INVALID, "fp8_linear: invalid dtype");
  if (M == 0) return MLXR_OK;
  if (!x_dev || !w_dev || !w_scale_dev || !y_dev) return set_error(MLXR_E_INVALID, "null buffer");
  if (((uintptr_t)w_dev | (uintptr_t)y_dev | (uintptr_t)workspace_dev) & 15)
    return set_error(MLXR_E_SHAPE, "fp8_linear: w, y and workspace must lie at multiples of 16 bytes");
  if (workspace_bytes < need || !workspace_dev)
    return set_error(MLXR_E_INVALID, "fp8_linear: the workspace is smaller than mlxr_fp8_linear_workspace_size");
  uint8_t* rows = (uint8_t*)workspace_dev;
  float* scales = (float*)(rows + row_bytes(M, K));
  uint8_t* rest = (uint8_t*)scales + scale_bytes(M, K);
  if (const int rc = mlxr_quantize_fp8(M, K, x_dev, x_dtype, x_stride, rows, scales, stream)) return rc;
  return mlxr_fp8_matmul(M, N, K, rows, scales, w_dev, w_scale_dev, bias_dev, bias_dtype, y_dev, y_dtype, rest,
                         workspace_bytes - (size_t)(rest - rows), stream);
}
