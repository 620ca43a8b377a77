// Low-rank adapters of many requests beside shared projections (include/mlxr_lora.h).
//
//   out[t] = y[t] + s_a h_t B_a^T,   h_t = x_t A_a^T,   a = ids[t]
//
// Three launches: the tokens are sorted by adapter into tiles of up to 16 tokens of one adapter;
// h for each tile, K split over workgroups (fp32 partial sums in the workspace); the second
// product with the partial sums added up, and y.  Both products take the adapter's rows as the
// A operand and the tile's tokens as columns of the matrix instructions.
#include <hip/hip_runtime.h>

#include "../../include/mlxr_lora.h"
#include "mfma16.h"
#include "qgemm_internal.h"

namespace mlxr {

namespace {

constexpr int kTokens = 16;  // of a tile
constexpr int kItems = 4;    // projections of one launch
constexpr int kPlanThreads = 1024;

struct Tile {
  int adapter, first, count;  // tokens order[first .. first + count)
};
struct LoraArgs {
  mlxr_lora_item item[kItems];
  const uint16_t* x;
  int64_t x_stride;
  const int32_t *ids, *ranks;
  const float* scales;
  int32_t* order;   // [tokens]
  int32_t* counts;  // tiles with an adapter, all tiles
  Tile* tiles;
  float* h;  // [count][splits][tokens][rank]
  int count, tokens, K, adapters, rank, splits, chunk;
};

__device__ __forceinline__ int rank_of(const LoraArgs& a, int adapter) {
  return a.ranks ? min(max(a.ranks[adapter], 0), a.rank) : a.rank;
}

// Tokens sorted by adapter, and the tiles; the last bucket holds the tokens without one.
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(LoraArgs a) {
  extern __shared__ int sh[];
  const int nb = a.adapters + 1, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int *count = sh, *next = sh + nb;
  __shared__ int part[2 * kPlanThreads / 64];
  for (int b = tid; b < nb; b += kPlanThreads) count[b] = 0;
  __syncthreads();
  auto bucket = [&](int t) {
    const int id = a.ids[t];
    return id >= 0 && id < a.adapters ? id : a.adapters;
  };
  for (int t = tid; t < a.tokens; t += kPlanThreads) atomicAdd(&count[bucket(t)], 1);
  __syncthreads();
  const int per = (nb + kPlanThreads - 1) / kPlanThreads, b0 = min(tid * per, nb), b1 = min(b0 + per, nb);
  int n = 0, m = 0;
  for (int b = b0; b < b1; ++b) n += count[b], m += (count[b] + kTokens - 1) / kTokens;
  int sn = n, sm = m;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int u = __shfl_up(sn, d), v = __shfl_up(sm, d);
    if (lane >= d) sn += u, sm += v;
  }
  if (lane == 63) part[2 * wave] = sn, part[2 * wave + 1] = sm;
  __syncthreads();
  int at = sn - n, tile = sm - m;
  for (int w = 0; w < wave; ++w) at += part[2 * w], tile += part[2 * w + 1];
  for (int b = b0; b < b1; ++b) {
    const int c = count[b];
    next[b] = at;
    if (b == a.adapters) {
      a.counts[0] = tile;
      a.counts[1] = tile + (c + kTokens - 1) / kTokens;
    }
    for (int i = 0; i < c; i += kTokens) a.tiles[tile++] = {b, at + i, min(kTokens, c - i)};
    at += c;
  }
  __syncthreads();
  for (int t = tid; t < a.tokens; t += kPlanThreads) a.order[atomicAdd(&next[bucket(t)], 1)] = t;
}

// h of one tile over one chunk of K: four wavefronts take a quarter each and add up in LDS.
// RT: tiles of 16 ranks.
template <bool F16, int RT>
__global__ __launch_bounds__(256) void shrink_kernel(LoraArgs a) {
  if ((int)blockIdx.x >= a.counts[0]) return;
  __shared__ float sh[3][RT][64][4];
  const Tile t = a.tiles[blockIdx.x];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const int split = blockIdx.y, item = blockIdx.z, rank = rank_of(a, t.adapter);
  const int k_end = min((split + 1) * a.chunk, a.K);
  const bool tok = col < t.count;
  const uint16_t* x = a.x + (int64_t)a.order[t.first + (tok ? col : 0)] * a.x_stride;
  const uint16_t* A = (const uint16_t*)a.item[item].a_dev + (int64_t)t.adapter * a.rank * a.K;
  f32x4_t acc[RT] = {};
  for (int k = split * a.chunk + wave * 32; k < k_end; k += 4 * 32) {
    const int kk = k + 8 * g;
    const bool in = kk < k_end;
    const u32x4_t xf = tok && in ? *(const u32x4_t*)(x + kk) : u32x4_t{0, 0, 0, 0};
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int row = 16 * r + col;
      const u32x4_t af = in && row < rank ? *(const u32x4_t*)(A + (int64_t)row * a.K + kk) : u32x4_t{0, 0, 0, 0};
      acc[r] = mfma16<F16>(af, xf, acc[r]);
    }
  }
  if (wave)
#pragma unroll
    for (int r = 0; r < RT; ++r) *(f32x4_t*)sh[wave - 1][r][lane] = acc[r];
  __syncthreads();
  if (wave || !tok) return;
  float* h = a.h + (((int64_t)item * a.splits + split) * a.tokens + t.first + col) * a.rank;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
#pragma unroll
    for (int w = 0; w < 3; ++w) acc[r] += *(const f32x4_t*)sh[w][r][lane];
    if (16 * r + 4 * g < a.rank) *(f32x4_t*)(h + 16 * r + 4 * g) = acc[r];
  }
}

// 64 columns of one tile for each wavefront.  Row 4 g + i of the c-th product is column 16 g + 4 c + i
// of the 64, so a lane ends with 16 neighbouring columns of its token.
template <bool F16, int RT>
__global__ __launch_bounds__(256) void expand_kernel(LoraArgs a) {
  if ((int)blockIdx.x >= a.counts[1]) return;
  constexpr int KT = (RT + 1) / 2;
  const Tile t = a.tiles[blockIdx.x];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const mlxr_lora_item& it = a.item[blockIdx.z];
  const int n0 = (blockIdx.y * 4 + wave) * 64;
  if (n0 >= it.N) return;
  f32x4_t acc[4] = {};
  float back = 1.f;
  if (t.adapter < a.adapters) {
    const int rank = rank_of(a, t.adapter);
    const float scale = a.scales ? a.scales[t.adapter] : 1.f;
    float h[KT][8];
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      const int at = 32 * k + 8 * g;
#pragma unroll
      for (int e = 0; e < 8; ++e) h[k][e] = 0.f;
      if (col < t.count && at < rank)
        for (int s = 0; s < a.splits; ++s) {
          const float* p = a.h + (((int64_t)blockIdx.z * a.splits + s) * a.tokens + t.first + col) * a.rank + at;
          const f32x4_t lo = *(const f32x4_t*)p, hi = *(const f32x4_t*)(p + 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) h[k][e] += lo[e], h[k][4 + e] += hi[e];
        }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        h[k][e] *= scale;
        top = fmaxf(top, fabsf(h[k][e]));
      }
    }
    if constexpr (F16) {  // h may lie outside f16: a power of two brings the token's largest to [1/2, 1)
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      if (top > 0.f && top < INFINITY) {
        const int e = __builtin_amdgcn_frexp_expf(top);
        back = __builtin_amdgcn_ldexpf(1.f, e);
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int i = 0; i < 8; ++i) h[k][i] = __builtin_amdgcn_ldexpf(h[k][i], -e);
      }
    }
    const uint16_t* B = (const uint16_t*)it.b_dev + (int64_t)t.adapter * it.N * a.rank;
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      u32x4_t hi, lo;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        hi[e] = pack2<F16>(h[k][2 * e], h[k][2 * e + 1]);
        const float d0 = h[k][2 * e] - unpack<F16>(hi[e], 0), d1 = h[k][2 * e + 1] - unpack<F16>(hi[e], 1);
        lo[e] = pack2<F16>(d0 == d0 ? d0 : 0.f, d1 == d1 ? d1 : 0.f);  // an infinite h stays infinite
      }
      const int at = 32 * k + 8 * g, left = rank - at;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int n = n0 + 16 * (col >> 2) + 4 * c + (col & 3);
        u32x4_t bf = n < it.N && left > 0 ? *(const u32x4_t*)(B + (int64_t)n * a.rank + at) : u32x4_t{0, 0, 0, 0};
        if (left < 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) bf[e] &= (2 * e < left ? 0xffffu : 0u) | (2 * e + 1 < left ? 0xffff0000u : 0u);
        acc[c] = mfma16<F16>(bf, lo, acc[c]);
        acc[c] = mfma16<F16>(bf, hi, acc[c]);
      }
    }
  } else if (it.out_dev == it.y_dev) {
    return;
  }
  if (col >= t.count) return;
  const int64_t row = (int64_t)a.order[t.first + col] * it.N;
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = n0 + 16 * g + 4 * c + i;
      if (n < it.N) store_scalar(it.out_dev, it.y_dtype, row + n, load_scalar(it.y_dev, it.y_dtype, row + n) + acc[c][i] * back);
    }
}

struct Layout {
  int tiles, splits, chunk;  // most tiles a call may have; splits of K
  size_t order, counts, tile, h, bytes;
};
Layout layout_of(int count, int tokens, int K, int adapters, int rank) {
  Layout l;
  const int items = count < kItems ? count : kItems;
  const int buckets = tokens < adapters + 1 ? tokens : adapters + 1;
  l.tiles = tokens / kTokens + buckets;
  if (l.tiles > tokens) l.tiles = tokens;
  // enough workgroups for the device; a wavefront takes at least two steps of 32
  const long want = 512 / ((long)l.tiles * items) + 1;
  const int most = (K + 255) / 256;
  int splits = (int)(want < most ? want : most);
  l.chunk = ((K + splits - 1) / splits + 31) / 32 * 32;
  l.splits = (K + l.chunk - 1) / l.chunk;
  auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
  l.order = 0;
  l.counts = up((size_t)tokens * 4);
  l.tile = l.counts + 256;
  l.h = l.tile + up((size_t)l.tiles * sizeof(Tile));
  l.bytes = l.h + (size_t)items * l.splits * tokens * rank * 4;
  return l;
}

template <bool F16, int RT>
void launch(const LoraArgs& a, int tiles, hipStream_t s) {
  int wide = 0;
  for (int i = 0; i < a.count; ++i) wide = wide > a.item[i].N ? wide : a.item[i].N;
  shrink_kernel<F16, RT><<<dim3(tiles, a.splits, a.count), 256, 0, s>>>(a);
  expand_kernel<F16, RT><<<dim3(tiles, (wide + 255) / 256, a.count), 256, 0, s>>>(a);
}
template <bool F16>
void launch_rank(const LoraArgs& a, int tiles, hipStream_t s) {
  if (a.rank <= 16) launch<F16, 1>(a, tiles, s);
  else if (a.rank <= 32) launch<F16, 2>(a, tiles, s);
  else if (a.rank <= 64) launch<F16, 4>(a, tiles, s);
  else launch<F16, 8>(a, tiles, s);
}

int check_lora(int count, int tokens, int K, int adapters, int rank) {
  if (count < 0 || tokens < 0 || K <= 0 || adapters <= 0 || rank <= 0) return set_error(MLXR_E_INVALID, "lora: bad sizes");
  if (adapters > MLXR_LORA_MAX_ADAPTERS)
    return set_error(MLXR_E_SHAPE, "lora: at most %d adapters", MLXR_LORA_MAX_ADAPTERS);
  if (rank % 8 || rank > MLXR_LORA_MAX_RANK)
    return set_error(MLXR_E_SHAPE, "lora: rank must be a multiple of 8 and at most %d", MLXR_LORA_MAX_RANK);
  if (K % 8) return set_error(MLXR_E_SHAPE, "lora: K must be a multiple of 8");
  if (tokens > (1 << 24)) return set_error(MLXR_E_SHAPE, "lora: at most %d tokens", 1 << 24);
  return MLXR_OK;
}

}  // namespace

}  // namespace mlxr

using namespace mlxr;

extern "C" int mlxr_lora_workspace_size(int count, int tokens, int K, int adapters, int rank, size_t* bytes) {
  if (!bytes) return set_error(MLXR_E_INVALID, "null bytes");
  if (const int rc = check_lora(count, tokens, K, adapters, rank)) return rc;
  *bytes = count && tokens ? layout_of(count, tokens, K, adapters, rank).bytes : 0;
  return MLXR_OK;
}

extern "C" int mlxr_lora_apply(int count, const mlxr_lora_item* items, int tokens, int K, int adapters, int rank,
                               const void* x_dev, int x_dtype, int64_t x_stride, const int32_t* ids_dev,
                               const float* scales_dev, const int32_t* ranks_dev, void* workspace_dev,
                               size_t workspace_bytes, void* stream) {
  if (const int rc = check_lora(count, tokens, K, adapters, rank)) return rc;
  if (x_dtype != MLXR_F16 && x_dtype != MLXR_BF16) return set_error(MLXR_E_INVALID, "invalid activation dtype %d", x_dtype);
  if (count == 0 || tokens == 0) return MLXR_OK;
  if (!items || !x_dev || !ids_dev || !workspace_dev) return set_error(MLXR_E_INVALID, "null buffer");
  if (x_stride % 8 || ((uintptr_t)x_dev & 15) || ((uintptr_t)workspace_dev & 15))
    return set_error(MLXR_E_SHAPE, "lora: rows of x and the workspace must start at multiples of 16 bytes");
  for (int i = 0; i < count; ++i) {
    const mlxr_lora_item& t = items[i];
    if (!t.a_dev || !t.b_dev || !t.y_dev || !t.out_dev) return set_error(MLXR_E_INVALID, "null buffer");
    if (t.N <= 0) return set_error(MLXR_E_INVALID, "lora: N must be positive");
    if (t.y_dtype != MLXR_F32 && t.y_dtype != MLXR_F16 && t.y_dtype != MLXR_BF16)
      return set_error(MLXR_E_INVALID, "invalid output dtype %d", t.y_dtype);
    if (((uintptr_t)t.a_dev | (uintptr_t)t.b_dev) & 15)
      return set_error(MLXR_E_SHAPE, "lora: A and B must start at multiples of 16 bytes");
  }
  const Layout l = layout_of(count, tokens, K, adapters, rank);
  if (workspace_bytes < l.bytes)
    return set_error(MLXR_E_INVALID, "lora: the workspace is smaller than mlxr_lora_workspace_size");
  const hipStream_t s = (hipStream_t)stream;
  uint8_t* ws = (uint8_t*)workspace_dev;
  LoraArgs a;
  a.x = (const uint16_t*)x_dev, a.x_stride = x_stride;
  a.ids = ids_dev, a.ranks = ranks_dev, a.scales = scales_dev;
  a.order = (int32_t*)(ws + l.order), a.counts = (int32_t*)(ws + l.counts), a.tiles = (Tile*)(ws + l.tile);
  a.h = (float*)(ws + l.h);
  a.tokens = tokens, a.K = K, a.adapters = adapters, a.rank = rank, a.splits = l.splits, a.chunk = l.chunk;
  for (int i = 0; i < count; i += kItems) {
    a.count = count - i < kItems ? count - i : kItems;
    for (int j = 0; j < a.count; ++j) a.item[j] = items[i + j];
    if (i == 0) plan_kernel<<<1, kPlanThreads, (size_t)(adapters + 1) * 8, s>>>(a);
    if (x_dtype == MLXR_F16) launch_rank<true>(a, l.tiles, s);
    else launch_rank<false>(a, l.tiles, s);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(MLXR_E_HIP, "lora launch: %s", hipGetErrorString(e));
  return MLXR_OK;
}
