// Low-rank adapters of many requests beside shared projections (include/mlxr_lora.h).
//
//   out[t] = y[t] + s_a h_t B_a^T,   h_t = x_t A_a^T,   a = ids[t]
//
// Tokens of one adapter are brought together in tiles, the columns of the matrix instructions; the
// adapter's rows of A and B are their other operand, read once for a tile.  The first launch
// computes h, K split over workgroups (fp32 partial sums in the workspace); the second adds the
// partial sums up, multiplies with B and adds y.  Up to kInline tokens, each workgroup of the first
// finds its tile among the ids by itself; above, a launch before sorts the tokens.
//
// Bound by the bytes of A, B and y.  A load of a matrix operand as it lies in its lanes is 16 pieces of 16 bytes for
// each 16 lanes, which the address path serves at a quarter of what whole rows get: x, A and B are loaded by rows and
// turned in LDS (64 tokens of rank 128 of 16 adapters: K 28672, N 8192 57 -> 47 us, K 4096, two of 14336 49 -> 39).
// Measured, in a graph on the same tensors: 61 tokens of 24 adapters of rank 64, K 8192, two of 28672 (194 MB) 40 us; 2048 tokens
// of 6 adapters of rank 32, K 4096, two of 14336 (259 MB) 59 (plan 5, shrink 9, expand 44 by their own); 8 tokens of 16 adapters
// of rank 16, K 4096, 6144 together, one launch 8.3.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/mlxr_lora.h"
#include "mfma16.h"
#include "qgemm_internal.h"

namespace mlxr {

namespace {

constexpr int kItems = 4;      // projections of one launch
constexpr int kThreads = 256;  // of expand
constexpr int kWaves = kThreads / 64;
constexpr int kShrinkThreads = 512;
constexpr int kFusedThreads = 512;
constexpr int kInline = kThreads;  // tokens
// Groups of 16 tokens in a tile of the sorted tokens, for which expand reads its columns of B once; and those
// that a workgroup of shrink takes of it.
constexpr int kSub = 4;
constexpr int shrink_sub(int rank_groups, int sub) { return sub == 1 || rank_groups > 4 ? 1 : 2; }
constexpr int rank_groups_of(int rank) { return rank <= 16 ? 1 : rank <= 32 ? 2 : rank <= 64 ? 4 : 8; }
constexpr int kSplits = 8;  // most splits of K
constexpr int kPlanThreads = 1024;
// Workgroups of expand for each CU (61 tokens of rank 64 as above with four, six, eight: 55, 50, 52 us; 2000 tokens
// of 8 adapters of rank 64 164, 151, 149).
constexpr int kExpandPerCu = 6;

// A tile's adapter (number `adapters`: none), its rank and scale; `count` tokens, order[16 SUB index ..] (0: no tile).
struct __attribute__((aligned(16))) Tile {
  int adapter, count, rank;
  float scale;
};
struct LoraArgs {
  mlxr_lora_item item[kItems];
  const uint16_t* x;
  int64_t x_stride;
  const int32_t *ids, *ranks;
  const float* scales;
  int32_t* order;  // a tile's tokens, in places of its own
  Tile* tiles;
  float* h;  // [count][splits][tokens][rank]
  int count, tokens, K, adapters, rank, splits, chunk, columns, most_tiles;
};

__device__ __forceinline__ Tile tile_of(const LoraArgs& a, int adapter, int count) {
  if (adapter == a.adapters) return {adapter, count, 0, 0.f};
  return {adapter, count, a.ranks ? min(max(a.ranks[adapter], 0), a.rank) : a.rank, a.scales ? a.scales[adapter] : 1.f};
}

// counter[b] + 1 for each active lane with its own b; returns a place of its own, as atomicAdd would.  One atomic for the
// lanes that share the first one's b (a prompt's tokens, whose atomics would queue), one for each other lane (2048 tokens
// in runs of 341 4.8 us; 823 of 27 adapters in any order 3.5, with one atomic for each adapter in turn 7.3).
__device__ __forceinline__ int wave_add(int* counter, int b) {
  const int lane = threadIdx.x & 63, first = __builtin_amdgcn_readfirstlane(b);
  const uint64_t same = __ballot(b == first);
  if (b != first) return atomicAdd(&counter[b], 1);
  const int leader = __builtin_ctzll(same);
  int base = 0;
  if (lane == leader) base = atomicAdd(&counter[b], __popcll(same));
  return __shfl(base, leader) + __popcll(same & ((1ull << lane) - 1));
}

// Tokens sorted by adapter, in tiles; the last bucket holds the tokens without one.
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(LoraArgs a) {
  extern __shared__ int sh[];
  constexpr int TM = 16 * kSub, AHEAD = 4;  // ids of a thread on their way at once
  const int nb = a.adapters + 1, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int *count = sh, *next = sh + nb;
  __shared__ int part[kPlanThreads / 64];
  const int per = (nb + kPlanThreads - 1) / kPlanThreads, b0 = min(tid * per, nb), b1 = min(b0 + per, nb);
  auto load = [&](int (&id)[AHEAD], int t0) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) id[k] = a.ids[min(t0 + k * kPlanThreads, a.tokens - 1)];
  };
  int first[AHEAD];
  load(first, tid);
  const Tile mine = tile_of(a, min(b0, a.adapters), 0);  // on its way while the tokens are counted
  for (int b = tid; b < nb; b += kPlanThreads) count[b] = 0;
  __syncthreads();
  auto each = [&](auto&& f) {
    for (int t0 = tid; t0 < a.tokens; t0 += AHEAD * kPlanThreads) {
      int id[AHEAD];
      if (t0 == tid)
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) id[k] = first[k];
      else load(id, t0);
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        if (const int t = t0 + k * kPlanThreads; t < a.tokens) f(t, id[k] >= 0 && id[k] < a.adapters ? id[k] : a.adapters);
    }
  };
  each([&](int, int b) { wave_add(count, b); });
  __syncthreads();
  int m = 0;
  for (int b = b0; b < b1; ++b) m += (count[b] + TM - 1) / TM;
  int sum = m;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int v = __shfl_up(sum, d);
    if (lane >= d) sum += v;
  }
  if (lane == 63) part[wave] = sum;
  __syncthreads();
  int tile = sum - m, all = 0;
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w < wave) tile += part[w];
    all += part[w];
  }
  for (int b = b0; b < b1; ++b) {
    const int c = count[b];
    next[b] = tile * TM;
    Tile t = b == b0 ? mine : tile_of(a, b, 0);
    for (int i = 0; i < c; i += TM) {
      t.count = min(TM, c - i);
      a.tiles[tile++] = t;
    }
  }
  for (int i = all + tid; i < a.most_tiles; i += kPlanThreads) a.tiles[i] = {0, 0, 0, 0.f};
  __syncthreads();
  // which place of its adapter a token gets depends on the order of the atomics; no value does
  each([&](int t, int b) { a.order[wave_add(next, b)] = t; });
}

// Tile `index` as planned, its tokens in token[0 .. count).
template <int SUB>
__device__ __forceinline__ Tile planned_tile(const LoraArgs& a, int index, int* token) {
  const Tile t = a.tiles[index];
  if (threadIdx.x < 16 * SUB) token[threadIdx.x] = a.order[index * 16 * SUB + threadIdx.x];
  __syncthreads();
  return t;
}

// Up to kInline tokens, without a plan: every workgroup ranks the tokens among those of their adapter; tiles start at
// the tokens of rank 0, 16, 32 .., in the order of these tokens.  The dynamic LDS holds a counter for each adapter.
template <int WAVES>
__device__ __forceinline__ Tile found_tile(const LoraArgs& a, int index, int* token) {
  const int tid = threadIdx.x;
  extern __shared__ int seen[];
  __shared__ uint64_t starts[WAVES];
  __shared__ Tile chosen;
  __shared__ int chosen_rank;
  const int lane = tid & 63, wave = tid >> 6, waves = (a.tokens + 63) >> 6;
  const uint64_t below = (1ull << lane) - 1;
  int b = -1;
  Tile mine = {0, 0, 0, 0.f};
  if (tid < a.tokens) {
    b = a.ids[tid];
    b = b >= 0 && b < a.adapters ? b : a.adapters;
    mine = tile_of(a, b, 0);  // on its way while the tokens are ranked
  }
  for (int i = tid; i <= a.adapters; i += 64 * WAVES) seen[i] = 0;
  uint64_t peers = __ballot(b >= 0);  // lanes of the same adapter, bit by bit of its number
  for (int bit = 1; bit <= a.adapters; bit *= 2) {
    const uint64_t set = __ballot((b & bit) != 0);
    peers &= b & bit ? set : ~set;
  }
  __syncthreads();
  int rank = -1;
  for (int w = 0; w < waves; ++w) {
    if (wave == w && b >= 0) {
      const int before = seen[b];
      rank = before + __popcll(peers & below);
      if ((peers & below) == 0) seen[b] = before + __popcll(peers);
    }
    __syncthreads();
  }
  const bool start = b >= 0 && (rank & 15) == 0;
  const uint64_t vote = __ballot(start);
  if (lane == 0) starts[wave] = vote;
  __syncthreads();
  int at = 0, all = 0;  // starts before this token, all
  for (int w = 0; w < waves; ++w) {
    const int n = __popcll(starts[w]);
    at += w < wave ? n : w == wave ? __popcll(vote & below) : 0;
    all += n;
  }
  if (index >= all) return {0, 0, 0, 0.f};
  if (start && at == index) {
    mine.count = min(16, seen[b] - rank);
    chosen = mine, chosen_rank = rank;
  }
  __syncthreads();
  const Tile t = chosen;
  const int first = chosen_rank;
  if (b == t.adapter && rank >= first && rank < first + 16) token[rank - first] = tid;
  __syncthreads();
  return t;
}

// Stands between accesses of a wavefront to LDS by which one lane sees or replaces what another wrote or read.  The hardware
// keeps a wavefront's accesses in order; only the compiler has to be told, which sees one lane's addresses.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// 16 rows of x or A by 64 k: a lane loads 16 bytes of rows lane / 8 and 8 + lane / 8, part lane % 8 of the 128, so that
// rows are read whole; turn makes operands of them by way of 2 KiB of LDS that the wavefront has for itself.  Which k an
// operand's place stands for is free, alike for x and A.  (An operand's own load would be 16 pieces.)
__device__ __forceinline__ void turn(u32x4_t (&v)[2], u32x4_t* buf) {
  const int lane = threadIdx.x & 63, row = lane >> 3, part = lane & 7, col = lane & 15, g = lane >> 4;
  // 8 lanes that read or write at once, and so 128 bytes, lie in different banks
  buf[row * 8 + (part ^ row)] = v[0];
  buf[(row + 8) * 8 + (part ^ row)] = v[1];
  wave_sync();
  v[0] = buf[col * 8 + (g ^ (col & 7))];
  v[1] = buf[col * 8 + ((4 + g) ^ (col & 7))];
  wave_sync();
}

// h of SS groups of 16 tokens of a tile over one chunk of K: the wavefronts take turns over it in steps of 64
// and add up in LDS.  RT: groups of 16 ranks; SUB: of 16 tokens in a tile.
template <bool F16, int RT, int SUB, bool INLINE>
__global__ __launch_bounds__(kShrinkThreads) void shrink_kernel(LoraArgs a) {
  constexpr int kWaves = kShrinkThreads / 64, SS = shrink_sub(RT, SUB);
  __shared__ int tokens[16 * SUB];
  __shared__ f32x4_t sh[kWaves - 1][SS * RT][64];
  __shared__ u32x4_t turns[kWaves][128];
  Tile tile;
  if constexpr (INLINE) {
    tile = found_tile<kWaves>(a, blockIdx.x, tokens);
    if (blockIdx.y == 0 && blockIdx.z == 0) {  // for expand
      if (threadIdx.x == 0) a.tiles[blockIdx.x] = tile;
      if ((int)threadIdx.x < tile.count) a.order[blockIdx.x * 16 + threadIdx.x] = tokens[threadIdx.x];
    }
  } else {
    tile = planned_tile<SUB>(a, blockIdx.x / (SUB / SS), tokens);
  }
  const int sub = blockIdx.x % (SUB / SS) * SS * 16, count = min(tile.count - sub, 16 * SS), adapter = tile.adapter;
  if (count <= 0 || tile.rank == 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const int split = blockIdx.y, item = blockIdx.z, rank = __builtin_amdgcn_readfirstlane(tile.rank);
  const int k_end = min((split + 1) * a.chunk, a.K);
  const int row = lane >> 3, at = 8 * (lane & 7);
  const uint16_t* A = (const uint16_t*)a.item[item].a_dev + (int64_t)adapter * a.rank * a.K;
  const uint16_t* x[SS][2];
#pragma unroll
  for (int s = 0; s < SS; ++s)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = 16 * s + 8 * i + row;
      x[s][i] = a.x + (int64_t)tokens[sub + (t < count ? t : 0)] * a.x_stride;
    }
  f32x4_t acc[SS][RT] = {};
  // Two steps are on their way.  The loads are unconditional: ranks that the adapter has not read its last (their
  // sums are not kept), places past the chunk its last.
  const int last = (rank - 1) & ~7, last_row = min(row, rank - 1 - last);
  u32x4_t xf[2][SS][2], af[2][RT][2];
  auto load = [&](int b, int k) {
    const int kk = min(k + at, k_end - 8);
    int64_t whole = (int64_t)row * a.K + kk, part = (int64_t)last_row * a.K + kk;
    asm("" : "+v"(whole), "+v"(part));  // or each row's address is kept over the loop, in two registers
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int s = 0; s < SS; ++s) xf[b][s][i] = *(const u32x4_t*)(x[s][i] + kk);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const int n = min(16 * r + 8 * i, last);
        af[b][r][i] = *(const u32x4_t*)(A + (int64_t)n * a.K + (n < last ? whole : part));
      }
    }
  };
  auto add = [&](int b, int k) {
    if (k + 64 > k_end) {
      const bool in = k + at < k_end;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int s = 0; s < SS; ++s) xf[b][s][i] = in ? xf[b][s][i] : u32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int r = 0; r < RT; ++r) af[b][r][i] = in ? af[b][r][i] : u32x4_t{0, 0, 0, 0};
      }
    }
#pragma unroll
    for (int s = 0; s < SS; ++s) turn(xf[b][s], turns[wave]);
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      turn(af[b][r], turns[wave]);
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int s = 0; s < SS; ++s) acc[s][r] = mfma16<F16>(af[b][r][e], xf[b][s][e], acc[s][r]);
    }
  };
  constexpr int S = kWaves * 64;
  int k = split * a.chunk + wave * 64;
  if (k < k_end) {
    load(0, k);
    load(1, k + S);
    for (; k + 2 * S < k_end; k += 2 * S) {
      add(0, k);
      load(0, k + 2 * S);
      add(1, k + S);
      load(1, k + 3 * S);
      asm volatile("" ::: "memory");  // the loads stay at the loop's end, not shared with those before it
    }
    add(0, k);
    if (k + S < k_end) add(1, k + S);
  }
  if (wave)
#pragma unroll
    for (int s = 0; s < SS; ++s)
#pragma unroll
      for (int r = 0; r < RT; ++r) sh[wave - 1][s * RT + r][lane] = acc[s][r];
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int s = 0; s < SS; ++s) {
    if (16 * s + col >= count) continue;
    float* h = a.h + (((int64_t)item * a.splits + split) * a.tokens + tokens[sub + 16 * s + col]) * a.rank + 4 * g;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      f32x4_t v = acc[s][r];
#pragma unroll
      for (int w = 0; w < kWaves - 1; ++w) v += sh[w][s * RT + r][lane];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = 16 * r + 4 * g + i < rank ? v[i] : 0.f;
      if (16 * r + 4 * g < a.rank) *(f32x4_t*)(h + 16 * r) = v;
    }
  }
}

// CT neighbouring columns of a token's row of y, as they lie in memory (YT: the type), in accesses of up to 16 bytes at
// any element: rows of odd widths start anywhere.
template <int YT, int CT>
struct Cols {
  static constexpr int S = YT == DT_F32 ? 4 : 2, W = CT * S / 4;  // bytes of an element; words
  uint32_t w[W];
  // other: 16 bytes that are read, and not used, where `in` is false: the load is unconditional
  __device__ __forceinline__ void load(const mlxr_lora_item& it, int64_t at, bool in, const void* other) {
    const uint8_t* p = in ? (const uint8_t*)it.y_dev + at * S : (const uint8_t*)other;
    if constexpr (W <= 4) {
      __builtin_memcpy(w, p, 4 * W);
    } else {
#pragma unroll
      for (int k = 0; k < W; k += 4) __builtin_memcpy(w + k, p + (in ? 4 * k : 0), 16);
    }
  }
  // out = y + v * back
  __device__ __forceinline__ void store(const mlxr_lora_item& it, int64_t at, const float* v, float back) {
    uint32_t o[W];
#pragma unroll
    for (int k = 0; k < W; ++k) {
      if constexpr (YT == DT_F32) o[k] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, w[k]) + v[k] * back);
      else o[k] = pack2<YT == DT_F16>(unpack<YT == DT_F16>(w[k], 0) + v[2 * k] * back, unpack<YT == DT_F16>(w[k], 1) + v[2 * k + 1] * back);
    }
    uint8_t* p = (uint8_t*)it.out_dev + at * S;
#pragma unroll
    for (int k = 0; k < W; k += 4) __builtin_memcpy(p + 4 * k, o + k, W < 4 ? 4 * W : 16);
  }
};

// Columns of a wavefront's step, in units of 16: 64 for few tokens (more workgroups), 128 for many: 256 bytes of a
// row in one store of 16-bit outputs; fewer where B leaves few wavefronts on a SIMD.  us: 2048 tokens of rank 32, two
// projections of 14336, 64 and 128 columns 71 and 64; 2000 of rank 64 32, 64 and 128 columns 97, 85 and 94; 64 tokens of
// rank 64, two of 28672, 32 and 64 columns 46 and 42; of rank 128, two of 14336, 39 and 45.
constexpr int columns_of(int sub, int rank_groups) { return rank_groups == 8 ? 2 : sub == 1 || rank_groups == 4 ? 4 : 8; }

// The bits of x that bf16 has, in the upper half; NaN (whose upper bits may be those of an infinity) quieted.
__device__ __forceinline__ uint32_t cut_bf16(float x) {
  return (__builtin_bit_cast(uint32_t, x) | (x != x ? 0x400000u : 0u)) & 0xffff0000u;
}

// 16-bit parts of h that add up to it: rounded to one part h would lose what the fp32 sums kept.
constexpr int h_parts(bool f16) { return f16 ? 2 : 3; }
// Elements of a token's row of them: R of each part; padded against bank conflicts.
constexpr int h_row(bool f16, int rt) { return 16 * rt * h_parts(f16) + 8; }

// 8 ranks at .. of token t of a tile into LDS in parts.  A part is cut, not rounded, and those after it never 0 beside it nor
// of the other sign, so that an infinite element of B gives an infinity as h in one piece does, not NaN.
// bf16: three parts, all bits of fp32 (the least later part is 2^-125).  f16: two, relative to a power of two that brings
// the token's largest to [2^14, 2^15), the reciprocal in back[t]: off by 2^-22 of every rank above 2^-16 of the largest, 2^-20
// at 2^-18 of it.  A token with one below that (not 0), an infinite one or NaN, or a largest that leaves no room for the power
// of two has back[t] = 0 and its ranks in fp32 in place of the parts (Expand::wide_tokens); of ranks that are alike one in 2^17
// lies so low by chance.  The 2 RT threads of a token are neighbours.
template <bool F16, int RT>
__device__ __forceinline__ void split_h(f32x4_t (&v)[2], float scale, int t, int at, uint16_t* row, float* back) {
  constexpr int R = 16 * RT;
#pragma unroll
  for (int e = 0; e < 2; ++e) v[e] *= scale;
  if constexpr (F16) {
    constexpr uint32_t kInf = 0x7f800000, kOct = 1 << 23;
    uint32_t top = 0, least = ~0u;  // bits of the largest, of the least that is not 0 less 1
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = v[i >> 2][i & 3];  // of a vector's element itself, the compiler's bit cast takes the first's bits
      const uint32_t x = __builtin_bit_cast(uint32_t, f) & 0x7fffffff;
      top = max(top, x);
      least = min(least, x - 1);
    }
#pragma unroll
    for (int d = 1; d < 2 * RT; d *= 2) {
      top = max(top, (uint32_t)__shfl_xor((int)top, d));
      least = min(least, (uint32_t)__shfl_xor((int)least, d));
    }
    const bool wide = top && (top >= kInf || top < 27 * kOct || least + 1 < top - 18 * kOct);  // below 2^-100; 2^-18 apart
    const int e = top && !wide ? 141 - (int)(top >> 23) : 0;
    if (at == 0) back[t] = wide ? 0.f : __builtin_amdgcn_ldexpf(1.f, -e);
    if (wide) {
      *(f32x4_t*)(row + 2 * at) = v[0];
      *(f32x4_t*)(row + 2 * at + 8) = v[1];
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i >> 2][i & 3] = __builtin_amdgcn_ldexpf(v[i >> 2][i & 3], e);
  }
  constexpr float LEAST = F16 ? 0x1p-24f : 0x1p-125f;
  auto rest = [](float x, float part) {  // of an infinite x: finite, of its sign
    return x == 0.f ? 0.f : copysignf(fmaxf(fabsf(x - part), LEAST), x);
  };
  u32x4_t hi, lo;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float v0 = v[e >> 1][2 * (e & 1)], v1 = v[e >> 1][2 * (e & 1) + 1];
    if constexpr (F16) hi[e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(v0, v1));
    else hi[e] = cut_bf16(v0) >> 16 | cut_bf16(v1);
    v0 = rest(v0, unpack<F16>(hi[e], 0)), v1 = rest(v1, unpack<F16>(hi[e], 1));
    if constexpr (F16) {
      lo[e] = pack2<true>(v0, v1);
    } else {
      lo[e] = cut_bf16(v0) >> 16 | cut_bf16(v1);
      v[e >> 1][2 * (e & 1)] = rest(v0, unpack<false>(lo[e], 0)), v[e >> 1][2 * (e & 1) + 1] = rest(v1, unpack<false>(lo[e], 1));
    }
  }
  *(u32x4_t*)(row + at) = hi;
  *(u32x4_t*)(row + R + at) = lo;
  if constexpr (!F16) {
    constexpr float SHARE = RT == 1 ? 0.5f : 1.f;  // RT 1 multiplies it twice
#pragma unroll
    for (int e = 0; e < 4; ++e) lo[e] = cut_bf16(v[e >> 1][2 * (e & 1)] * SHARE) >> 16 | cut_bf16(v[e >> 1][2 * (e & 1) + 1] * SHARE);
    *(u32x4_t*)(row + 2 * R + at) = lo;
  }
}

// The second product of a tile: columns [n0, end) of an item in steps of 16 CT for each of WAVES wavefronts.
// Tokens are the rows of the products; column n of the c-th is column CT n + c of the step, so a lane ends
// with CT neighbouring columns of four tokens, and 16 lanes with a stretch of a row.
template <bool F16, int RT, int SUB, int WAVES>
struct Expand {
  static constexpr int R = 16 * RT, KT = RT == 1 ? 1 : RT / 2, CT = columns_of(SUB, RT), STEP = WAVES * 16 * CT;
  static constexpr int C = R / 8, NB = 16 * CT * C / 64;  // 16-byte parts of a column's row of B; loads of a step
  // Turns in which a step's B goes through LDS.  A tile of 64 tokens of rank 128 in bf16 has 49 KiB of h: beside 32
  // KiB of B a CU would hold one workgroup, beside 16 it holds two (2000 tokens, two projections of 14336, 212 us and 158).
  static constexpr int TURNS = !F16 && RT == 8 && SUB > 1 ? 2 : 1, CTT = CT / TURNS, NBT = NB / TURNS, ROWS = NBT * 64;
  const LoraArgs& a;
  const mlxr_lora_item& it;
  const uint16_t* B;
  int rank, ld, n0, end, col, g;
  // B of a step, on its way while h or the columns before are computed, and its place in LDS: loads of rows side by
  // side, brought into operand order there (an operand's own load would be 16 pieces of 64 bytes).
  u32x4_t next[NB];
  u32x4_t* rows;
  bool wide = false;  // a token of this lane's is left to wide_tokens

  __device__ __forceinline__ Expand(const LoraArgs& a_, const mlxr_lora_item& it_, const Tile& t, int begin, u32x4_t* lds)
      : a(a_), it(it_), B((const uint16_t*)it_.b_dev + (t.adapter == a_.adapters ? 0 : (int64_t)t.adapter * it_.N * a_.rank)),
        rank(t.rank), ld(t.rank ? a_.rank : 0) {
    const int lane = threadIdx.x & 63;
    col = lane & 15, g = lane >> 4;
    n0 = begin + (threadIdx.x >> 6) * 16 * CT;
    rows = lds + (threadIdx.x >> 6) * ROWS;
    end = min(begin + a.columns, it.N);
    load_b(n0, n0 < end);
  }
  // The loads are unconditional, so that they stay in flight: what a column or rank that is not there gets lies in a row
  // that is read anyway.
  __device__ __forceinline__ void load_b(int n0, bool more) {
    const int ld = more ? this->ld : 0;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int at = i % NBT * 64 + (threadIdx.x & 63), part = at % C, n = at / C;
      const int column = n / CTT * CT + i / NBT * CTT + n % CTT;
      next[i] = *(const u32x4_t*)(B + (int64_t)min(n0 + column, it.N - 1) * ld + (8 * part < rank ? 8 * part : 0));
    }
  }
  // Place of part `part` of column n of a turn: 8 lanes that read or write at once, and so 128 bytes, lie in different banks.
  static __device__ __forceinline__ int place(int n, int part) { return (n * C + part) ^ (n / CTT & 7); }
  __device__ __forceinline__ void store_b(int turn) {
    wave_sync();  // other lanes' reads of the turn before
#pragma unroll
    for (int i = 0; i < NBT; ++i) {
      const int at = i * 64 + (threadIdx.x & 63);
      rows[place(at / C, at % C)] = next[turn * NBT + i];
    }
    wave_sync();
  }
  // RT 1 multiplies the first two parts in one product, ranks 8 (g & 1) .., and in bf16 half of the third twice in another.
  __device__ __forceinline__ int rank_at(int k) const { return RT == 1 ? 8 * (g & 1) : 32 * k + 8 * g; }
  // Operand c of the ranks k, without what the adapter has not.
  __device__ __forceinline__ u32x4_t operand(int k, int c) const {
    u32x4_t b = rows[place(CTT * col + c % CTT, rank_at(k) / 8)];
    if (rank < R) {
      const int left = rank - rank_at(k);
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] &= left >= 2 * e + 2 ? ~0u : left > 2 * e ? 0xffffu : 0u;
    }
    return b;
  }
  // The steps before n0 = stop.  hs: the tile's rows of h; none: the tokens have no adapter.  VEC: these steps hold no
  // part of a group of CT columns.
  template <int YT, bool VEC>
  __device__ __forceinline__ void columns(int stop, const int* token, int count, bool none, const uint16_t* hs, const float* back) {
    constexpr bool AHEAD = VEC && SUB > 1 && YT != DT_F32;  // y of the next 16 tokens on its way: fp32 has no registers for it
    for (; n0 < stop; n0 += STEP) {
      u32x4_t bf[SUB > 1 ? KT : 1][SUB > 1 ? CT : 1];  // read once for all tokens
#pragma unroll
      for (int turn = 0; turn < TURNS; ++turn) {
        store_b(turn);
        if constexpr (TURNS > 1)
#pragma unroll
          for (int k = 0; k < KT; ++k)
#pragma unroll
            for (int c = turn * CTT; c < (turn + 1) * CTT; ++c) bf[k][c] = operand(k, c);
      }
      const int n = n0 + CT * col, left = it.N - n;
      Cols<YT, CT> y[4];
      uint32_t bits[VEC ? 1 : 4][VEC ? 1 : CT];  // of single elements of y
      auto load_y = [&](Cols<YT, CT>(&to)[4], int s) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int t = 16 * s + 4 * g + i;
          const int64_t at = (int64_t)token[t < count ? t : 0] * it.N + n;
          if constexpr (VEC) {
            to[i].load(it, at, left > 0 && t < count, B);
          } else {
#pragma unroll
            for (int c = 0; c < CT; ++c) {
              bits[i][c] = 0;
              if (t < count && c < left)
                bits[i][c] = YT == DT_F32 ? ((const uint32_t*)it.y_dev)[at + c] : ((const uint16_t*)it.y_dev)[at + c];
            }
          }
        }
      };
      load_y(y, 0);
      asm volatile("" ::: "memory");  // the loads stay in this order: what waits for y would wait for those before it too
      load_b(n0 + STEP, n0 + STEP < end);
      if constexpr (SUB > 1 && TURNS == 1)
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int c = 0; c < CT; ++c) bf[k][c] = operand(k, c);
#pragma unroll 1
      for (int s = 0; s < SUB; ++s) {
        if (SUB > 1 && 16 * s >= count) break;
        Cols<YT, CT> y_next[4];
        if (AHEAD && 16 * (s + 1) < count) load_y(y_next, s + 1);
        f32x4_t acc[CT] = {};
        if (!none) {
          const uint16_t* h = hs + (16 * s + col) * h_row(F16, RT);
#pragma unroll
          for (int k = 0; k < KT; ++k) {
            constexpr int PARTS = RT == 1 ? h_parts(F16) - 1 : h_parts(F16);  // operands
            u32x4_t f[PARTS];
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
              f[p] = *(const u32x4_t*)(h + (RT == 1 ? p ? 2 * R + rank_at(0) : 8 * g : p * R + 32 * k + 8 * g));
#pragma unroll
            for (int c = 0; c < CT; ++c) {
              u32x4_t b;
              if constexpr (SUB > 1) b = bf[k][c];
              else b = operand(k, c);
#pragma unroll
              for (int p = PARTS - 1; p >= 0; --p) acc[c] = mfma16<F16>(f[p], b, acc[c]);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int t = 16 * s + 4 * g + i;
          const float f = F16 && !none ? back[t] : 1.f;
          if (t >= count || left <= 0) continue;
          if (f == 0.f) {
            wide = true;
            continue;
          }
          const int64_t at = (int64_t)token[t] * it.N + n;
          if constexpr (VEC) {
            float v[CT];
#pragma unroll
            for (int c = 0; c < CT; ++c) v[c] = acc[c][i];
            y[i].store(it, at, v, f);
          } else {
#pragma unroll
            for (int c = 0; c < CT; ++c)
              if (c < left) {
                const uint32_t b = bits[i][c];
                const float y0 = YT == DT_F32 ? __builtin_bit_cast(float, b) : unpack<YT == DT_F16>(b, 0);
                store_scalar(it.out_dev, YT, at + c, y0 + acc[c][i] * f);
              }
          }
        }
        if constexpr (AHEAD) {
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = y_next[i];
        } else if (16 * (s + 1) < count) {
          load_y(y, s + 1);
        }
      }
    }
  }
  template <int YT>
  __device__ __forceinline__ void columns(const int* token, int count, bool none, const uint16_t* hs, const float* back) {
    // a row's last columns, where they are fewer than CT, one by one with the others of their step
    columns<YT, true>(it.N % CT ? min(end, it.N - 16 * CT + 1) : end, token, count, none, hs, back);
    if (it.N % CT) columns<YT, false>(end, token, count, none, hs, back);
  }
  // The wavefront's columns of the tokens whose ranks are in fp32 (split_h), a column a lane: few, or none.
  __device__ __forceinline__ void wide_tokens(int begin, const int* token, int count, const uint16_t* hs, const float* back) {
    static_assert(16 * SUB <= 64, "a token for each lane");
    const int lane = threadIdx.x & 63, first = begin + (threadIdx.x >> 6) * 16 * CT;
    for (uint64_t which = __ballot(lane < count && back[min(lane, count - 1)] == 0.f); which; which &= which - 1) {
      const int t = __builtin_ctzll(which);
      const float* h = (const float*)(hs + t * h_row(F16, RT));
      for (int at = lane; first + at / (16 * CT) * STEP < end; at += 64) {
        const int n = first + at / (16 * CT) * STEP + at % (16 * CT);
        if (n >= end) continue;
        const int64_t to = (int64_t)token[t] * it.N + n;
        u32x4_t b[C];  // all on their way at once
#pragma unroll
        for (int p = 0; p < C; ++p) b[p] = *(const u32x4_t*)(B + (int64_t)n * ld + (8 * p < rank ? 8 * p : 0));
        float sum = load_scalar(it.y_dev, it.y_dtype, to);
#pragma unroll
        for (int p = 0; p < C; ++p) {
          if (8 * p >= rank) break;
          const f32x4_t lower = *(const f32x4_t*)(h + 8 * p), upper = *(const f32x4_t*)(h + 8 * p + 4);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (8 * p + i < rank) sum = __builtin_fmaf(i < 4 ? lower[i & 3] : upper[i & 3], unpack<true>(b[p][i / 2], i % 2), sum);
        }
        store_scalar(it.out_dev, it.y_dtype, to, sum);
      }
    }
  }
  __device__ __forceinline__ void run(int begin, const int* token, int count, bool none, const uint16_t* hs, const float* back) {
    if (it.y_dtype == DT_BF16) columns<DT_BF16>(token, count, none, hs, back);
    else if (it.y_dtype == DT_F16) columns<DT_F16>(token, count, none, hs, back);
    else columns<DT_F32>(token, count, none, hs, back);
    if constexpr (F16)
      if (__ballot(wide)) wide_tokens(begin, token, count, hs, back);
  }
};

// One tile and a.columns columns of an item, h from the workspace.
template <bool F16, int RT, int SUB>
__global__ __launch_bounds__(kThreads, RT <= 4 && SUB == 1 ? 3 : 2) void expand_kernel(LoraArgs a) {
  __shared__ int token[16 * SUB];
  __shared__ float back[16 * SUB];
  __shared__ __attribute__((aligned(16))) uint16_t hs[16 * SUB * h_row(F16, RT)];
  const mlxr_lora_item& it = a.item[blockIdx.z];
  const int begin = blockIdx.x * a.columns;
  if (begin >= it.N) return;
  const Tile tile = planned_tile<SUB>(a, blockIdx.y, token);
  const int count = tile.count, rank = tile.rank;
  if (count == 0) return;
  const bool none = tile.adapter == a.adapters;
  if (none && it.out_dev == it.y_dev) return;
  using E = Expand<F16, RT, SUB, kWaves>;
  __shared__ u32x4_t rows[kWaves * E::ROWS];
  E e(a, it, tile, begin, rows);
  if (!none) {
    for (int u = threadIdx.x; u < 16 * SUB * 2 * RT; u += kThreads) {
      const int t = u / (2 * RT), at = 8 * (u % (2 * RT));
      f32x4_t v[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
      if (t < count && at < rank) {
        const float* p = a.h + ((int64_t)blockIdx.z * a.splits * a.tokens + token[t]) * a.rank + at;
        const int64_t step = (int64_t)a.tokens * a.rank;
        f32x4_t in[kSplits][2];
#pragma unroll
        for (int s = 0; s < kSplits; ++s)
#pragma unroll
          for (int k = 0; k < 2; ++k) in[s][k] = s < a.splits ? *(const f32x4_t*)(p + s * step + 4 * k) : f32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < kSplits; ++s)
#pragma unroll
          for (int k = 0; k < 2; ++k) v[k] += in[s][k];
      }
      split_h<F16, RT>(v, tile.scale, t, at, hs + t * h_row(F16, RT), back);
    }
    __syncthreads();
  }
  e.run(begin, token, count, none, hs, back);
}

// Both products of one tile and a.columns columns of an item: every workgroup of a tile computes its h for itself.
// For few tokens and small A, where that costs less than a launch, and no workspace.
template <bool F16, int RT>
__global__ __launch_bounds__(kFusedThreads) void fused_kernel(LoraArgs a) {
  constexpr int WAVES = kFusedThreads / 64, U = 4;  // steps of 64 k on their way at once
  __shared__ int token[16];
  __shared__ float back[16];
  __shared__ __attribute__((aligned(16))) uint16_t hs[16 * h_row(F16, RT)];
  __shared__ f32x4_t sh[WAVES][RT][64];
  const mlxr_lora_item& it = a.item[blockIdx.z];
  const int begin = blockIdx.x * a.columns;
  if (begin >= it.N) return;
  const Tile tile = found_tile<WAVES>(a, blockIdx.y, token);
  const int count = tile.count, rank = tile.rank;
  if (count == 0) return;
  const bool none = tile.adapter == a.adapters;
  if (none && it.out_dev == it.y_dev) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  using E = Expand<F16, RT, 1, WAVES>;
  static_assert(E::ROWS >= 128, "turn's room");
  __shared__ u32x4_t rows[WAVES * E::ROWS];
  E e(a, it, tile, begin, rows);
  if (!none) {
    const int row = lane >> 3, at = 8 * (lane & 7);
    const uint16_t* A = (const uint16_t*)it.a_dev + (int64_t)tile.adapter * a.rank * a.K;
    const uint16_t* x[2] = {a.x + (int64_t)token[row < count ? row : 0] * a.x_stride,
                            a.x + (int64_t)token[row + 8 < count ? row + 8 : 0] * a.x_stride};
    f32x4_t acc[RT] = {};
    for (int k0 = wave * 64; k0 < a.K; k0 += WAVES * U * 64) {
      u32x4_t xf[U][2], af[U][RT][2];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int kk = k0 + u * WAVES * 64 + at;
          const bool in = kk < a.K;
          xf[u][i] = in ? *(const u32x4_t*)(x[i] + kk) : u32x4_t{0, 0, 0, 0};
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const int n = 16 * r + 8 * i + row;
            af[u][r][i] = in && n < rank ? *(const u32x4_t*)(A + (int64_t)n * a.K + kk) : u32x4_t{0, 0, 0, 0};
          }
        }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        turn(xf[u], rows + wave * E::ROWS);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          turn(af[u][r], rows + wave * E::ROWS);
#pragma unroll
          for (int e = 0; e < 2; ++e) acc[r] = mfma16<F16>(af[u][r][e], xf[u][e], acc[r]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) sh[wave][r][lane] = acc[r];
    __syncthreads();
    if (threadIdx.x < 32 * RT) {
      const int t = threadIdx.x / (2 * RT), part = threadIdx.x % (2 * RT);
      f32x4_t v[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
      for (int w = 0; w < WAVES; ++w)
#pragma unroll
        for (int k = 0; k < 2; ++k) v[k] += sh[w][part >> 1][(2 * (part & 1) + k) * 16 + t];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i >> 2][i & 3] = 8 * part + i < rank ? v[i >> 2][i & 3] : 0.f;  // an infinite x gave NaN there
      split_h<F16, RT>(v, tile.scale, t, 8 * part, hs + t * h_row(F16, RT), back);
    }
    __syncthreads();
  }
  e.run(begin, token, count, none, hs, back);
}

struct Layout {
  bool fused;
  int tiles, splits, chunk, columns;  // most tiles that the call may have; splits of K; columns of a workgroup
  size_t order, tile, h, bytes;
};
Layout layout_of(int count, const mlxr_lora_item* item, int tokens, int K, int adapters, int rank) {
  Layout l{};
  const int items = count < kItems ? count : kItems, tm = tokens <= kInline ? 16 : 16 * kSub;
  const int buckets = std::min(tokens, adapters + 1), groups = rank_groups_of(rank);
  l.tiles = std::min(tokens, tokens / tm + buckets);
  long wide = 0, fused_groups = 0;
  for (int i = 0; i < count; ++i) {
    wide += item[i].N;
    fused_groups += ((long)item[i].N + kFusedThreads - 1) / kFusedThreads;  // 64 columns a wavefront
  }
  // One launch where each workgroup's reading of A (at most 128 KiB) is short beside a launch and all of it together
  // at most 16 MiB.  Measured, us, one launch and two (the host needs 4 more for two): rank 16, K 2048, three
  // projections of 2560 together, 1 token 5.8 and 7.6, 64 tokens 7.8 and 9.0; rank 16, K 4096, 6144, 4 tokens
  // 8.7 and 8.6, 16 tokens (24 MiB) 12.3 and 9.9; rank 16, K 8192, 10240, 1 token 8.4 and 7.8; K 14336, 4096, 11.3 and 8.1.
  l.fused = tokens <= kInline && groups <= 2 && (long)rank * K <= 1 << 16 && fused_groups * l.tiles * rank * K <= 1 << 23;
  if (l.fused) {
    l.columns = kFusedThreads;
    return l;
  }
  const bool sorted = tokens > kInline;
  const int group = sorted ? 16 * shrink_sub(groups, kSub) : 16;
  // As many splits as the device holds workgroups of shrink at once (two on a CU up to rank 32, else one; a quarter more
  // for sorted tokens, whose adapters' last tiles are partly empty), in chunks of whole steps of the workgroup, two at least.
  // us, at once, twice that, half: 64 tokens of 16 adapters of rank 128, K 8192, three projections of 10240 together 43,
  // 46, 51; 16 tokens of rank 64 there 23, 26, 27; 64 of rank 128, K 28672, 8192, 47, 45, 52; 2000 of rank 64 there 67, 73, 85.
  const long places = (long)device_cu_count() * (groups <= 2 ? 2 : 1) * (sorted ? 5 : 4) / 4;
  const long want = std::max(1L, places / ((long)std::min(tokens, tokens / group + buckets) * items));
  const int most = std::min(kSplits, (K + 1023) / 1024);
  int splits = (int)(want < most ? want : most);
  l.chunk = ((K + splits - 1) / splits + kShrinkThreads - 1) / kShrinkThreads * kShrinkThreads;
  l.splits = (K + l.chunk - 1) / l.chunk;
  // columns of a workgroup of expand: several steps where that leaves enough workgroups, so that what a
  // workgroup does first (its tile, h) is paid less often
  const int step = 16 * columns_of(sorted ? kSub : 1, groups) * kWaves;
  const long steps = (wide / count + step - 1) / step * items * l.tiles / (kExpandPerCu * device_cu_count());
  l.columns = step * (int)std::max(1L, std::min(16L, steps));
  auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
  l.order = 0;
  l.tile = up((size_t)l.tiles * tm * 4);
  l.h = l.tile + up((size_t)l.tiles * sizeof(Tile));
  l.bytes = l.h + (size_t)items * l.splits * tokens * rank * 4;
  return l;
}

int widest(const LoraArgs& a) {
  int n = 0;
  for (int i = 0; i < a.count; ++i) n = std::max(n, a.item[i].N);
  return n;
}
template <bool F16, int RT, int SUB, bool INLINE>
void launch(const LoraArgs& a, int tiles, hipStream_t s) {
  const int wide = widest(a);
  const size_t lds = INLINE ? (size_t)(a.adapters + 1) * sizeof(int) : 0;
  shrink_kernel<F16, RT, SUB, INLINE><<<dim3(tiles * (SUB / shrink_sub(RT, SUB)), a.splits, a.count), kShrinkThreads, lds, s>>>(a);
  expand_kernel<F16, RT, SUB><<<dim3((wide + a.columns - 1) / a.columns, tiles, a.count), kThreads, 0, s>>>(a);
}
template <bool F16, int RT>
void launch_tokens(const LoraArgs& a, const Layout& l, hipStream_t s) {
  const int tiles = l.tiles;
  if constexpr (RT <= 2)
    if (l.fused) {
      fused_kernel<F16, RT><<<dim3((widest(a) + a.columns - 1) / a.columns, tiles, a.count), kFusedThreads,
                              (size_t)(a.adapters + 1) * sizeof(int), s>>>(a);
      return;
    }
  if (a.tokens <= kInline) launch<F16, RT, 1, true>(a, tiles, s);
  else launch<F16, RT, kSub, false>(a, tiles, s);
}
template <bool F16>
void launch_rank(const LoraArgs& a, const Layout& l, hipStream_t s) {
  const int n = rank_groups_of(a.rank);
  if (n == 1) launch_tokens<F16, 1>(a, l, s);
  else if (n == 2) launch_tokens<F16, 2>(a, l, s);
  else if (n == 4) launch_tokens<F16, 4>(a, l, s);
  else launch_tokens<F16, 8>(a, l, s);
}

int check_lora(int count, const mlxr_lora_item* items, int tokens, int K, int adapters, int rank) {
  if (count < 0 || tokens < 0 || K <= 0 || adapters <= 0 || rank <= 0) return set_error(MLXR_E_INVALID, "lora: bad sizes");
  if (adapters > MLXR_LORA_MAX_ADAPTERS)
    return set_error(MLXR_E_SHAPE, "lora: at most %d adapters", MLXR_LORA_MAX_ADAPTERS);
  if (rank % 8 || rank > MLXR_LORA_MAX_RANK)
    return set_error(MLXR_E_SHAPE, "lora: rank must be a multiple of 8 and at most %d", MLXR_LORA_MAX_RANK);
  if (K > MLXR_LORA_MAX_SIZE) return set_error(MLXR_E_SHAPE, "lora: K must be at most %d", MLXR_LORA_MAX_SIZE);
  if (K % 8) return set_error(MLXR_E_SHAPE, "lora: K must be a multiple of 8");
  if (tokens > MLXR_LORA_MAX_TOKENS) return set_error(MLXR_E_SHAPE, "lora: at most %d tokens", MLXR_LORA_MAX_TOKENS);
  if (count && !items) return set_error(MLXR_E_INVALID, "null items");
  for (int i = 0; i < count; ++i)
    if (items[i].N <= 0 || items[i].N > MLXR_LORA_MAX_SIZE)
      return set_error(MLXR_E_INVALID, "lora: N must be positive and at most %d", MLXR_LORA_MAX_SIZE);
  return MLXR_OK;
}

}  // namespace

}  // namespace mlxr

using namespace mlxr;

extern "C" int mlxr_lora_workspace_size(int count, const mlxr_lora_item* items, int tokens, int K, int adapters, int rank,
                                        size_t* bytes) {
  if (!bytes) return set_error(MLXR_E_INVALID, "null bytes");
  if (const int rc = check_lora(count, items, tokens, K, adapters, rank)) return rc;
  *bytes = count && tokens ? layout_of(count, items, tokens, K, adapters, rank).bytes : 0;
  return MLXR_OK;
}

extern "C" int mlxr_lora_apply(int count, const mlxr_lora_item* items, int tokens, int K, int adapters, int rank,
                               const void* x_dev, int x_dtype, int64_t x_stride, const int32_t* ids_dev,
                               const float* scales_dev, const int32_t* ranks_dev, void* workspace_dev,
                               size_t workspace_bytes, void* stream) {
  if (const int rc = check_lora(count, items, tokens, K, adapters, rank)) return rc;
  if (x_dtype != MLXR_F16 && x_dtype != MLXR_BF16) return set_error(MLXR_E_INVALID, "invalid activation dtype %d", x_dtype);
  if (count == 0 || tokens == 0) return MLXR_OK;
  if (!x_dev || !ids_dev) return set_error(MLXR_E_INVALID, "null buffer");
  if (x_stride % 8 || ((uintptr_t)x_dev & 15) || ((uintptr_t)workspace_dev & 15))
    return set_error(MLXR_E_SHAPE, "lora: rows of x and the workspace must start at multiples of 16 bytes");
  for (int i = 0; i < count; ++i) {
    const mlxr_lora_item& t = items[i];
    if (!t.a_dev || !t.b_dev || !t.y_dev || !t.out_dev) return set_error(MLXR_E_INVALID, "null buffer");
    if (t.y_dtype != MLXR_F32 && t.y_dtype != MLXR_F16 && t.y_dtype != MLXR_BF16)
      return set_error(MLXR_E_INVALID, "invalid output dtype %d", t.y_dtype);
    if (((uintptr_t)t.a_dev | (uintptr_t)t.b_dev) & 15)
      return set_error(MLXR_E_SHAPE, "lora: A and B must start at multiples of 16 bytes");
  }
  const Layout l = layout_of(count, items, tokens, K, adapters, rank);
  if (workspace_bytes < l.bytes || (l.bytes && !workspace_dev))
    return set_error(MLXR_E_INVALID, "lora: the workspace is smaller than mlxr_lora_workspace_size");
  const hipStream_t s = (hipStream_t)stream;
  uint8_t* ws = (uint8_t*)workspace_dev;
  LoraArgs a{};
  a.x = (const uint16_t*)x_dev, a.x_stride = x_stride;
  a.ids = ids_dev, a.ranks = ranks_dev, a.scales = scales_dev;
  a.order = (int32_t*)(ws + l.order), a.tiles = (Tile*)(ws + l.tile);
  a.h = (float*)(ws + l.h);
  a.tokens = tokens, a.K = K, a.adapters = adapters, a.rank = rank, a.splits = l.splits, a.chunk = l.chunk;
  a.columns = l.columns, a.most_tiles = l.tiles;
  for (int i = 0; i < count; i += kItems) {
    a.count = count - i < kItems ? count - i : kItems;
    for (int j = 0; j < a.count; ++j) a.item[j] = items[i + j];
    if (i == 0 && tokens > kInline) plan_kernel<<<1, kPlanThreads, (size_t)(adapters + 1) * 8, s>>>(a);
    if (x_dtype == MLXR_F16) launch_rank<true>(a, l, s);
    else launch_rank<false>(a, l, s);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(MLXR_E_HIP, "lora launch: %s", hipGetErrorString(e));
  return MLXR_OK;
}
