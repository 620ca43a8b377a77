// Page tables and slot maps of a paged key-value cache, and the writes of new keys and values
// (include/mlxr_paged.h).
#include <hip/hip_runtime.h>

#include "../../include/mlxr_paged.h"
#include "paged_internal.h"

namespace mlxr {

namespace {

struct ResizeArgs {
  int32_t* table;
  int64_t stride;
  const int32_t *lens, *want, *free_count;
  int32_t* free;
  int32_t *lens_out, *count_out, *starts, *slots, *positions, *refused;
  int rows, page, pages, width, tokens, run;  // run: neighbouring tokens of a thread
  Divisor by_page;
};

constexpr int kResizeThreads = 256;

struct Sum3 {
  int a, b, c;
};
// Exclusive sums over the threads of a workgroup, and the totals.
__device__ Sum3 block_scan(Sum3 v, Sum3* total, int* part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Sum3 s = v;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int a = __shfl_up(s.a, d), b = __shfl_up(s.b, d), c = __shfl_up(s.c, d);
    if (lane >= d) s.a += a, s.b += b, s.c += c;
  }
  __syncthreads();  // part may still be read from the call before
  if (lane == 63) part[3 * wave] = s.a, part[3 * wave + 1] = s.b, part[3 * wave + 2] = s.c;
  __syncthreads();
  Sum3 before = {0, 0, 0}, all = {0, 0, 0};
  for (int w = 0; w < (int)(blockDim.x >> 6); ++w) {
    const Sum3 p = {part[3 * w], part[3 * w + 1], part[3 * w + 2]};
    if (w < wave) before.a += p.a, before.b += p.b, before.c += p.c;
    all.a += p.a, all.b += p.b, all.c += p.c;
  }
  *total = all;
  return {before.a + s.a - v.a, before.b + s.b - v.b, before.c + s.c - v.c};
}

// Largest r in [0, n) with first[r] <= k (first is nondecreasing, first[0] = 0).
__device__ __forceinline__ int row_of(const int* first, int n, int k) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= k) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int pages_of(const ResizeArgs& a, int tokens) { return tokens ? a.by_page.quotient(tokens - 1) + 1 : 0; }

// With P(n) = ceil(n / page): row r takes need = P(want) - P(lens) pages or gives back as many, and the
// exclusive sums of both over the rows say which place of the stack each page goes to or comes
// from: the i-th page given back by r lands at count + G_r + i, the i-th page that r takes lies
// at c1 - 1 - (N_r + i), c1 = count + all that is given back.  Every output element follows from
// the sums alone (a page taken from a place at or above `count` is read from the table of the row
// that gives it back), so nothing in the launch waits for anything else in it: each workgroup
// makes the sums for itself and fills its share of the outputs.  What bounds it is latency: lengths,
// two sums, table or stack, outputs, one after the other (256 rows that get a token each 4.8 us; 96 rows, half
// of them new prompts, 393317 places for tokens, 10.4).
__global__ __launch_bounds__(kResizeThreads) void resize_kernel(ResizeArgs a) {
  extern __shared__ int sh[];  // of each row: N_r, G_r, new tokens before it, P(lens), lens, want (-1: refused)
  int *first_need = sh, *first_give = sh + a.rows, *first_new = sh + 2 * a.rows, *held = sh + 3 * a.rows,
      *have = sh + 4 * a.rows, *want = sh + 5 * a.rows;
  __shared__ int part[3 * (kResizeThreads / 64)];
  __shared__ int most_taken;
  const int tid = threadIdx.x, nt = kResizeThreads, most = a.width * a.page;
  const int per = (a.rows + nt - 1) / nt, r0 = min(tid * per, a.rows), r1 = min(r0 + per, a.rows);
  if (tid == 0) most_taken = 0;
  const int count = min(max(a.free_count[0], 0), a.pages);
  for (int r = tid; r < a.rows; r += nt) {
    const int w = a.want[r], h = min(max(a.lens[r], 0), most);
    have[r] = h;
    want[r] = w < 0 || w > most ? -1 : w;
    held[r] = pages_of(a, h);
  }
  __syncthreads();
  auto change = [&](int r) { return want[r] < 0 ? 0 : pages_of(a, want[r]) - held[r]; };
  Sum3 mine = {0, 0, 0}, total;
  for (int r = r0; r < r1; ++r) {
    const int d = change(r);
    mine.a += max(d, 0);
    mine.b += max(-d, 0);
  }
  Sum3 before = block_scan(mine, &total, part);
  const int given = total.b, stack = count + min(given, a.pages - count);
  int taken = 0;
  mine = {0, 0, 0};
  for (int r = r0; r < r1; ++r) {
    const int d = change(r);
    first_need[r] = before.a;
    first_give[r] = before.b;
    before.a += max(d, 0);
    before.b += max(-d, 0);
    if (d > 0) {
      // the sums grow with r: the rows that get pages are a prefix of those that ask
      if (before.a <= stack) taken = before.a;
      else want[r] = -1;
    }
    if (want[r] < 0) mine.b += 1;
    else mine.c += max(want[r] - have[r], 0);
  }
  if (taken) atomicMax(&most_taken, taken);
  before = block_scan(mine, &total, part);
  const int new_tokens = total.c;
  for (int r = r0; r < r1; ++r) {
    first_new[r] = before.c;
    before.c += want[r] < 0 ? 0 : max(want[r] - have[r], 0);
  }
  __syncthreads();
  const int all_taken = most_taken;
  if (blockIdx.x == 0) {
    for (int r = tid; r < a.rows; r += nt) {
      a.starts[r] = first_new[r];
      a.lens_out[r] = want[r] < 0 ? have[r] : want[r];
    }
    if (tid == 0) {
      a.starts[a.rows] = new_tokens;
      a.count_out[0] = stack - all_taken;
      a.refused[0] = total.b;
    }
  }

  const uint32_t gid = blockIdx.x * nt + tid, gn = gridDim.x * nt;
  auto given_page = [&](int k) {  // the k-th page given back
    const int r = row_of(first_give, a.rows, k);
    return a.table[r * a.stride + pages_of(a, want[r]) + (k - first_give[r])];
  };
  auto taken_page = [&](int k) {  // the k-th page taken
    const int p = stack - 1 - k;
    return p < count ? a.free[p] : given_page(p - count);
  };
  const uint32_t tokens = a.tokens;
  for (uint32_t t = gid * a.run; t < tokens; t += gn * a.run) {
    int r = -1, j = -1, id = -1;
    for (int at = (int)t, end = (int)min(t + a.run, tokens); at < end; ++at) {
      int slot = -1, pos = -1;
      if (at < new_tokens) {
        if (r < 0 || (r + 1 < a.rows && first_new[r + 1] <= at)) {
          r = row_of(first_new, a.rows, at);
          j = -1;
        }
        pos = have[r] + (at - first_new[r]);
        const int page = a.by_page.quotient(pos);
        if (page != j) {
          j = page;
          id = j < held[r] ? a.table[r * a.stride + j] : taken_page(first_need[r] + j - held[r]);
        }
        slot = id < 0 || id >= a.pages ? -1 : id * a.page + (pos - j * a.page);
      }
      a.slots[at] = slot;
      a.positions[at] = pos;
    }
  }
  // from the far end of the launch, so that these are other workgroups than the next loop's
  for (uint32_t k = gn - 1 - gid; k < (uint32_t)all_taken; k += gn) {
    const int r = row_of(first_need, a.rows, k);
    a.table[r * a.stride + held[r] + (k - first_need[r])] = taken_page(k);
  }
  for (uint32_t k = gid; k < (uint32_t)(stack - count); k += gn) a.free[count + k] = given_page((int)k);
}

struct AppendSide {
  const void* x;
  int64_t token, head;          // strides of x
  uint8_t* store;
  int64_t s_page, s_head, s_token;  // strides of the store
  const float* scale;
};
struct AppendArgs {
  AppendSide side[2];  // keys, values
  const int32_t* slots;
  int items, slots_end;
  Divisor by_token, by_head, by_page;  // items of a token, of a head; tokens of a page
};

// Eight elements of a row as they lie in memory, and as floats.
template <int XT>
struct Eight {
  uint4 w[XT == DT_F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* x, int64_t at) {
    if constexpr (XT == DT_F32) w[0] = ((const uint4*)((const float*)x + at))[0], w[1] = ((const uint4*)((const float*)x + at))[1];
    else w[0] = *(const uint4*)((const uint16_t*)x + at);
  }
  __device__ __forceinline__ float get(int k) const {
    const uint4& q = w[XT == DT_F32 ? k >> 2 : 0];
    const uint32_t u[4] = {q.x, q.y, q.z, q.w};
    if constexpr (XT == DT_F32) return __builtin_bit_cast(float, u[k & 3]);
    const uint32_t h = (u[k >> 1] >> (16 * (k & 1))) & 0xffffu;
    return XT == DT_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
  }
};
__device__ __forceinline__ uint32_t e4m3x4(const float* v) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
}
template <int N>
__device__ __forceinline__ float largest(const float (&v)[N]) {
  float top = 0.f;
#pragma unroll
  for (int n = 0; n < N; ++n) top = fmaxf(top, fabsf(v[n]));
  return top;
}

// v / d rounded as division does, for what becomes e4m3: a reciprocal for all of them and two corrections each, the last
// of which is exact (Markstein's theorem: q within an ulp, r the rounded reciprocal, the residue exact).  That holds
// where nothing overflows or comes near the smallest numbers; quotients below 2^-10 become 0 whatever their bits, of v's
// sign.  (4099 tokens as below: 10.5 us with divisions and every value clamped, 8.3 now, 6.1 without scales.)
template <int N>
__device__ __forceinline__ void divide(float (&v)[N], float d) {
  const float r = 1.f / d;
  float q[N];
#pragma unroll
  for (int n = 0; n < N; ++n) q[n] = v[n] * r;
  if (largest(q) < 0x1p80f && fabsf(d) > 0x1p-40f && fabsf(d) < 0x1p40f) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const float q1 = __builtin_fmaf(__builtin_fmaf(-q[n], d, v[n]), r, q[n]);
      v[n] = copysignf(__builtin_fmaf(__builtin_fmaf(-q1, d, v[n]), r, q1), q[n]);
    }
  } else {
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] /= d;
  }
}

// One thread moves 16 bytes of a store, for the keys and the values: 8 or 16 elements of one head's row of one
// token.  Bound by memory for a prompt (4099 tokens
// of 8 heads of 128, bf16 to e4m3 with scales, 25 MB, 8.3 us) and by the launch for a decode batch (64 tokens 2.5 us).
template <int XT, int CT>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  constexpr int N = CT == MLXR_E4M3 ? 16 : 8;
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= a.items) return;
  const int t = a.by_token.quotient(i), e = i - t * (int)a.by_token.d, h = a.by_head.quotient(e), c = e - h * (int)a.by_head.d;
  Eight<XT> x[2][N / 8];  // on their way together with the slot
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int n = 0; n < N / 8; ++n) x[k][n].load(a.side[k].x, (int64_t)t * a.side[k].token + (int64_t)h * a.side[k].head + N * c + 8 * n);
  const int slot = a.slots[t];
  if (slot < 0 || slot >= a.slots_end) return;
  const int pg = a.by_page.quotient(slot);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const AppendSide& s = a.side[k];
    const int64_t to = (int64_t)pg * s.s_page + (int64_t)h * s.s_head + (int64_t)(slot - pg * (int)a.by_page.d) * s.s_token + N * c;
    if constexpr (XT == CT) {
      if (!s.scale) {  // same type: the bits
        *(uint4*)(s.store + 2 * to) = x[k][0].w[0];
        continue;
      }
    }
    float v[N];
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = x[k][n / 8].get(n % 8);
    if (s.scale) {
      const float d = s.scale[h];
      if constexpr (CT == MLXR_E4M3) {
        divide(v, d);
      } else {
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] /= d;
      }
    }
    if constexpr (CT == MLXR_E4M3) {
      if (largest(v) > 448.f)
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] = v[n] > 448.f ? 448.f : v[n] < -448.f ? -448.f : v[n];  // NaN stays
      *(uint4*)(s.store + to) = make_uint4(e4m3x4(v), e4m3x4(v + 4), e4m3x4(v + 8), e4m3x4(v + 12));
    } else {
      uint32_t o[4];
#pragma unroll
      for (int n = 0; n < 4; ++n)
        o[n] = CT == DT_BF16 ? pack_bf16x2(v[2 * n], v[2 * n + 1])
                             : (f32_to_f16_bits(v[2 * n]) | ((uint32_t)f32_to_f16_bits(v[2 * n + 1]) << 16));
      *(uint4*)(s.store + 2 * to) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

template <int XT>
void launch_append(const AppendArgs& a, int ct, unsigned grid, hipStream_t s) {
  if (ct == MLXR_F16) append_kernel<XT, DT_F16><<<grid, 256, 0, s>>>(a);
  else if (ct == MLXR_BF16) append_kernel<XT, DT_BF16><<<grid, 256, 0, s>>>(a);
  else append_kernel<XT, MLXR_E4M3><<<grid, 256, 0, s>>>(a);
}

}  // namespace

int check_cache(const mlxr_paged_cache* c) {
  if (!c) return set_error(MLXR_E_INVALID, "null cache");
  if (!c->k_dev || !c->v_dev) return set_error(MLXR_E_INVALID, "null buffer");
  if (c->dtype != MLXR_F16 && c->dtype != MLXR_BF16 && c->dtype != MLXR_E4M3)
    return set_error(MLXR_E_INVALID, "invalid cache dtype %d", c->dtype);
  if (c->num_pages <= 0 || c->page_size <= 0 || c->kv_heads <= 0 || c->head_dim <= 0)
    return set_error(MLXR_E_INVALID, "cache sizes must be positive");
  if ((int64_t)c->num_pages * c->page_size > INT32_MAX)
    return set_error(MLXR_E_SHAPE, "a cache holds at most %d tokens", INT32_MAX);
  const int unit = c->dtype == MLXR_E4M3 ? 16 : 8;
  if (c->head_dim % unit || c->head_dim > 256)
    return set_error(MLXR_E_SHAPE, "head_dim must be a multiple of %d and at most 256 (got %d)", unit, c->head_dim);
  for (int i = 0; i < 3; ++i)
    if (c->k_stride[i] < 0 || c->v_stride[i] < 0 || c->k_stride[i] % unit || c->v_stride[i] % unit)
      return set_error(MLXR_E_SHAPE, "cache strides must be multiples of 16 bytes");
  if (((uintptr_t)c->k_dev | (uintptr_t)c->v_dev) & 15)
    return set_error(MLXR_E_INVALID, "cache addresses must be multiples of 16 bytes");
  return MLXR_OK;
}

}  // namespace mlxr

using namespace mlxr;

extern "C" int mlxr_page_resize(int rows, int page_size, int num_pages, int32_t* table_dev, int64_t table_stride,
                                int table_width, const int32_t* lens_dev, const int32_t* want_dev, int32_t* free_dev,
                                const int32_t* free_count_dev, int32_t* lens_out_dev, int32_t* free_count_out_dev,
                                int32_t* starts_dev, int32_t* slots_dev, int32_t* positions_dev, int tokens,
                                int32_t* refused_dev, void* stream) {
  if (rows < 0 || tokens < 0 || page_size <= 0 || num_pages <= 0 || table_width <= 0)
    return set_error(MLXR_E_INVALID, "page_resize: bad sizes");
  if (!free_count_dev || !free_count_out_dev || !starts_dev || !refused_dev || !free_dev ||
      (rows && (!table_dev || !lens_dev || !want_dev || !lens_out_dev)) || (tokens && (!slots_dev || !positions_dev)))
    return set_error(MLXR_E_INVALID, "null buffer");
  if (rows > MLXR_PAGED_MAX_ROWS)
    return set_error(MLXR_E_SHAPE, "page_resize: at most %d rows", MLXR_PAGED_MAX_ROWS);
  if (rows > 1 && table_stride < table_width) return set_error(MLXR_E_SHAPE, "page_resize: table rows overlap");
  if ((int64_t)num_pages * page_size > INT32_MAX ||
      (__int128)(rows ? rows : 1) * table_width * page_size > INT32_MAX)
    return set_error(MLXR_E_SHAPE, "page_resize: a pool and a table cover at most %d tokens", INT32_MAX);
  if (lens_out_dev == lens_dev || free_count_out_dev == free_count_dev)
    return set_error(MLXR_E_INVALID, "page_resize: outputs must not be the inputs");
  ResizeArgs a{table_dev, table_stride, lens_dev, want_dev, free_count_dev, free_dev, lens_out_dev, free_count_out_dev,
               starts_dev, slots_dev, positions_dev, refused_dev, rows, page_size, num_pages, table_width, tokens, 1, Divisor(page_size)};
  // one token for each thread up to 64 workgroups; a prompt's neighbours, mostly of one page, share the search
  constexpr int kTokens = kResizeThreads * 64;
  if (tokens > kTokens) a.run = 4;
  const int64_t groups = ((int64_t)tokens + kResizeThreads * a.run - 1) / (kResizeThreads * a.run);
  const int grid = groups < 1 ? 1 : groups > 1024 ? 1024 : (int)groups;
  const size_t lds = (size_t)rows * 6 * sizeof(int);
  hipError_t e = hipSuccess;
  if (lds > 48 << 10)
    e = hipFuncSetAttribute((const void*)resize_kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                            MLXR_PAGED_MAX_ROWS * 6 * (int)sizeof(int));
  if (e == hipSuccess) {
    resize_kernel<<<grid, kResizeThreads, lds, (hipStream_t)stream>>>(a);
    e = hipGetLastError();
  }
  if (e != hipSuccess) return set_error(MLXR_E_HIP, "page_resize launch: %s", hipGetErrorString(e));
  return MLXR_OK;
}

extern "C" int mlxr_paged_append(const mlxr_paged_cache* cache, int tokens, const void* k_dev, int64_t k_token_stride,
                                 int64_t k_head_stride, const void* v_dev, int64_t v_token_stride, int64_t v_head_stride,
                                 int x_dtype, const int32_t* slots_dev, void* stream) {
  if (const int rc = check_cache(cache)) return rc;
  if (tokens < 0) return set_error(MLXR_E_INVALID, "paged_append: tokens must not be negative");
  if (tokens == 0) return MLXR_OK;
  if (!k_dev || !v_dev || !slots_dev) return set_error(MLXR_E_INVALID, "null buffer");
  if (x_dtype != MLXR_F32 && x_dtype != MLXR_F16 && x_dtype != MLXR_BF16)
    return set_error(MLXR_E_INVALID, "invalid dtype %d", x_dtype);
  const int unit = x_dtype == MLXR_F32 ? 4 : 8;
  if (k_token_stride % unit || k_head_stride % unit || v_token_stride % unit || v_head_stride % unit ||
      (((uintptr_t)k_dev | (uintptr_t)v_dev) & 15))
    return set_error(MLXR_E_SHAPE, "paged_append: rows must start at multiples of 16 bytes");
  const int of_head = cache->head_dim / (cache->dtype == MLXR_E4M3 ? 16 : 8);
  const int64_t items = (int64_t)tokens * cache->kv_heads * of_head;
  if ((int64_t)cache->kv_heads * of_head > INT32_MAX || items > INT32_MAX - 255)
    return set_error(MLXR_E_SHAPE, "paged_append: too many elements");
  AppendArgs a{{{k_dev, k_token_stride, k_head_stride, (uint8_t*)cache->k_dev, cache->k_stride[0], cache->k_stride[1],
                 cache->k_stride[2], cache->k_scale_dev},
                {v_dev, v_token_stride, v_head_stride, (uint8_t*)cache->v_dev, cache->v_stride[0], cache->v_stride[1],
                 cache->v_stride[2], cache->v_scale_dev}},
               slots_dev, (int)items, cache->num_pages * cache->page_size,
               Divisor(of_head * cache->kv_heads), Divisor(of_head), Divisor(cache->page_size)};
  const unsigned grid = (unsigned)((items + 255) / 256);
  const hipStream_t s = (hipStream_t)stream;
  if (x_dtype == MLXR_F32) launch_append<DT_F32>(a, cache->dtype, grid, s);
  else if (x_dtype == MLXR_F16) launch_append<DT_F16>(a, cache->dtype, grid, s);
  else launch_append<DT_BF16>(a, cache->dtype, grid, s);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(MLXR_E_HIP, "paged_append launch: %s", hipGetErrorString(e));
  return MLXR_OK;
}
