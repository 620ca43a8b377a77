// Decode attention over a paged cache: the C entry, and the join of the pieces that the kernel
// (paged_attn.h) leaves of rows dealt to several wavefronts.
#include <algorithm>

#include "paged_attn.h"

namespace mlxr {
namespace paged {

namespace {

// A part of a softmax average: sum of weights relative to 2^m, and the weighted values.
struct Part {
  float m, l;
  f32x4_t o;
};
__device__ __forceinline__ void add(Part& a, const Part& b) {
  const float m = fmaxf(a.m, b.m), ref = m == -INFINITY ? 0.f : m;
  const float fa = __builtin_amdgcn_exp2f(a.m - ref), fb = __builtin_amdgcn_exp2f(b.m - ref);
  a.m = m;
  a.l = a.l * fa + b.l * fb;
  a.o = a.o * fa + b.o * fb;
}

// One workgroup per (row, head): o = sum_w 2^(m_w - M) o_w / sum_w 2^(m_w - M) l_w over the wavefronts w
// that had a piece of the row, M the maximum of their m (-inf: no token counted).  Rows without tokens get zeros; rows that one
// wavefront covered are done.  Threads: four dims each (LANES, a power of two that covers head_dim), several
// pieces side by side, four of them on their way at once.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void join_kernel(AttnArgs a, int lanes) {
  constexpr int WAVES = THREADS / 64;
  __shared__ Part sh[WAVES][64];
  const int r = blockIdx.x / a.heads, h = blockIdx.x - r * a.heads, tid = threadIdx.x;
  const int kvh = h / a.group, hk = h - kvh * a.group, grp = hk / kHeads, row = hk - grp * kHeads;
  const int per_row = a.kv_heads * a.groups, before = a.prefix[r], tiles = a.prefix[r + 1] - before, per = a.prefix[a.rows + 1];
  const int64_t head = (int64_t)r * a.heads + h;
  if (tiles == 0) {
    for (int d = tid; d < a.dim; d += THREADS) store_scalar(a.out, a.out_dtype, head * a.dim + d, 0.f);
    if (a.lse && tid == 0) a.lse[head] = -INFINITY;
    return;
  }
  const int64_t s = (int64_t)before * per_row + (int64_t)(kvh * a.groups + grp) * tiles;
  const int w0 = quotient(s, per), w1 = quotient(s + tiles - 1, per);
  if (w0 == w1) return;
  const int count = w1 - w0 + 1;
  const bool late = (int64_t)w0 * per < s;  // the first of them had another row before this one
  const int x = tid & (lanes - 1), y = tid / lanes, across = THREADS / lanes;
  const bool in = 4 * x < a.dim;
  Part sum = {-INFINITY, 0.f, {0, 0, 0, 0}};
  for (int i = y; i < count; i += 4 * across) {
    Part p[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int w = i + k * across;
      const bool ok = w < count;
      const float* at = partial(a, w0 + (ok ? w : 0), (ok ? w : 0) == 0 && late ? 1 : 0);
      const float* st = at + (int64_t)a.part_rows * a.dim + 2 * row;
      p[k].m = ok ? st[0] : -INFINITY;
      p[k].l = ok ? st[1] : 0.f;
      p[k].o = ok && in ? *(const f32x4_t*)(at + (int64_t)row * a.dim + 4 * x) : f32x4_t{0, 0, 0, 0};
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) add(sum, p[k]);
  }
  for (int d = lanes; d < 64; d *= 2) {
    Part q;
    q.m = __shfl_xor(sum.m, d);
    q.l = __shfl_xor(sum.l, d);
#pragma unroll
    for (int c = 0; c < 4; ++c) q.o[c] = __shfl_xor(sum.o[c], d);
    add(sum, q);
  }
  sh[tid >> 6][tid & 63] = sum;
  __syncthreads();
  if (y || !in) return;
  for (int w = 1; w < WAVES; ++w) add(sum, sh[w][x]);
  const float f = average_factor(a, kvh, sum.m, sum.l);
  const f32x4_t v = sum.o * f;
  const float each[4] = {v[0], v[1], v[2], v[3]};
  store_values<4>(a.out, a.out_dtype, head * a.dim + 4 * x, each);
  if (a.lse && x == 0) a.lse[head] = (sum.m + __builtin_amdgcn_logf(sum.l)) * 0.69314718055994531f;
}

AttnKern& kern(const mlxr_paged_cache* c, int q_dtype) {
  const bool f16 = q_dtype == MLXR_F16, p8 = c->page_size % 8 == 0;
  if (c->dtype == MLXR_E4M3) return f16 ? kern_f16_e4m3(c->head_dim, p8) : kern_bf16_e4m3(c->head_dim, p8);
  return f16 ? kern_f16(c->head_dim, p8) : kern_bf16(c->head_dim, p8);
}

constexpr int kGridPerCu = 4;  // most workgroups of a CU that grid_of gives
constexpr int kJoinMany = 512;
constexpr int kMaxHeads = (1 << 24) - 64;  // rows times heads: a launch has fewer than 2^32 threads

// How a call runs: short rows in one launch without a workspace.
struct Plan {
  int group, groups, part_rows;
  bool one, two_of_cu, keys_in_lds;  // of one launch
  size_t bytes;                      // of the workspace
};
constexpr size_t prefix_bytes(int rows) { return (size_t)(rows + 2 + 3) / 4 * 4 * sizeof(int32_t); }
// By the longest row that the table can hold, or the window; a window never needs more workspace.  A workgroup alone
// gets about 38 GB/s, so few rows have to be cut unless they are short; many rows fill the device uncut, until the longest
// keeps it waiting.
// Measured, us, uncut and cut (which also takes the host 4 us more), rows up to the longest, ragged unless one; 8 kv heads of
// 128 in bf16, up to 512 tokens (256 KiB a head): one row 9.5 and 9.5, 64 rows 18 and 24; 1024: 15 and 11, 4 rows 18 and
// 12, 16 19 and 17, 64 30 and 37; 2048 (1 MiB): 32 rows 30 and 35, 64 55 and 58; 4096 (2 MiB): 64 rows 103 and 95, 128
// 171 and 176; 8192: 128 rows 335 and 319.  32 of 128, 4096: 33 rows 197 and 176, 64 315 and 342; 8192: 64 rows 627 and
// 624.  In e4m3, 2048 (512 KiB): 16 rows 22 and 23, 64 33 and 46; 8192: 128 rows 186 and 192.  4 of 64, 2048: one row
// 18 and 10, 64 20 and 26; 8192: 64 rows 63 and 54.
Plan plan_of(const mlxr_paged_cache* c, int rows, int heads, int width, int window) {
  Plan p;
  const int64_t held = (int64_t)width * c->page_size, most = window > 0 && window < held ? window : held;
  p.group = heads / c->kv_heads;
  p.groups = (p.group + kHeads - 1) / kHeads;
  p.part_rows = p.group < kHeads ? p.group : kHeads;
  const int64_t units = (int64_t)rows * c->kv_heads * p.groups;
  const int64_t bytes = 2 * most * c->head_dim * (c->dtype == MLXR_E4M3 ? 1 : 2);
  p.one = bytes <= 256 << 10 || (bytes <= 1 << 20 && units >= 256) || (bytes <= 2 << 20 && units >= 2048) || rows > kMaxCutRows ||
          (held / kTile + 1) * rows > INT32_MAX || (held / kTile + 1) * units / 64 > INT32_MAX;  // what a cut launch counts in 32 bits
  // Rows of more than 256 KiB: two workgroups of a CU, not the three or four that its registers hold, by LDS that they do
  // not use.  Later workgroups then start where rows turn out short, and lines that heads share stay in the L2.  us, three
  // or four and two: 32 kv heads of 80 in [token, head] order, 1024 tokens, 17 rows 57 and 43, 48 rows 112 and 104; 32 of
  // 128, up to 1024, 17 rows 38 and 36, 200 rows 259 and 262; 4 of 64, up to 2048, 200 rows 56 and 48; below: 32 of 80,
  // 256 tokens, 100 rows 40 and 47; 8 of 128, up to 300, 200 rows 30 and 33.  (Above 128 dims one is resident.)
  p.two_of_cu = bytes > 256 << 10 && c->head_dim <= 128;
  // Where latency does not count (load_k): a workgroup for each CU, two tiles for a wavefront.  us, straight and through
  // LDS, 128 rows of 8 kv heads of 128 in bf16, up to 34 tokens 10.1 and 11.2, 100 13.1 and 13.7, 200 17.2 and 16.9, 1000 55
  // and 47; of 256, 100 37.3 and 37.1, 400 65 and 57, 1000 119 and 94; in e4m3 of 128, 200 14.7 and 14.7, 1000 33 and 29.
  p.keys_in_lds = units >= device_cu_count() && most >= 2 * kWaves * kTile;
  p.bytes = p.one ? 0 : prefix_bytes(rows) + (size_t)device_cu_count() * kGridPerCu * kWaves * 2 *
                                                 partial_floats(p.part_rows, c->head_dim) * sizeof(float);
  return p;
}
// Workgroups of a cut launch: as many as the device holds at once.
int grid_of(AttnKern& k, hipError_t* e) {
  int dev = 0;
  *e = hipGetDevice(&dev);
  if (*e != hipSuccess) return 0;
  const int d = dev >= 0 && dev < 64 ? dev : 0;
  int occ = k.residents[d].load(std::memory_order_acquire);
  if (!occ) {
    *e = hipOccupancyMaxActiveBlocksPerMultiprocessor(&occ, k.fn, 64 * kWaves, 0);
    if (*e != hipSuccess) return 0;
    occ = std::max(1, std::min(occ, kGridPerCu));
    k.residents[d].store(occ, std::memory_order_release);
  }
  return occ * device_cu_count();
}

int check_attn(const mlxr_paged_cache* c, int rows, int heads, int width) {
  if (const int rc = check_cache(c)) return rc;
  if (rows < 0 || heads <= 0 || width <= 0) return set_error(MLXR_E_INVALID, "paged_attention: bad sizes");
  if (heads % c->kv_heads) return set_error(MLXR_E_SHAPE, "heads must be a multiple of kv_heads");
  for (int i = 0; i < 3; i += 2)
    if (c->k_stride[i] > UINT32_MAX / 2 || c->v_stride[i] > UINT32_MAX / 2)
      return set_error(MLXR_E_SHAPE, "paged_attention: pages and tokens must lie less than 4 GiB apart");
  if ((int64_t)width * c->page_size > INT32_MAX - 1024) return set_error(MLXR_E_SHAPE, "paged_attention: the table covers too many tokens");
  if ((int64_t)rows * heads > kMaxHeads) return set_error(MLXR_E_SHAPE, "paged_attention: at most %d rows times heads", kMaxHeads);
  return MLXR_OK;
}

}  // namespace
}  // namespace paged
}  // namespace mlxr

using namespace mlxr;
using namespace mlxr::paged;

extern "C" int mlxr_paged_attention_workspace_size(const mlxr_paged_cache* cache, int rows, int heads, int table_width,
                                                   size_t* bytes) {
  if (!bytes) return set_error(MLXR_E_INVALID, "null bytes");
  if (const int rc = check_attn(cache, rows, heads, table_width)) return rc;
  *bytes = rows ? plan_of(cache, rows, heads, table_width, 0).bytes : 0;
  return MLXR_OK;
}

extern "C" int mlxr_paged_attention(const mlxr_paged_cache* cache, int rows, int heads, const void* q_dev, int q_dtype,
                                    int64_t q_row_stride, int64_t q_head_stride, const int32_t* table_dev,
                                    int64_t table_stride, int table_width, const int32_t* lens_dev, float scale,
                                    int window, void* out_dev, int out_dtype, float* lse_dev, void* workspace_dev,
                                    size_t workspace_bytes, void* stream) {
  if (const int rc = check_attn(cache, rows, heads, table_width)) return rc;
  if (q_dtype != MLXR_F16 && q_dtype != MLXR_BF16) return set_error(MLXR_E_INVALID, "invalid query dtype %d", q_dtype);
  if (cache->dtype != MLXR_E4M3 && cache->dtype != q_dtype)
    return set_error(MLXR_E_INVALID, "queries must have the cache's type");
  if (out_dtype != MLXR_F32 && out_dtype != MLXR_F16 && out_dtype != MLXR_BF16)
    return set_error(MLXR_E_INVALID, "invalid output dtype %d", out_dtype);
  if (window < 0) return set_error(MLXR_E_INVALID, "paged_attention: window must not be negative");
  if (rows == 0) return MLXR_OK;
  if (!q_dev || !table_dev || !lens_dev || !out_dev) return set_error(MLXR_E_INVALID, "null buffer");
  if (q_row_stride % 8 || q_head_stride % 8 || (((uintptr_t)q_dev | (uintptr_t)out_dev | (uintptr_t)workspace_dev) & 15))
    return set_error(MLXR_E_SHAPE, "paged_attention: query rows, output and workspace must start at multiples of 16 bytes");
  const Plan p = plan_of(cache, rows, heads, table_width, window);
  if (workspace_bytes < p.bytes || (p.bytes && !workspace_dev))
    return set_error(MLXR_E_INVALID, "paged_attention: the workspace is smaller than mlxr_paged_attention_workspace_size");
  const int es = cache->dtype == MLXR_E4M3 ? 1 : 2;
  AttnArgs a{};
  a.k = (const uint8_t*)cache->k_dev, a.v = (const uint8_t*)cache->v_dev;
  a.k_scale = cache->k_scale_dev, a.v_scale = cache->v_scale_dev;
  a.k_head = cache->k_stride[1] * es, a.v_head = cache->v_stride[1] * es;
  a.k_page = (uint32_t)(cache->k_stride[0] * es), a.k_token = (uint32_t)(cache->k_stride[2] * es);
  a.v_page = (uint32_t)(cache->v_stride[0] * es), a.v_token = (uint32_t)(cache->v_stride[2] * es);
  a.q = (const uint16_t*)q_dev, a.q_row = q_row_stride, a.q_head = q_head_stride;
  a.table = table_dev, a.table_stride = table_stride, a.lens = lens_dev;
  a.out = out_dev, a.lse = lse_dev;
  a.rows = rows, a.heads = heads, a.kv_heads = cache->kv_heads;
  a.group = p.group, a.groups = p.groups, a.part_rows = p.part_rows;
  a.dim = cache->head_dim, a.page = cache->page_size, a.pages = cache->num_pages, a.width = table_width;
  a.by_page = Divisor(a.page);
  a.window = window, a.out_dtype = out_dtype;
  a.scale = scale * 1.44269504088896341f;
  const hipStream_t st = (hipStream_t)stream;
  AttnKern& k = kern(cache, q_dtype);
  void* args[] = {&a};
  hipError_t e = hipSuccess;
  if (p.one) {
    // neighbouring kv heads share lines where a token's heads lie side by side and are no whole lines
    a.near = 1;
    if (a.k_head % 128 || a.v_head % 128)
      while (a.near < 8 && a.kv_heads % (2 * a.near) == 0) a.near *= 2;
    const int n = a.near * a.groups, units = rows * a.kv_heads;
    const int grid = n > 1 ? (units / a.near + 7) / 8 * 8 * n : units;
    const int own = k.rows_lds[p.keys_in_lds], lds = p.two_of_cu ? (56 << 10) - own : 0;  // of 160 KiB
    e = hipLaunchKernel(k.rows_fn[p.keys_in_lds], dim3(grid), dim3(64 * kWaves), args, lds, st);
  } else {
    const int grid = grid_of(k, &e);
    if (e != hipSuccess) return set_error(MLXR_E_HIP, "paged_attention: %s", hipGetErrorString(e));
    a.workers = grid * kWaves;
    a.prefix = (int32_t*)workspace_dev, a.ws = (float*)((uint8_t*)workspace_dev + prefix_bytes(rows));
    e = hipLaunchKernel(k.fn, dim3(grid), dim3(64 * kWaves), args, (size_t)(rows + 1) * 4, st);
    if (e == hipSuccess) {
      // few heads of all: long rows, in many pieces each
      int lanes = 2;
      while (4 * lanes < a.dim) lanes *= 2;
      if (rows * heads >= kJoinMany) join_kernel<256><<<rows * heads, 256, 0, st>>>(a, lanes);
      else join_kernel<1024><<<rows * heads, 1024, 0, st>>>(a, lanes);
      e = hipGetLastError();
    }
  }
  if (e != hipSuccess) return set_error(MLXR_E_HIP, "paged_attention launch: %s", hipGetErrorString(e));
  return MLXR_OK;
}
