// Attention of drafted tokens over a paged cache: the C entries, the join of the pieces that the kernel (paged_tree.h)
// leaves of cut rows, and the masks of trees.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "paged_tree.h"

namespace mlxr {
namespace tree {
namespace {

// One token's head for each `lanes` threads, four dims a thread: o = sum_w 2^(m_w - M) o_w / sum_w 2^(m_w - M) l_w over the
// workgroups w that had a piece of its columns, M the maximum of their m (-inf: no token counted); the factors are never 0, so that
// an infinite sum stays infinite, as in the kernel (pieces that counted nothing are zeros).  Rows without
// tokens get zeros; columns that one workgroup covered are done.  Four pieces are on their way at
// once, MANY: 16 where there are more.
template <bool MANY>
__global__ __launch_bounds__(kThreads) void join_kernel(Args a, int lanes) {
  extern __shared__ int starts[];  // [rows + 1]: searched in LDS
  const int tid = threadIdx.x, x = tid & (lanes - 1);
  for (int r = tid; r <= a.rows; r += kThreads) starts[r] = a.starts[r];
  const int64_t per = a.prefix[a.rows + 1];
  __syncthreads();
  const int64_t at = (int64_t)blockIdx.x * (kThreads / lanes) + tid / lanes;  // token * heads + head, below 2^27
  if (at >= (int64_t)a.tokens * a.heads) return;
  const int token = (int)at / a.heads, h = (int)at - token * a.heads;
  if (token >= starts[a.rows]) return;
  int lo = 0, hi = a.rows;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= token) lo = mid;
    else hi = mid;
  }
  const Row row = row_of(a, lo);
  const int node = token - row.start;
  if (node < 0 || node >= row.n) return;
  const bool in = 4 * x < a.dim;
  float o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0.f;
  const int kvh = a.by_group.quotient(h);
  if (row.tiles) {
    const int c = node * a.group + (h - kvh * a.group), block = c / a.qb, i = c - block * a.qb;  // below 2^27
    const int64_t s = a.prefix[lo] + ((int64_t)kvh * row.blocks + block) * (row.tiles + kStart);
    const int w0 = quotient(s + kStart, per), w1 = quotient(s + kStart + row.tiles - 1, per);
    if (w0 == w1) return;
    auto take = [&](int w, auto pieces) {
      constexpr int N = decltype(pieces)::value;
      float pm[N], pl[N];
      f32x4_t po[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const bool ok = w + k <= w1;
        const int64_t v = ok ? w + k : w;
        const float* sums = a.ws + (v * 2 + (v * per < s ? 1 : 0)) * partial_floats(a.qb, a.dim);  // after another in its run
        pm[k] = ok ? sums[(int64_t)a.qb * a.dim + 2 * i] : -INFINITY;
        pl[k] = ok ? sums[(int64_t)a.qb * a.dim + 2 * i + 1] : 0.f;
        po[k] = ok && in ? *(const f32x4_t*)(sums + (int64_t)i * a.dim + 4 * x) : f32x4_t{0, 0, 0, 0};
      }
      float top = m;
#pragma unroll
      for (int k = 0; k < N; ++k) top = fmaxf(top, pm[k]);
      const float ref = top == -INFINITY ? 0.f : top, f0 = fmaxf(__builtin_amdgcn_exp2f(m - ref), FLT_MIN);
      m = top;
      l *= f0;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] *= f0;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float f = fmaxf(__builtin_amdgcn_exp2f(pm[k] - ref), FLT_MIN);
        l += pl[k] * f;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += po[k][e] * f;
      }
    };
    int w = w0;
    if constexpr (MANY)
      for (; w + 3 < w1; w += 16) take(w, std::integral_constant<int, 16>());
    for (; w <= w1; w += 4) take(w, std::integral_constant<int, 4>());
  }
  const float f = m == -INFINITY ? 0.f : l == 0.f ? NAN : (a.v_scale ? a.v_scale[kvh] : 1.f) / l;
  const float v[4] = {o[0] * f, o[1] * f, o[2] * f, o[3] * f};
  if (in) store_values<4>(a.out, a.out_dtype, at * a.dim + 4 * x, v);
  if (a.lse && x == 0) a.lse[at] = (m + __builtin_amdgcn_logf(l)) * 0.69314718055994531f;
}

// A token's ancestors: one thread walks from each node to its root, by the parents of the row in LDS where they fit.  Bound by the deepest
// node's walk: 64 rows of 16 nodes 2.7 us, a tree of 4096 209, a chain of 513 82, of 4096 3077 (chains need no mask).
struct MaskArgs {
  const int32_t *starts, *parents, *positions;
  uint64_t* mask;
  int32_t* out;
  int rows, tokens, words;
};
constexpr int kMaskNodes = 4096;  // of a row in LDS
__global__ __launch_bounds__(kThreads) void mask_kernel(MaskArgs a) {
  __shared__ int sh[kMaskNodes];
  const int r = blockIdx.x, tid = threadIdx.x;
  const int s0 = r < a.rows ? min(max(a.starts[r], 0), a.tokens) : min(max(a.starts[a.rows], 0), a.tokens);
  if (r == a.rows) {  // padding: nothing is seen
    for (int t = s0 + tid; t < a.tokens; t += kThreads) {
      for (int w = 0; w < a.words; ++w) a.mask[(int64_t)t * a.words + w] = 0;
      if (a.out) a.out[t] = -1;
    }
    return;
  }
  const int n = min(max(a.starts[r + 1], s0), a.tokens) - s0;
  for (int i = tid; i < min(n, kMaskNodes); i += kThreads) sh[i] = a.parents[s0 + i];
  __syncthreads();
  for (int i = tid; i < n; i += kThreads) {
    int at = i, depth = 0;
    for (int w = i >> 6; w >= 0; --w) {
      uint64_t bits = 0;
      while (at >= 0 && at >> 6 == w) {  // parents come before their children: the words are met from the last on
        bits |= 1ull << (at & 63);
        const int p = at < kMaskNodes ? sh[at] : a.parents[s0 + at];
        at = p < at ? p : -1;
        ++depth;
      }
      if (w < a.words) a.mask[(int64_t)(s0 + i) * a.words + w] = bits;
    }
    for (int w = (i >> 6) + 1; w < a.words; ++w) a.mask[(int64_t)(s0 + i) * a.words + w] = 0;
    if (a.out) {
      const int p = a.positions ? a.positions[s0 + i] : i;
      a.out[s0 + i] = p < 0 ? -1 : p - i + depth - 1;
    }
  }
}

TreeKern kern(const mlxr_paged_cache* c, int q_dtype, int columns, int longest) {
  const bool f16 = q_dtype == MLXR_F16;
  if (c->dtype == MLXR_E4M3) return f16 ? kern_f16_e4m3(c->head_dim, columns, longest) : kern_bf16_e4m3(c->head_dim, columns, longest);
  return f16 ? kern_f16(c->head_dim, columns, longest) : kern_bf16(c->head_dim, columns, longest);
}

// A launch has fewer than 2^32 threads: the join at most 64 for each of tokens times heads, the kernel 512 for each 64 of them and
// for each row's kv heads.
constexpr int kMaxHeads = 1 << 26, kMaxRowHeads = 1 << 22;
// Threads of the join that share a token's head.
int join_lanes(int dim) {
  int lanes = 2;
  while (4 * lanes < dim) lanes *= 2;
  return lanes;
}

// How a call runs.
struct Plan {
  TreeKern k;
  bool cut;
  int64_t units;  // at most: (row, kv head, QB columns)
  int least;      // tiles of a run
  size_t bytes;   // of the workspace
};
constexpr size_t prefix_bytes(int rows) { return (size_t)(rows + 2 + 1) / 2 * 2 * sizeof(int64_t); }
// chain: no mask; needs no more workspace than with one.
Plan plan_of(const mlxr_paged_cache* c, int rows, int tokens, int heads, int width, int q_dtype, bool chain) {
  Plan p;
  const int group = heads / c->kv_heads;
  // on average, padding included; an eighth more than a block of columns is still taken as one
  int64_t columns = (int64_t)tokens * group / rows * 8 / 9;
  const int64_t held = (int64_t)width * c->page_size;
  // Little work (tiles of 16 columns by 64 tokens, for a CU) wants many workgroups rather than few reads of a tile: us, 256 columns and
  // 64, a chain of 513 over 600 (72), 32 heads and 8 kv heads, 54 and 41; 64 drafts of one row of 8192 (64) 45 and 41; 145 of 8 rows of up to 1806,
  // 8 heads and 2 (40) 40 and 31; but 64 drafts of 32 rows of 1000 (256) 81 and 98, of 8 rows of 8192 (512) 155 and 182.  Ragged rows in between lose a
  // little by it: 64 drafts of 16 rows of up to 2048 (170) 69 and 63.
  if ((double)tokens * group / 16 * c->kv_heads * ((held + 63) / 64) < 96.0 * device_cu_count()) columns = std::min<int64_t>(columns, 64);
  p.k = kern(c, q_dtype, (int)std::min<int64_t>(columns, 1 << 20), (int)held);
  p.units = ((int64_t)tokens * group / p.k.qb + rows) * c->kv_heads;
  int64_t tiles = (held + p.k.tok - 1) / p.k.tok;
  // Cut where the longest rows that the table holds are more than 3 tiles and 20 for each of a CU's units: what a launch without cuts
  // leaves idle while its longest unit ends grows with the row, the pieces and their join with the units.  us, cut and not, 16
  // drafts a row of 32 heads and 8 kv heads: one row (8 units) of 250 13.8 and 15.4, 8 rows of 250 21 and 16, of 1000 27 and 38; rows
  // spread over the lengths, 32 rows (256 units) of up to 500 29 and 25, of 2000 44 and 66, of 8192 119 and 234; 128 rows (1024 units) 59
  // and 48, 129 and 137, 383 and 485; of one length of 2000 32 rows 78 and 73, 128 rows of 1000 130 and 117, of 4096 423 and 409.
  // Rows that are mostly a chain have half as many tiles on average, and a cut would deal all of them: a prompt of 4096
  // (512 units) cut 498, not 276.
  if (chain && 2 * (int64_t)tokens > rows * held) tiles /= 2;
  const int64_t units = std::max((int64_t)tokens * group / p.k.qb, (int64_t)rows) * c->kv_heads;  // about
  p.cut = (tiles - 3) * device_cu_count() > 20 * units;
  // Few columns of a long row: runs of one tile would leave the join more pieces than it takes at once.  Its time goes with
  // tiles / run / 16, that of a run with its tiles: least together at about the root.  us, runs of one tile and
  // these, 4 drafts of one row, 8 heads and 2: of 10893 tokens (3) 33 and 22, of 32000 (6) 47 and 32.
  p.least = std::max(1, (int)std::sqrt((double)tiles / 13));
  p.bytes = p.cut ? prefix_bytes(rows) + (size_t)device_cu_count() * p.k.occ * 2 * partial_floats(p.k.qb, c->head_dim) * sizeof(float) : 0;
  return p;
}

int check_tree(const mlxr_paged_cache* c, int rows, int tokens, int heads, int width) {
  if (const int rc = check_cache(c)) return rc;
  if (rows < 0 || tokens < 0 || heads <= 0 || width <= 0) return set_error(MLXR_E_INVALID, "paged_tree_attention: bad sizes");
  if (heads % c->kv_heads) return set_error(MLXR_E_SHAPE, "heads must be a multiple of kv_heads");
  if (rows > kMaxRows) return set_error(MLXR_E_SHAPE, "paged_tree_attention: at most %d rows", kMaxRows);
  if ((int64_t)width * c->page_size > INT32_MAX - 1024) return set_error(MLXR_E_SHAPE, "paged_tree_attention: the table covers too many tokens");
  if ((int64_t)tokens * heads > kMaxHeads - (join_lanes(c->head_dim) > 32))
    return set_error(MLXR_E_SHAPE, "paged_tree_attention: at most %d tokens times heads", kMaxHeads - (join_lanes(c->head_dim) > 32));
  if ((int64_t)rows * c->kv_heads > kMaxRowHeads)
    return set_error(MLXR_E_SHAPE, "paged_tree_attention: at most %d rows times kv heads", kMaxRowHeads);
  return MLXR_OK;
}
int check_types(const mlxr_paged_cache* c, int q_dtype, int out_dtype) {
  if (q_dtype != MLXR_F16 && q_dtype != MLXR_BF16) return set_error(MLXR_E_INVALID, "invalid query dtype %d", q_dtype);
  if (c->dtype != MLXR_E4M3 && c->dtype != q_dtype) return set_error(MLXR_E_INVALID, "queries must have the cache's type");
  if (out_dtype != MLXR_F32 && out_dtype != MLXR_F16 && out_dtype != MLXR_BF16)
    return set_error(MLXR_E_INVALID, "invalid output dtype %d", out_dtype);
  return MLXR_OK;
}

}  // namespace
}  // namespace tree
}  // namespace mlxr

using namespace mlxr;
using namespace mlxr::tree;

extern "C" int mlxr_tree_mask(int rows, int tokens, const int32_t* starts_dev, const int32_t* parents_dev,
                              const int32_t* positions_dev, int words, int64_t* mask_dev, int32_t* positions_out_dev, void* stream) {
  if (rows < 0 || tokens < 0 || words <= 0) return set_error(MLXR_E_INVALID, "tree_mask: bad sizes");
  if (rows > kMaxRows || words > MLXR_TREE_MAX_WORDS)
    return set_error(MLXR_E_SHAPE, "tree_mask: at most %d rows and %d words", kMaxRows, MLXR_TREE_MAX_WORDS);
  if (tokens == 0) return MLXR_OK;
  if (!starts_dev || !parents_dev || !mask_dev) return set_error(MLXR_E_INVALID, "null buffer");
  MaskArgs a{starts_dev, parents_dev, positions_dev, (uint64_t*)mask_dev, positions_out_dev, rows, tokens, words};
  mask_kernel<<<(unsigned)(rows + 1), kThreads, 0, (hipStream_t)stream>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(MLXR_E_HIP, "tree_mask launch: %s", hipGetErrorString(e));
  return MLXR_OK;
}

extern "C" int mlxr_paged_tree_attention_workspace_size(const mlxr_paged_cache* cache, int rows, int tokens, int heads,
                                                        int table_width, int q_dtype, int out_dtype, size_t* bytes) {
  if (!bytes) return set_error(MLXR_E_INVALID, "null bytes");
  if (const int rc = check_tree(cache, rows, tokens, heads, table_width)) return rc;
  if (const int rc = check_types(cache, q_dtype, out_dtype)) return rc;
  *bytes = rows && tokens ? plan_of(cache, rows, tokens, heads, table_width, q_dtype, false).bytes : 0;
  return MLXR_OK;
}

extern "C" int mlxr_paged_tree_attention(const mlxr_paged_cache* cache, int rows, int tokens, int heads, const void* q_dev,
                                         int q_dtype, int64_t q_token_stride, int64_t q_head_stride, const int32_t* table_dev,
                                         int64_t table_stride, int table_width, const int32_t* lens_dev, const int32_t* starts_dev,
                                         const int64_t* mask_dev, int words, float scale, void* out_dev, int out_dtype,
                                         float* lse_dev, void* workspace_dev, size_t workspace_bytes, void* stream) {
  if (const int rc = check_tree(cache, rows, tokens, heads, table_width)) return rc;
  if (const int rc = check_types(cache, q_dtype, out_dtype)) return rc;
  if (mask_dev && (words <= 0 || words > MLXR_TREE_MAX_WORDS))
    return set_error(MLXR_E_SHAPE, "paged_tree_attention: a mask has 1 to %d words", MLXR_TREE_MAX_WORDS);
  if (tokens == 0) return MLXR_OK;
  if (rows == 0) return set_error(MLXR_E_INVALID, "paged_tree_attention: tokens without rows");
  if (!q_dev || !table_dev || !lens_dev || !starts_dev || !out_dev) return set_error(MLXR_E_INVALID, "null buffer");
  if (q_token_stride % 8 || q_head_stride % 8 || (((uintptr_t)q_dev | (uintptr_t)out_dev | (uintptr_t)workspace_dev) & 15))
    return set_error(MLXR_E_SHAPE, "paged_tree_attention: query rows, output and workspace must start at multiples of 16 bytes");
  const Plan p = plan_of(cache, rows, tokens, heads, table_width, q_dtype, !mask_dev);
  if (workspace_bytes < p.bytes || (p.bytes && !workspace_dev))
    return set_error(MLXR_E_INVALID, "paged_tree_attention: the workspace is smaller than mlxr_paged_tree_attention_workspace_size");
  const int es = cache->dtype == MLXR_E4M3 ? 1 : 2;
  Args a{};
  a.k = (const uint8_t*)cache->k_dev, a.v = (const uint8_t*)cache->v_dev;
  a.k_scale = cache->k_scale_dev, a.v_scale = cache->v_scale_dev;
  a.k_page = cache->k_stride[0] * es, a.k_head = cache->k_stride[1] * es, a.k_token = cache->k_stride[2] * es;
  a.v_page = cache->v_stride[0] * es, a.v_head = cache->v_stride[1] * es, a.v_token = cache->v_stride[2] * es;
  a.q = (const uint16_t*)q_dev, a.q_token = q_token_stride, a.q_head = q_head_stride;
  a.table = table_dev, a.table_stride = table_stride, a.lens = lens_dev, a.starts = starts_dev;
  a.mask = (const uint64_t*)mask_dev, a.words = words;
  a.out = out_dev, a.lse = lse_dev, a.out_dtype = out_dtype;
  a.rows = rows, a.tokens = tokens, a.heads = heads, a.kv_heads = cache->kv_heads, a.group = heads / cache->kv_heads;
  a.dim = cache->head_dim, a.page = cache->page_size, a.pages = cache->num_pages, a.width = table_width;
  a.qb = p.k.qb, a.tok = p.k.tok, a.step = p.k.tok % a.page == 0 ? p.k.tok / a.page : 0;
  a.by_page = Divisor(a.page), a.by_group = Divisor(a.group);
  a.scale = scale * 1.44269504088896341f;
  const hipStream_t st = (hipStream_t)stream;
  // LDS: two tiles, the rows' prefix, the wavefronts' sums and words; the limit is raised to all that a workgroup may use, once on each device
  const int lds = p.k.lds + (rows + 1 + 16) * (int)sizeof(int64_t), most = (int)device_lds_limit();
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return set_error(MLXR_E_HIP, "paged_tree_attention: %s", hipGetErrorString(e));
  std::atomic<int>& residents = p.k.residents[dev & 63];
  int occ = residents.load(std::memory_order_acquire);
  if (!occ) {
    e = hipFuncSetAttribute(p.k.fn, hipFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e == hipSuccess) e = hipOccupancyMaxActiveBlocksPerMultiprocessor(&occ, p.k.fn, p.k.threads, p.k.lds + 1024);
    if (e != hipSuccess) return set_error(MLXR_E_HIP, "paged_tree_attention: %s", hipGetErrorString(e));
    occ = std::max(1, std::min(occ, p.k.occ));
    residents.store(occ, std::memory_order_release);
  }
  int64_t grid = p.units;
  if (p.cut) {
    grid = (int64_t)occ * device_cu_count();
    a.workers = (int)grid, a.least = p.least;
    a.prefix = (int64_t*)workspace_dev, a.ws = (float*)((uint8_t*)workspace_dev + prefix_bytes(rows));
  }
  void* args[] = {&a};
  e = hipLaunchKernel(p.k.fn, dim3((unsigned)grid), dim3(p.k.threads), args, (size_t)lds, st);
  if (e == hipSuccess && p.cut) {
    const int lanes = join_lanes(a.dim);
    const unsigned blocks = (unsigned)(((int64_t)tokens * heads * lanes + kThreads - 1) / kThreads);
    // A few workgroups wait for memory: more at once, though fewer fit a CU.  us of a call, 4 and 16: 8 drafts of one row of 1000 16.8
    // and 14.6, 76 of 3 rows of up to 7391, 4 heads of 256 47 and 41; 64 of 8 rows of 8192 156 and 157.
    const auto join = blocks <= 2 * (unsigned)device_cu_count() ? join_kernel<true> : join_kernel<false>;
    join<<<blocks, kThreads, (rows + 1) * sizeof(int), st>>>(a, lanes);
    e = hipGetLastError();
  }
  if (e != hipSuccess) return set_error(MLXR_E_HIP, "paged_tree_attention launch: %s", hipGetErrorString(e));
  return MLXR_OK;
}
