// Tokens of a paged cache moved from slots to slots, in every layer's stores by one launch: the accepted path of a
// drafted tree together behind its context (accept), and rows copied to other rows (copy, fork).  What a token holds is
// copied bit for bit, so one kernel serves every cache type: 16 bytes a lane.
//
// Bound by memory: each byte moved is read once and written once.  64 rows of Llama-3-8B's 32 layers (8 heads of 128, bf16),
// paths of up to 6 of 16 drafted tokens (37 MB read and written): 10 us, 3.7 TB/s; a row of 1501 tokens to three others
// (787 MB): 157 us, 5 TB/s.
#include "mfma16.h"
#include "paged_internal.h"

namespace mlxr {
namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 8;  // 16-byte pieces of a thread on their way at once

struct Stores {
  uint8_t* at[2];  // keys, values
  int64_t layer[2], page[2], head[2], token[2];  // strides, bytes
  int kv_heads, layers, slots_end, pieces;       // pieces: of 16 bytes of a head's row
  Divisor by_page;
};

// Byte offset of a slot in a store.
__device__ __forceinline__ int64_t slot_offset(const Stores& s, int side, int slot) {
  const int pg = s.by_page.quotient(slot);
  return (int64_t)pg * s.page[side] + (int64_t)(slot - pg * (int)s.by_page.d) * s.token[side];
}

struct AcceptArgs {
  Stores s;
  const int32_t* table;
  int64_t table_stride;
  const int32_t *lens, *starts, *path, *counts;
  int64_t path_stride;
  int32_t* lens_out;
  int depth, width, items;  // items: of a row, (side, layer, head, piece)
  Divisor by_store, by_head;  // items of one layer's store, of a head
};

// Row blockIdx.y, pieces blockIdx.x * 256 ..: its drafted tokens lie at positions c .. c + n - 1, c = lens - n; node
// path[j] moves to c + j.  The path ascends, so path[j] >= j and a source of a later move is never an earlier move's
// destination: a thread that reads kAhead pieces, writes them and goes on sees every token before it is overwritten, and
// no other thread touches its pieces.  A workgroup first makes the list of the row's moves in LDS (path, then table: two
// latencies), 256 path entries at a time.
__global__ __launch_bounds__(kThreads) void accept_kernel(AcceptArgs a) {
  __shared__ int64_t move[2][2][kThreads];  // [side][source, destination]
  __shared__ int stop, shared_first;
  const int r = blockIdx.y, tid = threadIdx.x;
  const int len = a.lens[r], n = max(a.starts[r + 1] - a.starts[r], 0), context = len - n;
  const int most = min(max(a.counts[r], 0), min(a.depth, n));
  const int32_t* path = a.path + (int64_t)r * a.path_stride;
  const int item = blockIdx.x * kThreads + tid;
  const int store = a.by_store.quotient(min(item, a.items - 1)), in_store = item - store * (int)a.by_store.d;
  const int side = store >= a.s.layers, layer = store - side * a.s.layers;
  const int head = a.by_head.quotient(in_store), piece = in_store - head * (int)a.by_head.d;
  uint8_t* at = a.s.at[side] + (int64_t)layer * a.s.layer[side] + (int64_t)head * a.s.head[side] + 16 * piece;
  int kept = 0;
  for (int j0 = 0; j0 < most; j0 += kThreads) {
    if (tid == 0) stop = min(most, j0 + kThreads), shared_first = kThreads;
    __syncthreads();
    const int j = j0 + tid;
    int node = -1;
    if (j < most) {
      node = path[j];
      const int before = j ? path[j - 1] : -1;
      if (node <= before || node >= n) atomicMin(&stop, j);
      else if (node > j) atomicMin(&shared_first, tid);  // from here on all move
    }
    __syncthreads();
    const int end = stop - j0, first = shared_first;  // the moves of this part: first .. end - 1
    if (tid < end && tid >= first) {
      int slot[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int pos = context + (k ? j : node), pg = pos < 0 ? -1 : a.s.by_page.quotient(pos);
        const int id = pos < 0 || pg >= a.width ? -1 : a.table[(int64_t)r * a.table_stride + pg];
        const int64_t at_slot = (int64_t)id * (int)a.s.by_page.d + (pos - pg * (int)a.s.by_page.d);
        slot[k] = id < 0 || at_slot >= a.s.slots_end ? -1 : (int)at_slot;
      }
      const bool ok = slot[0] >= 0 && slot[1] >= 0;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int k = 0; k < 2; ++k) move[x][k][tid] = ok ? slot_offset(a.s, x, slot[k]) : -1;
    }
    __syncthreads();
    if (item < a.items) {
      for (int m = first; m < end; m += kAhead) {
        u32x4_t v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int64_t from = m + k < end ? move[side][0][m + k] : -1;
          v[k] = *(const u32x4_t*)(at + (from < 0 ? 0 : from));  // of the first slot where there is no move: not used
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int64_t to = m + k < end ? move[side][1][m + k] : -1;
          if (to >= 0) *(u32x4_t*)(at + to) = v[k];
        }
      }
    }
    kept = stop;
    __syncthreads();
    if (kept < min(most, j0 + kThreads)) break;
  }
  if (blockIdx.x == 0 && tid == 0) a.lens_out[r] = max(context + kept, 0);
}

struct CopyArgs {
  Stores s;
  const int32_t *src, *dst;  // slots; a fork has positions and rows instead of src
  const int32_t *sources, *starts, *positions, *table;
  int64_t table_stride;
  int tokens, rows, width;
  int heads_first;  // neighbouring tokens of a head lie side by side
  Divisor by_row, by_head;  // pieces of a head; of the 16 tokens of a head, or of all heads of a token
};

constexpr int kTokens = 16;  // of a workgroup

// Slot that token t's copy comes from: given, or its position's in the row that its own row is copied from.
__device__ __forceinline__ int source_of(const CopyArgs& a, int t) {
  if (a.src) return a.src[t];
  if (t >= a.starts[a.rows]) return -1;
  int lo = 0, hi = a.rows;  // the last row that starts at or before t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.starts[mid] <= t) lo = mid;
    else hi = mid;
  }
  const int from = a.sources[lo], pos = a.positions[t];
  if (from < 0 || from >= a.rows || from == lo || pos < 0) return -1;
  const int pg = a.s.by_page.quotient(pos);
  const int id = pg < a.width ? a.table[(int64_t)from * a.table_stride + pg] : -1;
  const int64_t slot = (int64_t)id * (int)a.s.by_page.d + (pos - pg * (int)a.s.by_page.d);
  return id < 0 || slot >= a.s.slots_end ? -1 : (int)slot;
}

// 16 tokens of one layer's keys or values.  Neighbouring lanes take neighbouring bytes in either memory order.
__global__ __launch_bounds__(kThreads) void copy_kernel(CopyArgs a) {
  __shared__ int64_t move[2][kTokens];
  const int tid = threadIdx.x, t0 = blockIdx.x * kTokens;
  const int side = blockIdx.y >= (unsigned)a.s.layers, layer = blockIdx.y - side * a.s.layers;
  if (tid < kTokens) {
    const int t = t0 + tid;
    int from = -1, to = -1;
    if (t < a.tokens) to = a.dst[t], from = source_of(a, t);
    const bool ok = from >= 0 && from < a.s.slots_end && to >= 0 && to < a.s.slots_end;
    move[0][tid] = ok ? slot_offset(a.s, side, from) : -1;
    move[1][tid] = ok ? slot_offset(a.s, side, to) : -1;
  }
  __syncthreads();
  uint8_t* base = a.s.at[side] + (int64_t)layer * a.s.layer[side];
  const int items = kTokens * a.s.kv_heads * a.s.pieces;
  for (int i0 = tid; i0 < items; i0 += kThreads * kAhead) {
    u32x4_t v[kAhead];
    int64_t to[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + k * kThreads, row = a.by_row.quotient(i), piece = i - row * (int)a.by_row.d;
      const int outer = a.by_head.quotient(i), inner = row - outer * (a.heads_first ? kTokens : a.s.kv_heads);
      const int t = a.heads_first ? inner : outer, head = a.heads_first ? outer : inner;
      const int64_t from = i < items ? move[0][t & (kTokens - 1)] : -1, in_head = (int64_t)head * a.s.head[side] + 16 * piece;
      to[k] = from < 0 ? -1 : move[1][t & (kTokens - 1)] + in_head;
      v[k] = *(const u32x4_t*)(base + (from < 0 ? 0 : from + in_head));
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (to[k] >= 0) *(u32x4_t*)(base + to[k]) = v[k];
  }
}

int stores_of(const mlxr_paged_cache* c, int layers, int64_t k_layer, int64_t v_layer, Stores* s) {
  if (const int rc = check_cache(c)) return rc;
  const int es = c->dtype == MLXR_E4M3 ? 1 : 2;
  if (layers <= 0) return set_error(MLXR_E_INVALID, "cache sizes must be positive");
  if (layers > 1 && (k_layer < 0 || v_layer < 0 || k_layer * es % 16 || v_layer * es % 16))
    return set_error(MLXR_E_SHAPE, "cache strides must be multiples of 16 bytes");
  const int pieces = c->head_dim * es / 16;
  if ((int64_t)2 * layers * c->kv_heads * pieces > INT32_MAX / kTokens || 2 * (int64_t)layers > 65535)
    return set_error(MLXR_E_SHAPE, "too many layers and heads");
  *s = Stores{{(uint8_t*)c->k_dev, (uint8_t*)c->v_dev},
              {layers > 1 ? k_layer * es : 0, layers > 1 ? v_layer * es : 0},
              {c->k_stride[0] * es, c->v_stride[0] * es},
              {c->k_stride[1] * es, c->v_stride[1] * es},
              {c->k_stride[2] * es, c->v_stride[2] * es},
              c->kv_heads, layers, c->num_pages * c->page_size, pieces, Divisor(c->page_size)};
  return MLXR_OK;
}

int launch_copy(CopyArgs& a, const mlxr_paged_cache* c, const char* what, hipStream_t stream) {
  a.heads_first = c->k_stride[2] < c->k_stride[1];
  a.by_row = Divisor(a.s.pieces);
  a.by_head = Divisor(a.s.pieces * (a.heads_first ? kTokens : a.s.kv_heads));
  const dim3 grid((unsigned)((a.tokens + kTokens - 1) / kTokens), 2 * (unsigned)a.s.layers);
  copy_kernel<<<grid, kThreads, 0, stream>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(MLXR_E_HIP, "%s launch: %s", what, hipGetErrorString(e));
  return MLXR_OK;
}

constexpr int kMaxCopied = 1 << 27;  // tokens of a launch, whose threads have 32 bits

}  // namespace
}  // namespace mlxr

using namespace mlxr;

extern "C" int mlxr_paged_accept(const mlxr_paged_cache* cache, int layers, int64_t k_layer_stride, int64_t v_layer_stride,
                                 int rows, const int32_t* table_dev, int64_t table_stride, int table_width,
                                 const int32_t* lens_dev, const int32_t* starts_dev, const int32_t* path_dev,
                                 int64_t path_stride, int depth, const int32_t* counts_dev, int32_t* lens_out_dev,
                                 void* stream) {
  AcceptArgs a{};
  if (const int rc = stores_of(cache, layers, k_layer_stride, v_layer_stride, &a.s)) return rc;
  if (rows < 0 || depth < 0 || table_width <= 0) return set_error(MLXR_E_INVALID, "paged_accept: bad sizes");
  if (rows > MLXR_PAGED_MAX_ROWS) return set_error(MLXR_E_SHAPE, "paged_accept: at most %d rows", MLXR_PAGED_MAX_ROWS);
  if (rows == 0) return MLXR_OK;
  if (!table_dev || !lens_dev || !starts_dev || (depth && !path_dev) || !counts_dev || !lens_out_dev)
    return set_error(MLXR_E_INVALID, "null buffer");
  if (lens_out_dev == lens_dev) return set_error(MLXR_E_INVALID, "paged_accept: lens_out must not be lens");
  if ((int64_t)table_width * cache->page_size > INT32_MAX)
    return set_error(MLXR_E_SHAPE, "paged_accept: the table covers too many tokens");
  a.table = table_dev, a.table_stride = table_stride, a.width = table_width;
  a.lens = lens_dev, a.starts = starts_dev, a.path = path_dev, a.path_stride = path_stride, a.counts = counts_dev;
  a.lens_out = lens_out_dev, a.depth = depth;
  const int store = cache->kv_heads * a.s.pieces;
  a.items = 2 * layers * store;
  a.by_store = Divisor(store), a.by_head = Divisor(a.s.pieces);
  accept_kernel<<<dim3((unsigned)((a.items + kThreads - 1) / kThreads), (unsigned)rows), kThreads, 0, (hipStream_t)stream>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(MLXR_E_HIP, "paged_accept launch: %s", hipGetErrorString(e));
  return MLXR_OK;
}

extern "C" int mlxr_paged_copy(const mlxr_paged_cache* cache, int layers, int64_t k_layer_stride, int64_t v_layer_stride,
                               int tokens, const int32_t* src_dev, const int32_t* dst_dev, void* stream) {
  CopyArgs a{};
  if (const int rc = stores_of(cache, layers, k_layer_stride, v_layer_stride, &a.s)) return rc;
  if (tokens < 0) return set_error(MLXR_E_INVALID, "paged_copy: tokens must not be negative");
  if (tokens == 0) return MLXR_OK;
  if (!src_dev || !dst_dev) return set_error(MLXR_E_INVALID, "null buffer");
  if (tokens > kMaxCopied) return set_error(MLXR_E_SHAPE, "paged_copy: at most %d tokens", kMaxCopied);
  a.src = src_dev, a.dst = dst_dev, a.tokens = tokens;
  return launch_copy(a, cache, "paged_copy", (hipStream_t)stream);
}

extern "C" int mlxr_paged_fork(const mlxr_paged_cache* cache, int layers, int64_t k_layer_stride, int64_t v_layer_stride,
                               int rows, const int32_t* table_dev, int64_t table_stride, int table_width,
                               const int32_t* sources_dev, const int32_t* starts_dev, const int32_t* slots_dev,
                               const int32_t* positions_dev, int tokens, void* stream) {
  CopyArgs a{};
  if (const int rc = stores_of(cache, layers, k_layer_stride, v_layer_stride, &a.s)) return rc;
  if (rows < 0 || tokens < 0 || table_width <= 0) return set_error(MLXR_E_INVALID, "paged_fork: bad sizes");
  if (rows == 0 || tokens == 0) return MLXR_OK;
  if (!table_dev || !sources_dev || !starts_dev || !slots_dev || !positions_dev) return set_error(MLXR_E_INVALID, "null buffer");
  if (tokens > kMaxCopied) return set_error(MLXR_E_SHAPE, "paged_fork: at most %d tokens", kMaxCopied);
  a.dst = slots_dev, a.sources = sources_dev, a.starts = starts_dev, a.positions = positions_dev;
  a.table = table_dev, a.table_stride = table_stride, a.width = table_width, a.rows = rows, a.tokens = tokens;
  return launch_copy(a, cache, "paged_fork", (hipStream_t)stream);
}
