// Attention of the drafted tokens of many requests over a paged key-value cache.
//
//   o[i,h] = sum_t p_t v[t] / sum_t p_t,   p_t = exp(scale q[i,h] . k[t] - m),   m the running maximum
//
// for each drafted token (node) i of a row and head h, t over the row's cached tokens before its drafts and over the
// nodes that i's mask names.  The (node, head) pairs of a kv head are columns of the matrix instructions, QB of them a
// workgroup, so a key or value is read once for QB of them:
//   S^T[tokens, columns] = K Q^T       K from LDS, Q in registers for the whole row
//   O^T[dim, columns]   += V^T P^T     V^T by the transposing read of LDS, P from S^T without leaving the registers
// Which token an element of the second product's 32 is, is free: lane group g's eight are tokens 4 g .. 4 g + 3 of two
// neighbouring 16 x 16 tiles of S^T, as the first product leaves them.  P enters in 16-bit parts that add up to it, as in decode
// attention and for every output type: bf16 three, all 24 bits; f16 (and the values of an e4m3 cache, exact in f16) two, 22 bits.
// A part takes as many matrix instructions as the first product.  us, with a bf16 cache two parts (16 bits) and these: 16 drafts of 16
// ragged rows of up to 8192 73 and 76, a chain of 513 over 6001 112 and 132; with an e4m3 cache one (11 bits) and these: 64 drafts
// of 8 ragged rows of up to 16384 153 and 176.  16-bit outputs have the bits of fp32 ones, rounded once.
//
// A tile of TOK tokens goes memory -> registers -> LDS, one tile ahead: while tile t is multiplied, t + 1 is on its way to
// registers; it is written to the other half of LDS before the tile's one barrier.
//
// What bounds it: few columns, memory (16 drafts of 32 rows of 8192, 32 heads and 8 kv heads of 128, bf16: 220 us, 4.9 TB/s); many
// columns, the vector unit's work on each score beside the matrix unit's two products (64 drafts of 8 rows of 16384, 64 heads, e4m3
// cache: 388 us, 0.71 PFLOP/s; a chain of 513 over 6001 tokens 0.39); a few rows, the launches and the start of each
// workgroup (8 drafts of one row of 1000 14.5 us).
//
// The tiles of all (row, kv head, QB columns) are dealt to the workgroups of a launch that fills the device in equal
// contiguous runs; a run that covers all of its columns' tiles writes the output, others leave (m, sum, unnormalized o) in
// the workspace, at most two a workgroup, and a second launch joins them.  Short rows, or many (plan_of): a workgroup for
// each (row, kv head, QB columns).
//
// A chain's block of columns ends with its last node's token, and what a wavefront's columns all see takes no mask, what they all do
// not no products: a chain of 513 over 6001 tokens 139 -> 136 us, of 513 alone 34 -> 23, of 4096 over 400 609 -> 317.
#pragma once
#include <cfloat>
#include <type_traits>

#include "paged_attn.h"

namespace mlxr {
namespace tree {

using paged::load_words;
using paged::store_values;
using paged::widen;

constexpr int kThreads = 256;  // of the join and the masks
constexpr int kMaxRows = MLXR_PAGED_MAX_ROWS;
// Tiles that the start and the end of a row's columns (queries, outputs or partial sums) are counted for in the deal.  us at 0, 2, 4 and 8:
// 64 drafts of 8 ragged rows of up to 16384, e4m3, 206, 184, 179 and 184; a chain of 513 over 6001 138, 135, 136 and 138; 16 drafts of 16
// ragged rows of up to 8192 85, 77, 75 and 76.
constexpr int kStart = 4;

struct Args {
  const uint8_t *k, *v;  // element addresses in bytes
  const float *k_scale, *v_scale;
  int64_t k_head, v_head, k_page, k_token, v_page, v_token;  // strides, bytes
  const uint16_t* q;
  int64_t q_token, q_head;  // elements
  const int32_t* table;
  int64_t table_stride;
  const int32_t *lens, *starts;
  const uint64_t* mask;  // or null: a chain
  int words;
  void* out;
  float* lse;
  float* ws;        // partial sums of cut runs; null: not cut
  int64_t* prefix;  // [rows + 1] tiles before each row, then tiles of a workgroup, for the join
  int rows, tokens, heads, kv_heads, group;
  int dim, page, pages, width, out_dtype, qb, tok;
  int step;  // pages of a tile where they are whole, else 0
  Divisor by_page, by_group;
  int workers, least;  // of a cut launch; a run is at least so many tiles
  float scale;  // times log2(e)
};

// A row: its drafted tokens are n tokens from `start` on, the first of those behind its context; starts may go past the listed
// tokens (page_resize lists no more than it is given places for), its len cached ones hold the others too.
struct Row {
  int start, n, len, context, blocks, tiles;
};
__device__ __forceinline__ Row row_of(const Args& a, int r) {
  Row w;
  const int64_t most = (int64_t)a.width * a.page;
  const int u0 = max(a.starts[r], 0), u1 = max(a.starts[r + 1], u0), s0 = min(u0, a.tokens), s1 = min(u1, a.tokens);
  const int len = max(a.lens[r], 0);
  w.start = s0;
  w.n = s1 - s0;
  w.context = len - (u1 - u0);  // may be negative: the first nodes are then not in the cache
  w.len = len > most ? (int)most : len;
  w.blocks = (int)(((int64_t)w.n * a.group + a.qb - 1) / a.qb);
  w.tiles = (w.len + a.tok - 1) / a.tok;
  return w;
}

// Floats of a cut run's partial sums: QB rows of dim, then m and sum of each.
__host__ __device__ constexpr int partial_floats(int qb, int dim) { return qb * dim + 2 * qb; }

// n / d, d > 0; most calls stay within 32 bits, whose division takes a tenth of the instructions.
__device__ __forceinline__ int quotient(int64_t n, int64_t d) {
  return n < (1ll << 31) && d < (1ll << 31) ? (int)((uint32_t)n / (uint32_t)d) : (int)(n / d);
}

// What a node sees of its row's nodes: 64 bits from bit `at` on, 1s before the nodes (at < 0).  The first two words stay in
// registers; no mask: bits 0 .. i.
struct Seen {
  uint64_t w[2];
  __device__ __forceinline__ void start(const Args& a, int token) {
    const uint64_t* mask = a.mask + (int64_t)token * a.words;
    w[0] = a.mask ? mask[0] : 0;
    w[1] = a.mask && a.words > 1 ? mask[1] : 0;
  }
  __device__ __forceinline__ uint64_t word(const Args& a, int token, int k) const {
    return k < 0 ? ~0ull : k < 2 ? (k ? w[1] : w[0]) : k < a.words ? a.mask[(int64_t)token * a.words + k] : 0ull;
  }
  __device__ __forceinline__ uint64_t bits(const Args& a, int token, int i, int at) const {
    if (!a.mask) {
      const int more = i - at;  // the last bit that counts
      return more < 0 ? 0ull : more >= 63 ? ~0ull : (2ull << more) - 1;
    }
    const int k = at >> 6, s = at & 63;
    const uint64_t lo = word(a, token, k);
    return s ? lo >> s | word(a, token, k + 1) << (64 - s) : lo;
  }
};

// Two weights in 16-bit parts that add up to them (f16: the second rounded), none negative.  FLOOR, for caches whose values may be
// infinite: nor a later one 0 where the first is not, so that an infinite value gives an infinite output as a weight in one piece
// does, not NaN.  Parts of a weight of 0 are all 0: what a column does not see adds nothing to it, whatever its value.
template <bool P16, bool FLOOR>
__device__ __forceinline__ void split_parts(float p0, float p1, uint32_t (&out)[P16 ? 2 : 3]) {
  auto floor2 = [&](uint32_t w) { return FLOOR ? paged::pair_max(w, paged::pair_min(out[0], P16 ? 0x00010001u : 0x00800080u)) : w; };
  if constexpr (P16) {
    typedef __attribute__((ext_vector_type(2))) float F;
    typedef __attribute__((ext_vector_type(2))) _Float16 H;
    const H hi = __builtin_bit_cast(H, __builtin_amdgcn_cvt_pkrtz(p0, p1));
    float minus = -1.f;
    asm("" : "+s"(minus));  // not known to the compiler, which would widen hi and subtract: one instruction takes it as it is
    out[0] = __builtin_bit_cast(uint32_t, hi);
    out[1] = floor2(__builtin_bit_cast(uint32_t, __builtin_convertvector((F{__builtin_fmaf(hi[0], minus, p0), __builtin_fmaf(hi[1], minus, p1)}), H)));
  } else {
#pragma unroll
    for (int n = 0; n < 3; ++n) {  // each the upper half of what is left; the last holds all of it
      const uint32_t b0 = __builtin_bit_cast(uint32_t, p0), b1 = __builtin_bit_cast(uint32_t, p1);
      const uint32_t w = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
      out[n] = n ? floor2(w) : w;
      p0 -= __builtin_bit_cast(float, b0 & 0xffff0000u);
      p1 -= __builtin_bit_cast(float, b1 & 0xffff0000u);
    }
  }
}

// A 16-bit value that is infinite or NaN; a word of two with those cleared.
template <bool F16>
__device__ __forceinline__ bool odd_half(uint32_t h) {
  constexpr uint32_t E = F16 ? 0x7c00u : 0x7f80u;
  return (h & E) == E;
}
template <bool F16>
__device__ __forceinline__ bool odd_word(uint32_t w) {
  return odd_half<F16>(w) || odd_half<F16>(w >> 16);
}
template <bool F16>
__device__ __forceinline__ uint32_t clean2(uint32_t w) {
  if (odd_half<F16>(w)) w &= 0xffff0000u;
  if (odd_half<F16>(w >> 16)) w &= 0x0000ffffu;
  return w;
}

// DT: 64, 128 or 256, at least head_dim.  W: wavefronts.  CW: columns of a wavefront, by 16.  TOK: tokens of a tile (32, 64).  OCC: workgroups
// that a CU's registers and LDS hold.
template <bool F16, bool F8, int DT, int W, int CW, int TOK, int OCC>
struct Kern {
  static constexpr bool P16 = F16 || F8;                      // the second product's type, f16 or else bf16
  static constexpr int PARTS = P16 ? 2 : 3;                   // of a weight
  static constexpr int THREADS = 64 * W, QB = 16 * CW * W;
  static constexpr int NT = TOK / 16, KT = TOK / 32, KS = DT / 32, ND = DT / 16;
  static constexpr int CH = DT / 8;                           // 16-byte pieces of a row in LDS
  static constexpr int CG = F8 ? DT / 16 : DT / 8;            // and in memory
  static constexpr int R = THREADS / TOK;                     // threads that bring a token's key and value to LDS
  static constexpr int LR = R == 4 ? 2 : 3;
  static_assert(CG % R == 0, "a token's threads share its pieces evenly");
  static constexpr int NL = CG / R;                           // loads of a thread, tile and store
  static constexpr int AHEAD = F8 || CW == 1 ? 3 : 2;         // steps that reads of LDS go before their products
  static constexpr int STORE = TOK * DT * 2;                  // bytes of a tile's keys or values in LDS
  static constexpr int LDS = 4 * STORE;
  // The reference that weights are relative to follows the maximum only when that is 2^SLACK above it: weights are at most
  // 2^(SHIFT + SLACK), below f16's largest number, and down to 2^-22 of that they stay normal ones.
  static constexpr float SHIFT = P16 ? 8.f : 0.f, SLACK = 7.f;
  static constexpr float UNSHIFT = P16 ? 0x1p-8f : 1.f;

  // Places in LDS: 16-byte piece c of token t's key, 16 dims (32 bytes) p of its value.  What 16 lanes access at once lies in
  // different banks: 16 tokens' piece of an operand's read, four tokens' dims of the transposing read (eight for two lane
  // groups), and R pieces of 16 / R tokens of a write.
  static __device__ __forceinline__ int key_place(int t, int c) {
    constexpr int N = CH >= 16 ? 4 : 3;  // bits of a piece's place within 256 bytes of banks; shorter rows are two to those
    const int u = CH >= 16 ? t : t >> 1;
    int swap;
    if constexpr (!F8) swap = (u & ((1 << (N - LR)) - 1)) << LR | (u >> (N - LR) & (R - 1));
    else if constexpr (N - LR == 1) swap = u & ((1 << N) - 1);  // e4m3: of the two pieces that one widens to, every other at once
    else swap = (u & 1) | (u >> 2 & 3) << 1 | (u >> 1 & 1) << 3;
    return t * DT * 2 + (c ^ swap) * 16;
  }
  static __device__ __forceinline__ int value_place(int t, int p) {
    const int swap = ND < 8 ? (t & 2) | (t >> 2 & 1) : R == 8 ? (t & 1) << 2 | (t >> 1 & 3) : (t & 3) << 1 | (t >> 2 & 1);
    return t * DT * 2 + (p ^ swap) * 32;
  }
};

template <bool F16, bool F8, int DT, int W, int CW, int TOK, int OCC>
__global__ __launch_bounds__(64 * W, OCC) void tree_kernel(Args a) {
  using T = Kern<F16, F8, DT, W, CW, TOK, OCC>;
  constexpr int THREADS = T::THREADS, NT = T::NT, KT = T::KT, KS = T::KS, ND = T::ND, NL = T::NL, PARTS = T::PARTS;
  constexpr bool P16 = T::P16;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, col = lane & 15;

  const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;

  // ---- this workgroup's run of tiles
  int64_t* pre = (int64_t*)(lds + T::LDS);  // [rows + 1] before each row: tiles, or (not cut) blocks of columns
  int64_t* part = pre + a.rows + 1;         // [W]
  int* flag = (int*)(part + W);             // [2][W] of the tiles' wavefronts
  const bool cut = a.ws != nullptr;
  // a unit of the deal: kStart places, then its tiles
  auto weight = [&](const Row& w) { return (int64_t)a.kv_heads * w.blocks * (!cut ? 1 : w.tiles ? w.tiles + kStart : 0); };
  const int behind = min(max(a.starts[a.rows], 0), a.tokens);  // the first token behind the rows
  {
    const int per_thread = (a.rows + THREADS - 1) / THREADS;
    const int r0 = min(tid * per_thread, a.rows), r1 = min(r0 + per_thread, a.rows);
    int64_t n = 0;
    for (int r = r0; r < r1; ++r) n += weight(row_of(a, r));
    int64_t sum = n;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int64_t v = __shfl_up(sum, d);
      if (lane >= d) sum += v;
    }
    if (lane == 63) part[wave] = sum;
    __syncthreads();
    int64_t at = sum - n;
    for (int w = 0; w < wave; ++w) at += part[w];
    if (tid == THREADS - 1) pre[a.rows] = at + n;
    for (int r = r0; r < r1; ++r) {
      pre[r] = at;
      if (r + 1 < r1) at += weight(row_of(a, r));  // a thread of one row does not ask for it again
    }
    __syncthreads();
  }
  // tokens behind the last row's: zeros
  {
    const int64_t first = (int64_t)behind * a.heads * a.dim, count = (int64_t)(a.tokens - behind) * a.heads * a.dim;
    const int64_t id = (int64_t)blockIdx.x * THREADS + tid, step = (int64_t)gridDim.x * THREADS;
    for (int64_t i = id; i < count / 8; i += step) {
      const float z[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      store_values<8>(a.out, a.out_dtype, first + 8 * i, z);
    }
    if (a.lse)
      for (int64_t i = id; i < (int64_t)(a.tokens - behind) * a.heads; i += step) a.lse[(int64_t)behind * a.heads + i] = -INFINITY;
  }
  const int64_t total = pre[a.rows];
  const int64_t per = cut ? max((total + a.workers - 1) / a.workers, (int64_t)a.least) : 1;
  if (cut && blockIdx.x == 0) {
    for (int r = tid; r <= a.rows; r += THREADS) a.prefix[r] = pre[r];
    if (tid == 0) a.prefix[a.rows + 1] = per;
  }
  if (total == 0) return;
  // workgroup id % 8 is the XCD: each takes neighbouring runs, which read the same keys and values, and as many as any other
  const int nb = min((int)gridDim.x, quotient(total + per - 1, per));
  const int x = (int)blockIdx.x & 7, i = (int)blockIdx.x >> 3, each = nb >> 3, more = nb & 7;
  if (i >= each + (x < more)) return;
  const int w = x * each + min(x, more) + i;
  int64_t pos = (int64_t)w * per;
  const int64_t end = pos + per < total ? pos + per : total;
  int lo = 0, hi = a.rows;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] <= pos) lo = mid;
    else hi = mid;
  }
  int r = __builtin_amdgcn_readfirstlane(lo), slot = 0;

  while (pos < end) {
    const Row row = row_of(a, r);
    if (weight(row) == 0) {
      ++r;
      continue;
    }
    const int64_t in_row = pos - pre[r];
    const int span = row.tiles + kStart, unit = cut ? quotient(in_row, span) : (int)in_row, from = (int)(in_row - (int64_t)unit * span);
    const int places = cut ? (int)min((int64_t)(span - from), end - pos) : 0;  // of this run
    const int first = cut ? max(from - kStart, 0) : 0, dealt = cut ? max(from + places - kStart, 0) - first : row.tiles;
    if (cut && dealt == 0) {  // the run ends within a unit's first places
      pos += places;
      continue;
    }
    const int kvh = unit / row.blocks, nth = unit - kvh * row.blocks, block = cut ? nth : row.blocks - 1 - nth;  // a chain's longest first
    // Tokens below `full` are seen by all columns of the block (of this wavefront), those from `none` on by none.
    const int columns = row.n * a.group, wave_column = block * T::QB + wave * CW * 16;
    const bool idle = wave_column >= columns;  // the wavefront only brings tiles
    auto last_node = [&](int column) { return a.by_group.quotient(min(column, columns) - 1); };
    const int block_full = row.context + (a.mask ? 0 : a.by_group.quotient(block * T::QB) + 1);
    const int full = row.context + (a.mask ? 0 : a.by_group.quotient(min(wave_column, columns - 1)) + 1);
    const int none = a.mask ? INT32_MAX : row.context + last_node(wave_column + CW * 16) + 1;
    const int block_none = a.mask ? INT32_MAX : max(row.context + last_node((block + 1) * T::QB) + 1, 0);
    const int count = min(dealt, max((int)(((int64_t)block_none + TOK - 1) / TOK) - first, 0));  // of the tiles dealt, those that are seen
    const int32_t* trow = a.table + (int64_t)r * a.table_stride;
    const uint8_t *kh = a.k + (int64_t)kvh * a.k_head, *vh = a.v + (int64_t)kvh * a.v_head;
    // scores times sc, which is made positive by the queries' sign (and never 0: -inf stays -inf)
    const float signed_sc = a.scale * (a.k_scale ? a.k_scale[kvh] : 1.f);
    const float sc = fabsf(signed_sc) < FLT_MIN ? FLT_MIN : fabsf(signed_sc);
    const uint32_t flip = signed_sc < 0.f ? 0x80008000u : 0u;

    // columns of this wavefront: (node, head) pairs; those past the row's last are node 0's with queries of 0
    const int first_column = wave_column + col;
    int node[CW];
    Seen sees[CW];
    u32x4_t q[CW][KS];
#pragma unroll
    for (int j = 0; j < CW; ++j) {
      const int c = first_column + 16 * j;
      const bool has = c < columns;
      node[j] = has ? a.by_group.quotient(c) : 0;
      sees[j].start(a, row.start + node[j]);
      const uint16_t* p = a.q + (int64_t)(row.start + node[j]) * a.q_token + (int64_t)(kvh * a.group + (has ? c - node[j] * a.group : 0)) * a.q_head;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int d = 32 * s + 8 * g;
        q[j][s] = has && d < a.dim ? *(const u32x4_t*)(p + d) : u32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int n = 0; n < 4; ++n) q[j][s][n] ^= flip;
      }
    }
    f32x4_t o[ND][CW];
    float m[CW], l[CW];  // what weights are relative to, and their sum
    bool counts[CW];     // some token of the column counts
#pragma unroll
    for (int j = 0; j < CW; ++j) {
      m[j] = -INFINITY, l[j] = 0.f, counts[j] = false;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d][j] = f32x4_t{0, 0, 0, 0};
    }

    // ---- a tile's way to LDS: R threads for a token, each every R-th piece of its key and value
    const int rt = tid / T::R, rp = tid % T::R;  // this thread's token and first piece
    u32x4_t kr[NL], vr[NL];
    int id, seen_id;           // pages of this thread's token, and of token `lane`
    bool ok;                   // this thread's token counts
    uint64_t live, next_live;  // tokens of the tile that count
    // Where a tile is whole pages, a thread's place in its page is the same in every tile, and its page index goes on by
    // as many.
    const int lane_t = lane & (TOK - 1), own_page = a.by_page.quotient(rt), lane_page = a.by_page.quotient(lane_t), last_page = a.by_page.quotient(max(row.len - 1, 0));
    const int own_in = rt - own_page * a.page;
    const int64_t k_in = own_in * a.k_token, v_in = own_in * a.v_token;
    auto pages_of = [&](int t0) {
      if (a.step) {
        const int before = t0 / TOK * a.step;
        id = trow[min(before + own_page, last_page)];
        seen_id = trow[min(before + lane_page, last_page)];
      } else {
        id = trow[a.by_page.quotient(min(t0 + rt, row.len - 1))];
        seen_id = trow[a.by_page.quotient(min(t0 + lane_t, row.len - 1))];
      }
    };
    auto load = [&](int t0) {  // unconditional loads: of page 0 where a token does not count
      const int t = t0 + rt;
      next_live = __ballot(t0 + lane_t < row.len && (uint32_t)seen_id < (uint32_t)a.pages);
      ok = t < row.len && (uint32_t)id < (uint32_t)a.pages;
      const int64_t pg = ok ? id : 0;
      const uint8_t *kp = kh + pg * a.k_page, *vp = vh + pg * a.v_page;
      if (a.step) {
        kp += k_in, vp += v_in;
      } else {
        const int in = ok ? t - a.by_page.quotient(t) * a.page : 0;
        kp += in * a.k_token, vp += in * a.v_token;
      }
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int c = rp + T::R * i, piece = c * (F8 ? 16 : 8) < a.dim ? 16 * c : 0;
        kr[i] = *(const u32x4_t*)(kp + piece);
        vr[i] = *(const u32x4_t*)(vp + piece);
      }
    };
    // Whether a value of the tile is infinite or NaN (asked of tiles that hold nodes).
    auto store = [&](int half, bool nodes) {
      bool odd = false;
      uint8_t *ks = lds + half * 2 * T::STORE, *vs = ks + T::STORE;
      if (__ballot(!ok))  // zeros for values of tokens that do not count: their bits may be NaN, their weight is 0
#pragma unroll
        for (int i = 0; i < NL; ++i) vr[i] = ok ? vr[i] : u32x4_t{0, 0, 0, 0};
      if (a.dim < DT)  // keys past the head's dims are zeros (the queries are); what values hold there reaches no output
#pragma unroll
        for (int i = 0; i < NL; ++i) kr[i] = (rp + T::R * i) * (F8 ? 16 : 8) < a.dim ? kr[i] : u32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int c = rp + T::R * i;
        const u32x4_t kv = kr[i], vv = vr[i];
        if constexpr (F8) {
          u32x4_t wide[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t k0 = kv[2 * h], k1 = kv[2 * h + 1], v0 = vv[2 * h], v1 = vv[2 * h + 1];
            *(u32x4_t*)(ks + T::key_place(rt, 2 * c + h)) = u32x4_t{widen<F16, false>(k0), widen<F16, true>(k0), widen<F16, false>(k1), widen<F16, true>(k1)};
            wide[h] = u32x4_t{widen<P16, false>(v0), widen<P16, true>(v0), widen<P16, false>(v1), widen<P16, true>(v1)};
            *(u32x4_t*)(vs + T::value_place(rt, c) + 16 * h) = wide[h];
          }
          if (nodes)
#pragma unroll
            for (int k = 0; k < 8; ++k) odd |= odd_word<P16>(wide[k >> 2][k & 3]);
        } else {
          *(u32x4_t*)(ks + T::key_place(rt, c)) = kv;
          *(u32x4_t*)(vs + T::value_place(rt, c >> 1) + 16 * (c & 1)) = vv;
          if (nodes)
#pragma unroll
            for (int k = 0; k < 4; ++k) odd |= odd_word<P16>(vv[k]);
        }
      }
      live = next_live;
      return odd;
    };

    const int base = first * TOK, stop = (first + count) * TOK;
    // A value that is infinite or NaN counts for the columns that see its token only, but 0 times it would reach all: where
    // a tile with nodes holds one (odd), the products take 0 for it, and it is added to its columns by hand.
    bool odd = false;
    auto join_waves = [&](int half, bool nodes, bool any) {
      // words of this half are read before the next barrier, and written again only after it
      if (nodes && lane == 0) flag[W * half + wave] = 0;
      if (nodes && any) flag[W * half + wave] = 1;
      __syncthreads();
      int any_wave = 0;
      if (nodes)
#pragma unroll
        for (int w = 0; w < W; ++w) any_wave |= flag[W * half + w];
      odd = __builtin_amdgcn_readfirstlane(any_wave);
    };
    if (count > 0) {  // a row without tokens has no tile
      pages_of(base);
      load(base);
      __syncthreads();  // the run before may still be read
      const bool nodes = base + TOK > block_full, any = store(0, nodes);
      if (count > 1) {
        pages_of(base + TOK);
        load(base + TOK);
      }
      join_waves(0, nodes, any);
    }
    int half = 0;
    for (int t0 = base; t0 < stop; t0 += TOK) {
      const bool further = t0 + 2 * TOK < stop;
      if (further) pages_of(t0 + 2 * TOK);
      uint8_t *ks = lds + half * 2 * T::STORE, *vs = ks + T::STORE;
      constexpr uint64_t ALL = TOK < 64 ? (1ull << TOK) - 1 : ~0ull;
      const uint64_t valid = live & ALL;
      const bool plain = t0 + TOK <= full && valid == ALL;
      if (odd) {
        if (!idle)
#pragma unroll
          for (int j = 0; j < CW; ++j) {
            const uint64_t bits = sees[j].bits(a, row.start + node[j], node[j], t0 - row.context) & valid;
#pragma unroll 1
            for (int t = 0; t < TOK; ++t)
#pragma unroll
              for (int d = 0; d < ND; ++d) {
                const u32x2_t v = *(const u32x2_t*)(vs + T::value_place(t, d) + 8 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const uint32_t h = v[e >> 1] >> (16 * (e & 1)) & 0xffffu;
                  if (odd_half<P16>(h) && (bits >> t & 1)) o[d][j][e] += unpack<P16>(h, 0);
                }
              }
          }
        __syncthreads();
#pragma unroll 1
        for (int i = tid; i < T::STORE / 4; i += THREADS) ((uint32_t*)vs)[i] = clean2<P16>(((uint32_t*)vs)[i]);
        __syncthreads();
      }
      if (!idle && t0 < none) {
        // Reads of LDS go AHEAD steps before the products that take them, in the order written (sched_barrier): left to
        // itself the compiler saves registers and waits for each read.
        constexpr int AHEAD = T::AHEAD;
        u32x4_t p[KT][CW][PARTS];
        f32x4_t s[NT][CW];
        {
          constexpr int N = KS * NT;
          u32x4_t kf[AHEAD + 1];
          // of tokens 16 i + col, piece 4 k + g: its place is token col's, with 4 k in the exclusive or, 16 i rows further
          const uint32_t at = lds_at + half * 2 * T::STORE + T::key_place(col, g);
          auto key = [&](int n) { return *(const __attribute__((address_space(3))) u32x4_t*)(uintptr_t)((at ^ (n / NT * 64)) + n % NT * 16 * DT * 2); };
#pragma unroll
          for (int n = 0; n < AHEAD; ++n) kf[n] = key(n);
#pragma unroll
          for (int n = 0; n < N; ++n) {
            if (n + AHEAD < N) kf[(n + AHEAD) % (AHEAD + 1)] = key(n + AHEAD);
            const int k = n / NT, i = n % NT;
#pragma unroll
            for (int j = 0; j < CW; ++j) s[i][j] = mfma16<F16>(kf[n % (AHEAD + 1)], q[j][k], k ? s[i][j] : f32x4_t{0, 0, 0, 0});
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        float off[CW];
#pragma unroll
        for (int j = 0; j < CW; ++j) {
          if (!plain) {
            const uint64_t bits = (sees[j].bits(a, row.start + node[j], node[j], t0 - row.context) & valid) >> (4 * g);
            const uint32_t word[2] = {(uint32_t)bits, (uint32_t)(bits >> 32)};
            counts[j] |= bits != 0;
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) s[i][j][e] = word[i >> 1] & (1u << (16 * (i & 1) + e)) ? s[i][j][e] : -INFINITY;
          } else {
            counts[j] = true;
          }
          float top = -INFINITY;
#pragma unroll
          for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = fmaxf(top, s[i][j][e]);
          top = fmaxf(top, __shfl_xor(top, 16));
          top = fmaxf(top, __shfl_xor(top, 32)) * sc;
          if (__ballot(top > m[j] + T::SLACK)) {
            const float m_new = top > m[j] + T::SLACK ? top : m[j];
            // never 0: an infinite sum stays infinite
            const float alpha = m_new == m[j] ? 1.f : fmaxf(__builtin_amdgcn_exp2f(m[j] - m_new), FLT_MIN);
            m[j] = m_new;
            l[j] *= alpha;
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d][j] *= alpha;
          }
          off[j] = T::SHIFT - (m[j] == -INFINITY ? 0.f : m[j]);  // nothing but -inf so far: weights 0, not NaN
        }
        // Weights of pair u of 32 tokens k: two of a lane's eight, of a column.  Those of the next 32 tokens are made between the
        // products of these.
        auto weights = [&](int k, int u) {
          const int j = u % CW, i = 2 * k + u / CW / 2, h = u / CW % 2;
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][j][2 * h], sc, off[j]));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][j][2 * h + 1], sc, off[j]));
          l[j] += p0 + p1;
          uint32_t out[PARTS];
          split_parts<P16, !F8>(p0, p1, out);  // e4m3 has no infinities
#pragma unroll
          for (int n = 0; n < PARTS; ++n) p[k][j][n][2 * (i & 1) + h] = out[n];
        };
        constexpr int N = KT * ND, PAIRS = 4 * CW;
        // Of 16 tokens, lane group g's four: rows 4 g .. 4 g + 3, eight bytes a lane; the transposing read gives each lane its dim of the
        // four.  Dims d are in the exclusive or of the first row's place, later tokens rows further.
        const uint32_t at = lds_at + (half * 2 + 1) * T::STORE + T::value_place(4 * g + (col >> 2), 0) + 8 * (col & 3);
        auto value = [&](int n) {  // dims n % ND of 32 tokens n / ND
          typedef __attribute__((ext_vector_type(4))) short s16x4_t;
          typedef __attribute__((address_space(3))) s16x4_t* lds_p;
          u32x4_t vf;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const u32x2_t v = __builtin_bit_cast(
                u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(uintptr_t)((at ^ (n % ND * 32)) + (32 * (n / ND) + 16 * h) * DT * 2)));
            vf[2 * h] = v[0], vf[2 * h + 1] = v[1];
          }
          return vf;
        };
        u32x4_t vf[AHEAD + 1];
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) vf[n] = value(n);
#pragma unroll
        for (int u = 0; u < PAIRS; ++u) weights(0, u);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < N; ++n) {
          if (n + AHEAD < N) vf[(n + AHEAD) % (AHEAD + 1)] = value(n + AHEAD);
          const int k = n / ND, d = n % ND;
#pragma unroll
          for (int j = 0; j < CW; ++j)
#pragma unroll
            for (int part = PARTS - 1; part >= 0; --part) o[d][j] = mfma16<P16>(vf[n % (AHEAD + 1)], p[k][j][part], o[d][j]);
          if (k + 1 < KT)
#pragma unroll
            for (int u = d * PAIRS / ND; u < (d + 1) * PAIRS / ND; ++u) weights(k + 1, u);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (t0 + TOK < stop) {
        half ^= 1;
        const bool nodes = t0 + 2 * TOK > block_full, any = store(half, nodes);
        if (further) load(t0 + 2 * TOK);
        join_waves(half, nodes, any);
      }
    }
#pragma unroll
    for (int j = 0; j < CW; ++j) {
      // a token of any lane group counts, whatever its score: m is then finite (average_factor)
      const uint64_t any = __ballot(counts[j]);
      if (any >> col & 0x0001000100010001ull) m[j] = fmaxf(m[j], -FLT_MAX);
      l[j] += __shfl_xor(l[j], 16);
      l[j] += __shfl_xor(l[j], 32);
    }
    // ---- outputs, or this run's part of them
    const bool whole = first == 0 && dealt == row.tiles;
    {
      float* part_sums = whole ? nullptr : a.ws + ((int64_t)w * 2 + slot) * partial_floats(T::QB, a.dim);
#pragma unroll
      for (int j = 0; j < CW; ++j) {
        const int column = first_column + 16 * j, c = (wave * CW + j) * 16 + col;
        if (column >= columns) continue;
        if (part_sums) {
#pragma unroll
          for (int d = 0; d < ND; ++d)
            if (16 * d + 4 * g < a.dim) *(f32x4_t*)(part_sums + (int64_t)c * a.dim + 16 * d + 4 * g) = o[d][j] * T::UNSHIFT;
          if (g == 0) {
            float* st = part_sums + (int64_t)T::QB * a.dim + 2 * c;
            st[0] = m[j];
            st[1] = l[j] * T::UNSHIFT;
          }
        } else {
          const int64_t at = (int64_t)(row.start + node[j]) * a.heads + kvh * a.group + (column - node[j] * a.group);
          const float f = m[j] == -INFINITY ? 0.f : l[j] == 0.f ? NAN : (a.v_scale ? a.v_scale[kvh] : 1.f) / l[j];
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            const float e[4] = {o[d][j][0] * f, o[d][j][1] * f, o[d][j][2] * f, o[d][j][3] * f};
            if (16 * d + 4 * g < a.dim) store_values<4>(a.out, a.out_dtype, at * a.dim + 16 * d + 4 * g, e);
          }
          if (a.lse && g == 0) a.lse[at] = (m[j] + __builtin_amdgcn_logf(l[j] * T::UNSHIFT)) * 0.69314718055994531f;
        }
      }
    }
    slot = 1;
    if (!cut) return;
    pos += places;
    if (pos >= pre[r + 1]) ++r;
  }
}

struct TreeKern {
  const void* fn;
  int qb, tok, lds, threads, occ;  // occ: workgroups of a CU at most, which the workspace goes by
  std::atomic<int>* residents;     // workgroups of a CU, by device; 0: not asked yet
};

// The kernel for head_dim, about `columns` columns of a row and the longest row that the table holds.
// Eight wavefronts of two groups of 16 columns share a tile where there are columns for them and rows are long: a quarter of the loads,
// widenings and LDS writes a column that four of one group have, but a quarter as many workgroups.  us, four (64 columns) and eight (256): 64
// drafts of 8 rows of 16384, e4m3, 495 and 387; of 8192, bf16, 182 and 155; of 32 rows of 1000 98 and 81, of 500 59 and 51; a chain of 513
// over 6001 148 and 135; but 64 drafts of 128 ragged rows of up to 300 100 and 114, of 8 rows of 256 17 and 29.  Four wavefronts of two groups
// need more than the 256 registers there are and lose at every size between: 32 drafts of 16 ragged rows of up to 8192 (128 columns) 102, with two
// groups 120; of 64 rows of up to 2048 116 and 147; 64 drafts of 64 rows of up to 500 69 and 87.  Heads of up to 64 dims have registers for two.
TreeKern kern_bf16(int dim, int columns, int longest);
TreeKern kern_f16(int dim, int columns, int longest);
TreeKern kern_bf16_e4m3(int dim, int columns, int longest);
TreeKern kern_f16_e4m3(int dim, int columns, int longest);

template <bool F16, bool F8, int DT, int W, int CW, int TOK, int OCC>
TreeKern kern_t() {
  using T = Kern<F16, F8, DT, W, CW, TOK, OCC>;
  static std::atomic<int> residents[64];
  return TreeKern{(const void*)tree_kernel<F16, F8, DT, W, CW, TOK, OCC>, T::QB, TOK, T::LDS, T::THREADS, OCC, residents};
}
template <bool F16, bool F8>
TreeKern kern_of(int dim, int columns, int longest) {
  if (dim > 128) return kern_t<F16, F8, 256, 4, 1, 32, 2>();
  if (dim > 64) {
    return columns > 128 && longest > 512 ? kern_t<F16, F8, 128, 8, 2, 64, 1>() : kern_t<F16, F8, 128, 4, 1, 64, 2>();
  }
  return columns > 64 ? kern_t<F16, F8, 64, 4, 2, 64, 2>() : kern_t<F16, F8, 64, 4, 1, 64, 4>();
}

}  // namespace tree
}  // namespace mlxr
