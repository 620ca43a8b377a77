// Decode attention over a paged key-value cache: one new token per row.
//
//   o[h] = sum_t p_t v[t] / sum_t p_t,   p_t = exp(scale q[h] . k[t] - m),   m the running maximum
//
// in one pass over keys and values.  The heads that share a kv head (up to 16 of them) are the
// columns of the matrix instructions, so a key or value is read once for all of them:
//   S^T[32 tokens, 16 heads] = K Q^T        rows of K from memory straight into A operands
//   O^T[dim, 16 heads]      += V^T P^T      V^T by exchanging 16-bit halves between registers
// Which token a row of the first product stands for is free: row 4 b + i of its half hh is token
// 8 b + 4 hh + i, so the scores that a lane holds (heads across lanes, rows 4 g .. 4 g + 3 for lane
// group g) are those of tokens 8 g .. 8 g + 7, which is what the second product wants in that lane
// as its operand: P never leaves the registers, and the softmax's factors are one value per lane.
// P is split in 16-bit parts that add up to it: three in bf16 (all bits of fp32), two in f16 (22 bits), which an e4m3
// cache's values, exact in either type, take too.  More products cost matrix cycles that the kernel, bound by memory, has to
// spare.
//
// Short rows: a workgroup for each (row, kv head), merged in LDS (attn_rows_kernel).  Long ones are cut
// evenly (attn_kernel): the tiles (32 tokens) of all rows and kv heads, in one sequence, are dealt to the
// wavefronts of a launch that fills the device, in equal contiguous runs.  A run that covers a whole (row,
// kv head) writes the output; others leave (m, sum, unnormalized o) in the workspace, at most two for
// a wavefront, and a second launch joins them.  Lengths are read on the device; the host chooses by the longest
// row that the table can hold.
//
// Bound by memory: 64 rows of 8 kv heads of 128 in bf16, up to 8192 tokens (961 MB), 158 us and 7 of the join, 6.1 TB/s;
// one row of 120001 tokens (492 MB) 78 and 6; 32 rows of an e4m3 cache, up to 16384 tokens (547 MB), 100 and 7; 17 rows of 32
// heads of 80, window 1024, in one launch 33 (158 MB; lines that heads share).  One row of 4 kv heads of 64, 700
// tokens, 7.6: latency.
#pragma once
#include <cfloat>

#include "mfma16.h"
#include "paged_internal.h"

namespace mlxr {
namespace paged {

constexpr int kTile = 32;     // tokens
constexpr int kWaves = 4;     // of a workgroup
constexpr int kHeads = 16;    // columns of the products
constexpr int kMaxCutRows = 4096;  // rows of a cut launch: their tiles are summed up in LDS

struct AttnArgs {
  const uint8_t *k, *v;  // element addresses in bytes
  const float *k_scale, *v_scale;
  int64_t k_head, v_head;  // strides, bytes
  uint32_t k_page, k_token, v_page, v_token;
  const uint16_t* q;
  int64_t q_row, q_head;  // elements
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;
  void* out;
  float* lse;
  float* ws;        // partials
  int32_t* prefix;  // [rows + 1] tiles before each row, then tiles of a wavefront, for the join
  int rows, heads, kv_heads, group, groups;  // groups: of 16 heads, of a kv head
  int dim, page, pages, width, window, out_dtype;
  Divisor by_page;
  int part_rows, workers, near;
  float scale;  // times log2(e)
};

// Tokens [first, len) of row r; the first tile starts at base.
struct Span {
  int first, base, len, tiles;
};
__device__ __forceinline__ Span span_of(const AttnArgs& a, int r) {
  Span s;
  const int64_t most = (int64_t)a.width * a.page;
  const int n = a.lens[r];
  s.len = n < 0 ? 0 : n > most ? (int)most : n;
  s.first = a.window > 0 && s.len > a.window ? s.len - a.window : 0;
  s.base = s.first & ~7;  // a block of eight tokens lies in one page where page % 8 == 0
  s.tiles = (s.len - s.base + kTile - 1) / kTile;
  return s;
}

// Partial of slot `slot` of worker w: part_rows rows of dim floats, then m and sum of each.
__host__ __device__ constexpr int partial_floats(int part_rows, int dim) { return part_rows * dim + (2 * part_rows + 3) / 4 * 4; }
__device__ __forceinline__ float* partial(const AttnArgs& a, int w, int slot) {
  return a.ws + ((int64_t)w * 2 + slot) * partial_floats(a.part_rows, a.dim);
}
// What makes an average of a row's weighted values.  A row none of whose tokens counts (m is -inf) gets zeros; one whose
// scores are all -inf (its weights, and so l, are 0) NaN, by the formula.
__device__ __forceinline__ float average_factor(const AttnArgs& a, int kvh, float m, float l) {
  return m == -INFINITY ? 0.f : l == 0.f ? NAN : (a.v_scale ? a.v_scale[kvh] : 1.f) / l;
}
// n / d, d > 0; most calls stay within 32 bits, whose division takes a tenth of the instructions.
__device__ __forceinline__ int quotient(int64_t n, int d) {
  return n < (1ll << 31) ? (int)((uint32_t)n / (uint32_t)d) : (int)(n / d);
}

// Two e4m3 values (half `h` of w) as two 16-bit floats: exact in either type.
template <bool F16, bool H>
__device__ __forceinline__ uint32_t widen(uint32_t w) {
  if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, H));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, H));
}

// The larger of the 16-bit halves: of floats that are not negative, the larger float.
__device__ __forceinline__ uint32_t pair_max(uint32_t a, uint32_t b) {
  typedef __attribute__((ext_vector_type(2))) uint16_t V;
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b)));
}

// N (1, 2, 4) words at a multiple of 4 N bytes.
template <int N>
struct Words {
  uint32_t w[N];
};
template <int N, bool NT>
__device__ __forceinline__ Words<N> load_words(const void* p) {
  Words<N> r;
  if constexpr (N == 1) {
    r.w[0] = NT ? __builtin_nontemporal_load((const uint32_t*)p) : *(const uint32_t*)p;
  } else {
    typedef __attribute__((ext_vector_type(N))) uint32_t V;
    const V v = NT ? __builtin_nontemporal_load((const V*)p) : *(const V*)p;
#pragma unroll
    for (int k = 0; k < N; ++k) r.w[k] = v[k];
  }
  return r;
}
template <int N>
__device__ __forceinline__ void store_words(void* p, const Words<N>& v) {
  __builtin_memcpy(__builtin_assume_aligned(p, 4 * N), &v, 4 * N);
}
// N (4, 8) neighbouring values from element i, a multiple of N, of an output on.
template <int N>
__device__ __forceinline__ void store_values(void* out, int dtype, int64_t i, const float* v) {
  if (dtype == DT_F32) {
#pragma unroll
    for (int c = 0; c < N; c += 4) *(f32x4_t*)((float*)out + i + c) = f32x4_t{v[c], v[c + 1], v[c + 2], v[c + 3]};
  } else {
    Words<N / 2> w;
#pragma unroll
    for (int k = 0; k < N / 2; ++k)
      w.w[k] = dtype == DT_F16 ? pack2<true>(v[2 * k], v[2 * k + 1]) : pack2<false>(v[2 * k], v[2 * k + 1]);
    store_words<N / 2>((uint16_t*)out + i, w);
  }
}

// F16: the type of the queries' product (else bf16).  F8: the cache is e4m3.  DT: 64, 96, 128 or 256, at least dim (DIM:
// equal; 96: above 64, not for e4m3; 128: above that).  P8: page_size % 8 == 0.
// LK: keys through LDS (load_k).
template <bool F16, bool F8, int DT, bool DIM, bool P8, bool LK>
struct Attn {
  static constexpr int KS = DT / 32;               // steps of the first product
  static constexpr int VE = DT == 64 ? 4 : 8;      // neighbouring values of a token that a lane loads
  static constexpr int VH = DT == 256 ? 2 : 1;     // times that
  static constexpr int NC = VH * VE;               // accumulators
  static constexpr bool P16 = F16 || F8;           // the second product's type, f16 or else bf16
  static constexpr int PARTS = P16 ? 2 : 3;        // of P
  // p times 2^14 in f16: weights down to 2^-28 of the largest stay normal numbers (bf16 has the range)
  static constexpr float SHIFT = P16 ? 14.f : 0.f;
  static constexpr float UNSHIFT = P16 ? 0x1p-14f : 1.f;
  static constexpr bool NT = DIM && DT * (F8 ? 1 : 2) % 128 == 0;  // past the caches
  static constexpr int KL = F8 ? KS / 2 : KS;      // 16-byte parts of a key row in a lane's operands
  // Keys through LDS: parts of a row, tokens of a load, loads of a tile.
  static constexpr int CH = F8 ? DT / 16 : DT == 96 ? 16 : DT / 8, TPL = 64 / CH, NL = LK ? kTile / TPL : 2 * KL;

  const AttnArgs& a;
  const int lane, col;
  int g;
  u32x4_t q[KS];
  u32x4_t kr[NL];
  u32x4_t* keys;  // [32 tokens][CH] of this wavefront
  uint32_t vr[VH][8][F8 ? VE / 4 : VE / 2];
  f32x4_t o[NC];
  float m, l, sc;
  const uint8_t *kh, *vh;
  const int32_t* trow;

  __device__ Attn(const AttnArgs& a_, u32x4_t* keys_) : a(a_), lane(threadIdx.x & 63), col(lane & 15), g(lane >> 4), keys(keys_) {}

  // Whether all lanes' part of load j of a key's row lies within the head's dims.
  static constexpr bool whole(int j) { return DIM || ((DT == 96 || DT == 128) && j < KL - 1); }

  // First element of the k-th operand of step j that lane group g holds, as in the keys' loads.
  __device__ __forceinline__ int dim_of(int j) const {
    return F8 ? (j >> 1) * 64 + g * 16 + (j & 1) * 8 : j * 32 + g * 8;
  }

  __device__ __forceinline__ void start(int r, int kvh, int grp) {
    const int h = grp * kHeads + col;
    const bool ok = h < a.group;
    const uint16_t* p = a.q + (int64_t)r * a.q_row + (int64_t)(kvh * a.group + (ok ? h : 0)) * a.q_head;
#pragma unroll
    for (int j = 0; j < KS; ++j) {
      const int d = dim_of(j);
      q[j] = ok && (whole(F8 ? j >> 1 : j) || d < a.dim) ? *(const u32x4_t*)(p + d) : u32x4_t{0, 0, 0, 0};
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) o[c] = f32x4_t{0, 0, 0, 0};
    m = -INFINITY;
    l = 0.f;
    sc = a.scale * (a.k_scale ? a.k_scale[kvh] : 1.f);
    kh = a.k + (int64_t)kvh * a.k_head;
    vh = a.v + (int64_t)kvh * a.v_head;
    trow = a.table + (int64_t)r * a.table_stride;
  }

  // Keys and values are read once: past the caches (64 rows of 8 kv heads of 128, up to 8192 tokens, 187 -> 167 us), unless
  // a row of a head is not whole 128-byte lines and so shares them with rows that other wavefronts read (33 rows of 32
  // heads of 80 in [token, head] order, window 1024, 69 -> 75 us).
  template <class T>
  static __device__ __forceinline__ T stream_load(const T* p) {
    if constexpr (NT) return __builtin_nontemporal_load(p);
    else return *p;
  }
  // Index of a position's page among its row's.
  __device__ __forceinline__ int page_of(int pos) const { return a.by_page.quotient(pos); }
  // Table entry of a position of the row (of the row's last token, past it).
  __device__ __forceinline__ int entry_of(int pos, const Span& s) const { return trow[page_of(min(pos, s.len - 1))]; }
  // Byte offset of a position in a store whose page is `id` (page 0 for one outside the cache: read, not used).
  __device__ __forceinline__ uint64_t offset(int id, int pos, uint32_t page, uint32_t token) const {
    return (uint64_t)((uint32_t)id < (uint32_t)a.pages ? id : 0) * page + (uint64_t)(uint32_t)(pos - page_of(pos) * a.page) * token;
  }

  // Table entries of a tile's tokens: one for each block of eight where a block lies in one page, else one for
  // each token of the lane's values and keys.
  struct Ids {
    int id[P8 ? 1 : 10];
  };
  __device__ __forceinline__ Ids ids_of(int t0, const Span& s) const {
    Ids n;
    if constexpr (P8) {
      n.id[0] = entry_of(t0 + 8 * g, s);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) n.id[j] = entry_of(t0 + 8 * g + j, s);
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) n.id[8 + hh] = entry_of(t0 + key_token(hh), s);
    }
    return n;
  }
  // Token of the tile that is row `col` of half hh of the keys.
  __device__ __forceinline__ int key_token(int hh) const { return 8 * (col >> 2) + 4 * hh + (col & 3); }
  // Bits of this lane's eight tokens (t0 + 8 g + j) that count.
  __device__ __forceinline__ uint32_t live_of(const Ids& n, int t0, const Span& s) const {
    const int pos = t0 + 8 * g, from = min(max(s.first - pos, 0), 8), to = min(max(s.len - pos, 0), 8);
    uint32_t live = (1u << to) - (1u << from);  // from <= to: a window is no later than the row's end
    if constexpr (P8) {
      if ((uint32_t)n.id[0] >= (uint32_t)a.pages) live = 0;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if ((uint32_t)n.id[j] >= (uint32_t)a.pages) live &= ~(1u << j);
    }
    return live;
  }

  // First of the VE neighbouring dims of row m of the second product's operand, half x; rows past the head's dims
  // repeat the first, their sums are not stored.
  __device__ __forceinline__ bool has_row(int x, int m) const { return DIM || x * 128 + VE * m < a.dim; }
  __device__ __forceinline__ int dims_of(int x, int m) const { return has_row(x, m) ? x * 128 + VE * m : 0; }

  // The loads of a tile are unconditional, from an address within the stores for whatever does not count, so
  // that they stay in flight over the branches: what they bring for tokens that do not count is left out later.
  // more: false where there is no further tile; all lanes then read the first page's first rows again.
  //
  // Keys: an operand's lanes are 16 tokens at a time, so that a load of it is 16 pieces of 64 bytes.  LK: loads of whole
  // rows side by side instead, brought into operand order through LDS; blocks of eight tokens lie side by side, their
  // offsets come from the lane groups by readlane.  us, straight and through LDS: 64 rows of 32 kv heads of 128, up to 1024
  // tokens, 93 and 82; of 32 of 80, window 1024, 137 and 121; 8 of 128, up to 8192, 172 and 168; but a row of 4 kv heads
  // of 64, 700 tokens, 7.3 and 8.6: nothing hides the way through LDS there.
  __device__ __forceinline__ void load_k(const Ids& n, int t0, bool more) {
    if constexpr (LK) {
      const int c = lane % CH, tk = lane / CH;
      const uint64_t at = (uint64_t)a.k_token * (tk & 7) + (DIM || c * (F8 ? 16 : 8) < a.dim ? c : 0) * 16;
      const uint64_t mine = more ? offset(n.id[0], t0 + 8 * g, a.k_page, a.k_token) : 0;  // of the block of eight tokens g
      const uint32_t lo = (uint32_t)mine, hi = (uint32_t)(mine >> 32);
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int from = 16 * (i * TPL / 8);
        uint64_t row;
        if constexpr (TPL > 8)
          row = (uint64_t)(uint32_t)__shfl((int)hi, from + 2 * (tk & 8)) << 32 | (uint32_t)__shfl((int)lo, from + 2 * (tk & 8));
        else
          row = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)hi, from) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)lo, from);
        kr[i] = stream_load((const u32x4_t*)(kh + row + (uint64_t)a.k_token * (i * TPL & 7) + at));
      }
    } else {
      const uint8_t* block = nullptr;
      if constexpr (P8) block = kh + (more ? offset(__shfl(n.id[0], (col & 12) * 4), t0 + key_token(0), a.k_page, a.k_token) : 0);
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const uint8_t* p = P8 ? block + (uint64_t)a.k_token * (4 * hh)
                              : kh + (more ? offset(n.id[P8 ? 0 : 8 + hh], t0 + key_token(hh), a.k_page, a.k_token) : 0);
#pragma unroll
        for (int j = 0; j < KL; ++j) {
          int d = F8 ? j * 64 + g * 16 : j * 32 + g * 8;
          if (!whole(j) && d >= a.dim) d = 0;
          kr[hh * KL + j] = stream_load((const u32x4_t*)(p + d * (F8 ? 1 : 2)));
        }
      }
    }
  }
  // Place of part c of a token's key: 8 lanes that read or write at once, and so 128 bytes, lie in different banks.
  static __device__ __forceinline__ int place(int token, int c) {
    const int swap = CH == 4 ? (token >> 1 & 1) | (token >> 2 & 2) : (token & 3) | (token >> 1 & 4);
    return token * CH + (c ^ swap);
  }
  __device__ __forceinline__ void store_k() {
    if constexpr (LK) {
      const int c = lane % CH, tk = lane / CH;
#pragma unroll
      for (int i = 0; i < NL; ++i) keys[place(i * TPL + tk, c)] = kr[i];
      // a wavefront's accesses to LDS are in order: only the compiler has to keep them so
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
  }
  __device__ __forceinline__ u32x4_t key_part(int hh, int j) const {
    if constexpr (LK) return keys[place(key_token(hh), 4 * j + g)];
    else return kr[hh * KL + j];
  }
  __device__ __forceinline__ void load_v(const Ids& n, int t0, bool more) {
    constexpr int W = F8 ? VE / 4 : VE / 2;
    const uint8_t* block = vh + (P8 && more ? offset(n.id[0], t0 + 8 * g, a.v_page, a.v_token) : 0);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint8_t* p = P8 ? block + (uint64_t)a.v_token * j
                            : vh + (more ? offset(n.id[P8 ? 0 : j], t0 + 8 * g + j, a.v_page, a.v_token) : 0);
#pragma unroll
      for (int x = 0; x < VH; ++x) {
        const Words<W> w = load_words<W, NT>(p + dims_of(x, col) * (F8 ? 1 : 2));
#pragma unroll
        for (int k = 0; k < W; ++k) vr[x][j][k] = w.w[k];
      }
    }
  }

  // Word w (dims 2 w, 2 w + 1 of the lane's VE) of token j, as a pair of 16-bit floats.
  template <int W>
  __device__ __forceinline__ uint32_t v_word(int x, int j) const {
    if constexpr (F8) return widen<P16, (W & 1) != 0>(vr[x][j][W >> 1]);
    else return vr[x][j][W];
  }
  template <int W>
  __device__ __forceinline__ void add_v(int x, const u32x4_t (&p)[PARTS]) {
    if constexpr (W < VE / 2) {
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = v_word<W>(x, j);
#pragma unroll
      for (int odd = 0; odd < 2; ++odd) {
        u32x4_t f;
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] = __builtin_amdgcn_perm(w[2 * k + 1], w[2 * k], odd ? 0x07060302u : 0x05040100u);
        const int c = x * VE + 2 * W + odd;
#pragma unroll
        for (int k = PARTS - 1; k >= 0; --k) o[c] = mfma16<P16>(f, p[k], o[c]);
      }
      add_v<W + 1>(x, p);
    }
  }

  // Tiles first .. first + count of the row: while a tile's weights are computed its values and the next
  // tile's keys are on their way, while its values are added up the next tile's keys and values.  Table
  // entries are read a tile before they are needed: loads return in order, waiting for one that was
  // asked for last would wait for all.
  __device__ __forceinline__ void run(const Span& s, int first, int count) {
    int t0 = s.base + first * kTile;
    const int last = s.base + (first + count - 1) * kTile;
    int t1 = t0 + kTile;
    Ids ids = ids_of(t0, s), next = ids_of(t1, s);
    load_k(ids, t0, true);
    __builtin_amdgcn_sched_barrier(0);  // the order of the loop's loads, which its waits count
    load_v(ids, t0, true);
    uint32_t live = live_of(ids, t0, s);
    uint64_t any = 0;
    while (true) {
      // Between 96 and 128 dims what follows from g is computed again for each tile: kept over the loop, it would cost a
      // third workgroup's registers (128 rows of 8 kv heads of 112, up to 200 tokens, 15.4 us and 14.4; other sizes lose 1 to 4 %).
      if constexpr (DT == 128 && !DIM && !LK && P8) asm("" : "+v"(g));
      const bool more = t0 != last;
      ids = next;
      next = ids_of(t1 + kTile, s);
      f32x4_t x[2];
      store_k();
      scores(x);
      load_k(ids, t1, more);
      const bool full = __ballot(live != 0xff) == 0;
      any |= __ballot(live != 0);
      u32x4_t p[PARTS];
      weights(x, live, full, p);
      if (!full) drop(live);
#pragma unroll
      for (int xh = 0; xh < VH; ++xh) add_v<0>(xh, p);
      load_v(ids, t1, more);
      asm volatile("" ::: "memory");  // the loads stay here, or what waits for the keys would wait for the values too
      if (!more) break;
      live = live_of(ids, t1, s);
      t0 = t1;
      t1 += kTile;
    }
    if (any) m = fmaxf(m, -FLT_MAX);  // a token counts, whatever its score (average_factor)
  }

  // Pair k of two weights in parts, none of them negative nor a later one 0: an infinite value then gives an infinite output
  // as a weight in one piece does, not NaN.  (The least later part, 2^-126 or 2^-38 of the largest weight, is far below the
  // rounding of the sums.)
  static __device__ __forceinline__ void split2(float p0, float p1, u32x4_t (&p)[PARTS], int k) {
    auto floor2 = [](uint32_t w) { return pair_max(w, P16 ? 0x00010001u : 0x00800080u); };
    if constexpr (P16) {
      const uint32_t hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(p0, p1));
      p[0][k] = hi;
      p[1][k] = floor2(pack2<true>(p0 - unpack<true>(hi, 0), p1 - unpack<true>(hi, 1)));
    } else {
#pragma unroll
      for (int n = 0; n < PARTS; ++n) {  // each the upper half of what is left; the last holds all of it
        const uint32_t b0 = __builtin_bit_cast(uint32_t, p0), b1 = __builtin_bit_cast(uint32_t, p1);
        const uint32_t w = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
        p[n][k] = n ? floor2(w) : w;
        p0 -= __builtin_bit_cast(float, b0 & 0xffff0000u);
        p1 -= __builtin_bit_cast(float, b1 & 0xffff0000u);
      }
    }
  }

  // Zeros for the values of tokens that do not count: their weight is 0, their bits may be NaN.
  __device__ __forceinline__ void drop(uint32_t live) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int x = 0; x < VH; ++x)
#pragma unroll
        for (int w = 0; w < (F8 ? VE / 4 : VE / 2); ++w) vr[x][j][w] = live >> j & 1 ? vr[x][j][w] : 0u;
  }

  __device__ __forceinline__ void scores(f32x4_t (&s)[2]) {
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      s[hh] = f32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        u32x4_t kf = key_part(hh, F8 ? j >> 1 : j);
        if constexpr (F8) {
          const uint32_t w0 = kf[2 * (j & 1)], w1 = kf[2 * (j & 1) + 1];
          kf = u32x4_t{widen<F16, false>(w0), widen<F16, true>(w0), widen<F16, false>(w1), widen<F16, true>(w1)};
        }
        if (!whole(F8 ? j >> 1 : j) && dim_of(j) >= a.dim) kf = u32x4_t{0, 0, 0, 0};
        s[hh] = mfma16<F16>(kf, q[j], s[hh]);
      }
    }
  }

  __device__ __forceinline__ void weights(const f32x4_t (&s)[2], uint32_t live, bool full, u32x4_t (&p)[PARTS]) {
    float x[8], top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = s[j >> 2][j & 3] * sc;
    if (!full)
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = live >> j & 1 ? x[j] : -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, x[j]);
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const float m_new = fmaxf(m, top);
    const float ref = m_new == -INFINITY ? 0.f : m_new;  // nothing but -inf so far: p = 0, not NaN
    const float alpha = __builtin_amdgcn_exp2f(m - ref);
    m = m_new;
    const float off = SHIFT - ref;
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float p0 = __builtin_amdgcn_exp2f(x[2 * k] + off), p1 = __builtin_amdgcn_exp2f(x[2 * k + 1] + off);
      sum += p0 + p1;
      split2(p0, p1, p, k);
    }
    l = l * alpha + sum;
#pragma unroll
    for (int c = 0; c < NC; ++c) o[c] *= alpha;
  }

  // This lane's sums to LDS, and those of another wavefront of the same row and heads added to its own.
  static constexpr int PARK = 4 * NC + 2;  // floats of a lane
  __device__ __forceinline__ void park(float* to) const {
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) to[(4 * c + i) * 64 + lane] = o[c][i];
    to[4 * NC * 64 + lane] = m;
    to[(4 * NC + 1) * 64 + lane] = l;
  }
  __device__ __forceinline__ void merge(const float* from) {
    const float m2 = from[4 * NC * 64 + lane], m_new = fmaxf(m, m2), ref = m_new == -INFINITY ? 0.f : m_new;
    const float f = __builtin_amdgcn_exp2f(m - ref), f2 = __builtin_amdgcn_exp2f(m2 - ref);
    m = m_new;
    l = l * f + from[(4 * NC + 1) * 64 + lane] * f2;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[c][i] = o[c][i] * f + from[(4 * c + i) * 64 + lane] * f2;
  }


  __device__ __forceinline__ void finish(int r, int kvh, int grp, float* part) {
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    const int h = grp * kHeads + col;
    if (h >= a.group) return;
    if (part) {
      float* row = part + (int64_t)col * a.dim;
#pragma unroll
      for (int x = 0; x < VH; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v[VE];
#pragma unroll
          for (int c = 0; c < VE; ++c) v[c] = o[x * VE + c][i] * UNSHIFT;
          if (has_row(x, 4 * g + i)) store_values<VE>(row, DT_F32, dims_of(x, 4 * g + i), v);
        }
      if (g == 0) {
        float* st = part + (int64_t)a.part_rows * a.dim + 2 * col;
        st[0] = m;
        st[1] = l * UNSHIFT;
      }
      return;
    }
    const int64_t head = (int64_t)r * a.heads + kvh * a.group + h;
    const float f = average_factor(a, kvh, m, l);
#pragma unroll
    for (int x = 0; x < VH; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v[VE];
#pragma unroll
        for (int c = 0; c < VE; ++c) v[c] = o[x * VE + c][i] * f;
        if (has_row(x, 4 * g + i)) store_values<VE>(a.out, a.out_dtype, head * a.dim + dims_of(x, 4 * g + i), v);
      }
    if (a.lse && g == 0) a.lse[head] = (m + __builtin_amdgcn_logf(l * UNSHIFT)) * 0.69314718055994531f;
  }
};

template <bool F16, bool F8, int DT, bool DIM, bool P8>
__global__ __launch_bounds__(64 * kWaves, DT == 256 ? 1 : 2) void attn_kernel(AttnArgs a) {
  extern __shared__ int pre[];  // [rows + 1] tiles before each row
  __shared__ int part[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per_thread = (a.rows + 64 * kWaves - 1) / (64 * kWaves);
  const int r0 = min(tid * per_thread, a.rows), r1 = min(r0 + per_thread, a.rows);
  int n = 0;
  for (int r = r0; r < r1; ++r) n += span_of(a, r).tiles;
  int sum = n;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int v = __shfl_up(sum, d);
    if (lane >= d) sum += v;
  }
  if (lane == 63) part[wave] = sum;
  __syncthreads();
  int at = sum - n;
  for (int w = 0; w < wave; ++w) at += part[w];
  for (int r = r0; r < r1; ++r) {
    pre[r] = at;
    at += span_of(a, r).tiles;
  }
  if (tid == 64 * kWaves - 1) pre[a.rows] = at;  // the last thread's sum is the total
  __syncthreads();
  const int per_row = a.kv_heads * a.groups;  // sequences of tiles of one row
  const int64_t total = (int64_t)pre[a.rows] * per_row;
  const int per = quotient(total + a.workers - 1, a.workers);
  if (blockIdx.x == 0) {  // for the join
    for (int r = tid; r <= a.rows; r += 64 * kWaves) a.prefix[r] = pre[r];
    if (tid == 0) a.prefix[a.rows + 1] = per;
  }
  const int w = __builtin_amdgcn_readfirstlane(wave) * (int)gridDim.x + (int)blockIdx.x;
  int64_t pos = (int64_t)w * per;
  const int64_t end = pos + per < total ? pos + per : total;
  if (pos >= end) return;
  int lo = 0, hi = a.rows;  // the row of pos
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if ((int64_t)pre[mid] * per_row <= pos) lo = mid;
    else hi = mid;
  }
  int r = __builtin_amdgcn_readfirstlane(lo);
  constexpr bool LK = P8;
  using T = Attn<F16, F8, DT, DIM, P8, LK>;
  __shared__ u32x4_t keys[LK ? kWaves : 1][LK ? kTile * T::CH : 1];
  T t(a, keys[LK ? wave : 0]);
  int slot = 0;
  while (pos < end) {
    const Span s = span_of(a, r);
    if (s.tiles == 0) {
      ++r;
      continue;
    }
    const int64_t in_row = pos - (int64_t)pre[r] * per_row;
    const int hg = quotient(in_row, s.tiles), first = (int)(in_row - (int64_t)hg * s.tiles);
    const int count = (int)min((int64_t)(s.tiles - first), end - pos);
    const int kvh = hg / a.groups, grp = hg - kvh * a.groups;
    t.start(r, kvh, grp);
    t.run(s, first, count);
    const bool whole = first == 0 && count == s.tiles;
    t.finish(r, kvh, grp, whole ? nullptr : partial(a, w, slot));
    slot = 1;
    pos += count;
    if (first + count == s.tiles && hg + 1 == per_row) ++r;
  }
}

// One launch for short rows: a workgroup for each (row, kv head, 16 heads), its wavefronts take equal runs of
// tiles and are merged in LDS.  Four wavefronts: of eight, half as many workgroups fit a CU (64 rows of
// 32 kv heads, up to 1024 tokens, keys not by way of LDS: 101 us, four 95).
template <class T, bool LK>
union RowsLds {
  float park[kWaves / 2][T::PARK * 64];
  u32x4_t keys[LK ? kWaves : 1][LK ? kTile * T::CH : 1];
};
template <bool F16, bool F8, int DT, bool DIM, bool P8, bool LK>
__global__ __launch_bounds__(64 * kWaves, DT == 256 ? 1 : 2) void attn_rows_kernel(AttnArgs a) {
  constexpr int WAVES = kWaves;
  using T = Attn<F16, F8, DT, DIM, P8, LK>;
  __shared__ RowsLds<T, LK> sh;
  // Workgroup i runs on XCD i % 8, each with its own L2.  Those that read the same lines follow each other on
  // one: the groups of 16 heads of a kv head, and a.near kv heads whose rows share lines.
  int unit = blockIdx.x, grp = 0;
  if (const int n = a.near * a.groups; n > 1) {
    const int set = unit / (8 * n), at = unit - set * 8 * n, k = at >> 3;
    grp = k % a.groups;
    unit = (set * 8 + (at & 7)) * a.near + k / a.groups;
    if (unit >= a.rows * a.kv_heads) return;
  }
  const int r = unit / a.kv_heads, kvh = unit - r * a.kv_heads;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Span s = span_of(a, r);
  if (s.tiles == 0) {
    const int h0 = kvh * a.group + grp * kHeads, n = min(kHeads, a.group - grp * kHeads);
    const int64_t head = (int64_t)r * a.heads + h0;
    for (int d = threadIdx.x; d < n * a.dim; d += 64 * WAVES) store_scalar(a.out, a.out_dtype, head * a.dim + d, 0.f);
    if (a.lse && (int)threadIdx.x < n) a.lse[head + threadIdx.x] = -INFINITY;
    return;
  }
  T t(a, sh.keys[LK ? wave : 0]);
  t.start(r, kvh, grp);
  const int per = (s.tiles + WAVES - 1) / WAVES, first = wave * per, count = min(per, s.tiles - first);
  if (count > 0) t.run(s, first, count);
  if constexpr (LK) __syncthreads();
#pragma unroll
  for (int half = WAVES / 2; half; half /= 2) {
    if (wave >= half && wave < 2 * half) t.park(sh.park[wave - half]);
    __syncthreads();
    if (wave < half) t.merge(sh.park[wave]);
    __syncthreads();
  }
  if (wave == 0) t.finish(r, kvh, grp, nullptr);
}

struct AttnKern {
  const void *fn, *rows_fn[2];  // rows_fn[1]: keys through LDS
  int rows_lds[2];
  std::atomic<int> residents[64];  // workgroups of a CU, by device; 0: not asked yet
};
// The kernel for head_dim at a page size; F16/F8 as above.
AttnKern& kern_bf16(int dim, bool p8);
AttnKern& kern_f16(int dim, bool p8);
AttnKern& kern_bf16_e4m3(int dim, bool p8);
AttnKern& kern_f16_e4m3(int dim, bool p8);

template <bool F16, bool F8>
AttnKern& kern_of(int dim, bool p8) {
#define MLXR_ATTN(DT, DIM, P8)                                                                                              \
  {                                                                                                                        \
    constexpr bool LK = P8;                                                                                    \
    static AttnKern k{(const void*)attn_kernel<F16, F8, DT, DIM, P8>,                                                      \
                      {(const void*)attn_rows_kernel<F16, F8, DT, DIM, P8, false>,                                         \
                       (const void*)attn_rows_kernel<F16, F8, DT, DIM, P8, LK>},                                           \
                      {(int)sizeof(RowsLds<Attn<F16, F8, DT, DIM, P8, false>, false>),                                     \
                       (int)sizeof(RowsLds<Attn<F16, F8, DT, DIM, P8, LK>, LK>)},                                          \
                      {}};                                                                                                 \
    return k;                                                                                                              \
  }
  if (dim == 64 && p8) MLXR_ATTN(64, true, true)
  if (dim == 128 && p8) MLXR_ATTN(128, true, true)
  if (dim == 256 && p8) MLXR_ATTN(256, true, true)
  if (p8) {
    if (dim < 64) MLXR_ATTN(64, false, true)
    if constexpr (!F8)
      if (dim <= 96) MLXR_ATTN(96, false, true)
    if (dim < 128) MLXR_ATTN(128, false, true)
    MLXR_ATTN(256, false, true)
  }
  if (dim <= 64) MLXR_ATTN(64, false, false)
  if constexpr (!F8)
    if (dim <= 96) MLXR_ATTN(96, false, false)
  if (dim <= 128) MLXR_ATTN(128, false, false)
  MLXR_ATTN(256, false, false)
#undef MLXR_ATTN
}

}  // namespace paged
}  // namespace mlxr
