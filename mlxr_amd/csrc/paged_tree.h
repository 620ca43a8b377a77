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
// neighbouring 16 x 16 tiles of S^T, as the first product leaves them.  P enters in 16-bit parts: f16 (and the values of an
// e4m3 cache, exact in f16) two parts, 22 bits; bf16 three, 24 bits, for fp32 outputs, two, 16 bits, for 16-bit outputs, whose
// own half step (2^-9, 2^-12) is far larger than what that leaves out of each weight (2^-17).
//
// A tile of TOK tokens goes memory -> registers -> LDS, one tile ahead: while tile t is multiplied, t + 1 is on its way to
// registers; it is written to the other half of LDS before the tile's one barrier.  Four wavefronts are WQ groups of
// columns times WT groups of the tile's tokens (merged at the end), by the columns that a row has on average.
//
// The tiles of all (row, kv head, QB columns) are dealt to the workgroups of a launch that fills the device in equal
// contiguous runs; a run that covers all of its columns' tiles writes the output, others leave (m, sum, unnormalized o) in
// the workspace, at most two a workgroup, and a second launch joins them.  Short rows, or many: a workgroup for each
// (row, kv head, QB columns).
#pragma once
#include <cfloat>

#include "paged_attn.h"

namespace mlxr {
namespace tree {

using paged::load_words;
using paged::store_values;
using paged::widen;

constexpr int kThreads = 256;
constexpr int kMaxRows = MLXR_PAGED_MAX_ROWS;

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
  Divisor by_page, by_group;
  int workers;
  float scale;  // times log2(e)
};

// A row: its drafted tokens are n tokens from `start` on, the last of its len cached ones.
struct Row {
  int start, n, len, context, blocks, tiles;
};
__device__ __forceinline__ Row row_of(const Args& a, int r) {
  Row w;
  const int64_t most = (int64_t)a.width * a.page;
  const int s0 = min(max(a.starts[r], 0), a.tokens), s1 = min(max(a.starts[r + 1], s0), a.tokens);
  const int len = a.lens[r];
  w.start = s0;
  w.n = s1 - s0;
  w.context = len - w.n;  // may be negative: the first nodes are then not in the cache
  w.len = len < 0 ? 0 : len > most ? (int)most : len;
  w.blocks = (int)(((int64_t)w.n * a.group + a.qb - 1) / a.qb);
  w.tiles = (w.len + a.tok - 1) / a.tok;
  return w;
}

// Floats of a cut run's partial sums: QB rows of dim, then m and sum of each.
__host__ __device__ constexpr int partial_floats(int qb, int dim) { return qb * dim + 2 * qb; }

// The 64 bits from bit `at` on of what node i sees: 1s before its row's drafts (at < 0), the mask's words, then 0s.
__device__ __forceinline__ uint64_t mask_word(const Args& a, const uint64_t* mask, int w) {
  return w < 0 ? ~0ull : w < a.words ? mask[w] : 0ull;
}
__device__ __forceinline__ uint64_t seen(const Args& a, int token, int i, int at) {
  if (!a.mask) {
    const int more = i - at;  // the last bit that counts
    return more < 0 ? 0ull : more >= 63 ? ~0ull : (2ull << more) - 1;
  }
  const uint64_t* m = a.mask + (int64_t)token * a.words;
  const int w = at >> 6, s = at & 63;
  const uint64_t lo = mask_word(a, m, w);
  return s ? lo >> s | mask_word(a, m, w + 1) << (64 - s) : lo;
}

// Two weights in PARTS 16-bit parts that add up to them (the last rounded), none negative nor a later one 0: an infinite
// value then gives an infinite output as a weight in one piece does, not NaN.
template <bool P16, int PARTS>
__device__ __forceinline__ void split_parts(float p0, float p1, uint32_t (&out)[PARTS]) {
  auto floor2 = [](uint32_t w) { return paged::pair_max(w, P16 ? 0x00010001u : 0x00800080u); };
  if constexpr (P16) {
    static_assert(PARTS == 2, "f16: two parts");
    const uint32_t hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(p0, p1));
    out[0] = hi;
    out[1] = floor2(pack2<true>(p0 - unpack<true>(hi, 0), p1 - unpack<true>(hi, 1)));
  } else {
#pragma unroll
    for (int n = 0; n < PARTS - 1; ++n) {  // each the upper half of what is left
      const uint32_t b0 = __builtin_bit_cast(uint32_t, p0), b1 = __builtin_bit_cast(uint32_t, p1);
      const uint32_t w = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
      out[n] = n ? floor2(w) : w;
      p0 -= __builtin_bit_cast(float, b0 & 0xffff0000u);
      p1 -= __builtin_bit_cast(float, b1 & 0xffff0000u);
    }
    out[PARTS - 1] = floor2(pack2<false>(p0, p1));
  }
}

// A 16-bit value that is infinite or NaN; a word of two with those cleared.
template <bool F16>
__device__ __forceinline__ bool odd_half(uint32_t h) {
  constexpr uint32_t E = F16 ? 0x7c00u : 0x7f80u;
  return (h & E) == E;
}
template <bool F16>
__device__ __forceinline__ uint32_t clean2(uint32_t w) {
  if (odd_half<F16>(w)) w &= 0xffff0000u;
  if (odd_half<F16>(w >> 16)) w &= 0x0000ffffu;
  return w;
}

template <bool F16, bool F8, int DT, int WQ, int WT, int CW, int PARTS>
struct Kern {
  static constexpr bool P16 = F16 || F8;                      // the second product's type, f16 or else bf16
  static constexpr int TPW = WT == 1 && DT < 256 ? 64 : 32;   // tokens of a tile and wavefront
  static constexpr int TOK = TPW * WT, QB = 16 * CW * WQ;
  static constexpr int NT = TPW / 16, KT = TPW / 32, KS = DT / 32, ND = DT / 16;
  static constexpr int CH = DT / 8;                           // 16-byte pieces of a row in LDS
  static constexpr int CG = F8 ? DT / 16 : DT / 8;            // and in memory
  static constexpr int NL = TOK * CG / kThreads;              // loads of a thread, tile and store
  static constexpr int SETS = (TOK + 63) / 64;
  static constexpr int STORE = TOK * DT * 2;                  // bytes of a tile's keys or values in LDS
  static constexpr int PARK = (4 * ND + 2) * CW * 256;        // bytes of a wavefront's sums
  static constexpr int LDS = 4 * STORE > (WT > 1 ? WQ * WT / 2 * PARK : 0) ? 4 * STORE : WQ * WT / 2 * PARK;
  static constexpr float SHIFT = P16 ? 14.f : 0.f;            // f16: weights down to 2^-28 stay normal numbers
  static constexpr float UNSHIFT = P16 ? 0x1p-14f : 1.f;

  // Place of 16-byte piece c of token t's key: the 16 rows of an operand's read lie in different banks.
  static __device__ __forceinline__ int key_place(int t, int c) {
    return t * DT * 2 + (CH >= 16 ? c ^ (t & 15) : c ^ (t >> 1 & 7)) * 16;
  }
  // Place of 16 dims (32 bytes) p of token t's value: the four tokens of two lane groups' transposing read likewise.
  static __device__ __forceinline__ int value_place(int t, int p) {
    return t * DT * 2 + (ND >= 8 ? p ^ (t & 7) : p ^ (t >> 1 & 3)) * 32;
  }
};

template <bool F16, bool F8, int DT, int WQ, int WT, int CW, int PARTS>
__global__ __launch_bounds__(kThreads, DT == 256 ? 1 : 2) void tree_kernel(Args a) {
  using T = Kern<F16, F8, DT, WQ, WT, CW, PARTS>;
  constexpr int NT = T::NT, KT = T::KT, KS = T::KS, ND = T::ND, NL = T::NL, CG = T::CG, TOK = T::TOK;
  constexpr bool P16 = T::P16;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wq = wave / WT, wt = wave - wq * WT, g = lane >> 4, col = lane & 15;

  // ---- this workgroup's run of tiles
  int64_t* pre = (int64_t*)(lds + T::LDS);  // [rows + 1] before each row: tiles, or (not cut) blocks of columns
  int64_t* part = pre + a.rows + 1;         // [4]
  const bool cut = a.ws != nullptr;
  auto weight = [&](const Row& w) { return (int64_t)a.kv_heads * w.blocks * (cut ? w.tiles : 1); };
  {
    const int per_thread = (a.rows + kThreads - 1) / kThreads;
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
    for (int r = r0; r < r1; ++r) {
      pre[r] = at;
      at += weight(row_of(a, r));
    }
    if (tid == kThreads - 1) pre[a.rows] = at;
    __syncthreads();
  }
  // tokens behind the last row's: zeros
  {
    const int from = min(max(a.starts[a.rows], 0), a.tokens);
    const int64_t first = (int64_t)from * a.heads * a.dim, count = (int64_t)(a.tokens - from) * a.heads * a.dim;
    const int64_t id = (int64_t)blockIdx.x * kThreads + tid, step = (int64_t)gridDim.x * kThreads;
    for (int64_t i = id; i < count / 8; i += step) {
      const float z[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      store_values<8>(a.out, a.out_dtype, first + 8 * i, z);
    }
    if (a.lse)
      for (int64_t i = id; i < (int64_t)(a.tokens - from) * a.heads; i += step) a.lse[(int64_t)from * a.heads + i] = -INFINITY;
  }
  const int64_t total = pre[a.rows];
  const int64_t per = cut ? (total + a.workers - 1) / a.workers : 1;
  if (cut && blockIdx.x == 0) {
    for (int r = tid; r <= a.rows; r += kThreads) a.prefix[r] = pre[r];
    if (tid == 0) a.prefix[a.rows + 1] = per;
  }
  // workgroup id % 8 is the XCD: each takes neighbouring runs, which read the same keys and values
  const int nb = (int)gridDim.x, x = (int)blockIdx.x & 7, each = nb >> 3, more = nb & 7;
  const int w = x * each + min(x, more) + ((int)blockIdx.x >> 3);
  int64_t pos = (int64_t)w * per;
  const int64_t end = pos + per < total ? pos + per : total;
  if (pos >= end) return;
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
    const int unit = (int)(cut ? in_row / row.tiles : in_row);
    const int first = cut ? (int)(in_row - (int64_t)unit * row.tiles) : 0;
    const int count = cut ? (int)min((int64_t)(row.tiles - first), end - pos) : row.tiles;
    const int kvh = unit / row.blocks, block = unit - kvh * row.blocks;
    const int32_t* trow = a.table + (int64_t)r * a.table_stride;
    const uint8_t *kh = a.k + (int64_t)kvh * a.k_head, *vh = a.v + (int64_t)kvh * a.v_head;
    const float sc = a.scale * (a.k_scale ? a.k_scale[kvh] : 1.f);

    // columns of this wavefront: (node, head) pairs
    int node[CW], head[CW];
    bool has[CW];
    u32x4_t q[CW][KS];
#pragma unroll
    for (int j = 0; j < CW; ++j) {
      const int c = block * T::QB + (wq * CW + j) * 16 + col;
      has[j] = c < row.n * a.group;
      node[j] = has[j] ? a.by_group.quotient(c) : 0;
      head[j] = kvh * a.group + (has[j] ? c - node[j] * a.group : 0);
      const uint16_t* p = a.q + (int64_t)(row.start + node[j]) * a.q_token + (int64_t)head[j] * a.q_head;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int d = 32 * s + 8 * g;
        q[j][s] = has[j] && d < a.dim ? *(const u32x4_t*)(p + d) : u32x4_t{0, 0, 0, 0};
      }
    }
    f32x4_t o[ND][CW];
    float m[CW], l[CW];
    bool counts[CW];  // some token of the column counts
#pragma unroll
    for (int j = 0; j < CW; ++j) {
      m[j] = -INFINITY, l[j] = 0.f, counts[j] = false;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d][j] = f32x4_t{0, 0, 0, 0};
    }

    // ---- a tile's way to LDS
    u32x4_t kr[NL], vr[NL];
    int id[T::SETS];     // page of token `lane` (+ 64) of the tile, or -1
    uint64_t live[T::SETS], next_live[T::SETS];
    auto pages_of = [&](int t0) {
#pragma unroll
      for (int s = 0; s < T::SETS; ++s) {
        const int t = t0 + 64 * s + lane;
        const int e = trow[a.by_page.quotient(min(t, row.len - 1))];
        id[s] = t < row.len && 64 * s + lane < TOK && (uint32_t)e < (uint32_t)a.pages ? e : -1;
      }
    };
    auto load = [&](int t0) {  // unconditional loads: of page 0 where a token does not count
#pragma unroll
      for (int s = 0; s < T::SETS; ++s) next_live[s] = __ballot(id[s] >= 0);
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int at = i * kThreads + tid, t = at / CG, c = at - t * CG;
        const int pg = __shfl(id[(i * kThreads / CG) >> 6], t & 63);
        const int p = t0 + t, in = p - a.by_page.quotient(p) * a.page;
        const bool ok = pg >= 0;
        const int64_t piece = c * (F8 ? 16 : 8) < a.dim ? 16 * c : 0;
        kr[i] = *(const u32x4_t*)(kh + (ok ? pg * a.k_page + in * a.k_token : 0) + piece);
        vr[i] = *(const u32x4_t*)(vh + (ok ? pg * a.v_page + in * a.v_token : 0) + piece);
      }
    };
    auto store = [&](int half) {
      uint8_t *ks = lds + half * 2 * T::STORE, *vs = ks + T::STORE;
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int at = i * kThreads + tid, t = at / CG, c = at - t * CG;
        // zeros for values of tokens that do not count (their bits may be NaN, their weight is 0) and past the head's dims
        const bool in = c * (F8 ? 16 : 8) < a.dim, ok = in && (next_live[(i * kThreads / CG) >> 6] >> (t & 63) & 1);
        const u32x4_t zero = {0, 0, 0, 0}, kv = in ? kr[i] : zero, vv = ok ? vr[i] : zero;
        if constexpr (F8) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t k0 = kv[2 * h], k1 = kv[2 * h + 1], v0 = vv[2 * h], v1 = vv[2 * h + 1];
            *(u32x4_t*)(ks + T::key_place(t, 2 * c + h)) = u32x4_t{widen<F16, false>(k0), widen<F16, true>(k0), widen<F16, false>(k1), widen<F16, true>(k1)};
            *(u32x4_t*)(vs + T::value_place(t, c) + 16 * h) = u32x4_t{widen<P16, false>(v0), widen<P16, true>(v0), widen<P16, false>(v1), widen<P16, true>(v1)};
          }
        } else {
          *(u32x4_t*)(ks + T::key_place(t, c)) = kv;
          *(u32x4_t*)(vs + T::value_place(t, c >> 1) + 16 * (c & 1)) = vv;
        }
      }
#pragma unroll
      for (int s = 0; s < T::SETS; ++s) live[s] = next_live[s];
    };

    const int base = first * TOK, stop = (first + count) * TOK;
    if (count > 0) {  // a row without tokens has no tile
      pages_of(base);
      load(base);
      __syncthreads();  // the run before may still be read
      store(0);
      if (count > 1) {
        pages_of(base + TOK);
        load(base + TOK);
      }
      __syncthreads();
    }
    int half = 0;
    for (int t0 = base; t0 < stop; t0 += TOK) {
      const bool further = t0 + 2 * TOK < stop;
      if (further) pages_of(t0 + 2 * TOK);
      const uint8_t *ks = lds + half * 2 * T::STORE, *vs = ks + T::STORE;
      const int mine = wt * T::TPW;  // this wavefront's tokens of the tile
      f32x4_t s[NT][CW];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int j = 0; j < CW; ++j) s[i][j] = f32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const u32x4_t kf = *(const u32x4_t*)(ks + T::key_place(mine + 16 * i + col, 4 * k + g));
#pragma unroll
          for (int j = 0; j < CW; ++j) s[i][j] = mfma16<F16>(kf, q[j][k], s[i][j]);
        }
      }
      uint64_t valid = (T::SETS > 1 && mine >= 64 ? live[T::SETS - 1] : live[0]) >> (mine & 63);
      if constexpr (T::TPW < 64) valid &= (1ull << T::TPW) - 1;
      constexpr uint64_t ALL = T::TPW < 64 ? (1ull << T::TPW) - 1 : ~0ull;
      const bool plain = t0 + TOK <= row.context && valid == ALL;
      // A value that is infinite or NaN counts for the columns that see its token only, but 0 times it would reach all: where
      // a tile that is not seen by all holds one, the products take 0 for it, and it is added to its columns by hand.
      bool odd = false;
      if (!plain) {
#pragma unroll 1
        for (int i = lane; i < T::TPW * T::CH; i += 64) {
          const u32x4_t w = *(const u32x4_t*)(vs + mine * DT * 2 + 16 * i);
#pragma unroll
          for (int k = 0; k < 4; ++k) odd |= odd_half<P16>(w[k]) || odd_half<P16>(w[k] >> 16);
        }
        odd = __ballot(odd) != 0;
      }
      u32x4_t p[KT][CW][PARTS];
#pragma unroll
      for (int j = 0; j < CW; ++j) {
        float v[NT][4], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[i][e] = s[i][j][e] * sc;
        if (!plain) {
          const uint64_t bits = (seen(a, row.start + node[j], node[j], t0 + mine - row.context) & valid) >> (4 * g);
          counts[j] |= bits != 0;
#pragma unroll
          for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][e] = bits >> (16 * i + e) & 1 ? v[i][e] : -INFINITY;
        } else {
          counts[j] = true;
        }
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) top = fmaxf(top, v[i][e]);
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float m_new = fmaxf(m[j], top);
        const float ref = m_new == -INFINITY ? 0.f : m_new;  // nothing but -inf so far: p = 0, not NaN
        if (__ballot(m_new != m[j])) {
          const float alpha = __builtin_amdgcn_exp2f(m[j] - ref);
          m[j] = m_new;
          l[j] *= alpha;
#pragma unroll
          for (int d = 0; d < ND; ++d) o[d][j] *= alpha;
        }
        const float off = T::SHIFT - ref;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float p0 = __builtin_amdgcn_exp2f(v[i][2 * h] + off), p1 = __builtin_amdgcn_exp2f(v[i][2 * h + 1] + off);
            sum += p0 + p1;
            uint32_t out[PARTS];
            split_parts<P16, PARTS>(p0, p1, out);
#pragma unroll
            for (int n = 0; n < PARTS; ++n) p[i >> 1][j][n][2 * (i & 1) + h] = out[n];
          }
        l[j] += sum;
      }
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          typedef __attribute__((ext_vector_type(4))) short s16x4_t;
          typedef __attribute__((address_space(3))) s16x4_t* lds_p;
          u32x2_t v[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            // rows 4 g .. 4 g + 3 of 16 tokens, eight bytes a lane; the read gives each lane its dim of the four
            const int t = mine + 32 * k + 16 * h + 4 * g + (col >> 2);
            v[h] = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                   (lds_p)(vs + T::value_place(t, d) + 8 * (col & 3))));
          }
          u32x4_t vf = {v[0][0], v[0][1], v[1][0], v[1][1]};
          if (odd)
#pragma unroll
            for (int n = 0; n < 4; ++n) vf[n] = clean2<P16>(vf[n]);
#pragma unroll
          for (int j = 0; j < CW; ++j)
#pragma unroll
            for (int n = PARTS - 1; n >= 0; --n) o[d][j] = mfma16<P16>(vf, p[k][j][n], o[d][j]);
        }
      if (odd) {
#pragma unroll
        for (int j = 0; j < CW; ++j) {
          const uint64_t bits = seen(a, row.start + node[j], node[j], t0 + mine - row.context) & valid;
#pragma unroll 1
          for (int t = 0; t < T::TPW; ++t)
#pragma unroll
            for (int d = 0; d < ND; ++d) {
              const u32x2_t v = *(const u32x2_t*)(vs + T::value_place(mine + t, d) + 8 * g);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t h = v[e >> 1] >> (16 * (e & 1)) & 0xffffu;
                if (odd_half<P16>(h) && (bits >> t & 1)) o[d][j][e] += unpack<P16>(h, 0);
              }
            }
        }
      }
      if (t0 + TOK < stop) {
        half ^= 1;
        store(half);
        if (further) load(t0 + 2 * TOK);
        __syncthreads();
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
    // ---- wavefronts of the same columns
    if constexpr (WT > 1) {
      __syncthreads();
#pragma unroll
      for (int step = WT / 2; step; step /= 2) {
        float* at = (float*)lds + (wq * (WT / 2) + (wt < step ? wt : wt - step)) * (T::PARK / 4) + lane;
        if (wt >= step && wt < 2 * step) {
#pragma unroll
          for (int j = 0; j < CW; ++j) {
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
              for (int e = 0; e < 4; ++e) at[((j * ND + d) * 4 + e) * 64] = o[d][j][e];
            at[(4 * ND * CW + 2 * j) * 64] = m[j];
            at[(4 * ND * CW + 2 * j + 1) * 64] = l[j];
          }
        }
        __syncthreads();
        if (wt < step) {
#pragma unroll
          for (int j = 0; j < CW; ++j) {
            const float m2 = at[(4 * ND * CW + 2 * j) * 64], l2 = at[(4 * ND * CW + 2 * j + 1) * 64];
            const float mx = fmaxf(m[j], m2), ref = mx == -INFINITY ? 0.f : mx;
            const float f = __builtin_amdgcn_exp2f(m[j] - ref), f2 = __builtin_amdgcn_exp2f(m2 - ref);
            m[j] = mx;
            l[j] = l[j] * f + l2 * f2;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[d][j][e] = o[d][j][e] * f + at[((j * ND + d) * 4 + e) * 64] * f2;
          }
        }
        __syncthreads();
      }
    }
    // ---- outputs, or this run's part of them
    const bool whole = first == 0 && count == row.tiles;
    if (wt == 0) {
      float* sums = whole ? nullptr : a.ws + ((int64_t)w * 2 + slot) * partial_floats(T::QB, a.dim);
#pragma unroll
      for (int j = 0; j < CW; ++j) {
        if (!has[j]) continue;
        const int c = (wq * CW + j) * 16 + col;
        if (sums) {
#pragma unroll
          for (int d = 0; d < ND; ++d)
            if (16 * d + 4 * g < a.dim) *(f32x4_t*)(sums + (int64_t)c * a.dim + 16 * d + 4 * g) = o[d][j] * T::UNSHIFT;
          if (g == 0) {
            float* st = sums + (int64_t)T::QB * a.dim + 2 * c;
            st[0] = m[j];
            st[1] = l[j] * T::UNSHIFT;
          }
        } else {
          const int64_t at = (int64_t)(row.start + node[j]) * a.heads + head[j];
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
    pos += count;
    if (pos >= pre[r + 1]) ++r;
  }
}

struct TreeKern {
  const void* fn;
  int qb, tok, lds;
  std::atomic<int>* residents;  // workgroups of a CU, by device; 0: not asked yet
};

// The kernel for head_dim and about `columns` columns of a row; three: P in three parts where its type is bf16.
TreeKern kern_bf16(int dim, int columns, bool three);
TreeKern kern_f16(int dim, int columns, bool three);
TreeKern kern_bf16_e4m3(int dim, int columns, bool three);
TreeKern kern_f16_e4m3(int dim, int columns, bool three);

template <bool F16, bool F8, int DT, int WQ, int WT, int CW, int PARTS>
TreeKern kern_t() {
  using T = Kern<F16, F8, DT, WQ, WT, CW, PARTS>;
  static std::atomic<int> residents[64];
  return TreeKern{(const void*)tree_kernel<F16, F8, DT, WQ, WT, CW, PARTS>, T::QB, T::TOK, T::LDS, residents};
}
template <bool F16, bool F8, int PARTS>
TreeKern kern_of(int dim, int columns) {
  if (dim > 128) return columns > 32 ? kern_t<F16, F8, 256, 4, 1, 1, PARTS>() : kern_t<F16, F8, 256, 2, 2, 1, PARTS>();
  if (dim > 64) {
    if (columns > 64) return kern_t<F16, F8, 128, 4, 1, 2, PARTS>();
    if (columns > 32) return kern_t<F16, F8, 128, 2, 2, 2, PARTS>();
    if (columns > 16) return kern_t<F16, F8, 128, 1, 4, 2, PARTS>();
    return kern_t<F16, F8, 128, 1, 4, 1, PARTS>();
  }
  if (columns > 64) return kern_t<F16, F8, 64, 4, 1, 2, PARTS>();
  if (columns > 32) return kern_t<F16, F8, 64, 2, 2, 2, PARTS>();
  if (columns > 16) return kern_t<F16, F8, 64, 1, 4, 2, PARTS>();
  return kern_t<F16, F8, 64, 1, 4, 1, PARTS>();
}

}  // namespace tree
}  // namespace mlxr
