// Attention of new tokens over what is cached and over one another: launch
// parameters, the split of the work over the grid, and the masks.  Shared by
// the 16-bit tensor-core kernel (extend_mma.cu) and the 32-bit kernel
// (extend_simt.cu).
//
// Sequence b has P_b cached tokens (in pages) and n_b new ones (packed).  The
// g query heads of a KV head are rows of one matrix, so the rows of one
// (sequence, KV head) are r = token * g + head, cut into row tiles of R rows;
// a tile reads the prefix and the new tokens up to its last one in key tiles
// of KT keys.
//
// The key tiles of all row tiles, laid end to end (each row tile with kFront
// more units in front, for its queries and its output), are cut into as many equal
// ranges as the grid has CTAs: a ragged batch, one long context and one long
// prompt all keep every SM busy for the same time, with no host knowledge of
// any length.  A row tile that crosses a cut leaves (m, l, o) pieces, which
// the combine kernel joins.
#pragma once

#include "kernels.h"

namespace adakv {

// two 32-bit operations in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

struct ExtSeq {
  int b;       // the sequence, and its
  int begin;   // first packed token
  int n;       // new tokens
  int prefix;  // cached tokens
  int slot;    // page table row
};

// A length, slot or offset that is out of range is reported and replaced by
// the nearest one that reads nothing out of bounds.
__device__ __forceinline__ ExtSeq ext_seq(const ExtParams& p, int b) {
  ExtSeq s;
  s.b = b;
  const int c0 = p.cu[b], c1 = p.cu[b + 1];
  s.begin = imin(imax(c0, 0), p.T);
  const int end = imin(imax(c1, s.begin), p.T);
  s.n = end - s.begin;
  s.prefix = 0;
  s.slot = 0;
  bool bad = c0 != s.begin || c1 != end;
  if (p.lens) {
    s.slot = p.slots ? p.slots[b] : b;
    if (s.slot < 0 || s.slot >= p.n_slots) {
      bad = true;
      s.slot = 0;
    } else {
      const int len = p.lens[s.slot];
      s.prefix = (int)(((int64_t)imax(len, 0) < p.max_prefix) ? (int64_t)imax(len, 0) : p.max_prefix);
      bad = bad || len != s.prefix;
    }
  }
  if (bad) report(p.status, ADAKV_ST_BAD_SEQ_LEN);
  return s;
}

// Page of prefix block j of a page table row; an id outside the pool is
// reported and replaced by page 0.
__device__ __forceinline__ int ext_page(const ExtParams& p, int slot, int j) {
  const int id = p.table[slot * p.table_stride + j];
  if (id >= 0 && id < p.n_pages) return id;
  report(p.status, ADAKV_ST_BAD_BLOCK_ID);
  return 0;
}

// What a row tile costs beside its key tiles, in key tiles: about 7,000 cycles
// where 128 keys take the 16-bit kernel 3,400.  (8192-token prompt: with 1 the
// CTAs that begin many short row tiles took 890 thousand cycles, the median 762
// thousand; with 2 every one takes 790 to 860 thousand.)  The 32-bit kernel, whose
// tiles are a half as large, uses it too; there, with 1, 2 and 3 (us): a 1500-token
// prompt 568, 601, 617, one of head_dim 64 309, 326, 335, trees of 1 to 64 tokens
// 58, 54, 54, 17 decode steps 253, 253, 265.
constexpr int kFront = 2;

// ---------------------------------------------------------------------------
// The cost of the row tiles in units (R = KT or R = 2 KT).
// ---------------------------------------------------------------------------
template <int R, int KT>
struct ExtCost {
  static_assert(R == KT || R == 2 * KT, "closed forms below");
  __device__ __forceinline__ static int row_tiles(int n, int g) {
    return (int)(((int64_t)n * g + R - 1) / R);
  }
  // key tiles of new tokens that row tile rt reads (those up to its last token)
  __device__ __forceinline__ static int new_tiles(int n, int g, int rt) {
    const int64_t row = ((int64_t)rt + 1) * R - 1;  // the tile's last row, and its token
    const int64_t last = (uint64_t)row >> 32 ? row / g : (int64_t)((uint32_t)row / (uint32_t)g);
    const int hi = (int)(last < n - 1 ? last : n - 1);
    return hi / KT + 1;
  }
  // sum of new_tiles over the row tiles before x: key tile j is read from row
  // tile floor(j KT g / R) on
  __device__ __forceinline__ static int64_t new_before(int n, int g, int64_t x) {
    const int64_t J = ((int64_t)n + KT - 1) / KT;
    const int64_t f = R / KT;
    const int64_t y = x * f + g - 1;
    int64_t jx = (uint64_t)y >> 32 ? y / g : (int64_t)((uint32_t)y / (uint32_t)g);
    jx = jx < J ? jx : J;
    int64_t starts = (int64_t)g * (jx * (jx - 1) / 2);
    if (f == 2) starts = (starts - ((g & 1) ? jx / 2 : 0)) / 2;
    return jx * x - starts;
  }
  __device__ __forceinline__ static int64_t before(const ExtSeq& s, int g, int64_t x) {
    return x * ((s.prefix + KT - 1) / KT + kFront) + new_before(s.n, g, x);
  }
  __device__ __forceinline__ static int64_t seq(const ExtSeq& s, int g) {
    return before(s, g, row_tiles(s.n, g));
  }
};

struct ExtStart {  // where a CTA's range begins
  int64_t units;   // of the range (0: nothing to do)
  ExtSeq s;
  int kvh, rt, off;
  int ctas;        // CTAs that have a range
};

// (64-bit division takes over 100 cycles; almost every sum here fits 32 bits)
__device__ __forceinline__ int64_t ext_div(int64_t a, int64_t b) {
  return (uint64_t)a >> 32 || (uint64_t)b >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

// One warp finds the start of CTA `c`'s range.
template <int R, int KT>
__device__ __forceinline__ ExtStart ext_locate(const ExtParams& p, int c, int grid, int lane) {
  using C = ExtCost<R, KT>;
  int64_t total = 0, own = 0;
  ExtSeq s{};
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    own = 0;
    if (b0 + lane < p.B) {
      s = ext_seq(p, b0 + lane);
      own = C::seq(s, p.g) * p.Hkv;
    }
    int64_t v = own;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    total += v;
  }
  ExtStart r{};
  r.ctas = (int)(total < grid ? total : grid);
  if (c >= r.ctas) return r;
  // c * total / ctas without overflowing: total = q ctas + m
  const int64_t q = ext_div(total, r.ctas);
  const int m = (int)(total - q * r.ctas);
  const int64_t lo = q * c + (uint32_t)(m * c) / (uint32_t)r.ctas;
  r.units = q * (c + 1) + (uint32_t)(m * (c + 1)) / (uint32_t)r.ctas - lo;
  int64_t base = 0;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    if (p.B > 32) {  // (else s and own are still those)
      own = 0;
      if (b0 + lane < p.B) {
        s = ext_seq(p, b0 + lane);
        own = C::seq(s, p.g) * p.Hkv;
      }
    }
    int64_t inc = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t t = __shfl_up_sync(~0u, inc, o);
      if (lane >= o) inc += t;
    }
    const uint32_t past = __ballot_sync(~0u, base + inc > lo);
    if (past) {
      const int l = __ffs(past) - 1;
      const int64_t at = lo - (base + __shfl_sync(~0u, inc - own, l));
      r.s.b = __shfl_sync(~0u, s.b, l);
      r.s.begin = __shfl_sync(~0u, s.begin, l);
      r.s.n = __shfl_sync(~0u, s.n, l);
      r.s.prefix = __shfl_sync(~0u, s.prefix, l);
      r.s.slot = __shfl_sync(~0u, s.slot, l);
      const int64_t per_head = C::seq(r.s, p.g);
      r.kvh = (int)ext_div(at, per_head);
      const int64_t rem = at - r.kvh * per_head;
      int x0 = 0, x1 = C::row_tiles(r.s.n, p.g);  // last x with before(x) <= rem
      while (x1 - x0 > 1) {
        const int mid = (x0 + x1) >> 1;
        if (C::before(r.s, p.g, mid) <= rem) x0 = mid; else x1 = mid;
      }
      r.rt = x0;
      r.off = (int)(rem - C::before(r.s, p.g, x0));
      return r;
    }
    base += __shfl_sync(~0u, inc, 31);
  }
  r.units = 0;
  return r;
}

// A CTA's row tiles, in order; every role of a CTA steps through the same ones.
template <int R, int KT>
struct ExtWalk {
  ExtSeq s;
  int kvh, rt;
  int k_lo, k_hi, k_all;  // this CTA's key tiles [k_lo, k_hi) of the row tile's k_all
  int p_tiles;            // the first p_tiles are the prefix's
  int take;               // units of the row tile in the range
  int64_t left;           // units of the range from this row tile on

  __device__ __forceinline__ void set(const ExtParams& p, int off) {
    p_tiles = (s.prefix + KT - 1) / KT;
    k_all = p_tiles + ExtCost<R, KT>::new_tiles(s.n, p.g, rt);
    take = (int)((int64_t)(k_all + kFront - off) < left ? k_all + kFront - off : left);
    k_lo = imax(off - kFront, 0);
    k_hi = imax(off + take - kFront, 0);
  }
  __device__ __forceinline__ void start(const ExtParams& p, const ExtStart& st) {
    left = st.units;
    if (left <= 0) return;
    s = st.s;
    kvh = st.kvh;
    rt = st.rt;
    set(p, st.off);
    // (units in front alone: the next range begins the row tile)
    if (k_lo == k_hi) left = 0;
  }
  __device__ __forceinline__ bool live() const { return left > 0; }
  __device__ __forceinline__ void next(const ExtParams& p) {
    left -= take;
    if (left <= 0) return;
    if (++rt >= ExtCost<R, KT>::row_tiles(s.n, p.g)) {
      rt = 0;
      if (++kvh >= p.Hkv) {
        kvh = 0;
        int b = s.b + 1;
        while (b < p.B) {
          s = ext_seq(p, b);
          if (s.n > 0) break;
          ++b;
        }
        if (b >= p.B) {
          left = 0;
          return;
        }
      }
    }
    set(p, 0);
    if (k_lo == k_hi) left = 0;
  }
  __device__ __forceinline__ bool begins() const { return k_lo == 0; }
  __device__ __forceinline__ bool ends() const { return k_hi == k_all; }
  __device__ __forceinline__ int rows(int g) const {
    const int64_t left_rows = (int64_t)s.n * g - (int64_t)rt * R;
    return (int)(left_rows < R ? left_rows : R);
  }
};

// Which of the new tokens [j0, j0 + 32 W) a new token sees.  Causal: those up
// to itself.  Tree: itself and its ancestors; a slot with a parent below -1 is
// unused, sees nothing and is seen by nothing.  A parent that is not an
// earlier token is reported and ends the walk.
template <int W>
__device__ __forceinline__ void ext_tree_mask(const ExtParams& p, const ExtSeq& s, int tok, int j0,
                                              uint32_t (&bits)[W]) {
#pragma unroll
  for (int w = 0; w < W; ++w) bits[w] = 0;
  const int* par = p.parents + s.begin;
  int at = tok;
  while (at >= j0) {
    const int up = par[at];
    if (up < -1) break;
    const int d = at - j0;
#pragma unroll
    for (int w = 0; w < W; ++w)
      if ((d >> 5) == w) bits[w] |= 1u << (d & 31);
    if (up >= at) {
      report(p.status, ADAKV_ST_BAD_PARENT);
      break;
    }
    at = up;
  }
}

// Is this slot of a tree in use?
__device__ __forceinline__ bool ext_live(const ExtParams& p, const ExtSeq& s, int tok) {
  return !p.parents || p.parents[s.begin + tok] >= -1;
}

// Values that are not finite.  0 times infinity is NaN, so a product over a tile
// would carry such a value of a new token to rows that do not see it.  Where a
// half or tile of new tokens has rows that see some of it and rows that do not
// (any of a tree's; a prompt's from the row tile's first token on), the kernels
// set these values to 0 in shared memory, which is rare, and add them to the
// outputs of the rows that see them afterwards: token `tok`'s columns [0, n) from
// the values v (row 0, same column) of the tokens that it sees in [lo, hi).
template <typename T, typename O>
__device__ __noinline__ void ext_add_infinite(const T* v, int64_t v_st, const int* par, int tok, int lo, int hi,
                                              O* dst, int n) {
  int at = par ? tok : imin(tok, hi - 1);
  while (at >= lo) {
    const int up = par ? par[at] : at - 1;
    if (up < -1) break;
    if (at < hi) {
      const T* row = v + at * v_st;
#pragma unroll 4
      for (int d = 0; d < n; ++d) {
        const float x = to_f32(row[d]);
        if (!(fabsf(x) < INFINITY)) dst[d] = from_f32<O>(to_f32(dst[d]) + x);
      }
    }
    if (up >= at) break;  // (reported where the masks are made)
    at = up;
  }
}

// ---------------------------------------------------------------------------
// Pieces.  A CTA leaves at most two: [0] of the row tile that began before its
// range, [1] of the row tile that ends after it (both of one tile: [0] only).
// ---------------------------------------------------------------------------
struct ExtRec {
  int tail;       // 1: piece [1] is there and begins a row tile, which the words below name
  int b, kvh, rt;
  int head;       // 1: piece [0] is there
  int head_ends;  // 1: and it is its row tile's last
  int pad[2];
};

}  // namespace adakv
