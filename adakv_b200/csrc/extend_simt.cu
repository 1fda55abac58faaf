// Attention of new tokens for 32-bit elements.
//
// One CTA of 256 threads per row tile piece: 64 rows x 64 keys, q.k as 4 x 4
// register tiles (16 x 16 threads, rows 16 apart), running maximum and sum in
// registers (each row belongs to 16 lanes of one warp), probabilities through
// shared memory, p.v as 4 x D/16 register tiles.  Row tiles of up to 16 or 32
// rows (decode steps, small trees) do one or two rows a thread: 17 decode steps
// over 200 to 5176 tokens, 64/8 heads, 253 us (four rows: 372), a tree of 8 tokens
// over 6,000, 32 rows, 63 us (four: 76).
//
// V of a key tile is copied (cp.async) while its scores are computed, K of the
// next one during its p.v; page ids are read a tile earlier still.  Rows of K
// are unpadded, their 16-byte words swapped by the row (16 rows are read at a
// time): two CTAs fit an SM at D = 128.
//
// Bound by the multiply-adds and the shared-memory reads that feed them (8
// 16-byte reads for 64 multiply-adds): 31 TFLOP/s on a 1500-token prompt of 32 /
// 8 heads of 128 (600 us), 43 % of the 72 that the SMs have at 1.9 GHz.
#include <type_traits>

#include "extend.cuh"

namespace adakv {
namespace {

constexpr int R = kExtSimtRows;
constexpr int KT = kExtSimtRows;
constexpr int kThreads = 256;

template <int D>
constexpr size_t simt_smem() {
  return sizeof(float) * (R * D + 2 * KT * D + R * KT) + 8 * R + sizeof(ExtStart);
}

template <int D>
__global__ void __launch_bounds__(kThreads, kExtSimtCtas) extend_simt_kernel(const ExtParams p) {
  constexpr int N16 = D / 4;  // 16-byte words of a row
  constexpr int NC = D / 64;
  extern __shared__ __align__(16) unsigned char raw[];
  float* sq = reinterpret_cast<float*>(raw);
  float* sk = sq + R * D;
  float* sv = sk + KT * D;
  float* sp = sv + KT * D;
  uint2* smask = reinterpret_cast<uint2*>(sp + R * KT);
  ExtStart* sstart = reinterpret_cast<ExtStart*>(smask + R);
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;

  if (tid < 32) {
    const ExtStart st = ext_locate<R, KT>(p, blockIdx.x, gridDim.x, tid);
    if (tid == 0) *sstart = st;
  }
  __syncthreads();
  ExtWalk<R, KT> w;
  w.start(p, *sstart);
  ExtRec rec{};
  const int page_mask = (1 << p.page_log2) - 1;

  const int p_swap = (ty & 1) << 2;  // a warp's two rows of probabilities lie in different banks
  constexpr int RP = kThreads / N16, NR = KT / RP;  // rows of a tile at a time, rows a thread copies
  const int c = tid % N16, r_first = tid / N16;
  for (; w.live(); w.next(p)) {
    const int rows = w.rows(p.g);
    const int row0 = w.rt * R;
    // Row r_first + i RP of key tile kt: its page, or that it is a new token (kNew), or nothing (-1).
    constexpr int kNew = 1 << 30;
    auto find = [&](int kt, int (&at)[NR]) {
      const bool cached = kt < w.p_tiles;
      const int j0 = (cached ? kt : kt - w.p_tiles) * KT;
      const int have = kt < w.k_hi ? imin(KT, (cached ? w.s.prefix : w.s.n) - j0) : 0;
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const int r = r_first + i * RP, j = j0 + r;
        at[i] = r >= have ? -1 : cached ? ext_page(p, w.s.slot, j >> p.page_log2) : ext_live(p, w.s, j) ? kNew : -1;
      }
    };
    auto copy = [&](int kt, const int (&at)[NR], bool is_v) {
      const int j0 = (kt < w.p_tiles ? kt : kt - w.p_tiles) * KT;
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const int r = r_first + i * RP, j = j0 + r;
        const float* src = static_cast<const float*>(p.q);  // (never read from where there is nothing)
        if (at[i] == kNew)
          src = is_v ? static_cast<const float*>(p.v) + (int64_t)(w.s.begin + j) * p.v_st + w.kvh * p.v_sh
                     : static_cast<const float*>(p.k) + (int64_t)(w.s.begin + j) * p.k_st + w.kvh * p.k_sh;
        else if (at[i] >= 0)
          src = is_v ? static_cast<const float*>(p.pv) + at[i] * p.pv_sp + w.kvh * p.pv_sh + (j & page_mask) * p.pv_st
                     : static_cast<const float*>(p.pk) + at[i] * p.pk_sp + w.kvh * p.pk_sh + (j & page_mask) * p.pk_st;
        cp_async16(is_v ? sv + r * D + c * 4 : sk + r * D + (c ^ (r & 7)) * 4, src + (at[i] >= 0 ? c * 4 : 0), at[i] >= 0);
      }
      cp_async_commit();
    };
    int at[NR], next[NR];
    int infinite = 0;  // (the same in every thread)
    find(w.k_lo, at);
    __syncthreads();  // (the row tile before this one is done with Q, K and V)
    for (int i = tid; i < R * N16; i += kThreads) {
      const int r = i / N16;
      const float* src = static_cast<const float*>(p.q);
      if (r < rows) {
        const int row = row0 + r, tok = row / p.g, h = w.kvh * p.g + row % p.g;
        src += (int64_t)(w.s.begin + tok) * p.q_st + h * p.q_sh + c * 4;
      }
      cp_async16(sq + r * D + c * 4, src, r < rows);
    }
    copy(w.k_lo, at, false);
    float m[4], l[4], o[4][NC * 4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
#pragma unroll
      for (int j = 0; j < NC * 4; ++j) o[i][j] = 0.f;
    }
    for (int kt = w.k_lo; kt < w.k_hi; ++kt) {
      const bool cached = kt < w.p_tiles;
      const int j0 = (cached ? kt : kt - w.p_tiles) * KT;
      const int have = imin(KT, (cached ? w.s.prefix : w.s.n) - j0);
      if (tid < R) {  // which keys of the tile row tid sees
        uint32_t bits[2] = {0u, 0u};
        if (tid < rows) {
          const int tok = (row0 + tid) / p.g;
          if (!cached && p.parents) {
            ext_tree_mask<2>(p, w.s, tok, j0, bits);
          } else if (ext_live(p, w.s, tok)) {
            const int see = cached ? have : imin(have, tok - j0 + 1);
            bits[0] = see >= 32 ? ~0u : see > 0 ? (1u << see) - 1u : 0u;
            bits[1] = see >= 64 ? ~0u : see > 32 ? (1u << (see - 32)) - 1u : 0u;
          }
        }
        smask[tid] = make_uint2(bits[0], bits[1]);
      }
      cp_async_wait_all();
      __syncthreads();  // K is there, and everyone is done with V of the tile before
      copy(kt, at, true);
      find(kt + 1, next);
      // with as many of the four rows of a thread as the row tile needs
      auto tile = [&](auto rows16) {
        constexpr int NI = decltype(rows16)::value;
        // scores: rows ty + 16 i, keys tx + 16 j
        // (two products an instruction: even and odd elements of the head dim)
        float2 s2[NI][4] = {};
#pragma unroll 8
        for (int d = 0; d < D; d += 4) {
          float4 a[NI], b[4];
#pragma unroll
          for (int i = 0; i < NI; ++i) a[i] = *reinterpret_cast<const float4*>(sq + (ty + 16 * i) * D + d);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            b[j] = *reinterpret_cast<const float4*>(sk + (tx + 16 * j) * D + (((d >> 2) ^ (tx & 7)) << 2));
#pragma unroll
          for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              s2[i][j] = fma2(make_float2(a[i].x, a[i].y), make_float2(b[j].x, b[j].y), s2[i][j]);
              s2[i][j] = fma2(make_float2(a[i].z, a[i].w), make_float2(b[j].z, b[j].w), s2[i][j]);
            }
        }
        float s[NI][4];
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[i][j] = s2[i][j].x + s2[i][j].y;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const uint2 see = smask[ty + 16 * i];
          float top = m[i];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t word = j < 2 ? see.x : see.y;
            const bool on = (word >> ((tx + 16 * j) & 31)) & 1u;
            s[i][j] = on ? s[i][j] * p.scale : -INFINITY;
            top = fmaxf(top, s[i][j]);
          }
#pragma unroll
          for (int x = 1; x < 16; x <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, x));
          // a row that has seen nothing yet keeps m at -inf: subtract 0 there
          const float ref = top == -INFINITY ? 0.f : top;
          const float keep = exp2f(m[i] - ref);
          m[i] = top;
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s[i][j] = exp2f(s[i][j] - ref);
            sum += s[i][j];
            sp[(ty + 16 * i) * KT + ((tx + 16 * j) ^ p_swap)] = s[i][j];
          }
          l[i] = l[i] * keep + sum;
#pragma unroll
          for (int j = 0; j < NC * 4; ++j) o[i][j] *= keep;
        }
        cp_async_wait_all();
        if (!cached && (p.parents ? w.s.n > 1 : j0 + have - 1 > row0 / p.g)) {  // (ext_add_infinite)
          uint32_t bad = 0;  // the sign bit: an exponent of all ones in what this thread has copied
          auto sign = [](uint32_t x) { return (x & 0x7F800000u) + 0x00800000u; };
#pragma unroll
          for (int i = 0; i < NR; ++i) {
            const uint4 x = *reinterpret_cast<const uint4*>(sv + (r_first + i * RP) * D + c * 4);
            bad |= sign(x.x) | sign(x.y) | sign(x.z) | sign(x.w);
          }
          if (bad >> 31) {
#pragma unroll 1
            for (int i = 0; i < NR * 4; ++i) {
              float* x = sv + (r_first + (i >> 2) * RP) * D + c * 4 + (i & 3);
              if (!(fabsf(*x) < INFINITY)) *x = 0.f;
            }
          }
          infinite |= __syncthreads_or(bad >> 31);
        } else {
          __syncthreads();  // V is there, and everyone is done with K
        }
        // (none behind the last tile: two asynchronous copies to one place have no
        // order, and the next row tile's K goes there without a wait in between)
        if (kt + 1 < w.k_hi) copy(kt + 1, next, false);
#pragma unroll
        for (int i = 0; i < NR; ++i) at[i] = next[i];
#pragma unroll 4
        for (int j = 0; j < KT; j += 4) {
          float4 a[NI];
#pragma unroll
          for (int i = 0; i < NI; ++i) a[i] = *reinterpret_cast<const float4*>(sp + (ty + 16 * i) * KT + (j ^ p_swap));
#pragma unroll
          for (int jj = 0; jj < 4; ++jj)
#pragma unroll
            for (int c = 0; c < NC; ++c) {
              const float4 b = *reinterpret_cast<const float4*>(sv + (j + jj) * D + c * 64 + tx * 4);
#pragma unroll
              for (int i = 0; i < NI; ++i) {
                const float x = jj == 0 ? a[i].x : jj == 1 ? a[i].y : jj == 2 ? a[i].z : a[i].w;
                float2* y = reinterpret_cast<float2*>(&o[i][c * 4]);
                y[0] = fma2(make_float2(x, x), make_float2(b.x, b.y), y[0]);
                y[1] = fma2(make_float2(x, x), make_float2(b.z, b.w), y[1]);
              }
            }
        }
      };
      if (rows <= 16) tile(std::integral_constant<int, 1>{});
      else if (rows <= 32) tile(std::integral_constant<int, 2>{});
      else tile(std::integral_constant<int, 4>{});
    }
    const bool whole = w.begins() && w.ends();
    const int piece = w.begins() ? 1 : 0;
    if (!whole) {
      if (piece) {
        rec.tail = 1;
        rec.b = w.s.b;
        rec.kvh = w.kvh;
        rec.rt = w.rt;
      } else {
        rec.head = 1;
        rec.head_ends = w.ends();
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int x = 1; x < 16; x <<= 1) l[i] += __shfl_xor_sync(~0u, l[i], x);
      const int r = ty + 16 * i;
      if (r >= rows) continue;
      if (l[i] == 0.f) {  // selected, not multiplied: V may be infinite where others see it
#pragma unroll
        for (int j = 0; j < NC * 4; ++j) o[i][j] = 0.f;
      }
      if (whole) {
        const int row = row0 + r, tok = w.s.begin + row / p.g, h = w.kvh * p.g + row % p.g;
        const float inv = l[i] != 0.f ? 1.f / l[i] : 0.f;  // (a NaN sum stays one)
        float* dst = static_cast<float*>(p.out) + (int64_t)tok * p.o_st + h * p.o_sh;
#pragma unroll
        for (int c = 0; c < NC; ++c)
          *reinterpret_cast<float4*>(dst + c * 64 + tx * 4) =
              make_float4(o[i][c * 4] * inv, o[i][c * 4 + 1] * inv, o[i][c * 4 + 2] * inv, o[i][c * 4 + 3] * inv);
        if (p.lse && tx == 0)
          p.lse[(int64_t)tok * p.Hq + h] = l[i] != 0.f ? (m[i] + log2f(l[i])) * 0.69314718055994531f : -INFINITY;
      } else {
        const int64_t at = ((int64_t)blockIdx.x * 2 + piece) * R + r;
#pragma unroll
        for (int c = 0; c < NC; ++c)
          *reinterpret_cast<float4*>(p.part_o + at * D + c * 64 + tx * 4) =
              make_float4(o[i][c * 4], o[i][c * 4 + 1], o[i][c * 4 + 2], o[i][c * 4 + 3]);
        if (tx == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m[i], l[i]);
      }
      if (infinite) {
        const int row = row0 + r, tok = row / p.g, h = w.kvh * p.g + row % p.g;
        const float* v = static_cast<const float*>(p.v) + (int64_t)w.s.begin * p.v_st + w.kvh * p.v_sh + tx * 4;
        const int* par = p.parents ? p.parents + w.s.begin : nullptr;
        const int lo = imax(imax(w.k_lo - w.p_tiles, 0) * KT, par ? 0 : (row0 / p.g) & ~(KT - 1));
        const int hi = imin(imax(w.k_hi - w.p_tiles, 0) * KT, w.s.n);
        float* dst = (whole ? static_cast<float*>(p.out) + (int64_t)(w.s.begin + tok) * p.o_st + h * p.o_sh
                            : p.part_o + (((int64_t)blockIdx.x * 2 + piece) * R + r) * D) + tx * 4;
#pragma unroll 1
        for (int c = 0; c < NC; ++c) ext_add_infinite(v + c * 64, p.v_st, par, tok, lo, hi, dst + c * 64, 4);
      }
    }
  }
  if (tid == 0) p.rec[blockIdx.x] = rec;
}

}  // namespace

cudaError_t ext_simt_init() {
  cudaError_t e = cudaFuncSetAttribute(extend_simt_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)simt_smem<64>());
  if (e != cudaSuccess) return e;
  return cudaFuncSetAttribute(extend_simt_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              (int)simt_smem<128>());
}

cudaError_t launch_extend_simt(const ExtParams& p, int D, int grid, cudaStream_t st) {
  if (D == 64) extend_simt_kernel<64><<<grid, kThreads, simt_smem<64>(), st>>>(p);
  else extend_simt_kernel<128><<<grid, kThreads, simt_smem<128>(), st>>>(p);
  return cudaGetLastError();
}

}  // namespace adakv
