// Joins the pieces of row tiles that the attention of new tokens has split.
#include "extend.cuh"

namespace adakv {
namespace {

constexpr int kRowsPerWarp = 2, kWarps = 4;

// Joins the pieces of each row tile that begins in one CTA's range and goes on
// into the next ones: out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i.
// Block (c, y): the row tile that CTA c began, two rows a warp.  A lane holds
// the weight of one piece (32 at a time), then E columns of every piece: the
// loads of a step do not wait for one another.  (One piece after the other took
// 17.5 us where 19 pieces meet, one token over 32K.)
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(32 * kWarps) extend_combine_kernel(const ExtParams p, int grid) {
  pdl_wait();
  const int c = blockIdx.x;
  const ExtRec rec = p.rec[c];
  if (!rec.tail) return;
  const int lane = threadIdx.x & 31;
  const int r0 = (blockIdx.y * kWarps + (threadIdx.x >> 5)) * kRowsPerWarp;
  const int begin = imin(imax(p.cu[rec.b], 0), p.T), end = imin(imax(p.cu[rec.b + 1], begin), p.T);
  const int64_t rows = (int64_t)(end - begin) * p.g - (int64_t)rec.rt * ROWS;
  if (r0 >= rows) return;
  // the pieces: [1] of CTA c, then [0] of the next ones up to the last
  int n = 1;
  while (c + n < grid) {
    const int i = c + n + lane;
    const bool last = i < grid && p.rec[i].head_ends;
    const uint32_t ends = __ballot_sync(~0u, last);
    if (ends) {
      n += __ffs(ends);
      break;
    }
    n += 32;
  }
  n = imin(n, grid - c);
  constexpr int E = D / 32;
  float M[kRowsPerWarp], L[kRowsPerWarp], o[kRowsPerWarp][E] = {};
#pragma unroll
  for (int x = 0; x < kRowsPerWarp; ++x) {
    M[x] = -INFINITY;
    L[x] = 0.f;
  }
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int i = i0 + lane;
    const int64_t at = ((int64_t)(c + i) * 2 + (i == 0)) * ROWS + r0;
    float2 ml[kRowsPerWarp];
#pragma unroll
    for (int x = 0; x < kRowsPerWarp; ++x)
      ml[x] = i < n && r0 + x < rows ? *reinterpret_cast<const float2*>(p.part_ml + (at + x) * 2)
                                     : make_float2(-INFINITY, 0.f);
    float w[kRowsPerWarp];
#pragma unroll
    for (int x = 0; x < kRowsPerWarp; ++x) {
      const float top = fmaxf(M[x], warp_max(ml[x].x));
      const float ref = top == -INFINITY ? 0.f : top;
      const float keep = exp2f(M[x] - ref);
      w[x] = exp2f(ml[x].x - ref);
      float l = ml[x].y * w[x];
#pragma unroll
      for (int k = 16; k; k >>= 1) l += __shfl_xor_sync(~0u, l, k);
      L[x] = L[x] * keep + l;
#pragma unroll
      for (int j = 0; j < E; ++j) o[x][j] *= keep;
      M[x] = top;
    }
    const int m = imin(32, n - i0);
#pragma unroll 4
    for (int k = 0; k < m; ++k) {
      const int64_t from = ((int64_t)(c + i0 + k) * 2 + (i0 + k == 0)) * ROWS + r0;
#pragma unroll
      for (int x = 0; x < kRowsPerWarp; ++x) {
        const float wk = __shfl_sync(~0u, w[x], k);
        if (r0 + x < rows) {
          const float* src = p.part_o + (from + x) * D + lane * E;
          if constexpr (E == 4) {
            const float4 f = *reinterpret_cast<const float4*>(src);
            o[x][0] = fmaf(f.x, wk, o[x][0]);
            o[x][1] = fmaf(f.y, wk, o[x][1]);
            o[x][2] = fmaf(f.z, wk, o[x][2]);
            o[x][3] = fmaf(f.w, wk, o[x][3]);
          } else {
            const float2 f = *reinterpret_cast<const float2*>(src);
            o[x][0] = fmaf(f.x, wk, o[x][0]);
            o[x][1] = fmaf(f.y, wk, o[x][1]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int x = 0; x < kRowsPerWarp; ++x) {
    if (r0 + x >= rows) break;
    const int64_t row = (int64_t)rec.rt * ROWS + r0 + x;
    const int tok = begin + (int)(row / p.g), h = rec.kvh * p.g + (int)(row % p.g);
    const float inv = L[x] != 0.f ? 1.f / L[x] : 0.f;
    T* dst = static_cast<T*>(p.out) + (int64_t)tok * p.o_st + h * p.o_sh + lane * E;
#pragma unroll
    for (int j = 0; j < E; ++j) dst[j] = from_f32<T>(o[x][j] * inv);
    if (p.lse && lane == 0)
      p.lse[(int64_t)tok * p.Hq + h] = L[x] != 0.f ? (M[x] + log2f(L[x])) * 0.69314718055994531f : -INFINITY;
  }
}

template <typename T, int D, int ROWS>
cudaError_t run(const ExtParams& p, int grid, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid, ROWS / (kWarps * kRowsPerWarp));
  cfg.blockDim = dim3(32 * kWarps);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, extend_combine_kernel<T, D, ROWS>, p, grid);
}

template <typename T>
cudaError_t run_t(const ExtParams& p, int D, int rows, int grid, cudaStream_t st) {
  constexpr int M = kExtMmaRows;
  if (D == 64) return rows == M ? run<T, 64, M>(p, grid, st) : run<T, 64, 2 * M>(p, grid, st);
  return rows == M ? run<T, 128, M>(p, grid, st) : run<T, 128, 2 * M>(p, grid, st);
}

}  // namespace

size_t ext_rec_bytes(int grid) { return sizeof(ExtRec) * (size_t)grid; }

cudaError_t launch_extend_combine(const ExtParams& p, int dtype, int D, int rows, int grid,
                                  cudaStream_t st) {
  if (dtype == ADAKV_DTYPE_F32)
    return D == 64 ? run<float, 64, kExtSimtRows>(p, grid, st) : run<float, 128, kExtSimtRows>(p, grid, st);
  if (dtype == ADAKV_DTYPE_F16) return run_t<__half>(p, D, rows, grid, st);
  return run_t<__nv_bfloat16>(p, D, rows, grid, st);
}

}  // namespace adakv
