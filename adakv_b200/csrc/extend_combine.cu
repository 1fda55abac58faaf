// Joins the pieces of row tiles that the attention of new tokens has split.
#include "extend.cuh"

namespace adakv {
namespace {

// Joins the pieces of each row tile that begins in one CTA's range and goes on
// into the next ones: out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i.
// Block (c, y): the row tile that CTA c began, rows y * 4 .. + 3, a warp each.
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(128) extend_combine_kernel(const ExtParams p, int grid) {
  pdl_wait();
  const int c = blockIdx.x;
  const ExtRec rec = p.rec[c];
  if (!rec.tail) return;
  const int lane = threadIdx.x & 31, r = blockIdx.y * 4 + (threadIdx.x >> 5);
  const ExtSeq s = ext_seq(p, rec.b);
  const int64_t row = (int64_t)rec.rt * ROWS + r;
  if (row >= (int64_t)s.n * p.g) return;
  constexpr int E = D / 32;
  float M = -INFINITY, L = 0.f, o[E] = {};
  for (int i = c; i < grid; ++i) {
    const int piece = i == c ? 1 : 0;
    bool last = false;
    if (i != c) {
      const int2 h = *reinterpret_cast<const int2*>(&p.rec[i].head);
      if (!h.x) break;  // cannot be: the row tile goes on
      last = h.y != 0;
    }
    const int64_t at = ((int64_t)i * 2 + piece) * ROWS + r;
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + at * 2);
    float x[E];
    if constexpr (E == 4) {
      const float4 f = *reinterpret_cast<const float4*>(p.part_o + at * D + lane * 4);
      x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
    } else {
      const float2 f = *reinterpret_cast<const float2*>(p.part_o + at * D + lane * 2);
      x[0] = f.x; x[1] = f.y;
    }
    const float top = fmaxf(M, ml.x);
    const float ref = top == -INFINITY ? 0.f : top;
    const float a = exp2f(M - ref), b = exp2f(ml.x - ref);
    L = L * a + ml.y * b;
#pragma unroll
    for (int j = 0; j < E; ++j) o[j] = o[j] * a + x[j] * b;
    M = top;
    if (last) break;
  }
  const int tok = s.begin + (int)(row / p.g), h = rec.kvh * p.g + (int)(row % p.g);
  const float inv = L != 0.f ? 1.f / L : 0.f;
  T* dst = static_cast<T*>(p.out) + (int64_t)tok * p.o_st + h * p.o_sh + lane * E;
#pragma unroll
  for (int j = 0; j < E; ++j) dst[j] = from_f32<T>(o[j] * inv);
  if (p.lse && lane == 0)
    p.lse[(int64_t)tok * p.Hq + h] = L != 0.f ? (M + log2f(L)) * 0.69314718055994531f : -INFINITY;
}

template <typename T, int D, int ROWS>
cudaError_t run(const ExtParams& p, int grid, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid, ROWS / 4);
  cfg.blockDim = dim3(128);
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
