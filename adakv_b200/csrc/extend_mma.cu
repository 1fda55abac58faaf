// Attention of new tokens for 16-bit element types on the tensor cores.
//
// One persistent CTA per SM walks the row tiles of its range.  A row tile is
// NQ x 128 rows (token, head of the KV head's group); keys come in tiles of
// 128, worked on in halves of 64 that come through a ring of shared-memory
// slots, a slot holding a half of K or of V.  Warp roles:
//
//   NQ x 4 warps    softmax, a thread a row: running maximum and sum in
//                   registers, S from tensor memory, P back into the first half
//                   of S's columns, the output at the end
//   two warps       load K, and Q and V: whole tiles of packed tokens, or 16-row
//                   boxes (a page holds one or more of them), by TMA
//   NQ warps        issue the MMAs of a row tile each:  S = Q K^T  (both from
//                   shared memory) and  O += P V  (P from tensor memory); while the
//                   softmax runs, they look through V of the new tokens that only
//                   some of the rows see
//
// O is rescaled only when a row's maximum has grown by more than 2^8 since it
// last was (P then stays below 2^8, and the sum in 32 bits): most tiles after
// the first leave O alone (a published way).  fp16 keeps 5 bits of exponent: there P, l and O are
// 2^7 times as large (at most 2^15), so that what is lost of a probability lies
// below 2^-32 of the largest one's and not below 2^-25, which thousands of keys
// beside one that outweighs them all add up to.
//
// Nothing behind a sequence's end can reach a result: scores are masked by
// selection, P V runs over whole groups of 16 keys only as far as there are
// keys, and a group that ends inside (or a tree's tile, with unused slots) has
// its V brought in by plain loads with zeros in the missing rows.  (Values that
// are not finite: ext_add_infinite.)
//
// What bounds it (B200).  Decode and small trees: HBM; a key tile of 64 KB takes
// 2,920 cycles of an SM, 2,810 at the measured copy rate, and the softmax of the
// one warp that has rows takes as long (one token over 32K tokens, 8 KV heads:
// 134 MB in about 25 us of 38 us with launch, start and combine).  Long prompts:
// the softmax and, for longer than a few milliseconds, the power limit (8192
// tokens, 32 / 8 heads of 128: 515 us, 1.07 PFLOP/s at 1.7 GHz; 595 us and 0.92
// PFLOP/s at 1.5 GHz when it runs on).  Half of a tile's time two softmax warps
// share a scheduler: 64 powers of two, 64 maxima, 32 conversions a thread.
#include <cuda.h>

#include "extend.cuh"

namespace adakv {
namespace {

constexpr int KT = 128;   // keys of a tile
constexpr int KH = 64;    // keys of a half: one step of the softmax
constexpr int G16 = 16;   // keys of a group: a TMA box, a step of P V

// ---------------------------------------------------------------------------
// tcgen05
// ---------------------------------------------------------------------------
__device__ __forceinline__ void tm_alloc(uint32_t* dst, int cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(dst)), "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tm_free(uint32_t at, int cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(cols));
}
__device__ __forceinline__ void tm_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// One lane of the (converged) warp.  tcgen05.mma, commit and TMA instructions
// take uniform registers: the loops around them run on the whole warp, so that
// descriptors and addresses are the warp's, and one elected lane issues.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}
// The same value in every lane, in a register that is the warp's.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __reduce_or_sync(~0u, x); }
// `bar` gets one arrival when every MMA issued so far by this thread is done
__device__ __forceinline__ void mma_commit(uint32_t on, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar)),
      "r"(on)
      : "memory");
}
template <bool ADD>
__device__ __forceinline__ void mma_ss(uint32_t on, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "n"(ADD ? 1 : 0), "r"(on)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t on, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(add), "r"(on)
      : "memory");
}

#define R8(x, i) "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3]), "=r"(x[i + 4]), "=r"(x[i + 5]), "=r"(x[i + 6]), "=r"(x[i + 7])
#define W8(x, i) "r"(x[i]), "r"(x[i + 1]), "r"(x[i + 2]), "r"(x[i + 3]), "r"(x[i + 4]), "r"(x[i + 5]), "r"(x[i + 6]), "r"(x[i + 7])
// 32 columns of this thread's row (tensor memory lane)
__device__ __forceinline__ void tm_ld32(uint32_t at, uint32_t* x) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : R8(x, 0), R8(x, 8), R8(x, 16), R8(x, 24)
      : "r"(at));
}
__device__ __forceinline__ void tm_st32(uint32_t at, const uint32_t* x) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::W8(x, 0),
      W8(x, 8), W8(x, 16), W8(x, 24), "r"(at)
      : "memory");
}
#undef R8
#undef W8

// Shared-memory operand descriptors, 128-byte swizzle, rows of 128 bytes in
// groups of 8 (1024 bytes).  K-major (Q, K: a row is 64 elements of the head
// dim): groups of 8 rows follow one another.  MN-major (V: a row is 64
// elements of the head dim at one key): groups of 8 keys follow one another,
// and the next 64 elements lie a half of a slot further.
constexpr uint64_t kDescBase = (1ull << 46) | (2ull << 61) | ((uint64_t)(1024 >> 4) << 32);
constexpr int kColsQ = KT * 128;  // bytes of 64 columns of a 128-row tile of Q
constexpr int kCols = KH * 128;   // and of a half of K or V
__device__ __forceinline__ uint64_t desc_k(uint32_t at) { return kDescBase | (1ull << 16) | ((at >> 4) & 0x3FFF); }
__device__ __forceinline__ uint64_t desc_mn(uint32_t at) {
  return kDescBase | ((uint64_t)(kCols >> 4) << 16) | ((at >> 4) & 0x3FFF);
}
template <typename T>
constexpr uint32_t idesc(int n, bool b_mn) {
  const uint32_t f = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;  // bf16 / f16 operands
  return (1u << 4) | (f << 7) | (f << 10) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

__device__ __forceinline__ void mbar_expect(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* m, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::
          "r"(dst),
      "l"(m), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void tma_4d(uint32_t dst, const CUtensorMap* m, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];" ::"r"(dst),
      "l"(m), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void st_global_32(void* at, const uint32_t* x) {  // 32 bytes: a whole sector
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at), "r"(x[0]), "r"(x[1]), "r"(x[2]),
               "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7])
               : "memory");
}

// A wait of the whole warp: one answer, and the warp together again (the
// tcgen05 loads and stores below are warp-wide).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(~0u, mbar_wait_bounded(bar, parity));
}

template <typename T> struct Pack2;
template <> struct Pack2<__nv_bfloat16> {
  static constexpr float up = 0.f;  // P, l and O are 2^up times softmax's terms
  __device__ __forceinline__ static uint32_t run(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};
template <> struct Pack2<__half> {
  static constexpr float up = 7.f;
  __device__ __forceinline__ static uint32_t run(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};

template <int D, int NQ>
struct Smem {
  static constexpr int q_tile = KT * D * 2;
  static constexpr int q = NQ * q_tile;
  static constexpr int slot = KH * D * 2;
  static constexpr int slots = (224 * 1024 - q) / slot < 16 ? (224 * 1024 - q) / slot : 16;
  static constexpr int bytes = q + slots * slot + 1024;  // + alignment; barriers are static
};

// An exponent of all ones in either half of x: one more carries into the sign bit,
// which is cleared.
template <typename T>
__device__ __forceinline__ uint32_t infinite(uint32_t x) {
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  return (x & (kBf16 ? 0x7F807F80u : 0x7C007C00u)) + (kBf16 ? 0x00800080u : 0x04000400u);
}

// Sets what is not finite in V of a half (n words of 16 bytes in each 64 columns) to
// 0, by a whole warp, and says so.  The other row tile's MMA warp may find zeros
// already; its softmax group finds the word.
template <typename T, int D>
__device__ __noinline__ void make_finite(unsigned char* v, int n, int lane, volatile uint32_t* found) {
  *found = 1;
  __threadfence_block();
#pragma unroll 1
  for (int c = 0; c < D / 64; ++c)
#pragma unroll 1
    for (int i = lane; i < 4 * n; i += 32) {
      uint32_t* x = reinterpret_cast<uint32_t*>(v + c * kCols) + i;
      const uint32_t bad = (infinite<T>(*x) & 0x80008000u) >> 15;
      if (bad) *x &= ~(bad * 0xFFFFu);
    }
  fence_async_smem();
  __syncwarp();
}

// a + 0 x in two halves: NaN from the first infinity or NaN on
template <typename T>
__device__ __forceinline__ uint32_t add_zero_times(uint32_t x, uint32_t a) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(a) : "r"(x), "r"(0u));
  else
    asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(a) : "r"(x), "r"(0u));
  return a;
}

// Looks for values that are not finite in V of a half; by a whole warp.  As little
// code as can be: the roles share the instruction caches.  A 17-token prompt takes
// 8.6 us with the look and 8.1 without, ten prompts of 0 to 1500 tokens 67.2 and 66.7,
// with this loop unrolled 76.
template <typename T, int D>
__device__ __forceinline__ void look_through(unsigned char* v, int n, int lane, volatile uint32_t* found) {
  uint32_t a[4] = {0u, 0u, 0u, 0u};
#pragma unroll 1
  for (int at = lane; at < n; at += 64)
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const uint4 x = *reinterpret_cast<const uint4*>(v + (c >> 1) * kCols + (at + (c & 1) * 32) * 16);
      a[0] = add_zero_times<T>(x.x, a[0]);
      a[1] = add_zero_times<T>(x.y, a[1]);
      a[2] = add_zero_times<T>(x.z, a[2]);
      a[3] = add_zero_times<T>(x.w, a[3]);
    }
  // (a half that is no NaN is 0, of either sign)
  if (__any_sync(~0u, (a[0] | a[1] | a[2] | a[3]) & 0x7FFF7FFFu)) make_finite<T, D>(v, n, lane, found);
  __threadfence_block();
}

struct Maps {
  CUtensorMap q;       // boxes of KT rows (token, head), where the group's heads divide KT

  CUtensorMap k, v;    // new tokens: boxes of KH rows
  CUtensorMap kg, vg;  // and of G16
  CUtensorMap pk, pv;  // pages: G16
};

template <int NQ>
constexpr int threads() {
  return 32 * (5 * NQ + 2);
}

template <typename T, int D, int NQ>
__global__ void __launch_bounds__(threads<NQ>(), 1)
    extend_mma_kernel(const ExtParams p, const __grid_constant__ Maps maps) {
  using S = Smem<D, NQ>;
  constexpr int R = 128 * NQ, NS = S::slots;
  constexpr int kLoadK = 4 * NQ, kLoadV = kLoadK + 1, kMma = kLoadK + 2;  // warps
  constexpr uint32_t kO = 256;  // tensor memory: S (and P) of row tile i at 128 i, O at 256 + 128 i
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ uint64_t full[NS], empty[NS], q_full, q_empty, s_full[NQ][2], p_full[NQ][2], o_done[NQ],
      o_last[NQ], drained[NQ];
  // Was anything of a row tile's V not finite?  By the row tile's number: V is
  // loaded at most two row tiles ahead of a softmax group's output.
  __shared__ volatile uint32_t v_infinite[4];
  __shared__ ExtStart start;
  __shared__ uint32_t tm_base;
  const uint32_t smem0 = (smem_addr(raw) + 1023u) & ~1023u;
  unsigned char* base = raw + (smem0 - smem_addr(raw));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (warp == kLoadK) {
    if (lane == 0) {
      for (int i = 0; i < NS; ++i) {
        mbar_init(&full[i], 1);
        mbar_init(&empty[i], NQ);
      }
      mbar_init(&q_full, 1);
      mbar_init(&q_empty, NQ);
      for (int i = 0; i < NQ; ++i) {
        for (int h = 0; h < 2; ++h) {
          mbar_init(&s_full[i][h], 1);
          mbar_init(&p_full[i][h], 128);
        }
        mbar_init(&o_done[i], 1);
        mbar_init(&o_last[i], 2);  // the products' end, and the MMA warp that has waited for every P
        mbar_init(&drained[i], 1);
      }
    }
    __syncwarp();
  } else if (warp == kMma) {
    tm_alloc(&tm_base, 512);
  } else if (warp == kLoadV) {
    const ExtStart st = ext_locate<R, KT>(p, blockIdx.x, gridDim.x, lane);
    if (lane == 0) start = st;
  }
  tm_before_sync();
  __syncthreads();
  tm_after_sync();
  const uint32_t tm = uniform(tm_base);
  // The combine kernel comes up meanwhile; it waits for this one's end.  Where none
  // follows, the next kernel is somebody else's and may read `out` before it waits.
  if (p.join) pdl_launch_dependents();
  ExtWalk<R, KT> w;
  w.start(p, start);
  bool ok = true;

  if (warp >= kLoadK) {
    if (warp == kLoadK || warp == kLoadV) {
      // ------------------------------------------------------------------ K, V
      const bool is_v = warp == kLoadV;
      uint32_t f = 0, sent = 0, phase = 0;  // slots that have had a tile of this warp's, and its parity
      const uint32_t leader = elect_one();
      // Page ids of a prefix tile, a lane a group: those of the tile before next
      // are on their way while one is loaded.
      auto fetch_ids = [&](int kt) {
        const int j = kt * KT + lane * G16;
        return lane < KT / G16 && kt < w.p_tiles && j < w.s.prefix ? ext_page(p, w.s.slot, j >> p.page_log2) : 0;
      };
      // half v of the range (page: the ids of its tile) into the ring, its `fill`-th
      auto load = [&](int v, uint32_t fill, int page) {
        const uint32_t slot = fill % NS, round = fill / NS;
        if (round && !warp_wait(&empty[slot], (round - 1) & 1)) return false;
        const uint32_t dst = smem0 + S::q + slot * S::slot;
        const int kt = w.k_lo + (v >> 1), g0 = (v & 1) * (KH / G16);  // first group of the half in its tile
        const bool cached = kt < w.p_tiles;
        const int j0 = (cached ? kt : kt - w.p_tiles) * KT + (v & 1) * KH;
        const int have = imax(0, imin(KH, (cached ? w.s.prefix : w.s.n) - j0));
        const int groups = (have + G16 - 1) / G16;
        // groups of V from here on come by plain loads
        const int plain = !is_v ? groups : !cached && p.parents ? 0 : have / G16;
        const int boxes = imin(groups, plain);
        // one box for a whole half of new tokens (K may read on behind the sequence)
        const bool whole = !cached && (is_v ? plain * G16 == KH : have > KH / 2);
        if (leader) mbar_expect(&full[slot], (whole ? KH / G16 : boxes) * (D / 64) * (G16 * 128));
        __syncwarp();
        if (whole) {
          if (lane < D / 64)
            tma_3d(dst + lane * kCols, is_v ? &maps.v : &maps.k, lane * 64, w.kvh, w.s.begin + j0, &full[slot]);
        } else {
          // a lane a box
          const int g = lane % (KH / G16), c = lane / (KH / G16);
          const int id = __shfl_sync(~0u, page, g0 + g);
          if (c < D / 64 && g < boxes) {
            if (cached)
              tma_4d(dst + c * kCols + g * (G16 * 128), is_v ? &maps.pv : &maps.pk, c * 64,
                     (j0 + g * G16) & ((1 << p.page_log2) - 1), w.kvh, id, &full[slot]);
            else
              tma_3d(dst + c * kCols + g * (G16 * 128), is_v ? &maps.vg : &maps.kg, c * 64, w.kvh,
                     w.s.begin + j0 + g * G16, &full[slot]);
          }
        }
        if (plain < groups) {
          unsigned char* out = base + S::q + slot * S::slot;
          constexpr int C = D / 8, RT = 32 / C;  // 16-byte words of a row, rows at a time
          const int c = lane % C;
          uint32_t live[KH / 32];  // rows that exist and are in use
#pragma unroll
          for (int i = 0; i < KH / 32; ++i) {
            const int r = i * 32 + lane;
            live[i] = __ballot_sync(~0u, r < have && (cached || ext_live(p, w.s, j0 + r)));
          }
          for (int r = plain * G16 + lane / C; r < groups * G16; r += RT) {
            const bool on = (live[r >> 5] >> (r & 31)) & 1;
            const T* src;
            if (cached) {
              const int id = __shfl_sync(~0u, page, g0 + r / G16);
              src = static_cast<const T*>(p.pv) + id * p.pv_sp + w.kvh * p.pv_sh +
                    ((j0 + r) & ((1 << p.page_log2) - 1)) * p.pv_st;
            } else {
              src = static_cast<const T*>(p.v) + (int64_t)(w.s.begin + j0 + r) * p.v_st + w.kvh * p.v_sh;
            }
            cp_async16(out + (c >> 3) * kCols + r * 128 + (((c & 7) ^ (r & 7)) << 4),
                       on ? src + c * 8 : static_cast<const T*>(cached ? p.pv : p.v), on);
          }
          cp_async_commit();
          cp_async_wait_all();
          fence_async_smem();
          __syncwarp();
        }
        if (leader) mbar_arrive(&full[slot]);
        sent |= 1u << slot;
        phase = (phase & ~(1u << slot)) | ((round & 1) << slot);
        return true;
      };
      // Q of a row tile
      auto load_q = [&]() {
        if (KT % p.g == 0) {
          // rows behind the sequence's last belong to other tokens, and to nobody here
          if (leader) mbar_expect(&q_full, S::q);
          __syncwarp();
          if (lane < NQ * (D / 64)) {
            const int i = lane / (D / 64), h = lane % (D / 64);
            tma_3d(smem0 + i * S::q_tile + h * kColsQ, &maps.q, h * 64, w.kvh * p.g,
                   w.s.begin + (w.rt * R + i * 128) / p.g, &q_full);
          }
          __syncwarp();
        } else {
          const int rows = w.rows(p.g);
          constexpr int C = D / 8, RT = 32 / C;  // 16-byte words of a row, rows at a time
          const int c = lane % C;
          const T* src = static_cast<const T*>(p.q) + (int64_t)w.s.begin * p.q_st + (int64_t)w.kvh * p.g * p.q_sh + c * 8;
          const int row = w.rt * R + lane / C;
          int tok = row / p.g, h = row - tok * p.g;
          const int step_tok = RT / p.g, step_h = RT - step_tok * p.g;
#pragma unroll 4
          for (int r = lane / C; r < R; r += RT) {
            cp_async16(base + (r >> 7) * S::q_tile + (c >> 3) * kColsQ + (r & 127) * 128 + (((c & 7) ^ (r & 7)) << 4),
                       r < rows ? src + tok * p.q_st + h * p.q_sh : src, r < rows);
            tok += step_tok;
            h += step_h;
            if (h >= p.g) {
              h -= p.g;
              ++tok;
            }
          }
          cp_async_commit();
          cp_async_wait_all();
          fence_async_smem();
          __syncwarp();
        }
        if (leader) mbar_arrive(&q_full);
      };
      uint32_t item = 0;
      for (; ok && w.live(); w.next(p), ++item) {
        const int n = w.k_hi - w.k_lo;
        if (is_v) {  // (V is needed later than K)
          ok = item == 0 || warp_wait(&q_empty, (item - 1) & 1);
          if (!ok) break;
          if (leader) v_infinite[item & 3] = 0;
          load_q();
        }
        // The ring's order is that in which the MMAs take the halves: both of the
        // first K tile, then V of a half and K of the same half of the next tile.
        int ids = fetch_ids(w.k_lo);
        for (int j = 0; ok && j < n; ++j) {
          const int next = fetch_ids(w.k_lo + j + 1);
          for (int h = 0; ok && h < 2; ++h) {
            const int at = is_v ? (j + 1 < n ? 2 + 4 * j + 2 * h : 2 + 4 * j + h) : j == 0 ? h : 4 * j - 1 + 2 * h;
            ok = load(2 * j + h, f + at, ids);
          }
          ids = next;
        }
        f += 4 * n;
      }
      if (!ok)  // copies in flight end before the CTA does
        for (int i = 0; i < NS; ++i)
          if ((sent >> i) & 1) warp_wait(&full[i], (phase >> i) & 1);
    } else if (warp >= kMma) {
      // ------------------------------------------------------------------ MMAs
      // The scores of a half are issued two halves ahead, as soon as the P V
      // that reads the half's place in tensor memory is: a softmax group finds
      // its next scores ready.
      const int i = warp - kMma;
      const uint32_t leader = elect_one();
      uint32_t item = 0, t = 0, ring = 0, turn = 0;  // next slot of the ring, and its parity
      const uint64_t qd = desc_k(smem0 + i * S::q_tile);
      const uint32_t s_at = tm + i * 128, o_at = tm + kO + i * 128;
      auto take = [&](uint32_t& slot) {  // the ring's next half, once it is there
        slot = ring;
        const bool there = warp_wait(&full[ring], turn);
        if (++ring == NS) {
          ring = 0;
          turn ^= 1;
        }
        return there;
      };
      auto qk = [&](int h, uint32_t ks, bool last) {  // the scores of half h of a tile
        const uint64_t kd = desc_k(smem0 + S::q + uniform(ks) * S::slot);
        mma_ss<false>(leader, s_at + h * KH, qd, kd, idesc<T>(KH, false));
#pragma unroll
        for (int k = 1; k < D / 16; ++k) {
          const uint32_t q_off = ((k >> 2) * kColsQ + (k & 3) * 32) >> 4, k_off = ((k >> 2) * kCols + (k & 3) * 32) >> 4;
          mma_ss<true>(leader, s_at + h * KH, qd + q_off, kd + k_off, idesc<T>(KH, false));
        }
        mma_commit(leader, &s_full[i][h]);
        mma_commit(leader, &empty[ks]);
        if (last) mma_commit(leader, &q_empty);
      };
      for (; ok && w.live(); w.next(p), ++item) {
        const int n = w.k_hi - w.k_lo;
        uint32_t vs = 0, ks = 0;
        // From this tile on the row tile's rows see the new tokens in part.
        const int part = w.p_tiles - w.k_lo + (w.s.n == 1 ? n : p.parents ? 0 : w.rt * R / p.g / KT);
        ok = warp_wait(&q_full, item & 1);
        for (int h = 0; ok && h < 2; ++h) {
          ok = take(ks);
          if (!ok) break;
          tm_after_sync();
          qk(h, ks, n == 1 && h);
        }
        for (int j = 0; ok && j < n; ++j) {
          const int kt = w.k_lo + j;
          const int left = imin(KT, kt < w.p_tiles ? w.s.prefix - kt * KT : w.s.n - (kt - w.p_tiles) * KT);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            // V of this half, K of the next tile's (there before the softmax is done)
            ok = take(vs) && (j + 1 == n || take(ks));
            if (!ok) break;
            if (__builtin_expect(j >= part && left > h * KH, 0))
              look_through<T, D>(base + S::q + vs * S::slot, imin(KH / G16, (left - h * KH + G16 - 1) / G16) * (G16 * 8),
                                 lane, &v_infinite[item & 3]);
            const uint64_t vd = desc_mn(smem0 + S::q + uniform(vs) * S::slot);
            ok = warp_wait(&p_full[i][h], (t + j) & 1);
            if (!ok) break;
            tm_after_sync();
#pragma unroll
            for (int k = 0; k < KH / G16; ++k) {
              const uint32_t on = left > h * KH + k * G16 ? leader : 0;
              mma_ts(on, o_at, s_at + h * KH + k * 8, vd + (k * G16 * 128 >> 4), idesc<T>(D, true), j > 0 || h + k > 0);
            }
            mma_commit(leader, &o_done[i]);
            mma_commit(leader, &empty[vs]);
            if (h && j + 1 == n) {
              mma_commit(leader, &o_last[i]);
              if (leader) mbar_arrive(&o_last[i]);
            }
            if (j + 1 < n) qk(h, ks, j + 2 == n && h);
          }
        }
        t += n;
      }
      if (!ok) {  // MMAs in flight end before the tensor memory is given back
        mma_commit(leader, &drained[i]);
        warp_wait(&drained[i], 0);
      }
    }
  } else {
    // --------------------------------------------------------------- softmax
    const int qi = warp >> 2;             // row tile of the NQ
    const int r = (warp & 3) * 32 + lane;       // row in it, and tensor memory lane
    const uint32_t lanes = tm + ((uint32_t)(warp & 3) << 21);  // lane (warp & 3) * 32, column 0
    const uint32_t o_at = lanes + kO + qi * 128;
    uint32_t t = 0, u = 0, item = 0;  // tiles, halves, row tiles so far
    ExtRec rec{};
    for (; ok && w.live(); w.next(p), ++item) {
      const int rows = w.rows(p.g);
      const int rr = qi * 128 + r;
      const bool mine = rr < rows;
      const bool idle = qi * 128 + (warp & 3) * 32 >= rows;  // no row of this warp exists
      const int tok = mine ? (w.rt * R + rr) / p.g : 0;
      const bool seen = mine && ext_live(p, w.s, tok);
      float m = -INFINITY, l = 0.f;  // maximum that O and l are scaled by (of q.k), sum
      for (int kt = w.k_lo; ok && kt < w.k_hi; ++kt, ++t) {
        const bool cached = kt < w.p_tiles;
        const bool tree = !cached && p.parents;
#pragma unroll 1
        for (int h = 0; h < 2; ++h, ++u) {
          const int j0 = (cached ? kt : kt - w.p_tiles) * KT + h * KH;
          const int have = imin(KH, (cached ? w.s.prefix : w.s.n) - j0);  // (none or fewer in a last half)
          ok = warp_wait(&s_full[qi][h], t & 1);
          if (!ok) break;
          tm_after_sync();
          if (!idle && have > 0) {
            const uint32_t s_at = lanes + qi * 128 + h * KH;
            uint32_t x[KH];
            tm_ld32(s_at, x);
            tm_ld32(s_at + 32, x + 32);
            const int see = !seen ? 0 : cached || tree ? have : imin(have, tok - j0 + 1);
            const bool cut = __any_sync(~0u, tree || (mine && see < KH));
            tm_wait_ld();
            if (cut) {
              uint32_t bits[2];
              if (tree) {
                if (seen) ext_tree_mask<2>(p, w.s, tok, j0, bits);
                else bits[0] = bits[1] = 0;
              } else {
                bits[0] = see >= 32 ? ~0u : see > 0 ? (1u << see) - 1u : 0u;
                bits[1] = see >= 64 ? ~0u : see > 32 ? (1u << (see - 32)) - 1u : 0u;
              }
#pragma unroll
              for (int i = 0; i < KH; ++i)
                if (!((bits[i >> 5] >> (i & 31)) & 1u)) x[i] = 0xFF800000u;
            }
            float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < KH; ++i) top[i & 3] = fmaxf(top[i & 3], __uint_as_float(x[i]));
            const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
            if (kt == w.k_lo && h == 0) {
              m = mx;
            } else if (__any_sync(~0u, (mx - m) * p.scale > 8.f)) {
              const float up = fmaxf(m, mx);
              const float keep = up == -INFINITY ? 1.f : exp2_fast((m - up) * p.scale);
              m = up;
              l *= keep;
              // (these scores were issued behind the P V of the half before the
              // last one: the phase waited for is the barrier's current one or
              // the one before)
              ok = warp_wait(&o_done[qi], (u - 1) & 1);
              if (!ok) break;
              tm_after_sync();
#pragma unroll 1
              for (int c = 0; c < D; c += 32) {
                uint32_t y[32];
                tm_ld32(o_at + c, y);
                tm_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * keep);
                tm_st32(o_at + c, y);
              }
            }
            __syncwarp();
            const float off = m == -INFINITY ? 0.f : m * p.scale - Pack2<T>::up;
            float2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
            uint32_t y[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              float2 v = fma2(make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])),
                              make_float2(p.scale, p.scale), make_float2(-off, -off));
              v.x = exp2_fast(v.x);
              v.y = exp2_fast(v.y);
              sum[i & 1] = add2(sum[i & 1], v);
              y[i] = Pack2<T>::run(v.x, v.y);
            }
            tm_st32(s_at, y);
            l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            tm_wait_st();
          }
          tm_before_sync();
          mbar_arrive(&p_full[qi][h]);
        }
      }
      if (!ok) break;
      // the row tile's output, or this CTA's piece of it
      ok = warp_wait(&o_last[qi], item & 1);
      if (!ok) break;
      tm_after_sync();
      const bool whole = w.begins() && w.ends(), spoilt = v_infinite[item & 3];
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
      if (idle) continue;
      const int row = w.rt * R + rr;
      const int64_t at = ((int64_t)blockIdx.x * 2 + piece) * R + rr;
      const int h = w.kvh * p.g + row % p.g;
      T* dst = static_cast<T*>(p.out) + (int64_t)(w.s.begin + tok) * p.o_st + h * p.o_sh;
      const bool wide = (reinterpret_cast<uintptr_t>(dst) & 31) == 0;  // (rows are 16-byte aligned)
      // (a row that has seen nothing has a sum of 0; one whose scores are all NaN
      // has m = -inf too, but its sum is NaN)
      const float inv = !whole ? 1.f : l != 0.f ? 1.f / l : 0.f;
#pragma unroll 1  // (less code: the ten prompts 67.4 us, unrolled 69.2)
      for (int c = 0; c < D; c += 32) {
        uint32_t y[32];
        __syncwarp();
        tm_ld32(o_at + c, y);
        tm_wait_ld();
        if (l == 0.f) {  // selected, not multiplied: V may be infinite where others see it
#pragma unroll
          for (int i = 0; i < 32; ++i) y[i] = 0;
        }
        if (!mine) {
        } else if (whole) {
          uint32_t z[16];
#pragma unroll
          for (int i = 0; i < 16; ++i)
            z[i] = Pack2<T>::run(__uint_as_float(y[2 * i]) * inv, __uint_as_float(y[2 * i + 1]) * inv);
          if (wide) {
            st_global_32(dst + c, z);
            st_global_32(dst + c + 16, z + 8);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<uint4*>(dst + c + i * 8) = make_uint4(z[4 * i], z[4 * i + 1], z[4 * i + 2], z[4 * i + 3]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) st_global_32(p.part_o + at * D + c + i * 8, y + i * 8);
        }
      }
      if (mine) {
        const float ml = m == -INFINITY ? -INFINITY : m * p.scale - Pack2<T>::up;
        if (!whole) {
          *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(ml, l);
        } else if (p.lse) {
          p.lse[(int64_t)(w.s.begin + tok) * p.Hq + h] =
              l != 0.f ? (ml + log2f(l)) * 0.69314718055994531f : -INFINITY;
        }
      }
      if (__builtin_expect(spoilt && seen, 0)) {
        const T* v = static_cast<const T*>(p.v) + (int64_t)w.s.begin * p.v_st + w.kvh * p.v_sh;
        const int* par = p.parents ? p.parents + w.s.begin : nullptr;
        const int lo = imax(imax(w.k_lo - w.p_tiles, 0) * KT, par ? 0 : (w.rt * R / p.g) & ~(KT - 1));
        const int hi = imin(imax(w.k_hi - w.p_tiles, 0) * KT, w.s.n);
        if (whole) ext_add_infinite(v, p.v_st, par, tok, lo, hi, dst, D);
        else ext_add_infinite(v, p.v_st, par, tok, lo, hi, p.part_o + at * D, D);
      }
    }
    if (tid == 0) p.rec[blockIdx.x] = rec;
  }
  if (!ok && lane == 0) report(p.status, ADAKV_ST_WAIT_TIMEOUT);
  tm_before_sync();
  __syncthreads();
  if (warp == kMma) tm_free(tm, 512);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn g_encode = nullptr;

template <int N>
cudaError_t encode(CUtensorMap* m, int dtype, const void* data, const int64_t (&dims)[N],
                   const int64_t (&strides)[N - 1], const int (&box)[N]) {
  cuuint64_t d[N], s[N - 1];
  cuuint32_t b[N], one[N];
  for (int i = 0; i < N; ++i) {
    d[i] = (cuuint64_t)dims[i];
    b[i] = (cuuint32_t)box[i];
    one[i] = 1;
  }
  // an axis of one entry may carry any stride: give it one that is allowed
  for (int i = 0; i + 1 < N; ++i) s[i] = dims[i + 1] > 1 ? (cuuint64_t)strides[i] * 2 : 16;
  const CUresult r = g_encode(
      m, dtype == ADAKV_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, N,
      const_cast<void*>(data), d, s, b, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <typename T, int D, int NQ>
cudaError_t run(const ExtParams& p, const Maps& maps, int grid, cudaStream_t st) {
  extend_mma_kernel<T, D, NQ><<<grid, threads<NQ>(), Smem<D, NQ>::bytes, st>>>(p, maps);
  return cudaGetLastError();
}

template <typename T>
cudaError_t run_t(const ExtParams& p, const Maps& maps, int D, int nq, int grid, cudaStream_t st) {
  if (D == 64) return nq == 1 ? run<T, 64, 1>(p, maps, grid, st) : run<T, 64, 2>(p, maps, grid, st);
  return nq == 1 ? run<T, 128, 1>(p, maps, grid, st) : run<T, 128, 2>(p, maps, grid, st);
}

template <typename T, int D, int NQ>
cudaError_t prepare() {
  return cudaFuncSetAttribute(extend_mma_kernel<T, D, NQ>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              Smem<D, NQ>::bytes);
}

}  // namespace

cudaError_t ext_mma_init() {
  cudaError_t e;
  if (!g_encode) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    if ((e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found))) return e;
    if (found != cudaDriverEntryPointSuccess) return cudaErrorNotSupported;
    g_encode = reinterpret_cast<EncodeFn>(fn);
  }
  if ((e = prepare<__half, 64, 1>()) || (e = prepare<__half, 64, 2>()) || (e = prepare<__half, 128, 1>()) ||
      (e = prepare<__half, 128, 2>()) || (e = prepare<__nv_bfloat16, 64, 1>()) ||
      (e = prepare<__nv_bfloat16, 64, 2>()) || (e = prepare<__nv_bfloat16, 128, 1>()))
    return e;
  return prepare<__nv_bfloat16, 128, 2>();
}

cudaError_t launch_extend_mma(const ExtParams& p, int dtype, int D, int row_tiles, int grid, cudaStream_t st) {
  Maps maps;
  cudaError_t e;
  if (KT % p.g == 0) {
    const int64_t dq[3] = {D, p.Hq, p.T};
    const int bq[3] = {64, p.g, KT / p.g};
    if ((e = encode<3>(&maps.q, dtype, p.q, dq, {p.q_sh, p.q_st}, bq))) return e;
  }
  const int64_t dn[3] = {D, p.Hkv, p.T};
  const int bn[3] = {64, 1, KH}, bg[3] = {64, 1, G16};
  if ((e = encode<3>(&maps.k, dtype, p.k, dn, {p.k_sh, p.k_st}, bn))) return e;
  if ((e = encode<3>(&maps.v, dtype, p.v, dn, {p.v_sh, p.v_st}, bn))) return e;
  if ((e = encode<3>(&maps.kg, dtype, p.k, dn, {p.k_sh, p.k_st}, bg))) return e;
  if ((e = encode<3>(&maps.vg, dtype, p.v, dn, {p.v_sh, p.v_st}, bg))) return e;
  if (p.lens) {
    const int64_t dp[4] = {D, 1 << p.page_log2, p.Hkv, p.n_pages};
    const int bp[4] = {64, G16, 1, 1};
    if ((e = encode<4>(&maps.pk, dtype, p.pk, dp, {p.pk_st, p.pk_sh, p.pk_sp}, bp))) return e;
    if ((e = encode<4>(&maps.pv, dtype, p.pv, dp, {p.pv_st, p.pv_sh, p.pv_sp}, bp))) return e;
  } else {
    maps.pk = maps.k;
    maps.pv = maps.v;
  }
  return dtype == ADAKV_DTYPE_F16 ? run_t<__half>(p, maps, D, row_tiles, grid, st)
                                  : run_t<__nv_bfloat16>(p, maps, D, row_tiles, grid, st);
}

}  // namespace adakv
