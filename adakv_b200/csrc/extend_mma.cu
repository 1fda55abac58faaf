// Attention of new tokens for 16-bit element types on the tensor cores.
//
// One persistent CTA per SM walks the row tiles of its range.  A row tile is
// NQ x 128 rows (token, head of the KV head's group); keys come in tiles of
// 128 through a ring of shared-memory slots, a slot holding one tile of K or
// of V.  Warp roles:
//
//   warps 0, 2      load K, and V: whole tiles of packed tokens, or 16-row boxes
//                   (a page holds one or more of them), by TMA
//   warp 1          issues the MMAs:  S = Q K^T  (both from shared memory) and
//                   O += P V  (P from tensor memory); S, P and O live there
//   warp 3          loads the next row tile's Q
//   warps 4..       NQ groups of four softmax warps, a thread a row: running
//                   maximum and sum in registers, S from tensor memory, P back
//                   into the first half of S's columns, the output at the end
//
// O is rescaled only when a row's maximum has grown by more than 2^8 since it
// last was (P then stays below 2^8, and the sum in 32 bits): most tiles after
// the first leave O alone.
//
// Nothing behind a sequence's end can reach a result: scores are masked by
// selection, P V runs over whole groups of 16 keys only as far as there are
// keys, and a group that ends inside (or a tree's tile, with unused slots) has
// its V brought in by plain loads with zeros in the missing rows.
#include <cuda.h>

#include "extend.cuh"

namespace adakv {
namespace {

constexpr int KT = 128;   // keys of a tile
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
__device__ __forceinline__ void tm_ld16(uint32_t at, uint32_t* x) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : R8(x, 0), R8(x, 8)
      : "r"(at));
}
__device__ __forceinline__ void tm_st16(uint32_t at, const uint32_t* x) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15};" ::W8(x, 0),
      W8(x, 8), "r"(at)
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
constexpr int kHalf = KT * 128;  // bytes of 64 columns of a 128-row tile
__device__ __forceinline__ uint64_t desc_k(uint32_t at) { return kDescBase | (1ull << 16) | ((at >> 4) & 0x3FFF); }
__device__ __forceinline__ uint64_t desc_mn(uint32_t at) {
  return kDescBase | ((uint64_t)(kHalf >> 4) << 16) | ((at >> 4) & 0x3FFF);
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

// A wait of the whole warp: one answer, and the warp together again (the
// tcgen05 loads and stores below are warp-wide).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(~0u, mbar_wait_bounded(bar, parity));
}

template <typename T> struct Pack2;
template <> struct Pack2<__nv_bfloat16> {
  __device__ __forceinline__ static uint32_t run(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};
template <> struct Pack2<__half> {
  __device__ __forceinline__ static uint32_t run(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};

template <int D, int NQ>
struct Smem {
  static constexpr int slot = KT * D * 2;
  static constexpr int q = NQ * slot;
  static constexpr int slots = (224 * 1024 - q) / slot < 12 ? (224 * 1024 - q) / slot : 12;
  static constexpr int bytes = q + slots * slot + 1024;  // + alignment; barriers are static
};

// The ring's order is the order in which the MMAs take the tiles of a row tile:
// K of the next key tile before V of this one (one row tile), or V of this one
// and then K of the next (two).  Counted from the row tile's first.
template <int NQ>
__device__ __forceinline__ uint32_t k_fill(int j) {
  return NQ == 2 || j == 0 ? 2 * j : 2 * j - 1;
}
template <int NQ>
__device__ __forceinline__ uint32_t v_fill(int j, int n) {
  return NQ == 2 || j + 1 == n ? 2 * j + 1 : 2 * j + 2;
}

struct Maps {
  CUtensorMap q;       // boxes of KT rows (token, head), where the group's heads divide KT

  CUtensorMap k, v;    // new tokens: boxes of KT rows
  CUtensorMap kg, vg;  // and of G16
  CUtensorMap pk, pv;  // pages: G16
};

template <typename T, int D, int NQ>
__global__ void __launch_bounds__(128 * (1 + NQ), 1)
    extend_mma_kernel(const ExtParams p, const __grid_constant__ Maps maps) {
  using S = Smem<D, NQ>;
  constexpr int R = 128 * NQ, NS = S::slots;
  constexpr uint32_t kO = 256;  // tensor memory: S (and P) at 0 and 128, O at 256 and 384
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ uint64_t full[NS], empty[NS], q_full, q_empty, s_full[2], p_full[2], o_done[NQ], o_last[NQ], drained;
  __shared__ ExtStart start;
  __shared__ uint32_t tm_base;
  const uint32_t smem0 = (smem_addr(raw) + 1023u) & ~1023u;
  unsigned char* base = raw + (smem0 - smem_addr(raw));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (warp == 0) {
    if (lane == 0) {
      for (int i = 0; i < NS; ++i) {
        mbar_init(&full[i], 1);
        mbar_init(&empty[i], 1);
      }
      mbar_init(&q_full, 1);
      mbar_init(&q_empty, 1);
      mbar_init(&drained, 1);
      for (int i = 0; i < 2; ++i) {
        mbar_init(&s_full[i], 1);
        mbar_init(&p_full[i], 128);
      }
      for (int i = 0; i < NQ; ++i) {
        mbar_init(&o_done[i], 1);
        mbar_init(&o_last[i], 1);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    tm_alloc(&tm_base, 512);
  } else if (warp == 3) {
    const ExtStart st = ext_locate<R, KT>(p, blockIdx.x, gridDim.x, lane);
    if (lane == 0) start = st;
  }
  tm_before_sync();
  __syncthreads();
  tm_after_sync();
  const uint32_t tm = uniform(tm_base);
  ExtWalk<R, KT> w;
  w.start(p, start);
  bool ok = true;

  // 384 threads start with 168 registers each; 128 x 80 + 256 x 208 is less
  if (warp < 4) {
    if constexpr (NQ == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == 0 || warp == 2) {
      // ------------------------------------------------------------------ K, V
      const bool is_v = warp == 2;
      uint32_t f = 0, sent = 0, phase = 0;  // slots that have had a tile of this warp's, and its parity
      const uint32_t leader = elect_one();
      // Page ids of a prefix tile, a lane a group: those of the tile before next
      // are on their way while one is loaded.
      auto fetch_ids = [&](int kt) {
        const int j = kt * KT + lane * G16;
        return lane < KT / G16 && kt < w.p_tiles && j < w.s.prefix ? ext_page(p, w.s.slot, j >> p.page_log2) : 0;
      };
      // tile kt of K or V into the ring: its `fill`-th tile
      auto load = [&](int kt, uint32_t fill, int page) {
        const uint32_t slot = fill % NS, round = fill / NS;
        if (round && !warp_wait(&empty[slot], (round - 1) & 1)) return false;
        const uint32_t dst = smem0 + S::q + slot * S::slot;
        const bool cached = kt < w.p_tiles;
        const int j0 = (cached ? kt : kt - w.p_tiles) * KT;
        const int have = imin(KT, (cached ? w.s.prefix : w.s.n) - j0);
        const int groups = (have + G16 - 1) / G16;
        // groups of V from here on come by plain loads
        const int plain = !is_v ? groups : !cached && p.parents ? 0 : have / G16;
        const int boxes = imin(groups, plain);
        // one box for a whole tile of new tokens (K may read on behind the sequence)
        const bool whole = !cached && (is_v ? plain * G16 == KT : have > KT / 2);
        if (leader) mbar_expect(&full[slot], (whole ? KT / G16 : boxes) * (D / 64) * (G16 * 128));
        __syncwarp();
        if (cached) {
          // a lane a box
          const int g = lane % (KT / G16), h = lane / (KT / G16);
          const int id = __shfl_sync(~0u, page, g);
          if (h < D / 64 && g < boxes)
            tma_4d(dst + h * kHalf + g * (G16 * 128), is_v ? &maps.pv : &maps.pk, h * 64,
                   (j0 + g * G16) & ((1 << p.page_log2) - 1), w.kvh, id, &full[slot]);
        } else if (whole) {
          if (lane < D / 64)
            tma_3d(dst + lane * kHalf, is_v ? &maps.v : &maps.k, lane * 64, w.kvh, w.s.begin + j0, &full[slot]);
        } else {
          const int g = lane % (KT / G16), h = lane / (KT / G16);
          if (h < D / 64 && g < boxes)
            tma_3d(dst + h * kHalf + g * (G16 * 128), is_v ? &maps.vg : &maps.kg, h * 64, w.kvh,
                   w.s.begin + j0 + g * G16, &full[slot]);
        }
        if (plain < groups) {
          unsigned char* out = base + S::q + slot * S::slot;
          constexpr int C = D / 8;  // 16-byte words of a row
          for (int i = plain * G16 * C + lane; i < groups * G16 * C; i += 32) {
            const int r = i / C, c = i % C, j = j0 + r;
            uint4 x = make_uint4(0, 0, 0, 0);
            if (r < have && (cached || ext_live(p, w.s, j))) {
              const T* src;
              if (cached) {
                const int page = ext_page(p, w.s.slot, j >> p.page_log2);
                src = static_cast<const T*>(p.pv) + page * p.pv_sp + w.kvh * p.pv_sh +
                      (j & ((1 << p.page_log2) - 1)) * p.pv_st;
              } else {
                src = static_cast<const T*>(p.v) + (int64_t)(w.s.begin + j) * p.v_st + w.kvh * p.v_sh;
              }
              x = *reinterpret_cast<const uint4*>(src + c * 8);
            }
            *reinterpret_cast<uint4*>(out + (c >> 3) * kHalf + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = x;
          }
          fence_async_smem();
          __syncwarp();
        }
        if (leader) mbar_arrive(&full[slot]);
        sent |= 1u << slot;
        phase = (phase & ~(1u << slot)) | ((round & 1) << slot);
        return true;
      };
      for (; ok && w.live(); w.next(p)) {
        const int n = w.k_hi - w.k_lo;
        int ids = fetch_ids(w.k_lo);
        for (int j = 0; ok && j < n; ++j) {
          const int next = fetch_ids(w.k_lo + j + 1);
          ok = load(w.k_lo + j, f + (is_v ? v_fill<NQ>(j, n) : k_fill<NQ>(j)), ids);
          ids = next;
        }
        f += 2 * n;
      }
      if (!ok)  // copies in flight end before the CTA does
        for (int i = 0; i < NS; ++i)
          if ((sent >> i) & 1) warp_wait(&full[i], (phase >> i) & 1);
    } else if (warp == 1) {
      // ------------------------------------------------------------------ MMAs
      const uint32_t leader = elect_one();
      uint32_t f = 0, item = 0, t = 0;
      auto slot_at = [&](uint32_t i) { return smem0 + S::q + uniform(i % NS) * S::slot; };
      auto wait_slot = [&](uint32_t i) { return warp_wait(&full[i % NS], (i / NS) & 1); };
      auto qk = [&](int i, uint32_t s, uint32_t fill) {  // S of row tile i, buffer s
        const uint64_t a = desc_k(smem0 + i * S::slot), b = desc_k(slot_at(fill));
        const uint32_t d = tm + uniform(s) * 128;
        mma_ss<false>(leader, d, a, b, idesc<T>(KT, false));
  #pragma unroll
        for (int k = 1; k < D / 16; ++k) {
          const uint32_t o = ((k >> 2) * kHalf + (k & 3) * 32) >> 4;
          mma_ss<true>(leader, d, a + o, b + o, idesc<T>(KT, false));
        }
      };
      auto pv = [&](int i, uint32_t s, uint32_t fill, int steps, bool first) {
        const uint64_t b = desc_mn(slot_at(fill));
        const uint32_t d = tm + kO + i * 128, a = tm + uniform(s) * 128;
        mma_ts(leader, d, a, b, idesc<T>(D, true), !first);
        if (steps == KT / G16) {
  #pragma unroll
          for (int k = 1; k < KT / G16; ++k) mma_ts(leader, d, a + k * 8, b + k * (G16 * 128 >> 4), idesc<T>(D, true), 1);
        } else {
          for (int k = 1; k < steps; ++k) mma_ts(leader, d, a + k * 8, b + k * (G16 * 128 >> 4), idesc<T>(D, true), 1);
        }
      };
      for (; ok && w.live(); w.next(p), ++item) {
        const int n = w.k_hi - w.k_lo;
        ok = warp_wait(&q_full, item & 1);
        if (NQ == 1) {
          for (int j = -1; ok && j < n; ++j) {
            if (j + 1 < n) {  // the next tile's scores, beside this one's softmax
              const uint32_t fill = f + k_fill<1>(j + 1);
              const uint32_t tt = t + j + 1;
              ok = wait_slot(fill);
              if (!ok) break;
              tm_after_sync();
              qk(0, tt & 1, fill);
              mma_commit(leader, &empty[fill % NS]);
              mma_commit(leader, &s_full[tt & 1]);
              if (j + 2 == n) mma_commit(leader, &q_empty);
            }
            if (j < 0) continue;
            const uint32_t fill = f + v_fill<1>(j, n);
            const uint32_t tt = t + j;
            const int kt = w.k_lo + j;
            const int left = kt < w.p_tiles ? w.s.prefix - kt * KT : w.s.n - (kt - w.p_tiles) * KT;
            ok = wait_slot(fill) && warp_wait(&p_full[tt & 1], (tt >> 1) & 1);
            if (!ok) break;
            tm_after_sync();
            pv(0, tt & 1, fill, (imin(KT, left) + G16 - 1) / G16, j == 0);
            mma_commit(leader, &empty[fill % NS]);
            mma_commit(leader, &o_done[0]);
            if (j + 1 == n) mma_commit(leader, &o_last[0]);
          }
        } else {
          for (int j = -1; ok && j < n; ++j) {
            const uint32_t fk = f + k_fill<2>(j + 1), fv = f + v_fill<2>(j, n), tt = t + j;
            const int kt = w.k_lo + j;
            const int left = kt < w.p_tiles ? w.s.prefix - kt * KT : w.s.n - (kt - w.p_tiles) * KT;
            const int steps = (imin(KT, left) + G16 - 1) / G16;
  #pragma unroll
            for (int i = 0; i < NQ; ++i) {
              if (j >= 0) {
                ok = (i || wait_slot(fv)) && warp_wait(&p_full[i], tt & 1);
                if (!ok) break;
                tm_after_sync();
                pv(i, i, fv, steps, j == 0);
                if (i == NQ - 1) mma_commit(leader, &empty[fv % NS]);
                mma_commit(leader, &o_done[i]);
                if (j + 1 == n) mma_commit(leader, &o_last[i]);
              }
              if (j + 1 < n) {
                ok = i || wait_slot(fk);
                if (!ok) break;
                tm_after_sync();
                qk(i, i, fk);
                if (i == NQ - 1) mma_commit(leader, &empty[fk % NS]);
                mma_commit(leader, &s_full[i]);
                if (i == NQ - 1 && j + 2 == n) mma_commit(leader, &q_empty);
              }
            }
          }
        }
        f += 2 * n;
        t += n;
      }
      if (!ok) {  // MMAs in flight end before the tensor memory is given back
        mma_commit(leader, &drained);
        warp_wait(&drained, 0);
      }
    } else {
      // --------------------------------------------------------------------- Q
      const uint32_t leader = elect_one();
      uint32_t item = 0;
      for (; ok && w.live(); w.next(p), ++item) {
        if (item) ok = warp_wait(&q_empty, (item - 1) & 1);
        if (!ok) break;
        if (KT % p.g == 0) {
          // rows behind the sequence's last belong to other tokens, and to nobody here
          if (leader) mbar_expect(&q_full, S::q);
          __syncwarp();
          if (lane < NQ * (D / 64)) {
            const int i = lane / (D / 64), h = lane % (D / 64);
            tma_3d(smem0 + i * S::slot + h * kHalf, &maps.q, h * 64, w.kvh * p.g,
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
            cp_async16(base + (r >> 7) * S::slot + (c >> 3) * kHalf + (r & 127) * 128 + (((c & 7) ^ (r & 7)) << 4),
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
      }
    }
  } else {
    // --------------------------------------------------------------- softmax
    if constexpr (NQ == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int qi = (warp - 4) >> 2;             // row tile of the NQ
    const int r = (warp & 3) * 32 + lane;       // row in it, and tensor memory lane
    const uint32_t lanes = tm + ((uint32_t)(warp & 3) << 21);  // lane (warp & 3) * 32, column 0
    const uint32_t o_at = lanes + kO + qi * 128;
    uint32_t t = 0, item = 0;
    ExtRec rec{};
    for (; ok && w.live(); w.next(p), ++item) {
      const int rows = w.rows(p.g);
      const int rr = qi * 128 + r;
      const bool mine = rr < rows;
      const bool idle = qi * 128 + (warp & 3) * 32 >= rows;  // no row of this warp exists
      const int tok = mine ? (w.rt * R + rr) / p.g : 0;
      const bool seen = mine && ext_live(p, w.s, tok);
      float m = -INFINITY, l = 0.f;  // maximum that O and l are scaled by (of q.k), sum
      for (int kt = w.k_lo; kt < w.k_hi; ++kt, ++t) {
        const uint32_t sb = NQ == 1 ? t & 1 : qi, par = NQ == 1 ? (t >> 1) & 1 : t & 1;
        ok = warp_wait(&s_full[sb], par);
        if (!ok) break;
        tm_after_sync();
        if (!idle) {
          const uint32_t s_at = lanes + sb * 128;
          uint32_t x[128];
#pragma unroll
          for (int i = 0; i < 4; ++i) tm_ld32(s_at + i * 32, x + i * 32);
          const bool cached = kt < w.p_tiles;
          const int j0 = (cached ? kt : kt - w.p_tiles) * KT;
          const int have = imin(KT, (cached ? w.s.prefix : w.s.n) - j0);
          const bool tree = !cached && p.parents;
          const int see = !seen ? 0 : cached || tree ? have : imin(have, tok - j0 + 1);
          const bool cut = __any_sync(~0u, tree || (mine && see < KT));
          tm_wait_ld();
          if (cut) {
            uint32_t bits[4];
            if (tree) {
              if (seen) ext_tree_mask<4>(p, w.s, tok, j0, bits);
              else bits[0] = bits[1] = bits[2] = bits[3] = 0;
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                bits[i] = see >= 32 * (i + 1) ? ~0u : see > 32 * i ? (1u << (see - 32 * i)) - 1u : 0u;
            }
#pragma unroll
            for (int i = 0; i < 128; ++i)
              if (!((bits[i >> 5] >> (i & 31)) & 1u)) x[i] = 0xFF800000u;
          }
          float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 128; i += 4)
#pragma unroll
            for (int j = 0; j < 4; ++j) top[j] = fmaxf(top[j], __uint_as_float(x[i + j]));
          const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
          const bool first = kt == w.k_lo;
          if (first) {
            m = mx;
          } else if (__any_sync(~0u, (mx - m) * p.scale > 8.f)) {
            const float up = fmaxf(m, mx);
            const float keep = up == -INFINITY ? 1.f : exp2_fast((m - up) * p.scale);
            m = up;
            l *= keep;
            // (this tile's scores were issued behind the P V of the tile before
            // the last one: the phase waited for is the barrier's current one or the one before)
            ok = warp_wait(&o_done[qi], (t - 1) & 1);
            if (!ok) break;
            tm_after_sync();
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {  // (few registers are left beside x)
              uint32_t y[16];
              tm_ld16(o_at + c, y);
              tm_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * keep);
              tm_st16(o_at + c, y);
            }
          }
          __syncwarp();
          const float off = m == -INFINITY ? 0.f : m * p.scale;
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t y[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float a = exp2_fast(fmaf(__uint_as_float(x[c * 64 + 2 * i]), p.scale, -off));
              const float b = exp2_fast(fmaf(__uint_as_float(x[c * 64 + 2 * i + 1]), p.scale, -off));
              sum[(2 * i) & 3] += a;
              sum[(2 * i + 1) & 3] += b;
              y[i] = Pack2<T>::run(a, b);
            }
            tm_st32(s_at + c * 32, y);
          }
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          tm_wait_st();
        }
        tm_before_sync();
        mbar_arrive(&p_full[sb]);
      }
      if (!ok) break;
      // the row tile's output, or this CTA's piece of it
      ok = warp_wait(&o_last[qi], item & 1);
      if (!ok) break;
      tm_after_sync();
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
      if (idle) continue;
      const int row = w.rt * R + rr;
      const int64_t at = ((int64_t)blockIdx.x * 2 + piece) * R + rr;
      const int h = w.kvh * p.g + row % p.g;
      T* dst = static_cast<T*>(p.out) + (int64_t)(w.s.begin + tok) * p.o_st + h * p.o_sh;
      const float inv = whole ? (l != 0.f ? 1.f / l : 0.f) : 1.f;
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        uint32_t y[32];
        __syncwarp();
        tm_ld32(o_at + c, y);
        tm_wait_ld();
        if (!mine) {
        } else if (whole) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t z[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
              z[j] = Pack2<T>::run(__uint_as_float(y[i * 8 + j * 2]) * inv, __uint_as_float(y[i * 8 + j * 2 + 1]) * inv);
            *reinterpret_cast<uint4*>(dst + c + i * 8) = make_uint4(z[0], z[1], z[2], z[3]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *reinterpret_cast<uint4*>(p.part_o + at * D + c + i * 4) =
                make_uint4(y[i * 4], y[i * 4 + 1], y[i * 4 + 2], y[i * 4 + 3]);
        }
      }
      if (mine) {
        const float ml = m == -INFINITY ? -INFINITY : m * p.scale;
        if (!whole) {
          *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(ml, l);
        } else if (p.lse) {
          p.lse[(int64_t)(w.s.begin + tok) * p.Hq + h] =
              l != 0.f ? (ml + log2f(l)) * 0.69314718055994531f : -INFINITY;
        }
      }
    }
    if (tid == 128) p.rec[blockIdx.x] = rec;
  }
  if (!ok && lane == 0) report(p.status, ADAKV_ST_WAIT_TIMEOUT);
  tm_before_sync();
  __syncthreads();
  if (warp == 1) tm_free(tm, 512);
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
  extend_mma_kernel<T, D, NQ><<<grid, 128 * (1 + NQ), Smem<D, NQ>::bytes, st>>>(p, maps);
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
  const int bn[3] = {64, 1, KT}, bg[3] = {64, 1, G16};
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
