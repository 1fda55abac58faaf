// Pages of a cache: copying, forking, freeing and compacting them, and
// appending tokens.
//
// A pool of pages [layers, n_pages] is shared by sequences: row s of the page
// table names sequence s's pages in order, lens[s] its tokens, ref[p] how many
// rows name page p (0: free).  Full pages are shared between forks, the last,
// partly filled page of a sequence never is.  Free pages are taken lowest id
// first in the order of the request, so that every result is determined by
// its inputs.
//
// Fork, compact and append first plan in one CTA (which pages, in which
// order; nothing is changed if the request cannot be met as a whole) and then
// move the data from a second kernel over the whole GPU, launched
// programmatically behind the first.
//
// Bound by HBM where pages move (a CTA moves 32 KB with all loads in flight:
// copying 367 MB takes 117 us, 6.3 TB/s of reads and writes, 96 % of a plain
// copy's rate), by launches and round trips elsewhere: the plan reads its lists in one
// CTA (5 to 7 us with the reference counts of 2,048 to 16,384 pages), freeing 24
// sequences of 190 pages takes 5 us.
#include "kernels.h"

namespace adakv {
namespace {

constexpr int kPageThreads = 1024;
constexpr int kPer = 8;  // reference counts a thread reads at a time

// the plan's lists in the workspace
struct Lists {
  int* head;   // [0] pairs (or tokens) to move, [1] 1 if the request is met, [2] live pages
  int* src;    // [n_pages]
  int* dst;    // [n_pages]
  int* seq;    // [3 * kPagesMaxBatch + 2]
};
__host__ __device__ inline Lists lists_of(int* ws, int n_pages) {
  Lists l;
  l.head = ws;
  l.src = ws + 64;
  l.dst = l.src + n_pages;
  l.seq = l.dst + n_pages;
  return l;
}

struct PlanShared {
  int warp[32];
  uint32_t bad;  // ADAKV_ST_* bits of the request
  uint32_t bits[kPagesMaxSlots / 32];
};

// exclusive sum of v over the block; `total` is the whole sum
__device__ __forceinline__ int block_scan(int v, int* warp, int& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(~0u, inc, o);
    if (lane >= o) inc += t;
  }
  if (lane == 31) warp[w] = inc;
  __syncthreads();
  if (w == 0) {
    int x = warp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(~0u, x, o);
      if (lane >= o) x += t;
    }
    warp[lane] = x;
  }
  __syncthreads();
  total = warp[31];
  const int r = inc - v + (w ? warp[w - 1] : 0);
  __syncthreads();
  return r;
}

// The `want` lowest free pages, ascending, into out; how many there are (at
// most `want`).  Stops at the chunk that holds the last one.
__device__ __forceinline__ int find_free(const int* ref, int n_pages, int want, int* out,
                                         PlanShared& sh) {
  int found = 0;
  for (int at = 0; at < n_pages && found < want; at += kPageThreads * kPer) {
    const int id0 = at + threadIdx.x * kPer;
    int c[kPer], mine = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      c[i] = id0 + i < n_pages ? ref[id0 + i] : 1;
      mine += c[i] == 0;
    }
    int total;
    int r = found + block_scan(mine, sh.warp, total);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (c[i] == 0) {
        if (r < want) out[r] = id0 + i;
        ++r;
      }
    found += total;
  }
  __syncthreads();
  return found < want ? found : want;
}

// Marks slot s; false if it is out of range or was marked before.
__device__ __forceinline__ bool mark_slot(PlanShared& sh, int s, int n_slots) {
  if (s < 0 || s >= n_slots) return false;
  const uint32_t bit = 1u << (s & 31);
  return !(atomicOr(&sh.bits[s >> 5], bit) & bit);
}

__device__ __forceinline__ void clear_bits(PlanShared& sh, int n_slots) {
  for (int i = threadIdx.x; i < (n_slots + 31) / 32; i += kPageThreads) sh.bits[i] = 0;
  if (threadIdx.x == 0) sh.bad = 0;
  __syncthreads();
}

// The whole block's bits.
__device__ __forceinline__ uint32_t all_bits(PlanShared& sh, uint32_t bad) {
  if (bad) atomicOr(&sh.bad, bad);
  __syncthreads();
  return sh.bad;
}

// ---------------------------------------------------------------------------
// moving whole pages
// ---------------------------------------------------------------------------
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 8;
constexpr int kCopyChunk = kCopyThreads * kCopyUnroll * 16;  // bytes a CTA moves at a time

// One chunk of the page of one (pair, layer, k or v): task = ((pair * layers +
// layer) * 2 + which) * chunks + chunk.
__device__ __forceinline__ void copy_task(const PagePool& p, int from, int to, int layer, int which,
                                          int64_t off) {
  unsigned char* base = which ? p.v + layer * p.v_sl : p.k + layer * p.k_sl;
  const int64_t sp = which ? p.v_sp : p.k_sp;
  const unsigned char* src = base + from * sp;
  unsigned char* dst = base + to * sp;
  uint4 x[kCopyUnroll];
#pragma unroll
  for (int i = 0; i < kCopyUnroll; ++i) {
    const int64_t at = off + ((int64_t)i * kCopyThreads + threadIdx.x) * 16;
    if (at < p.page_bytes) x[i] = __ldcs(reinterpret_cast<const uint4*>(src + at));
  }
#pragma unroll
  for (int i = 0; i < kCopyUnroll; ++i) {
    const int64_t at = off + ((int64_t)i * kCopyThreads + threadIdx.x) * 16;
    if (at < p.page_bytes) __stcs(reinterpret_cast<uint4*>(dst + at), x[i]);
  }
}

__device__ __forceinline__ void copy_pairs(const PagePool& p, const int* src, const int* dst, int n,
                                           uint32_t* status) {
  const int chunks = (int)((p.page_bytes + kCopyChunk - 1) / kCopyChunk);
  const int per_pair = p.layers * 2 * chunks;
  const int64_t tasks = (int64_t)n * per_pair;
  for (int64_t t = blockIdx.x; t < tasks; t += gridDim.x) {
    const int pair = (int)(t / per_pair), rest = (int)(t % per_pair);
    const int from = src[pair], to = dst[pair];
    if (from < 0 || from >= p.n_pages || to < 0 || to >= p.n_pages) {
      if (threadIdx.x == 0) report(status, ADAKV_ST_BAD_BLOCK_ID);
      continue;
    }
    const int chunk = rest % chunks, plane = rest / chunks;
    copy_task(p, from, to, plane >> 1, plane & 1, (int64_t)chunk * kCopyChunk);
  }
}

__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const PagePool p, const int* src,
                                                            const int* dst, int n, uint32_t* status) {
  copy_pairs(p, src, dst, n, status);
}

// ---------------------------------------------------------------------------
// fork
// ---------------------------------------------------------------------------
// seq[i]: tokens of pair i's source; seq[kPagesMaxBatch + i]: the fresh page
// of its last, partly filled page (-1: it has none)
__global__ void __launch_bounds__(kPageThreads) fork_plan_kernel(const PageTable t, int n_pages,
                                                                 int page_size, const int* src,
                                                                 const int* dst, int n,
                                                                 uint32_t* status, int* ws) {
  extern __shared__ __align__(16) unsigned char raw[];
  PlanShared& sh = *reinterpret_cast<PlanShared*>(raw);
  const Lists L = lists_of(ws, n_pages);
  clear_bits(sh, t.n_slots);
  uint32_t bad = 0;
  int want = 0;
  for (int i0 = 0; i0 < n; i0 += kPageThreads) {
    const int i = i0 + threadIdx.x;
    int part = 0, len = 0;
    if (i < n) {
      const int s = src[i], d = dst[i];
      if (s < 0 || s >= t.n_slots || !mark_slot(sh, d, t.n_slots)) {
        bad |= ADAKV_ST_BAD_SLOT;
      } else {
        len = t.lens[s];
        if (t.lens[d] != 0) bad |= ADAKV_ST_BAD_SLOT;
        if (len < 0 || len > (int64_t)t.width * page_size) {
          bad |= ADAKV_ST_BAD_SEQ_LEN;
          len = 0;
        }
        part = len % page_size != 0;
      }
    }
    int total;
    const int r = want + block_scan(part, sh.warp, total);
    want = imin(want + total, n_pages + 1);
    if (i < n) {
      L.seq[i] = len;
      L.seq[kPagesMaxBatch + i] = part ? r : -1;
    }
  }
  bad = all_bits(sh, bad);
  int found = 0;
  if (!bad) {
    found = want > n_pages ? 0 : find_free(t.ref, n_pages, want, L.dst, sh);
    if (found < want) bad = ADAKV_ST_NO_PAGES;
  }
  if (bad) {
    if (threadIdx.x == 0) {
      report(status, bad);
      L.head[0] = 0;
      L.head[1] = 0;
    }
    return;
  }
  for (int i = threadIdx.x; i < n; i += kPageThreads) {
    const int len = L.seq[i], r = L.seq[kPagesMaxBatch + i];
    if (r >= 0) {
      const int page = L.dst[r];
      L.src[r] = t.table[src[i] * t.stride + len / page_size];
      L.seq[kPagesMaxBatch + i] = page;
      t.ref[page] = 1;
    }
    t.lens[dst[i]] = len;
  }
  if (threadIdx.x == 0) {
    L.head[0] = want;
    L.head[1] = 1;
  }
}

__global__ void __launch_bounds__(kCopyThreads) fork_move_kernel(const PagePool p, const PageTable t,
                                                                 const int* src, const int* dst, int n,
                                                                 uint32_t* status, int* ws) {
  pdl_wait();
  const Lists L = lists_of(ws, p.n_pages);
  if (!L.head[1]) return;
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    const int len = L.seq[i], fresh = L.seq[kPagesMaxBatch + i];
    const int full = len / p.page_size;
    const int* from = t.table + src[i] * t.stride;
    int* to = t.table + dst[i] * t.stride;
    if (len == 0) continue;
    for (int j = threadIdx.x; j < t.width; j += kCopyThreads) {
      int id = from[j];
      if (j < full) {
        if (id >= 0 && id < p.n_pages) atomicAdd(&t.ref[id], 1);
        else report(status, ADAKV_ST_BAD_BLOCK_ID);
      } else {
        id = j == full && fresh >= 0 ? fresh : -1;
      }
      to[j] = id;
    }
  }
  copy_pairs(p, L.src, L.dst, L.head[0], status);
}

// ---------------------------------------------------------------------------
// free
// ---------------------------------------------------------------------------
// A row's entries are taken out with an exchange, so a slot that is listed
// twice gives its pages back once.
__global__ void __launch_bounds__(256) free_kernel(const PageTable t, int n_pages, const int* slots,
                                                   uint32_t* status) {
  const int s = slots[blockIdx.x];
  if (s < 0 || s >= t.n_slots) {
    if (threadIdx.x == 0 && blockIdx.y == 0) report(status, ADAKV_ST_BAD_SLOT);
    return;
  }
  int* row = t.table + s * t.stride;
  for (int j = blockIdx.y * 256 + threadIdx.x; j < t.width; j += gridDim.y * 256) {
    if (row[j] < 0) continue;
    const int id = atomicExch(&row[j], -1);
    if (id < 0) continue;
    if (id >= n_pages || atomicSub(&t.ref[id], 1) <= 0) report(status, ADAKV_ST_BAD_BLOCK_ID);
  }
  if (threadIdx.x == 0 && blockIdx.y == 0) t.lens[s] = 0;
}

// ---------------------------------------------------------------------------
// compact
// ---------------------------------------------------------------------------
// The i-th live page at or above the number of live pages goes to the i-th
// hole below it; seq is not used, src / dst list the moves.
__global__ void __launch_bounds__(kPageThreads) compact_plan_kernel(const PageTable t, int n_pages,
                                                                    int* ws) {
  extern __shared__ __align__(16) unsigned char raw[];
  PlanShared& sh = *reinterpret_cast<PlanShared*>(raw);
  const Lists L = lists_of(ws, n_pages);
  int mine = 0;
  for (int i = threadIdx.x; i < n_pages; i += kPageThreads) mine += t.ref[i] > 0;
  int live;
  block_scan(mine, sh.warp, live);
  int holes = 0, movers = 0;
  for (int at = 0; at < n_pages; at += kPageThreads * kPer) {
    const int id0 = at + threadIdx.x * kPer;
    int c[kPer], h = 0, m = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int id = id0 + i;
      c[i] = id < n_pages ? t.ref[id] : 0;
      h += id < live && c[i] <= 0;
      m += id >= live && c[i] > 0;
    }
    int total;  // both counts at once: at most 8192 each
    const int r = block_scan(h | (m << 16), sh.warp, total);
    int rh = holes + (r & 0xFFFF), rm = movers + (r >> 16);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int id = id0 + i;
      if (id < live && c[i] <= 0) L.dst[rh++] = id;
      if (id >= live && id < n_pages && c[i] > 0) L.src[rm++] = id;
    }
    holes += total & 0xFFFF;
    movers += total >> 16;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < movers; i += kPageThreads) {
    t.ref[L.dst[i]] = t.ref[L.src[i]];
    t.ref[L.src[i]] = 0;
  }
  if (threadIdx.x == 0) {
    L.head[0] = movers;
    L.head[1] = 1;
    L.head[2] = live;
  }
}

__global__ void __launch_bounds__(kCopyThreads) compact_move_kernel(const PagePool p, const PageTable t,
                                                                    uint32_t* status, int* ws) {
  pdl_wait();
  const Lists L = lists_of(ws, p.n_pages);
  const int moves = L.head[0], live = L.head[2];
  if (moves == 0) return;
  const int64_t cells = (int64_t)t.n_slots * t.width;
  for (int64_t i = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x; i < cells;
       i += (int64_t)gridDim.x * kCopyThreads) {
    int* cell = t.table + (i / t.width) * t.stride + i % t.width;
    const int id = *cell;
    if (id < live) continue;  // stays (or none)
    int lo = 0, hi = moves;   // the move whose source is id
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (L.src[mid] <= id) lo = mid; else hi = mid;
    }
    if (L.src[lo] == id) *cell = L.dst[lo];
    else report(status, ADAKV_ST_BAD_BLOCK_ID);
  }
  copy_pairs(p, L.src, L.dst, moves, status);
}

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
// seq[b]: accepted tokens before sequence b (b <= B); seq[kPagesMaxBatch + 1 +
// b]: its length before; seq[2 kPagesMaxBatch + 1 + b]: fresh pages before it
__global__ void __launch_bounds__(kPageThreads) append_plan_kernel(const PageTable t, int n_pages,
                                                                   int page_size, const PageAppend a,
                                                                   uint32_t* status, int* ws) {
  extern __shared__ __align__(16) unsigned char raw[];
  PlanShared& sh = *reinterpret_cast<PlanShared*>(raw);
  const Lists L = lists_of(ws, n_pages);
  int* len0 = L.seq + kPagesMaxBatch + 1;
  int* first = L.seq + 2 * kPagesMaxBatch + 1;
  clear_bits(sh, t.n_slots);
  uint32_t bad = 0;
  int tokens = 0, want = 0;
  // the positions that are used, an entry a thread (a thread a sequence would
  // wait for each of its entries)
  for (int64_t x = threadIdx.x; a.index && x < (int64_t)a.B * a.index_width; x += kPageThreads) {
    const int b = (int)(x / a.index_width), i = (int)(x % a.index_width);
    const int n = a.counts ? a.counts[b] : a.index_width;
    const int at = a.index[b * a.index_stride + i];
    if (i < n && (at < 0 || at >= a.cu[b + 1] - a.cu[b])) bad |= ADAKV_ST_BAD_SEQ_LEN;
  }
  for (int b0 = 0; b0 < a.B; b0 += kPageThreads) {
    const int b = b0 + threadIdx.x;
    int n = 0, need = 0, len = 0;
    if (b < a.B) {
      const int s = a.slots ? a.slots[b] : b;
      const int c0 = a.cu[b], c1 = a.cu[b + 1];
      n = a.counts ? a.counts[b] : a.index ? a.index_width : c1 - c0;
      if (!mark_slot(sh, s, t.n_slots)) bad |= ADAKV_ST_BAD_SLOT;
      else len = t.lens[s];
      if (c0 < 0 || c1 < c0 || c1 > a.T || n < 0 || n > (a.index ? a.index_width : c1 - c0) || len < 0 ||
          (int64_t)len + n > (int64_t)t.width * page_size) {
        bad |= ADAKV_ST_BAD_SEQ_LEN;
        n = 0;
        len = 0;
      }
      if (n > 0 && len % page_size != 0) {  // the page that is written on has no other owner
        const int tail = t.table[s * t.stride + len / page_size];
        if (tail < 0 || tail >= n_pages || t.ref[tail] != 1) bad |= ADAKV_ST_BAD_BLOCK_ID;
      }
      need = (len + n + page_size - 1) / page_size - (len + page_size - 1) / page_size;
    }
    int total;
    const int at = tokens + block_scan(n, sh.warp, total);
    tokens += total;
    const int page_at = want + block_scan(imin(need, n_pages + 1), sh.warp, total);
    want = imin(want + total, n_pages + 1);
    if (b < a.B) {
      L.seq[b] = at;
      len0[b] = len;
      first[b] = page_at;
    }
  }
  bad = all_bits(sh, bad);
  int found = 0;
  if (!bad) {
    if (want <= n_pages) found = find_free(t.ref, n_pages, want, L.dst, sh);
    if (found < want) bad = ADAKV_ST_NO_PAGES;
  }
  if (bad) {
    if (threadIdx.x == 0) {
      report(status, bad);
      L.head[0] = 0;
      L.head[1] = 0;
    }
    return;
  }
  if (threadIdx.x == 0) {
    L.seq[a.B] = tokens;
    L.head[0] = tokens;
    L.head[1] = 1;
  }
  __syncthreads();
  for (int b = threadIdx.x; b < a.B; b += kPageThreads) {
    const int s = a.slots ? a.slots[b] : b;
    const int n = L.seq[b + 1] - L.seq[b], len = len0[b];
    const int have = (len + page_size - 1) / page_size, last = (len + n + page_size - 1) / page_size;
    for (int j = have; j < last; ++j) {
      const int page = L.dst[first[b] + j - have];
      t.table[s * t.stride + j] = page;
      t.ref[page] = 1;
    }
    t.lens[s] = len + n;
  }
}

__global__ void __launch_bounds__(kCopyThreads) append_move_kernel(const PagePool p, const PageTable t,
                                                                   const PageAppend a, uint32_t* status,
                                                                   int* ws) {
  pdl_wait();
  const Lists L = lists_of(ws, p.n_pages);
  const int tokens = L.head[0];
  const int* len0 = L.seq + kPagesMaxBatch + 1;
  const int row16 = a.row_bytes / 16;
  const int units = p.layers * 2 * a.Hkv * row16;  // 16-byte words of a token
  for (int x = blockIdx.x; x < tokens; x += gridDim.x) {
    int lo = 0, hi = a.B;  // last b with seq[b] <= x
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (L.seq[mid] <= x) lo = mid; else hi = mid;
    }
    const int i = x - L.seq[lo];
    const int s = a.slots ? a.slots[lo] : lo;
    const int tok = a.cu[lo] + (a.index ? a.index[lo * a.index_stride + i] : i);
    const int pos = len0[lo] + i;
    const int page = t.table[s * t.stride + pos / p.page_size];
    if (page < 0 || page >= p.n_pages) {
      if (threadIdx.x == 0) report(status, ADAKV_ST_BAD_BLOCK_ID);
      continue;
    }
    const int64_t place = (int64_t)(pos % p.page_size) * a.row_bytes;
    for (int u = threadIdx.x; u < units; u += kCopyThreads) {
      const int c = u % row16, r = u / row16;
      const int h = r % a.Hkv, plane = r / a.Hkv;
      const int layer = plane >> 1;
      const unsigned char* src = (plane & 1)
          ? a.v + layer * a.v_sl + tok * a.v_st + h * a.v_sh
          : a.k + layer * a.k_sl + tok * a.k_st + h * a.k_sh;
      unsigned char* dst = (plane & 1) ? p.v + layer * p.v_sl + page * p.v_sp
                                       : p.k + layer * p.k_sl + page * p.k_sp;
      dst += (int64_t)h * p.page_size * a.row_bytes + place + c * 16;
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src + c * 16);
    }
  }
}

int move_grid(int64_t tasks) { return (int)std::min<int64_t>(std::max<int64_t>(tasks, 1), 148 * 8); }

int64_t pair_tasks(const PagePool& p) {
  return (int64_t)p.layers * 2 * ((p.page_bytes + kCopyChunk - 1) / kCopyChunk);
}

template <typename... KArgs, typename... Args>
cudaError_t launch_behind(void (*k)(KArgs...), int grid, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kCopyThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k, args...);
}

}  // namespace

size_t page_ws_bytes(int n_pages) {
  return sizeof(int) * (64 + 2 * (size_t)n_pages + 3 * (size_t)kPagesMaxBatch + 2);
}

cudaError_t launch_pages_copy(const PagePool& p, const int* src, const int* dst, int n,
                              uint32_t* status, cudaStream_t st) {
  const int64_t tasks = n * pair_tasks(p);
  copy_kernel<<<(int)std::min<int64_t>(tasks, 1 << 20), kCopyThreads, 0, st>>>(p, src, dst, n, status);
  return cudaGetLastError();
}

cudaError_t launch_pages_fork(const PagePool& p, const PageTable& t, const int* src, const int* dst,
                              int n, uint32_t* status, int* lists, cudaStream_t st) {
  fork_plan_kernel<<<1, kPageThreads, sizeof(PlanShared), st>>>(t, p.n_pages, p.page_size, src, dst, n,
                                                                status, lists);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  return launch_behind(fork_move_kernel, move_grid(std::max<int64_t>(n, n * pair_tasks(p))), st, p, t,
                       src, dst, n, status, lists);
}

cudaError_t launch_pages_free(const PageTable& t, int n_pages, const int* slots, int n,
                              uint32_t* status, cudaStream_t st) {
  const int split = std::min(std::max(t.width / 1024, 1), 16);
  free_kernel<<<dim3(n, split), 256, 0, st>>>(t, n_pages, slots, status);
  return cudaGetLastError();
}

cudaError_t launch_pages_compact(const PagePool& p, const PageTable& t, uint32_t* status, int* lists,
                                 cudaStream_t st) {
  compact_plan_kernel<<<1, kPageThreads, sizeof(PlanShared), st>>>(t, p.n_pages, lists);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  return launch_behind(compact_move_kernel, move_grid((int64_t)p.n_pages / 2 * pair_tasks(p)), st, p, t,
                       status, lists);
}

cudaError_t launch_pages_append(const PagePool& p, const PageTable& t, const PageAppend& a,
                                uint32_t* status, int* lists, cudaStream_t st) {
  append_plan_kernel<<<1, kPageThreads, sizeof(PlanShared), st>>>(t, p.n_pages, p.page_size, a, status,
                                                                  lists);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int64_t most = a.index ? (int64_t)a.B * a.index_width : a.T;
  return launch_behind(append_move_kernel, move_grid(most), st, p, t, a, status, lists);
}

}  // namespace adakv
