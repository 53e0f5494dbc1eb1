// Pages of a paged cache while its sequences live: copies inside the pool, forks,
// frees and compaction, all from tensors that stay on the device.
//
// The state is the pool [L, 2, NB, page], the block tables [B, MB] (-1 padded),
// the context lengths [B] and one count per block, ref_counts [NB]: how many table
// rows (or other holders) keep it.  A block whose count is not above 0 is free.  A
// fork shares a parent's full blocks (counts go up) and copies the tokens of the
// last, unfinished one into a fresh block; a free takes the counts down again;
// free blocks are found, lowest first, by a scan of the counts; a compaction moves
// the highest live blocks into the lowest holes.  Counts change by integer
// atomics, whose order changes no result.
//
// The copies are HBM-bound (copies of 128 blocks of 32 layers, 537 MB read and written:
// 95.6 us, 5.6 TB/s; a large copy reaches 6.6); everything else is a few microseconds
// of latency, so each operation is one launch (a compaction two).  The scans need each
// chunk's number of blocks before it: every workgroup counts them itself, a stream of
// reads from L2, which is shorter than a second launch would be (131072 blocks: 8.7 us
// in all, 18 with one load in flight a thread).
#include "hs_kernels.h"
#include "hs_kvrows.h"
#include "hs_private.h"

#include <algorithm>

namespace hs {

namespace {

constexpr int kCopyThreads = 256;
constexpr int64_t kPiece = kCopyThreads * 16;   // bytes that a workgroup copies at once
constexpr int kScanThreads = 1024;
constexpr int kScanPer = 4;                     // counts per thread: one 16-byte load
constexpr int kScanChunk = kScanThreads * kScanPer;
constexpr int kMaxScan = 1 << 22;               // counts: every workgroup reads all before it
constexpr int kInlinePairs = HS_KV_HOST_IDS / 2;

// bytes [piece * kPiece, ...) of a page of `bytes` (vec: 16 bytes a thread)
__device__ inline void copy_piece(const uint8_t* src, uint8_t* dst, int64_t bytes, int64_t piece,
                                  bool vec) {
  if (vec) {
    const int64_t off = piece * kPiece + (int64_t)threadIdx.x * 16;
    if (off < bytes) store16_stream(dst + off, load16_stream(src + off));
  } else {
    const int64_t end = min(bytes, (piece + 1) * kPiece);
    for (int64_t off = piece * kPiece + threadIdx.x; off < end; off += kCopyThreads)
      dst[off] = src[off];
  }
}

// Workgroup b of n runs on XCD b % 8: each XCD takes one contiguous run of the jobs
// (128 blocks of 32 layers, 32-KB pages: 100.9 us in grid order, 95.6 so; whole pages a
// workgroup 101.2; stores without the streaming hint 101.2).
__device__ inline int64_t xcd_run(int64_t b, int64_t n) {
  const int64_t x = b % 8, q = n / 8, r = n % 8;
  return x * q + (x < r ? x : r) + b / 8;
}

// `bytes` by one workgroup, 8 loads of a thread at a time.
template <bool kVec>
__device__ inline void copy_bytes(const uint8_t* src, uint8_t* dst, int64_t bytes) {
  if constexpr (kVec) {
    constexpr int kU = 8;
    for (int64_t base = (int64_t)threadIdx.x * 16; base < bytes; base += kU * kPiece) {
      uint4 v[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (base + u * kPiece < bytes) v[u] = load16_stream(src + base + u * kPiece);
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (base + u * kPiece < bytes) store16_stream(dst + base + u * kPiece, v[u]);
    }
  } else {
    for (int64_t off = threadIdx.x; off < bytes; off += kCopyThreads) dst[off] = src[off];
  }
}

// ---- copies inside the pool -------------------------------------------------

struct PairsInMemory {
  const int64_t *src, *dst;
  __device__ int64_t from(int64_t i) const { return src[i]; }
  __device__ int64_t to(int64_t i) const { return dst[i]; }
};
struct PairsInArguments {
  int32_t src[kInlinePairs], dst[kInlinePairs];
  __device__ int64_t from(int64_t i) const { return src[i]; }
  __device__ int64_t to(int64_t i) const { return dst[i]; }
};

// Workgroup w copies piece (w % pieces) of page (w / pieces) = (i * 2 L) + (l, c).
template <bool kVec, typename Pairs>
__global__ __launch_bounds__(kCopyThreads) void copy_blocks_kernel(uint8_t* pool, Pairs ids, int first,
                                                                   int L2, int NB, int64_t page,
                                                                   int64_t pieces) {
  const int64_t w = xcd_run(blockIdx.x, gridDim.x);
  const int64_t pg = w / pieces, piece = w - pg * pieces;
  const int64_t i = pg / L2, lc = pg - i * L2;
  const int64_t s = ids.from(first + i), d = ids.to(first + i);
  if (s < 0 || s >= NB || d < 0 || d >= NB) return;
  copy_piece(pool + (lc * NB + s) * page, pool + (lc * NB + d) * page, page, piece, kVec);
}

// ---- scans of the counts ----------------------------------------------------

// Sum over the workgroup, in every thread.
__device__ inline int block_sum(int x, int* part) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
  __syncthreads();
  int s = 0;
#pragma unroll
  for (int i = 0; i < kScanThreads / 64; ++i) s += part[i];
  __syncthreads();
  return s;
}

// Sum of the threads before this one, and of all.
__device__ inline int block_scan(int x, int* part, int& total) {
  int inc = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(inc, o);
    if ((int)(threadIdx.x & 63) >= o) inc += y;
  }
  if ((threadIdx.x & 63) == 63) part[threadIdx.x >> 6] = inc;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kScanThreads / 64; ++i) {
    if (i < (int)(threadIdx.x >> 6)) before += part[i];
    total += part[i];
  }
  __syncthreads();
  return before + inc - x;
}

// Live blocks among [first, end), this thread's share; first is a multiple of
// kScanChunk, so 16-byte loads start as aligned as refs does (vec).
__device__ inline int count_live(const int32_t* refs, int first, int end, bool vec) {
  int live = 0;
  int i = first;
  if (vec) {
    const int4* v = reinterpret_cast<const int4*>(refs) + threadIdx.x;
#pragma unroll 8
    for (; i + kScanChunk <= end; i += kScanChunk) {
      const int4 x = v[i / 4];
      live += (x.x > 0) + (x.y > 0) + (x.z > 0) + (x.w > 0);
    }
  }
#pragma unroll 4
  for (i += threadIdx.x; i < end; i += kScanThreads) live += refs[i] > 0;
  return live;
}

// out[0 .. n): the lowest free blocks, -1 past the last.
__global__ __launch_bounds__(kScanThreads) void find_free_kernel(const int32_t* refs, int NB,
                                                                 int32_t* out, int n, bool vec) {
  __shared__ int part[kScanThreads / 64];
  const int first = blockIdx.x * kScanChunk;
  const int before = first - block_sum(count_live(refs, 0, first, vec), part);   // free blocks
  const bool last = blockIdx.x == gridDim.x - 1;
  if (before >= n && !last) return;
  const int i0 = first + threadIdx.x * kScanPer;
  bool free_[kScanPer];
  int mine = 0;
#pragma unroll
  for (int e = 0; e < kScanPer; ++e) {
    free_[e] = i0 + e < NB && refs[i0 + e] <= 0;
    mine += free_[e];
  }
  int total;
  int at = before + block_scan(mine, part, total);
#pragma unroll
  for (int e = 0; e < kScanPer; ++e)
    if (free_[e]) {
      if (at < n) out[at] = i0 + e;
      ++at;
    }
  if (last)
    for (int64_t i = (int64_t)before + total + threadIdx.x; i < n; i += kScanThreads) out[i] = -1;
}

// ---- fork -------------------------------------------------------------------

struct ForkArgs {
  uint8_t* pool;
  int L2, NB, BS;
  int64_t page;
  int32_t* bt;          // [B, MB]
  int32_t* ctx;         // [B]
  int32_t* refs;        // [NB]
  const int32_t *parents, *children, *fresh;   // [n]
  int32_t* forked;      // [n]
  int B, MB;
};

// A child's plan, the same in every workgroup that works for it: the parent's
// full blocks, the tokens of its last one and where they lie.  False: no fork, and
// without `rows` (a row that is none, or its own parent) no row to empty either.
struct ForkPlan {
  bool rows;
  int parent, child, full, rem, last, fresh, ctx;
};
__device__ inline bool fork_plan(const ForkArgs& a, int i, ForkPlan& p) {
  p.parent = a.parents[i];
  p.child = a.children[i];
  p.rows = p.parent >= 0 && p.parent < a.B && p.child >= 0 && p.child < a.B && p.parent != p.child;
  if (!p.rows) return false;
  p.ctx = (int)max((int64_t)0, min((int64_t)a.ctx[p.parent], (int64_t)a.MB * a.BS));
  p.full = p.ctx / a.BS;
  p.rem = p.ctx - p.full * a.BS;
  p.last = p.fresh = -1;
  if (p.rem) {
    p.last = a.bt[(int64_t)p.parent * a.MB + p.full];
    p.fresh = a.fresh[i];
    if (p.last < 0 || p.last >= a.NB || p.fresh < 0 || p.fresh >= a.NB || p.last == p.fresh)
      return false;
  }
  return true;
}

// y 0: the child's table row and the counts; y 1 + (l, c): the tokens of the last
// block's page, whose loads are all on their way behind one walk of dependent reads
// (us, a workgroup per 4 KB / per page: 16 children, 32 layers, 32-KB pages 12.5 / 5.7, 64
// children 42 / 27).
template <bool kVec>
__global__ __launch_bounds__(kCopyThreads) void fork_kernel(ForkArgs a) {
  const int i = blockIdx.x;
  ForkPlan p;
  const bool ok = fork_plan(a, i, p);
  if (blockIdx.y > 0) {
    if (!ok || !p.rem) return;
    const int64_t lc = blockIdx.y - 1;
    copy_bytes<kVec>(a.pool + (lc * a.NB + p.last) * a.page, a.pool + (lc * a.NB + p.fresh) * a.page,
                     a.page / a.BS * p.rem);
    return;
  }
  if (threadIdx.x == 0) a.forked[i] = ok;
  if (!p.rows) return;
  int32_t* row = a.bt + (int64_t)p.child * a.MB;
  const int32_t* from = a.bt + (int64_t)p.parent * a.MB;   // read only where ok
  for (int j = threadIdx.x; j < a.MB; j += kCopyThreads) {
    int id = -1;
    if (ok && j < p.full) id = from[j];
    else if (ok && j == p.full && p.rem) id = p.fresh;
    row[j] = id;
    if (id >= 0 && id < a.NB) atomicAdd(&a.refs[id], 1);
  }
  if (threadIdx.x == 0) a.ctx[p.child] = ok ? p.ctx : 0;
}

// ---- free -------------------------------------------------------------------

// Row rows[x], entries of chunk y.  An entry is taken out of the table by an
// exchange, so a row that is named twice is freed once; a count that is 0 already
// stays there.
__global__ __launch_bounds__(kCopyThreads) void free_kernel(int32_t* bt, int32_t* ctx,
                                                            int32_t* refs, const int32_t* rows,
                                                            int B, int MB, int NB) {
  const int b = rows[blockIdx.x];
  if (b < 0 || b >= B) return;
  const int64_t j = (int64_t)blockIdx.y * kCopyThreads + threadIdx.x;
  if (j == 0) ctx[b] = 0;
  if (j >= MB) return;
  const int id = atomicExch(&bt[(int64_t)b * MB + j], -1);
  if (id >= 0 && id < NB && atomicSub(&refs[id], 1) <= 0) atomicAdd(&refs[id], 1);
}

// ---- compaction -------------------------------------------------------------

// The plan, in the caller's workspace: with `live` blocks in all, rank r of the
// holes below `live` (ascending) is filled by rank r of the live blocks at or
// above it (descending).
struct CompactPlan {
  int32_t* n;        // [1] moves
  int32_t* hole;     // [NB] by rank
  int32_t* mover;    // [NB] by rank
  int32_t* to;       // [NB] the block's new id; -1: free; -2 - r: the r-th hole
};

__global__ __launch_bounds__(kScanThreads) void compact_plan_kernel(const int32_t* refs, int NB,
                                                                    CompactPlan p, int32_t* live_out,
                                                                    bool vec) {
  __shared__ int part[kScanThreads / 64];
  const int first = blockIdx.x * kScanChunk;
  const int own_before = count_live(refs, 0, first, vec);
  const int rest = count_live(refs, first, NB, vec);
  const int before = block_sum(own_before, part);
  const int live = before + block_sum(rest, part);
  const int i0 = first + threadIdx.x * kScanPer;
  bool on[kScanPer];
  int mine = 0;
#pragma unroll
  for (int e = 0; e < kScanPer; ++e) {
    on[e] = i0 + e < NB && refs[i0 + e] > 0;
    mine += on[e];
  }
  int total;
  int at = before + block_scan(mine, part, total);   // live blocks before this one
#pragma unroll
  for (int e = 0; e < kScanPer; ++e) {
    const int id = i0 + e;
    if (id < NB) {
      int to = -1;
      if (on[e]) {
        to = id;
        if (id >= live) {
          const int r = live - 1 - at;
          p.mover[r] = id;
          to = -2 - r;
        }
        ++at;
      } else if (id < live) {
        p.hole[id - at] = id;
      }
      p.to[id] = to;
      if (id == live - 1) *p.n = live - at;   // the live blocks that lie above
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    *live_out = live;
    if (live == 0) *p.n = 0;
  }
}

template <bool kVec>
__global__ __launch_bounds__(kCopyThreads) void compact_move_kernel(uint8_t* pool, int L2, int NB,
                                                                    int64_t page, int32_t* bt, int64_t entries,
                                                                    int32_t* refs, CompactPlan p,
                                                                    int32_t* moved_to) {
  const int moves = *p.n;
  const int64_t t0 = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x;
  const int64_t step = (int64_t)gridDim.x * kCopyThreads;
  auto resolve = [&](int id) {
    const int to = p.to[id];
    return to < -1 ? p.hole[-2 - to] : to;
  };
  for (int64_t i = t0; i < NB; i += step) moved_to[i] = resolve((int)i);
  for (int64_t i = t0; i < entries; i += step) {
    const int id = bt[i];
    if (id >= 0 && id < NB) bt[i] = resolve(id);
  }
  for (int64_t i = t0; i < moves; i += step) {   // holes and movers are disjoint
    const int m = p.mover[i];
    refs[p.hole[i]] = refs[m];
    refs[m] = 0;
  }
  const int64_t jobs = (int64_t)moves * L2;
  for (int64_t w = blockIdx.x; w < jobs; w += gridDim.x) {
    const int64_t i = w / L2, lc = w - i * L2;
    copy_bytes<kVec>(pool + (lc * NB + p.mover[i]) * page, pool + (lc * NB + p.hole[i]) * page, page);
  }
}

bool pool_fits(int L, int NB, int64_t page) { return sat_mul(L, 2, NB, page) != INT64_MAX; }

bool pool_vec(const void* pool, int64_t page) { return page % 16 == 0 && aligned16(pool); }

template <typename Pairs>
int launch_copy(void* pool, int L, int NB, int64_t page, const Pairs& ids, int n, hipStream_t stream) {
  const int64_t pieces = ceil_div(page, kPiece);
  const int64_t per_block = sat_mul(2, L, pieces);
  if (!grid_fits(per_block, kCopyThreads)) return fail(HS_EUNSUPPORTED, "page copy grid too large");
  if (!pool_fits(L, NB, page)) return fail(HS_EUNSUPPORTED, "pool too large for 64-bit offsets");
  uint8_t* p = static_cast<uint8_t*>(pool);
  // as many blocks as one launch holds (64 GiB of copies)
  const int most = (int)std::min((int64_t)n, (((int64_t)1 << 32) / kCopyThreads - 1) / per_block);
  profile_begin(stream);
  for (int first = 0; first < n; first += std::min(most, n - first)) {
    const dim3 g((unsigned)(std::min(most, n - first) * per_block)), t(kCopyThreads);
    if (pool_vec(pool, page))
      hipLaunchKernelGGL((copy_blocks_kernel<true, Pairs>), g, t, 0, stream, p, ids, first, 2 * L, NB, page,
                         pieces);
    else
      hipLaunchKernelGGL((copy_blocks_kernel<false, Pairs>), g, t, 0, stream, p, ids, first, 2 * L, NB, page,
                         pieces);
  }
  profile_end(stream);
  return check_launch("kv copy");
}

}  // namespace

int launch_copy_blocks(void* pool, int L, int NB, int64_t page, const int64_t* src,
                       const int64_t* dst, int n, hipStream_t stream) {
  return launch_copy(pool, L, NB, page, PairsInMemory{src, dst}, n, stream);
}

int launch_copy_blocks_host_ids(void* pool, int L, int NB, int64_t page, const int64_t* src,
                                const int64_t* dst, int n, hipStream_t stream) {
  if (n > kInlinePairs) return fail(HS_EUNSUPPORTED, "too many host block ids for one launch");
  PairsInArguments ids;
  for (int i = 0; i < kInlinePairs; ++i) {   // an id outside the pool is skipped by the kernel
    const bool ok = i < n && src[i] >= 0 && src[i] < NB && dst[i] >= 0 && dst[i] < NB;
    ids.src[i] = ok ? (int32_t)src[i] : -1;
    ids.dst[i] = ok ? (int32_t)dst[i] : -1;
  }
  return launch_copy(pool, L, NB, page, ids, n, stream);
}

int launch_find_free(const int32_t* refs, int NB, int32_t* out, int n, hipStream_t stream) {
  const int64_t chunks = ceil_div(NB, kScanChunk);
  if (NB > kMaxScan)
    return fail(HS_EUNSUPPORTED, "at most " + std::to_string(kMaxScan) + " blocks in a scan");
  hipLaunchKernelGGL(find_free_kernel, dim3((unsigned)chunks), dim3(kScanThreads), 0, stream, refs, NB,
                     out, n, aligned16(refs));
  return check_launch("free block search");
}

int launch_fork(void* pool, int L, int NB, int64_t page, int BS, int32_t* bt, int B, int MB,
                int32_t* ctx, int32_t* refs, const int32_t* parents, const int32_t* children,
                const int32_t* fresh, int n, int32_t* forked, hipStream_t stream) {
  if (!pool_fits(L, NB, page)) return fail(HS_EUNSUPPORTED, "pool too large for 64-bit offsets");
  if (L > 32767 || !grid_fits(n, kCopyThreads)) return fail(HS_EUNSUPPORTED, "fork grid too large");
  ForkArgs a{static_cast<uint8_t*>(pool), 2 * L, NB, BS, page, bt, ctx, refs, parents, children, fresh,
             forked, B, MB};
  const dim3 g((unsigned)n, (unsigned)(1 + 2 * L)), t(kCopyThreads);
  profile_begin(stream);
  if (pool_vec(pool, page) && page / BS % 16 == 0)
    hipLaunchKernelGGL(fork_kernel<true>, g, t, 0, stream, a);
  else
    hipLaunchKernelGGL(fork_kernel<false>, g, t, 0, stream, a);
  profile_end(stream);
  return check_launch("kv fork");
}

int launch_free(int32_t* bt, int B, int MB, int32_t* ctx, int32_t* refs, int NB, const int32_t* rows,
                int n, hipStream_t stream) {
  const int64_t chunks = ceil_div(MB, kCopyThreads);
  if (chunks > 65535 || !grid_fits(n, kCopyThreads))
    return fail(HS_EUNSUPPORTED, "block table too wide, or too many rows, for one launch");
  hipLaunchKernelGGL(free_kernel, dim3((unsigned)n, (unsigned)chunks), dim3(kCopyThreads), 0, stream, bt,
                     ctx, refs, rows, B, MB, NB);
  return check_launch("kv free");
}

int64_t compact_workspace_bytes(int NB) { return sat_mul(sat_add(sat_mul(3, NB), 64), 4); }

int launch_compact(void* pool, int L, int NB, int64_t page, int32_t* bt, int B, int MB, int32_t* refs,
                   int32_t* moved_to, int32_t* live, void* workspace, int cus, hipStream_t stream) {
  if (!pool_fits(L, NB, page))
    return fail(HS_EUNSUPPORTED, "pool too large for 64-bit offsets");
  if (NB > kMaxScan)
    return fail(HS_EUNSUPPORTED, "at most " + std::to_string(kMaxScan) + " blocks in a scan");
  int32_t* ws = static_cast<int32_t*>(workspace);
  const CompactPlan p{ws, ws + 64, ws + 64 + (int64_t)NB, ws + 64 + 2 * (int64_t)NB};
  hipLaunchKernelGGL(compact_plan_kernel, dim3((unsigned)ceil_div(NB, kScanChunk)), dim3(kScanThreads), 0,
                     stream, refs, NB, p, live, aligned16(refs));
  // The number of moves, at most NB / 2, stays on the device, so up to 64 workgroups a CU
  // take the pages in turn.  32 layers, 432 moves of 32-KB pages, us at 8 / 64 / 512: 190 /
  // 173 / 166; without a move 7 / 10 / 35.
  const int64_t most = sat_mul((NB + 1) / 2, 2, L);
  const dim3 g((unsigned)std::min((int64_t)64 * cus, std::max((int64_t)cus, most))), t(kCopyThreads);
  uint8_t* pl = static_cast<uint8_t*>(pool);
  const int64_t entries = (int64_t)B * MB;
  profile_begin(stream);
  if (pool_vec(pool, page))
    hipLaunchKernelGGL(compact_move_kernel<true>, g, t, 0, stream, pl, 2 * L, NB, page, bt, entries,
                       refs, p, moved_to);
  else
    hipLaunchKernelGGL(compact_move_kernel<false>, g, t, 0, stream, pl, 2 * L, NB, page, bt,
                       entries, refs, p, moved_to);
  profile_end(stream);
  return check_launch("kv compaction");
}

}  // namespace hs
