// Blocks of a paged cache that several requests map: forking a request, giving blocks
// back, moving the blocks in use together, and the copies of rows that these name.
//
//   shares[blk] = table entries that map block blk beyond the first (0: one request's
//   own, or free), so that a program without shared blocks has zeros there for good and
//   dsr_paged_plan, which only ever maps free blocks, leaves it alone.
//
// A move (source row, destination row, rows, 0) names up to one block of rows to copy.
// The tables are changed once for all layers; dsr_paged_copy then runs per cache, or for
// the pools of many layers at once.
//
// Small calls are bound by their launches: all kernels here are launched while the one
// before them runs (programmatic dependent launch) and wait for its end before their first
// access, and small tables are released and compacted by one CTA in one launch.  A fork of one
// child, its copy and its release: 12.4 us from a graph, 16 us as three calls of the extension.
#include "common.cuh"
#include "host_common.h"

namespace dsr {
namespace {

constexpr int kShareMaxBatch = 16384;  // as the plan's
constexpr int kShareShift = 6;
static_assert(DSR_BLOCK_TOKENS == 1 << kShareShift, "64-row blocks");
constexpr int4 kNoMove = {-1, -1, 0, 0};

__device__ __forceinline__ int32_t blocks_of(int64_t tokens) {
  return int32_t((tokens + DSR_BLOCK_TOKENS - 1) >> kShareShift);
}

struct ShareArgs {
  const int32_t* parent;  // fork only
  const int32_t* lengths;
  int32_t* held;
  int32_t* table;
  int64_t stride;
  int32_t* ring;
  int32_t* state;  // head, count, ticket (0 between calls), unused
  int32_t* shares;
  int64_t blocks;
  int4* moves;
  int32_t* count;
  int32_t* err;
  int batch;
};

__device__ __forceinline__ int64_t ring_at(const ShareArgs& a, int64_t i) { return i < a.blocks ? i : i - a.blocks; }

struct Pair {
  int64_t x, y;
};

// Exclusive sums over the CTA's threads; `all` the totals.  Each warp sums up the warps'
// totals by itself; the barrier at the end lets `part` be used again.
template <int Threads>
__device__ __forceinline__ Pair cta_scan(const Pair& mine, Pair* part, Pair& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto inclusive = [&](Pair run) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const Pair up{__shfl_up_sync(~0u, run.x, d), __shfl_up_sync(~0u, run.y, d)};
      if (lane >= d) run.x += up.x, run.y += up.y;
    }
    return run;
  };
  const Pair run = inclusive(mine);
  if (lane == 31) part[warp] = run;
  __syncthreads();
  const Pair one = lane < Threads / 32 ? part[lane] : Pair{0, 0}, upto = inclusive(one);
  all = Pair{__shfl_sync(~0u, upto.x, 31), __shfl_sync(~0u, upto.y, 31)};
  const Pair before{__shfl_sync(~0u, upto.x - one.x, warp), __shfl_sync(~0u, upto.y - one.y, warp)};
  __syncthreads();
  return Pair{before.x + run.x - mine.x, before.y + run.y - mine.y};
}

// The largest b with cu[b] <= i (cu[0] = 0, cu increasing weakly, i < cu[n]).
__device__ __forceinline__ int share_owner(const int32_t* cu, int n, int32_t i) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

// ---------------------------------------------------------------------------
// Fork.  Every CTA scans all requests itself, as the plan does; an entry of a child is
// read from its parent's row, which no child's is.  held and the ring's state are written
// by the CTA that is the last to have read them (a ticket in the ring state, drawn when a
// CTA has its sums: it runs beside the entries).  Bound by latency: 64 children of 513 blocks
// 8 us with cold inputs, one child 6 us.
// ---------------------------------------------------------------------------
constexpr int kForkThreads = 512;

// Blocks of request b when it is a child (else 0), and whether its last one is a copy;
// false when it is refused.
__device__ __forceinline__ bool fork_request(const ShareArgs& a, int b, int32_t& parent, int32_t& len, int32_t& need) {
  parent = a.parent[b];
  len = need = 0;
  if (parent == -1) return true;
  if (parent < 0 || parent >= a.batch || parent == b || a.parent[parent] != -1 || a.held[b] != 0) return false;
  const int32_t have = a.held[parent], most = a.lengths[parent];
  len = a.lengths[b];
  if (have < 0 || have > a.stride || len < 0 || len > most || most > int64_t(have) * DSR_BLOCK_TOKENS) return false;
  need = blocks_of(len);
  return true;
}

__global__ void __launch_bounds__(kForkThreads) fork_kernel(const ShareArgs a) {
  extern __shared__ int32_t fork_smem[];
  int32_t* cu_entry = fork_smem;               // [batch + 1] entries before each request
  int32_t* cu_take = cu_entry + a.batch + 1;   // [batch + 1] fresh blocks before it
  __shared__ Pair part[kForkThreads / 32];
  __shared__ int bad, last;
  const int tid = threadIdx.x;
  pdl_launch_dependents();
  if (tid == 0) bad = 0;
  pdl_wait();
  __syncthreads();
  const int per = (a.batch + kForkThreads - 1) / kForkThreads;
  const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
  Pair mine{0, 0};
  for (int b = b0; b < b1; ++b) {
    int32_t parent, len, need;
    if (!fork_request(a, b, parent, len, need)) bad = 1;
    mine.x += need, mine.y += (len & (DSR_BLOCK_TOKENS - 1)) != 0;
  }
  const int64_t head = a.state[0], count = a.state[1];
  Pair all, at = cta_scan<kForkThreads>(mine, part, all);
  const bool ok = bad == 0 && all.x < (int64_t(1) << 31) && all.y <= count && head >= 0 && head < a.blocks &&
                  count >= 0 && count <= a.blocks;
  if (ok) {
    for (int b = b0; b < b1; ++b) {
      int32_t parent, len, need;
      fork_request(a, b, parent, len, need);
      cu_entry[b] = int32_t(at.x);
      cu_take[b] = int32_t(at.y);
      at.x += need, at.y += (len & (DSR_BLOCK_TOKENS - 1)) != 0;
    }
    if (tid == 0) cu_entry[a.batch] = int32_t(all.x), cu_take[a.batch] = int32_t(all.y);
  } else if (blockIdx.x == 0 && tid == 0) {
    flag(a.err, DSR_ERR_ID);
  }
  __syncthreads();  // all of this CTA have read
  if (tid == 0) last = atomicAdd(a.state + 2, 1) == int(gridDim.x) - 1;
  const int64_t step = int64_t(gridDim.x) * kForkThreads, first = int64_t(blockIdx.x) * kForkThreads + tid;
  const int64_t moved = ok ? all.y : 0;
  for (int64_t i = moved + first; i < a.batch; i += step) a.moves[i] = kNoMove;
  if (first == 0) *a.count = int32_t(moved);
  if (ok) {
    for (int64_t i = first; i < all.x; i += step) {
      const int b = share_owner(cu_entry, a.batch, int32_t(i));
      const int32_t j = int32_t(i) - cu_entry[b], len = a.lengths[b];
      int32_t blk = a.table[int64_t(a.parent[b]) * a.stride + j];
      const bool good = blk >= 0 && blk < a.blocks;
      if (!good) flag(a.err, DSR_ERR_ID);
      if (j < len >> kShareShift) {
        if (good) atomicAdd(a.shares + blk, 1);
      } else {
        const int32_t source = blk;
        blk = a.ring[ring_at(a, head + cu_take[b])];
        const bool fresh = blk >= 0 && blk < a.blocks;
        if (!fresh) flag(a.err, DSR_ERR_ID);
        a.moves[cu_take[b]] = good && fresh ? make_int4(source * DSR_BLOCK_TOKENS, blk * DSR_BLOCK_TOKENS,
                                                        len & (DSR_BLOCK_TOKENS - 1), 0)
                                            : kNoMove;
        if (!fresh) blk = -1;
      }
      a.table[int64_t(b) * a.stride + j] = blk >= 0 && blk < a.blocks ? blk : -1;
    }
  }
  __syncthreads();
  if (!last) return;
  if (ok) {
    for (int b = b0; b < b1; ++b)
      if (a.parent[b] >= 0) a.held[b] = blocks_of(a.lengths[b]);
    if (tid == 0) {
      a.state[0] = int32_t((head + all.y) % a.blocks);
      a.state[1] = int32_t(count - all.y);
    }
  }
  if (tid == 0) a.state[2] = 0;
}

// ---------------------------------------------------------------------------
// Release.  One CTA decides: which last blocks are shared, before any count changes, and
// what is dropped.  Then the entries are dropped, and the blocks that nobody maps any more
// go to the ring, in the order of their ids, so that the order in which the counts were
// lowered does not matter.  Tables of up to kWholeEntries entries: by the same CTA, with
// its bit per freed block in shared memory; larger ones by two more launches.
// Scratch of three launches: {ok, taken, dropped} and cu_drop[batch + 1], then the bits.
// Bound by latency: 512 requests cut somewhere, 41000 entries dropped, 22 us with cold inputs
// (7.5, 7.6 and 6.7; the freed blocks by the last CTA of the second launch took 16 instead).
// ---------------------------------------------------------------------------
constexpr int kScanThreads = 1024, kDropThreads = 512;
constexpr int kScanPer = kShareMaxBatch / kScanThreads;
static_assert(kScanPer <= 32, "a bit for each of a thread's requests");
// (One CTA takes some 1 ns an entry, the second launch 5 us and more.)
constexpr int64_t kWholeEntries = 8192, kWholeBlocks = 65536;  // bits: 8 KB

struct ReleaseScratch {
  int32_t* head;      // {ok, taken, dropped}
  int32_t* cu_drop;   // [batch + 1]
  uint32_t* freed;    // [words]
  int64_t words;
};

__device__ __forceinline__ void drop_block(const ShareArgs& a, uint32_t* freed, int32_t blk) {
  if (blk < 0 || blk >= a.blocks) {
    flag(a.err, DSR_ERR_ID);
    return;
  }
  const int32_t others = atomicSub(a.shares + blk, 1);
  if (others < 0) flag(a.err, DSR_ERR_ID);  // mapped more often than its count says
  if (others <= 0) atomicOr(freed + (blk >> 5), 1u << (blk & 31));
}

// The dropped entries, `per` of a thread at a time: their chains of accesses run side by side.
template <int Threads>
__device__ __forceinline__ void drop_entries(const ShareArgs& a, const int32_t* cu_drop, uint32_t* freed,
                                             int32_t dropped) {
  constexpr int kPer = 4;
  const int64_t step = int64_t(gridDim.x) * Threads;
  for (int64_t i0 = int64_t(blockIdx.x) * Threads + threadIdx.x; i0 < dropped; i0 += step * kPer) {
    int32_t blk[kPer];
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      const int64_t i = i0 + q * step;
      if (i >= dropped) continue;
      const int b = share_owner(cu_drop, a.batch, int32_t(i));
      int32_t* entry = a.table + int64_t(b) * a.stride + blocks_of(a.lengths[b]) + (int32_t(i) - cu_drop[b]);
      blk[q] = *entry;
      *entry = -1;
    }
#pragma unroll
    for (int q = 0; q < kPer; ++q)
      if (i0 + q * step < dropped) drop_block(a, freed, blk[q]);
  }
}

// The freed blocks behind the ring's tail, held, and the ring's state.  Every CTA has a run of
// words and counts the blocks before it itself; a warp takes a word, so that its stores are to
// neighbours.  The state is written by the CTA that is the last to have read it (a ticket).
// Own: the bits are this CTA's, in shared memory.
template <int Threads, bool Own>
__device__ __forceinline__ void free_blocks(const ShareArgs& a, const uint32_t* freed, int64_t words, int64_t taken,
                                            Pair* part, int* last) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t head = a.state[0], count = a.state[1];
  const int64_t slice = (words + gridDim.x - 1) / gridDim.x;
  const int64_t w0 = min(blockIdx.x * slice, words), w1 = min(w0 + slice, words);
  auto bits = [&](int64_t w) { return Own ? freed[w] : __ldcg(freed + w); };
  Pair mine{0, 0}, all;  // blocks before this CTA's, and all
  for (int64_t w = threadIdx.x; w < words; w += Threads) {
    const int n = __popc(bits(w));
    mine.x += w < w0 ? n : 0, mine.y += n;
  }
  cta_scan<Threads>(mine, part, all);  // all of this CTA have read the state
  if (threadIdx.x == 0) *last = gridDim.x == 1 || atomicAdd(a.state + 2, 1) == int(gridDim.x) - 1;
  int64_t to = head + count + all.x;
  for (int64_t c = w0; c < w1; c += Threads / 32) {
    const uint32_t word = lane < Threads / 32 && c + lane < w1 ? bits(c + lane) : 0u;
    int upto = __popc(word);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(~0u, upto, d);
      if (lane >= d) upto += up;
    }
    const uint32_t own = __shfl_sync(~0u, word, warp);
    const int end = __shfl_sync(~0u, upto, warp);
    if (own >> lane & 1) {
      int64_t place = to + end - __popc(own >> lane);
      while (place >= a.blocks) place -= a.blocks;
      const int32_t blk = int32_t(c + warp) * 32 + lane;
      a.ring[place] = blk;
      a.shares[blk] = 0;
    }
    __syncwarp();
    to += __shfl_sync(~0u, upto, 31);
  }
  for (int64_t b = int64_t(blockIdx.x) * Threads + threadIdx.x; b < a.batch; b += int64_t(gridDim.x) * Threads)
    a.held[b] = blocks_of(a.lengths[b]);
  __syncthreads();
  if (*last && threadIdx.x == 0) {
    const int64_t now = count - taken + all.y;
    if (now > a.blocks) flag(a.err, DSR_ERR_ID);  // the ring held blocks that were mapped
    a.state[0] = int32_t((head + taken) % a.blocks);
    a.state[1] = int32_t(now < a.blocks ? now : a.blocks);
    a.state[2] = 0;
  }
}

template <bool Whole>
__global__ void __launch_bounds__(kScanThreads, 1) release_scan_kernel(const ShareArgs a, const ReleaseScratch s) {
  extern __shared__ int32_t release_smem[];  // Whole: cu_drop, then the bits
  __shared__ Pair part[kScanThreads / 32];
  __shared__ int bad, last;
  const int tid = threadIdx.x;
  int32_t* cu_drop = Whole ? release_smem : s.cu_drop;
  uint32_t* freed = Whole ? reinterpret_cast<uint32_t*>(release_smem + a.batch + 1) : s.freed;
  pdl_launch_dependents();
  if (tid == 0) bad = 0;
  pdl_wait();
  for (int64_t w = tid; w < s.words; w += kScanThreads) freed[w] = 0u;
  __syncthreads();
  const int per = (a.batch + kScanThreads - 1) / kScanThreads;
  const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
  uint32_t copies = 0;  // of this thread's requests, those whose last block is exchanged
  Pair mine{0, 0};
  for (int b = b0; b < b1; ++b) {
    const int32_t len = a.lengths[b], have = a.held[b], need = blocks_of(len);
    if (len < 0 || have < 0 || have > a.stride || need > have) {
      bad = 1;
      continue;
    }
    if (len & (DSR_BLOCK_TOKENS - 1)) {
      const int32_t blk = a.table[int64_t(b) * a.stride + need - 1];
      if (blk < 0 || blk >= a.blocks) flag(a.err, DSR_ERR_ID);
      else if (a.shares[blk] > 0) copies |= 1u << (b - b0);
    }
    mine.x += have - need, mine.y += copies >> (b - b0) & 1;
  }
  const int64_t head = a.state[0], count = a.state[1];
  Pair all, at = cta_scan<kScanThreads>(mine, part, all);
  const bool ok = bad == 0 && all.x < (int64_t(1) << 31) && all.y <= count && head >= 0 && head < a.blocks &&
                  count >= 0 && count <= a.blocks;
  const int64_t moved = ok ? all.y : 0;
  for (int64_t i = moved + tid; i < a.batch; i += kScanThreads) a.moves[i] = kNoMove;
  if (tid == 0) {
    if constexpr (!Whole) {
      s.head[0] = ok;
      s.head[1] = int32_t(moved);
      s.head[2] = ok ? int32_t(all.x) : 0;
    }
    *a.count = int32_t(moved);
    if (!ok) flag(a.err, DSR_ERR_ID);
  }
  if (!ok) return;
  // every count has been read: it may change now
  for (int b = b0; b < b1; ++b) {
    const int32_t len = a.lengths[b], need = blocks_of(len);
    cu_drop[b] = int32_t(at.x);
    at.x += a.held[b] - need;
    if (!(copies >> (b - b0) & 1)) continue;
    int32_t* entry = a.table + int64_t(b) * a.stride + need - 1;
    const int32_t source = *entry, blk = a.ring[ring_at(a, head + at.y)];
    const bool good = blk >= 0 && blk < a.blocks;
    if (!good) flag(a.err, DSR_ERR_ID);
    a.moves[at.y] = good ? make_int4(source * DSR_BLOCK_TOKENS, blk * DSR_BLOCK_TOKENS, len & (DSR_BLOCK_TOKENS - 1), 0)
                         : kNoMove;
    *entry = good ? blk : -1;
    drop_block(a, freed, source);
    ++at.y;
  }
  if (tid == 0) cu_drop[a.batch] = int32_t(all.x);
  if constexpr (Whole) {
    __syncthreads();
    drop_entries<kScanThreads>(a, cu_drop, freed, int32_t(all.x));
    __syncthreads();
    free_blocks<kScanThreads, true>(a, freed, s.words, all.y, part, &last);
  }
}

__global__ void __launch_bounds__(kDropThreads, 1) release_drop_kernel(const ShareArgs a, const ReleaseScratch s) {
  extern __shared__ int32_t drop_smem[];  // cu_drop
  pdl_launch_dependents();
  pdl_wait();
  const int32_t dropped = __ldcg(s.head + 2);
  if (dropped == 0) return;
  for (int b = threadIdx.x; b <= a.batch; b += kDropThreads) drop_smem[b] = __ldcg(s.cu_drop + b);
  __syncthreads();
  drop_entries<kDropThreads>(a, drop_smem, s.freed, dropped);
}

__global__ void __launch_bounds__(kDropThreads, 1) release_free_kernel(const ShareArgs a, const ReleaseScratch s) {
  __shared__ Pair part[kDropThreads / 32];
  __shared__ int last;
  pdl_launch_dependents();
  pdl_wait();
  if (__ldcg(s.head) == 0) return;  // alike in all CTAs
  free_blocks<kDropThreads, false>(a, s.freed, s.words, __ldcg(s.head + 1), part, &last);
}

// ---------------------------------------------------------------------------
// Compaction.  With L live blocks (mapped by an entry below its row's held), the i-th
// live id from L on goes to the i-th id below L that is not live: the fewest copies, and
// no destination is a source.  A bit per live block; every CTA sums the bits of 256-block
// groups itself and finds ranks and free ids by search.  Tables of up to kWholeEntries
// entries: one CTA, with its bits in shared memory, in one launch.
// ---------------------------------------------------------------------------
constexpr int kCompactThreads = 512;
constexpr int kCompactMaxGroups = 32768;  // of 256 blocks: 128 KB of shared memory

struct CompactScratch {
  uint32_t* live;  // [8 groups]
  int32_t* bad;
  int groups;
};

__device__ __forceinline__ void mark_live(const ShareArgs& a, uint32_t* live, int* bad) {
  const int64_t step = int64_t(gridDim.x) * kCompactThreads, first = int64_t(blockIdx.x) * kCompactThreads + threadIdx.x;
  for (int64_t b = first; b < a.batch; b += step)
    if (a.held[b] < 0 || a.held[b] > a.stride) {
      flag(a.err, DSR_ERR_ID);
      *bad = 1;
    }
  for (int64_t i = first; i < int64_t(a.batch) * a.stride; i += step) {
    const int64_t b = i / a.stride;
    if (i - b * a.stride >= a.held[b]) continue;
    const int32_t blk = a.table[i];
    if (blk < 0 || blk >= a.blocks) {
      flag(a.err, DSR_ERR_ID);
      continue;
    }
    const uint32_t bit = 1u << (blk & 31);
    if (!(*reinterpret_cast<volatile uint32_t*>(live + (blk >> 5)) & bit)) atomicOr(live + (blk >> 5), bit);
  }
}

__global__ void __launch_bounds__(kCompactThreads) compact_mark_kernel(const ShareArgs a, const CompactScratch s) {
  mark_live(a, s.live, s.bad);
}

template <bool Whole>
__global__ void __launch_bounds__(kCompactThreads) compact_apply_kernel(const ShareArgs a, const CompactScratch s) {
  extern __shared__ uint4 compact_smem[];  // Whole: the bits; [groups + 1] live blocks before each group
  uint32_t* live = Whole ? reinterpret_cast<uint32_t*>(compact_smem) : s.live;
  int32_t* before = reinterpret_cast<int32_t*>(compact_smem + (Whole ? 2 * s.groups : 0));
  __shared__ Pair part[kCompactThreads / 32];
  __shared__ int refused;
  const int tid = threadIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  if constexpr (Whole) {
    if (tid == 0) refused = 0;
    for (int w = tid; w < 8 * s.groups; w += kCompactThreads) live[w] = 0u;
    __syncthreads();
    mark_live(a, live, &refused);
  } else if (tid == 0) {
    refused = __ldcg(s.bad);
  }
  __syncthreads();
  const int64_t step = int64_t(gridDim.x) * kCompactThreads, first = int64_t(blockIdx.x) * kCompactThreads + tid;
  const int64_t room = a.blocks < 2 ? 1 : a.blocks / 2;
  if (refused != 0) {
    for (int64_t i = first; i < room; i += step) a.moves[i] = kNoMove;
    if (first == 0) *a.count = 0;
    return;
  }
  auto words = [&](int g, uint32_t (&w)[8]) {
    const uint4* from = reinterpret_cast<const uint4*>(live) + 2 * g;
    const uint4 lo = Whole ? from[0] : __ldcg(from), hi = Whole ? from[1] : __ldcg(from + 1);
    w[0] = lo.x, w[1] = lo.y, w[2] = lo.z, w[3] = lo.w, w[4] = hi.x, w[5] = hi.y, w[6] = hi.z, w[7] = hi.w;
  };
  int32_t used = 0;
  for (int g0 = 0; g0 < s.groups; g0 += kCompactThreads) {
    const int g = g0 + tid;
    int n = 0;
    if (g < s.groups) {
      uint32_t w[8];
      words(g, w);
#pragma unroll
      for (int q = 0; q < 8; ++q) n += __popc(w[q]);
    }
    Pair all;
    const Pair at = cta_scan<kCompactThreads>(Pair{n, 0}, part, all);
    if (g < s.groups) before[g] = used + int32_t(at.x);
    used += int32_t(all.x);
  }
  if (tid == 0) before[s.groups] = used;
  __syncthreads();
  // live ids below id
  auto rank = [&](int32_t id) {
    uint32_t w[8];
    words(id >> 8, w);
    int32_t n = before[id >> 8];
    const int in = id & 255;
#pragma unroll
    for (int q = 0; q < 8; ++q) n += __popc(in >= 32 * (q + 1) ? w[q] : in > 32 * q ? w[q] & ((1u << (in & 31)) - 1u) : 0u);
    return n;
  };
  // the i-th id that is not live
  auto hole = [&](int32_t i) {
    int lo = 0, hi = s.groups;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (mid * 256 - before[mid] <= i) lo = mid;
      else hi = mid;
    }
    uint32_t w[8];
    words(lo, w);
    i -= lo * 256 - before[lo];
    int32_t id = lo * 256;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int n = __popc(~w[q]);
      if (i >= n) {
        i -= n;
        id += 32;
      } else if (i >= 0) {
        uint32_t left = ~w[q];
        for (; i > 0; --i) left &= left - 1;
        id += __ffs(left) - 1;
        i = -1;
      }
    }
    return id;
  };
  const int32_t kept = used < a.blocks ? rank(used) : used;  // live ids that stay
  const int32_t moved = used - kept;
  auto target = [&](int32_t id) { return hole(rank(id) - kept); };
  for (int64_t i = moved + first; i < room; i += step) a.moves[i] = kNoMove;
  if (first == 0) {
    *a.count = moved;
    a.state[0] = 0;
    a.state[1] = int32_t(a.blocks) - used;
  }
  for (int64_t i = first; i < a.blocks; i += step) a.ring[i] = i < a.blocks - used ? int32_t(i) + used : -1;
  for (int64_t i = used + first; i < a.blocks; i += step) {
    if (!((Whole ? live[i >> 5] : __ldcg(s.live + (i >> 5))) >> (i & 31) & 1)) {
      a.shares[i] = 0;  // free, whatever it was
      continue;
    }
    const int32_t n = rank(int32_t(i)) - kept, to = hole(n);
    a.moves[n] = make_int4(int32_t(i) * DSR_BLOCK_TOKENS, to * DSR_BLOCK_TOKENS, DSR_BLOCK_TOKENS, 0);
    a.shares[to] = a.shares[i];
    a.shares[i] = 0;
  }
  for (int64_t i = first; i < int64_t(a.batch) * a.stride; i += step) {
    const int64_t b = i / a.stride;
    if (i - b * a.stride >= a.held[b]) continue;
    const int32_t blk = a.table[i];
    if (blk >= used && blk < a.blocks) a.table[i] = target(blk);
  }
}

// ---------------------------------------------------------------------------
// Copies.  A work item is a piece of one move's rows in one pool, four 16-byte units a thread
// on their way at once; the generations of the written rows are a move's last item.  Bound by
// memory: 4039 blocks of 90 KB with their generations, 732 MB read and written, 118 us (6.2 TB/s,
// 95% of the rate of a 2 GB copy and 99% of one of this size); 489 copies of up to 63 rows in four
// layers, 178 MB, 30.5 us (5.8 TB/s).
// ---------------------------------------------------------------------------
constexpr int kCopyThreads = 256, kCopyPiece = 16384;  // bytes of an item
constexpr int kCopyMax = 64;                           // pools, and generations, of a call

struct CopyArgs {
  uint8_t* data[kCopyMax];
  int64_t* generations[kCopyMax];
  int32_t row_bytes[kCopyMax];
  int32_t first[kCopyMax + 1];  // items of a move before each pool's
  const int4* moves;
  const int32_t* count;
  int64_t rows;
  int32_t* err;
  int32_t pools, gens, room;
};

__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const __grid_constant__ CopyArgs a) {
  const int tid = threadIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  int32_t n = *a.count;
  if (n < 0 || n > a.room) {
    if (blockIdx.x == 0 && tid == 0) flag(a.err, DSR_ERR_ID);
    return;
  }
  const int per = a.first[a.pools] + (a.gens > 0);
  for (int64_t item = blockIdx.x; item < int64_t(n) * per; item += gridDim.x) {
    const int64_t k = item / per;
    const int in = int(item - k * per);
    const int4 m = a.moves[k];
    if (m.z == 0) continue;
    if (m.z < 0 || m.z > DSR_BLOCK_TOKENS || m.x < 0 || m.y < 0 || m.x > a.rows - m.z || m.y > a.rows - m.z) {
      if (tid == 0) flag(a.err, DSR_ERR_ID);
      continue;
    }
    if (in == a.first[a.pools]) {
      for (int i = tid; i < a.gens * DSR_BLOCK_TOKENS; i += kCopyThreads)
        if ((i & (DSR_BLOCK_TOKENS - 1)) < m.z) ++a.generations[i / DSR_BLOCK_TOKENS][m.y + (i & (DSR_BLOCK_TOKENS - 1))];
      continue;
    }
    int p = 0;
    while (in >= a.first[p + 1]) ++p;
    const int64_t width = a.row_bytes[p], begin = int64_t(in - a.first[p]) * kCopyPiece;
    const int units = int((min(begin + kCopyPiece, width * m.z) - begin) / 16);
    const uint4* src = reinterpret_cast<const uint4*>(a.data[p] + m.x * width + begin);
    uint4* dst = reinterpret_cast<uint4*>(a.data[p] + m.y * width + begin);
    uint4 v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (tid + q * kCopyThreads < units) v[q] = __ldg(src + tid + q * kCopyThreads);
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (tid + q * kCopyThreads < units) dst[tid + q * kCopyThreads] = v[q];
  }
}
static_assert(kCopyPiece == 4 * 16 * kCopyThreads, "four 16-byte units a thread");

int64_t freed_words(int64_t blocks) { return (blocks + 31) / 32; }
int64_t live_groups(int64_t blocks) { return (blocks + 255) / 256; }
size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }

// What fork, release and compaction have in common: the checks, and the arguments.
int share_args(ShareArgs* out, int32_t* held, int32_t* table, int64_t stride, int32_t* ring, int32_t* state,
               int32_t* shares, int64_t blocks, int32_t* moves, int32_t* count, int32_t* err, int64_t batch,
               const char* what) {
  PoolAddr pa;  // the range checks of every paged entry point
  const int rc = paged_addr(&pa, table, stride, blocks, what);
  if (rc != DSR_OK) return rc;
  DSR_REQUIRE(held && ring && state && shares && moves && count && err, "%s: null pointer", what);
  DSR_REQUIRE(batch > 0 && batch <= kShareMaxBatch, "%s: batch %lld outside [1, %d]", what, (long long)batch,
              kShareMaxBatch);
  DSR_REQUIRE(aligned16(moves), "%s: moves must be 16-byte aligned", what);
  *out = ShareArgs{nullptr, nullptr, held, table, stride, ring, state, shares, blocks, reinterpret_cast<int4*>(moves),
                   count, err, int(batch)};
  return DSR_OK;
}

int check_scratch(const void* workspace, size_t have, size_t need, const char* what) {
  DSR_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0,
              "%s: workspace must be 256-byte aligned", what);
  DSR_REQUIRE(have >= need, "%s: workspace %zu < %zu bytes", what, have, need);
  return DSR_OK;
}

// A table that one CTA takes in one launch.
bool whole_table(int64_t batch, int64_t stride, int64_t blocks) {
  return batch * stride <= kWholeEntries && blocks <= kWholeBlocks;
}

// CTAs for `items` of which a thread takes `per`, up to one per SM.
unsigned share_grid(int64_t items, int64_t per) {
  const int64_t grid = (items + per - 1) / per;
  return unsigned(grid < 1 ? 1 : grid < sm_count() ? grid : sm_count());
}

}  // namespace
}  // namespace dsr

extern "C" int dsr_paged_fork(const int32_t* parent, const int32_t* lengths, int32_t* held, int32_t* block_table,
                              int64_t table_stride, int32_t* free_ring, int32_t* ring_state, int32_t* shares,
                              int64_t pool_blocks, int32_t* moves, int32_t* count, int32_t* err, int64_t batch,
                              void* stream) {
  using namespace dsr;
  clear_error();
  ShareArgs a;
  int rc = share_args(&a, held, block_table, table_stride, free_ring, ring_state, shares, pool_blocks, moves, count, err,
                      batch, "paged_fork");
  if (rc != DSR_OK) return rc;
  DSR_REQUIRE(parent && lengths, "paged_fork: null pointer");
  a.parent = parent;
  a.lengths = lengths;
  rc = set_max_smem(fork_kernel, 2 * size_t(kShareMaxBatch + 1) * sizeof(int32_t), "paged_fork");
  if (rc != DSR_OK) return rc;
  const unsigned grid = share_grid(batch * table_stride, kForkThreads);
  return launch_after(fork_kernel, grid, kForkThreads, 2 * size_t(batch + 1) * sizeof(int32_t), as_stream(stream),
                      "paged_fork", a);
}

extern "C" size_t dsr_paged_release_workspace_bytes(int64_t batch, int64_t pool_blocks) {
  using namespace dsr;
  if (batch <= 0 || pool_blocks <= 0) return 0;
  return 256 + rounded(size_t(batch + 1) * 4) + size_t(freed_words(pool_blocks)) * 4;
}

extern "C" int dsr_paged_release(const int32_t* lengths, int32_t* held, int32_t* block_table, int64_t table_stride,
                                 int32_t* free_ring, int32_t* ring_state, int32_t* shares, int64_t pool_blocks,
                                 int32_t* moves, int32_t* count, void* workspace, size_t workspace_bytes,
                                 int32_t* err, int64_t batch, void* stream) {
  using namespace dsr;
  clear_error();
  ShareArgs a;
  int rc = share_args(&a, held, block_table, table_stride, free_ring, ring_state, shares, pool_blocks, moves, count, err,
                      batch, "paged_release");
  if (rc != DSR_OK) return rc;
  DSR_REQUIRE(lengths, "paged_release: null pointer");
  rc = check_scratch(workspace, workspace_bytes, dsr_paged_release_workspace_bytes(batch, pool_blocks), "paged_release");
  if (rc != DSR_OK) return rc;
  a.lengths = lengths;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const ReleaseScratch s{reinterpret_cast<int32_t*>(ws), reinterpret_cast<int32_t*>(ws + 256),
                         reinterpret_cast<uint32_t*>(ws + 256 + rounded(size_t(batch + 1) * 4)), freed_words(pool_blocks)};
  if (whole_table(batch, table_stride, pool_blocks)) {
    const size_t smem = (size_t(batch + 1) + size_t(s.words)) * 4, most = (kShareMaxBatch + 1 + kWholeBlocks / 32) * 4;
    rc = set_max_smem(release_scan_kernel<true>, most, "paged_release");
    if (rc != DSR_OK) return rc;
    return launch_after(release_scan_kernel<true>, 1, kScanThreads, smem, as_stream(stream), "paged_release", a, s);
  }
  rc = set_max_smem(release_drop_kernel, size_t(kShareMaxBatch + 1) * sizeof(int32_t), "paged_release");
  if (rc != DSR_OK) return rc;
  rc = launch_after(release_scan_kernel<false>, 1, kScanThreads, 0, as_stream(stream), "paged_release", a, s);
  if (rc != DSR_OK) return rc;
  rc = launch_after(release_drop_kernel, share_grid(batch * table_stride, kDropThreads), kDropThreads,
                    size_t(batch + 1) * sizeof(int32_t), as_stream(stream), "paged_release", a, s);
  if (rc != DSR_OK) return rc;
  // two words a warp and more
  return launch_after(release_free_kernel, share_grid(s.words, 2 * kDropThreads / 32), kDropThreads, 0,
                      as_stream(stream), "paged_release", a, s);
}

extern "C" size_t dsr_paged_compact_workspace_bytes(int64_t pool_blocks) {
  return pool_blocks <= 0 ? 0 : 256 + size_t(dsr::live_groups(pool_blocks)) * 32;
}

extern "C" int dsr_paged_compact(int32_t* held, int32_t* block_table, int64_t table_stride, int32_t* free_ring,
                                 int32_t* ring_state, int32_t* shares, int64_t pool_blocks, int32_t* moves,
                                 int32_t* count, void* workspace, size_t workspace_bytes, int32_t* err, int64_t batch,
                                 void* stream) {
  using namespace dsr;
  clear_error();
  ShareArgs a;
  int rc = share_args(&a, held, block_table, table_stride, free_ring, ring_state, shares, pool_blocks, moves, count, err,
                      batch, "paged_compact");
  if (rc != DSR_OK) return rc;
  const int64_t groups = live_groups(pool_blocks);
  DSR_REQUIRE(groups <= kCompactMaxGroups, "paged_compact: pool blocks %lld above %d", (long long)pool_blocks,
              kCompactMaxGroups * 256);
  const size_t need = dsr_paged_compact_workspace_bytes(pool_blocks);
  rc = check_scratch(workspace, workspace_bytes, need, "paged_compact");
  if (rc != DSR_OK) return rc;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const CompactScratch s{reinterpret_cast<uint32_t*>(ws + 256), reinterpret_cast<int32_t*>(ws), int(groups)};
  if (whole_table(batch, table_stride, pool_blocks)) {
    const size_t smem = size_t(groups) * 36 + 4;
    rc = set_max_smem(compact_apply_kernel<true>, kWholeBlocks / 256 * 36 + 4, "paged_compact");
    if (rc != DSR_OK) return rc;
    return launch_after(compact_apply_kernel<true>, 1, kCompactThreads, smem, as_stream(stream), "paged_compact", a, s);
  }
  rc = set_max_smem(compact_apply_kernel<false>, size_t(kCompactMaxGroups + 1) * sizeof(int32_t), "paged_compact");
  if (rc != DSR_OK) return rc;
  const cudaError_t e = cudaMemsetAsync(ws, 0, need, as_stream(stream));
  if (e != cudaSuccess) return fail(DSR_ECUDA, "paged_compact: %s", cudaGetErrorString(e));
  const int64_t entries = batch * table_stride;
  compact_mark_kernel<<<share_grid(entries, kCompactThreads), kCompactThreads, 0, as_stream(stream)>>>(a, s);
  rc = launch_status("paged_compact launch");
  if (rc != DSR_OK) return rc;
  return launch_after(compact_apply_kernel<false>, share_grid(entries > pool_blocks ? entries : pool_blocks, kCompactThreads),
                      kCompactThreads, size_t(groups + 1) * sizeof(int32_t), as_stream(stream), "paged_compact", a, s);
}

extern "C" int dsr_paged_copy(void* const* pools, const int64_t* row_bytes, int64_t pool_count,
                              int64_t* const* generations, int64_t generation_count, int64_t pool_rows,
                              const int32_t* moves, const int32_t* count, int64_t max_moves, int32_t* err,
                              void* stream) {
  using namespace dsr;
  clear_error();
  DSR_REQUIRE(moves && count && err, "paged_copy: null pointer");
  DSR_REQUIRE(aligned16(moves), "paged_copy: moves must be 16-byte aligned");
  DSR_REQUIRE(pool_count >= 0 && pool_count <= kCopyMax && generation_count >= 0 && generation_count <= kCopyMax,
              "paged_copy: more than %d pools or generations", kCopyMax);
  DSR_REQUIRE((pool_count == 0 || (pools && row_bytes)) && (generation_count == 0 || generations),
              "paged_copy: null pointer");
  DSR_REQUIRE(pool_rows > 0 && pool_rows < (int64_t(1) << 31), "paged_copy: pool rows %lld outside [1, 2^31)",
              (long long)pool_rows);
  DSR_REQUIRE(max_moves >= 0 && max_moves < (int64_t(1) << 25), "paged_copy: moves %lld outside [0, 2^25)",
              (long long)max_moves);
  CopyArgs a = {};
  for (int64_t i = 0; i < pool_count; ++i) {
    DSR_REQUIRE(pools[i] && aligned16(pools[i]), "paged_copy: pools must be 16-byte aligned");
    DSR_REQUIRE(row_bytes[i] > 0 && row_bytes[i] <= 65536 && row_bytes[i] % 16 == 0,
                "paged_copy: rows of %lld bytes, not a multiple of 16 in [16, 65536]", (long long)row_bytes[i]);
    a.data[i] = static_cast<uint8_t*>(pools[i]);
    a.row_bytes[i] = int32_t(row_bytes[i]);
    a.first[i + 1] = a.first[i] + int32_t((row_bytes[i] * DSR_BLOCK_TOKENS + kCopyPiece - 1) / kCopyPiece);
  }
  for (int64_t i = 0; i < generation_count; ++i) {
    DSR_REQUIRE(generations[i], "paged_copy: null pointer");
    for (int64_t j = 0; j < i; ++j) {  // two threads would add to one entry
      const int64_t apart = reinterpret_cast<intptr_t>(generations[i]) - reinterpret_cast<intptr_t>(generations[j]);
      DSR_REQUIRE((apart < 0 ? -apart : apart) >= pool_rows * int64_t(sizeof(int64_t)),
                  "paged_copy: the same generations twice");
    }
    a.generations[i] = generations[i];
  }
  if (max_moves == 0 || pool_count + generation_count == 0) return DSR_OK;
  a.moves = reinterpret_cast<const int4*>(moves);
  a.count = count;
  a.rows = pool_rows;
  a.err = err;
  a.pools = int32_t(pool_count);
  a.gens = int32_t(generation_count);
  a.room = int32_t(max_moves);
  const int64_t items = max_moves * (a.first[pool_count] + 1), most = int64_t(sm_count()) * 8;
  return launch_after(copy_kernel, unsigned(items < most ? items : most), kCopyThreads, 0, as_stream(stream),
                      "paged_copy", a);
}
