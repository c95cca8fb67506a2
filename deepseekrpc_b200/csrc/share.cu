// Blocks of a paged cache that several requests map: forking a request, giving blocks
// back, moving the blocks in use together, and the copies of rows that these name.
//
//   shares[blk] = table entries that map block blk beyond the first (0: one request's
//   own, or free), so that a program without shared blocks has zeros there for good and
//   dsr_paged_plan, which only ever maps free blocks, need not know of it.
//
// A move (source row, destination row, rows, 0) names up to one block of rows to copy.
// The tables are changed once for all layers; dsr_paged_copy then runs per cache, or for
// the pools of many layers at once.
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
__device__ __forceinline__ Pair operator+(const Pair& a, const Pair& b) { return Pair{a.x + b.x, a.y + b.y}; }

// Exclusive sums over the CTA's threads; `all` the totals.  `part` holds one pair a warp.
template <int Threads>
__device__ __forceinline__ Pair cta_scan(const Pair& mine, Pair* part, Pair& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Pair run = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const Pair up{__shfl_up_sync(~0u, run.x, d), __shfl_up_sync(~0u, run.y, d)};
    if (lane >= d) run = run + up;
  }
  if (lane == 31) part[warp] = run;
  __syncthreads();
  Pair before{0, 0};
  all = Pair{0, 0};
  for (int w = 0; w < Threads / 32; ++w) {
    if (w < warp) before = before + part[w];
    all = all + part[w];
  }
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

// True in all threads of the last CTA to get here (a ticket in the ring state).
__device__ __forceinline__ bool last_cta(const ShareArgs& a, int* last) {
  __syncthreads();
  if (threadIdx.x == 0) {
    *last = gridDim.x == 1;
    if (!*last) {
      __threadfence();
      *last = atomicAdd(a.state + 2, 1) == int(gridDim.x) - 1;
      __threadfence();
    }
  }
  __syncthreads();
  return *last != 0;
}

// ---------------------------------------------------------------------------
// Fork.  Every CTA scans all requests itself, as the plan does; an entry of a child is
// read from its parent's row, which no child's is.  held and the ring's state are written
// by the last CTA, since all have read them.
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
  if (tid == 0) bad = 0;
  __syncthreads();
  const int per = (a.batch + kForkThreads - 1) / kForkThreads;
  const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
  Pair mine{0, 0};
  for (int b = b0; b < b1; ++b) {
    int32_t parent, len, need;
    if (!fork_request(a, b, parent, len, need)) bad = 1;
    mine = mine + Pair{need, (len & (DSR_BLOCK_TOKENS - 1)) != 0};
  }
  Pair all, at = cta_scan<kForkThreads>(mine, part, all);
  const int64_t head = a.state[0], count = a.state[1];
  const bool ok = bad == 0 && all.x < (int64_t(1) << 31) && all.y <= count && head >= 0 && head < a.blocks &&
                  count >= 0 && count <= a.blocks;
  if (ok) {
    for (int b = b0; b < b1; ++b) {
      int32_t parent, len, need;
      fork_request(a, b, parent, len, need);
      cu_entry[b] = int32_t(at.x);
      cu_take[b] = int32_t(at.y);
      at = at + Pair{need, (len & (DSR_BLOCK_TOKENS - 1)) != 0};
    }
    if (tid == 0) cu_entry[a.batch] = int32_t(all.x), cu_take[a.batch] = int32_t(all.y);
  } else if (blockIdx.x == 0 && tid == 0) {
    flag(a.err, DSR_ERR_ID);
  }
  __syncthreads();
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
  if (!last_cta(a, &last)) return;
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
// Release, in two launches.  The first (one CTA) decides: which last blocks are shared,
// before any count changes, and what is dropped.  The second drops the entries; the last
// of its CTAs gives the blocks that nobody maps any more to the ring, in the order of
// their ids, so that the order in which the counts were lowered does not matter.
// Scratch: {ok, taken, dropped} and cu_drop[batch + 1], then a bit per freed block.
// ---------------------------------------------------------------------------
constexpr int kScanThreads = 1024, kDropThreads = 512;
constexpr int kScanPer = kShareMaxBatch / kScanThreads;

struct ReleaseScratch {
  int32_t* head;      // {ok, taken, dropped}
  int32_t* cu_drop;   // [batch + 1]
  uint32_t* freed;    // [words]
  int64_t words;      // a multiple of 4
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

__global__ void __launch_bounds__(kScanThreads, 1) release_scan_kernel(const ShareArgs a, const ReleaseScratch s) {
  __shared__ Pair part[kScanThreads / 32];
  __shared__ int bad;
  const int tid = threadIdx.x;
  if (tid == 0) bad = 0;
  for (int64_t w = tid; w < s.words; w += kScanThreads) s.freed[w] = 0u;
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
    mine = mine + Pair{have - need, copies >> (b - b0) & 1};
  }
  Pair all, at = cta_scan<kScanThreads>(mine, part, all);
  const int64_t head = a.state[0], count = a.state[1];
  const bool ok = bad == 0 && all.x < (int64_t(1) << 31) && all.y <= count && head >= 0 && head < a.blocks &&
                  count >= 0 && count <= a.blocks;
  const int64_t moved = ok ? all.y : 0;
  for (int64_t i = moved + tid; i < a.batch; i += kScanThreads) a.moves[i] = kNoMove;
  if (tid == 0) {
    s.head[0] = ok;
    s.head[1] = int32_t(moved);
    s.head[2] = ok ? int32_t(all.x) : 0;
    *a.count = int32_t(moved);
    if (!ok) flag(a.err, DSR_ERR_ID);
  }
  if (ok) {
    // every count has been read: it may change now
    for (int b = b0; b < b1; ++b) {
      const int32_t len = a.lengths[b], need = blocks_of(len);
      s.cu_drop[b] = int32_t(at.x);
      at.x += a.held[b] - need;
      if (!(copies >> (b - b0) & 1)) continue;
      int32_t* entry = a.table + int64_t(b) * a.stride + need - 1;
      const int32_t source = *entry, blk = a.ring[ring_at(a, head + at.y)];
      const bool good = blk >= 0 && blk < a.blocks;
      if (!good) flag(a.err, DSR_ERR_ID);
      a.moves[at.y] = good ? make_int4(source * DSR_BLOCK_TOKENS, blk * DSR_BLOCK_TOKENS,
                                       len & (DSR_BLOCK_TOKENS - 1), 0)
                           : kNoMove;
      *entry = good ? blk : -1;
      drop_block(a, s.freed, source);
      ++at.y;
    }
    if (tid == 0) s.cu_drop[a.batch] = int32_t(all.x);
  }
}

__global__ void __launch_bounds__(kDropThreads, 1) release_drop_kernel(const ShareArgs a, const ReleaseScratch s) {
  extern __shared__ int32_t drop_smem[];  // cu_drop
  __shared__ Pair part[kDropThreads / 32];
  __shared__ int last;
  const int tid = threadIdx.x;
  pdl_wait();
  const bool ok = __ldcg(s.head) != 0;
  const int32_t dropped = __ldcg(s.head + 2);
  if (ok && dropped > 0) {
    for (int b = tid; b <= a.batch; b += kDropThreads) drop_smem[b] = __ldcg(s.cu_drop + b);
    __syncthreads();
    for (int64_t i = int64_t(blockIdx.x) * kDropThreads + tid; i < dropped; i += int64_t(gridDim.x) * kDropThreads) {
      const int b = share_owner(drop_smem, a.batch, int32_t(i));
      int32_t* entry = a.table + int64_t(b) * a.stride + blocks_of(a.lengths[b]) + (int32_t(i) - drop_smem[b]);
      const int32_t blk = *entry;
      *entry = -1;
      drop_block(a, s.freed, blk);
    }
  }
  if (!last_cta(a, &last)) return;
  if (ok) {
    const int64_t head = a.state[0], count = a.state[1], taken = __ldcg(s.head + 1);
    int64_t free = 0;
    // 128 blocks a thread at a time
    for (int64_t w0 = 0; w0 < s.words; w0 += 4 * kDropThreads) {
      const int64_t w = w0 + 4 * tid;
      uint4 bits = make_uint4(0u, 0u, 0u, 0u);
      if (w < s.words) bits = __ldcg(reinterpret_cast<const uint4*>(s.freed + w));
      const int n = __popc(bits.x) + __popc(bits.y) + __popc(bits.z) + __popc(bits.w);
      if (!__syncthreads_or(n)) continue;
      Pair all, at = cta_scan<kDropThreads>(Pair{n, 0}, part, all);
      int64_t to = head + count + free + at.x;
      const uint32_t word[4] = {bits.x, bits.y, bits.z, bits.w};
#pragma unroll
      for (int q = 0; q < 4; ++q)
        for (uint32_t left = word[q]; left != 0; left &= left - 1, ++to) {
          const int32_t blk = int32_t(w + q) * 32 + __ffs(left) - 1;
          a.ring[to % a.blocks] = blk;
          a.shares[blk] = 0;
        }
      free += all.x;
    }
    for (int b = tid; b < a.batch; b += kDropThreads) a.held[b] = blocks_of(a.lengths[b]);
    if (tid == 0) {
      const int64_t now = count - taken + free;
      if (now > a.blocks) flag(a.err, DSR_ERR_ID);  // the ring held blocks that were mapped
      a.state[0] = int32_t((head + taken) % a.blocks);
      a.state[1] = int32_t(now < a.blocks ? now : a.blocks);
    }
  }
  if (tid == 0) a.state[2] = 0;
}

// ---------------------------------------------------------------------------
// Compaction.  With L live blocks (mapped by an entry below its row's held), the i-th
// live id from L on goes to the i-th id below L that is not live: the fewest copies, and
// no destination is a source.  A bit per live block; every CTA sums the bits of 256-block
// groups itself and finds ranks and free ids by search.
// ---------------------------------------------------------------------------
constexpr int kCompactThreads = 512;
constexpr int kCompactMaxGroups = 32768;  // of 256 blocks: 128 KB of shared memory

struct CompactScratch {
  uint32_t* live;  // [8 groups]
  int32_t* bad;
  int groups;
};

__global__ void __launch_bounds__(kCompactThreads) compact_mark_kernel(const ShareArgs a, const CompactScratch s) {
  const int64_t step = int64_t(gridDim.x) * kCompactThreads, first = int64_t(blockIdx.x) * kCompactThreads + threadIdx.x;
  for (int64_t b = first; b < a.batch; b += step)
    if (a.held[b] < 0 || a.held[b] > a.stride) {
      flag(a.err, DSR_ERR_ID);
      *s.bad = 1;
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
    if (!(__ldcg(s.live + (blk >> 5)) & bit)) atomicOr(s.live + (blk >> 5), bit);
  }
}

__global__ void __launch_bounds__(kCompactThreads) compact_apply_kernel(const ShareArgs a, const CompactScratch s) {
  extern __shared__ int32_t before[];  // [groups + 1] live blocks before each group
  __shared__ Pair part[kCompactThreads / 32];
  const int tid = threadIdx.x;
  pdl_wait();
  const int64_t step = int64_t(gridDim.x) * kCompactThreads, first = int64_t(blockIdx.x) * kCompactThreads + tid;
  const int64_t room = a.blocks < 2 ? 1 : a.blocks / 2;
  if (__ldcg(s.bad) != 0) {
    for (int64_t i = first; i < room; i += step) a.moves[i] = kNoMove;
    if (first == 0) *a.count = 0;
    return;
  }
  auto words = [&](int g, uint32_t (&w)[8]) {
    const uint4 lo = __ldcg(reinterpret_cast<const uint4*>(s.live) + 2 * g);
    const uint4 hi = __ldcg(reinterpret_cast<const uint4*>(s.live) + 2 * g + 1);
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
    if (!(__ldcg(s.live + (i >> 5)) >> (i & 31) & 1)) continue;
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
// Copies.  A work item is a piece of one move's rows in one pool; the generations of the
// written rows are a pool's last items.
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

int64_t freed_words(int64_t blocks) { return (blocks + 127) / 128 * 4; }
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

// CTAs for `items` of which a thread takes `per`, up to one per SM.
unsigned share_grid(int64_t items, int64_t per) {
  const int64_t grid = (items + per - 1) / per;
  return unsigned(grid < 1 ? 1 : grid < sm_count() ? grid : sm_count());
}

template <typename... P, typename... A>
int launch_after(void (*kernel)(P...), unsigned grid, int threads, size_t smem, cudaStream_t stream, const char* what,
                 const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) return fail(DSR_ECUDA, "%s launch: %s", what, cudaGetErrorString(e));
  return DSR_OK;
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
  fork_kernel<<<grid, kForkThreads, 2 * size_t(batch + 1) * sizeof(int32_t), as_stream(stream)>>>(a);
  return launch_status("paged_fork launch");
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
  rc = set_max_smem(release_drop_kernel, size_t(kShareMaxBatch + 1) * sizeof(int32_t), "paged_release");
  if (rc != DSR_OK) return rc;
  release_scan_kernel<<<1, kScanThreads, 0, as_stream(stream)>>>(a, s);
  rc = launch_status("paged_release launch");
  if (rc != DSR_OK) return rc;
  return launch_after(release_drop_kernel, share_grid(batch * table_stride, kDropThreads), kDropThreads,
                      size_t(batch + 1) * sizeof(int32_t), as_stream(stream), "paged_release", a, s);
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
  rc = set_max_smem(compact_apply_kernel, size_t(kCompactMaxGroups + 1) * sizeof(int32_t), "paged_compact");
  if (rc != DSR_OK) return rc;
  const cudaError_t e = cudaMemsetAsync(ws, 0, need, as_stream(stream));
  if (e != cudaSuccess) return fail(DSR_ECUDA, "paged_compact: %s", cudaGetErrorString(e));
  const int64_t entries = batch * table_stride;
  compact_mark_kernel<<<share_grid(entries, kCompactThreads), kCompactThreads, 0, as_stream(stream)>>>(a, s);
  rc = launch_status("paged_compact launch");
  if (rc != DSR_OK) return rc;
  return launch_after(compact_apply_kernel, share_grid(entries > pool_blocks ? entries : pool_blocks, kCompactThreads),
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
