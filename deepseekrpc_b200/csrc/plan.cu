// Block tables and slot maps of a paged batch, built on the GPU from the request
// lengths: dsr_paged_plan sets every request's number of mapped 64-row blocks to
// what its length needs and maps the new tokens to pool rows.
//
//   need_b = ceil((length_b + new_b) / 64)
//   need_b > held_b: blocks [held_b, need_b) come from the head of the free ring,
//   need_b < held_b: blocks [need_b, held_b) go back to its tail (entries -> -1),
//   both in request order, then block order.  Token i of the batch belongs to the
//   request b with cu_b <= i < cu_{b+1}, sits at position p = length_b + i - cu_b
//   and in pool row table[b][p / 64] * 64 + p % 64.
//
// One launch.  Every CTA scans all requests itself (batch <= 16384: at most 192 KB
// that come from L2 after the first CTA), so that no CTA waits for another: a
// token whose block is new reads its id from the free ring, never from the table
// entry that another CTA may be writing.  Blocks are taken from the ring's head
// and given back behind its tail, which are disjoint entries.  What all CTAs read
// and the call changes (held, the ring's head and count) is written by the last
// CTA to finish (a ticket in the ring state).  Bound by latency: one scan, one
// dependent read of the block id, one store.  Measured: 7 us a call for 1 request as for
// 256 with 8 tokens each (launch and the extension's allocation); 1M tokens of 256
// requests 15.6 us, 12 MB written (0.8 TB/s).
#include "common.cuh"
#include "host_common.h"

namespace dsr {
namespace {

constexpr int kPlanThreads = 512;
constexpr int kPlanMaxBatch = 16384;
constexpr int kBlockShift = 6;
static_assert(DSR_BLOCK_TOKENS == 1 << kBlockShift, "64-row blocks");

struct PlanArgs {
  const int32_t* lengths;
  const int32_t* new_tokens;
  int32_t* held;
  int32_t* table;
  int64_t stride;
  int32_t* ring;
  int32_t* state;  // head, count, ticket (0 between calls), unused
  int64_t blocks;
  int32_t* seq;
  int32_t* positions;
  int32_t* slots;
  int32_t* cu;       // [batch + 1]
  int32_t* visible;  // [batch]
  int32_t* err;
  int64_t tokens;
  int batch;
};

struct Sums {
  int64_t tokens, take, give;
};

__device__ __forceinline__ Sums operator+(const Sums& a, const Sums& b) {
  return Sums{a.tokens + b.tokens, a.take + b.take, a.give + b.give};
}
__device__ __forceinline__ Sums shfl_up(const Sums& s, int d) {
  return Sums{__shfl_up_sync(~0u, s.tokens, d), __shfl_up_sync(~0u, s.take, d), __shfl_up_sync(~0u, s.give, d)};
}

// Request b's sizes; false when they are out of range (then all zero).
__device__ __forceinline__ bool plan_request(const PlanArgs& a, int b, int32_t& len, int32_t& fresh, int32_t& have,
                                             int32_t& need) {
  len = a.lengths[b];
  fresh = a.new_tokens[b];
  have = a.held[b];
  const int64_t total = int64_t(len) + fresh;
  if (len < 0 || fresh < 0 || total > a.stride * DSR_BLOCK_TOKENS || have < 0 || have > a.stride) {
    len = fresh = have = need = 0;
    return false;
  }
  need = int32_t((total + DSR_BLOCK_TOKENS - 1) >> kBlockShift);
  return true;
}

// The largest b with cu[b] <= i (cu[0] = 0, cu increasing weakly, i < cu[n]).
__device__ __forceinline__ int plan_owner(const int32_t* cu, int n, int32_t i) {
  int lo = 0, hi = n;  // cu[lo] <= i < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanArgs a) {
  extern __shared__ int32_t plan_smem[];
  int32_t* cu_tokens = plan_smem;                  // [batch + 1]
  int32_t* cu_take = cu_tokens + a.batch + 1;      // [batch + 1]
  int32_t* cu_give = cu_take + a.batch + 1;        // [batch + 1]
  __shared__ Sums warp_sums[kPlanThreads / 32];
  __shared__ int bad, last;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) bad = 0;
  __syncthreads();

  // ---- exclusive sums over the requests (each thread a run of consecutive ones)
  const int per = (a.batch + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
  Sums mine{0, 0, 0};
  for (int b = b0; b < b1; ++b) {
    int32_t len, fresh, have, need;
    if (!plan_request(a, b, len, fresh, have, need)) bad = 1;
    mine = mine + Sums{fresh, max(need - have, 0), max(have - need, 0)};
  }
  Sums run = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const Sums up = shfl_up(run, d);
    if (lane >= d) run = run + up;
  }
  if (lane == 31) warp_sums[warp] = run;
  __syncthreads();
  Sums before{0, 0, 0}, all{0, 0, 0};
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w < warp) before = before + warp_sums[w];
    all = all + warp_sums[w];
  }
  const int64_t head = a.state[0], count = a.state[1];
  const bool ok = bad == 0 && all.tokens <= a.tokens && all.take <= count && head >= 0 && head < a.blocks &&
                  count >= 0 && count + all.give <= a.blocks;
  Sums at = before + run;
  at = Sums{at.tokens - mine.tokens, at.take - mine.take, at.give - mine.give};
  if (ok) {
    for (int b = b0; b < b1; ++b) {
      int32_t len, fresh, have, need;
      plan_request(a, b, len, fresh, have, need);
      cu_tokens[b] = int32_t(at.tokens);
      cu_take[b] = int32_t(at.take);
      cu_give[b] = int32_t(at.give);
      at = at + Sums{fresh, max(need - have, 0), max(have - need, 0)};
      if (blockIdx.x == 0) {
        a.cu[b] = cu_tokens[b];
        a.visible[b] = len + fresh;
      }
    }
    if (tid == 0) {
      cu_tokens[a.batch] = int32_t(all.tokens);
      cu_take[a.batch] = int32_t(all.take);
      cu_give[a.batch] = int32_t(all.give);
      if (blockIdx.x == 0) a.cu[a.batch] = int32_t(all.tokens);
    }
  } else if (blockIdx.x == 0) {
    // refused: nothing of the tables changes, no token is mapped
    if (tid == 0) {
      flag(a.err, DSR_ERR_ID);
      a.cu[a.batch] = 0;
    }
    for (int b = b0; b < b1; ++b) {
      a.cu[b] = 0;
      a.visible[b] = a.lengths[b];
    }
  }
  __syncthreads();

  const int64_t step = int64_t(gridDim.x) * kPlanThreads, first = int64_t(blockIdx.x) * kPlanThreads + tid;
  auto ring_at = [&](int64_t i) { return int64_t(i < a.blocks ? i : i - a.blocks); };
  // ---- the map of the new tokens, four consecutive ones a thread, stored 16 bytes at a time
  // where all three outputs allow (1M tokens: 15.6 us, off that grid 19.8; 16K: 10.3 both)
  const int64_t mapped = ok ? all.tokens : 0;
  const bool vec = ((reinterpret_cast<uintptr_t>(a.seq) | reinterpret_cast<uintptr_t>(a.positions) |
                     reinterpret_cast<uintptr_t>(a.slots)) & 15u) == 0;
  for (int64_t i0 = first * 4; i0 < a.tokens; i0 += step * 4) {
    int32_t seq[4], pos[4], slot[4];
    int32_t s = i0 < mapped ? plan_owner(cu_tokens, a.batch, int32_t(i0)) : 0;
    int32_t len = 0, have = 0, start = 0, next = 0, last_j = -1, blk = -1;
    bool fetch = true;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t i = i0 + q;
      seq[q] = pos[q] = slot[q] = -1;
      if (i >= mapped) continue;
      if (!fetch && i >= next) {
        do ++s;
        while (cu_tokens[s + 1] <= i);
        fetch = true;
      }
      if (fetch) {
        len = a.lengths[s], have = a.held[s], start = cu_tokens[s], next = cu_tokens[s + 1];
        last_j = -1;
        fetch = false;
      }
      const int32_t p = len + int32_t(i) - start, j = p >> kBlockShift;
      if (j != last_j) {
        blk = j < have ? a.table[int64_t(s) * a.stride + j] : a.ring[ring_at(head + cu_take[s] + (j - have))];
        last_j = j;
      }
      seq[q] = s;
      pos[q] = p;
      if (blk >= 0 && blk < a.blocks) slot[q] = blk * DSR_BLOCK_TOKENS + (p & (DSR_BLOCK_TOKENS - 1));
      else flag(a.err, DSR_ERR_ID);
    }
    if (vec && i0 + 4 <= a.tokens) {
      *reinterpret_cast<int4*>(a.seq + i0) = make_int4(seq[0], seq[1], seq[2], seq[3]);
      *reinterpret_cast<int4*>(a.positions + i0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      *reinterpret_cast<int4*>(a.slots + i0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (i0 + q < a.tokens) a.seq[i0 + q] = seq[q], a.positions[i0 + q] = pos[q], a.slots[i0 + q] = slot[q];
    }
  }
  if (ok) {
    // ---- blocks moved, four of a thread at a time: their chains of reads run side by side
    constexpr int kMoves = 4;
    // taken from the ring's head
    for (int64_t i0 = first; i0 < all.take; i0 += step * kMoves) {
      int32_t blk[kMoves], *entry[kMoves];
#pragma unroll
      for (int q = 0; q < kMoves; ++q) {
        const int64_t i = i0 + q * step;
        entry[q] = nullptr;
        if (i >= all.take) continue;
        blk[q] = a.ring[ring_at(head + i)];
        const int b = plan_owner(cu_take, a.batch, int32_t(i));
        entry[q] = a.table + int64_t(b) * a.stride + a.held[b] + (int32_t(i) - cu_take[b]);
      }
#pragma unroll
      for (int q = 0; q < kMoves; ++q) {
        if (entry[q] == nullptr) continue;
        const bool good = blk[q] >= 0 && blk[q] < a.blocks;
        if (!good) flag(a.err, DSR_ERR_ID);
        *entry[q] = good ? blk[q] : -1;
      }
    }
    // given back behind its tail
    for (int64_t i0 = first; i0 < all.give; i0 += step * kMoves) {
      int32_t blk[kMoves], *entry[kMoves];
#pragma unroll
      for (int q = 0; q < kMoves; ++q) {
        const int64_t i = i0 + q * step;
        entry[q] = nullptr;
        if (i >= all.give) continue;
        const int b = plan_owner(cu_give, a.batch, int32_t(i));
        const int32_t need = (a.lengths[b] + a.new_tokens[b] + DSR_BLOCK_TOKENS - 1) >> kBlockShift;
        entry[q] = a.table + int64_t(b) * a.stride + need + (int32_t(i) - cu_give[b]);
        blk[q] = *entry[q];
      }
#pragma unroll
      for (int q = 0; q < kMoves; ++q) {
        if (entry[q] == nullptr) continue;
        const bool good = blk[q] >= 0 && blk[q] < a.blocks;
        if (!good) flag(a.err, DSR_ERR_ID);
        a.ring[ring_at(ring_at(head + count) + i0 + q * step)] = good ? blk[q] : -1;
        *entry[q] = -1;
      }
    }
  }
  // ---- the last CTA to get here writes what every CTA has read
  __syncthreads();
  if (tid == 0) {
    last = gridDim.x == 1;
    if (!last) {
      __threadfence();
      last = atomicAdd(a.state + 2, 1) == int(gridDim.x) - 1;
      __threadfence();
    }
  }
  __syncthreads();
  if (!last) return;
  if (ok) {
    for (int b = b0; b < b1; ++b) {
      int32_t len, fresh, have, need;
      plan_request(a, b, len, fresh, have, need);
      if (need != have) a.held[b] = need;
    }
    if (tid == 0) {
      a.state[0] = int32_t((head + all.take) % a.blocks);
      a.state[1] = int32_t(count - all.take + all.give);
    }
  }
  if (tid == 0) a.state[2] = 0;
}

}  // namespace
}  // namespace dsr

extern "C" int dsr_paged_plan(const int32_t* lengths, const int32_t* new_tokens, int32_t* held, int32_t* block_table,
                              int64_t table_stride, int32_t* free_ring, int32_t* ring_state, int64_t pool_blocks,
                              int32_t* seq, int32_t* positions, int32_t* slots, int64_t tokens, int32_t* cu_tokens,
                              int32_t* visible, int32_t* err, int64_t batch, void* stream) {
  using namespace dsr;
  clear_error();
  PoolAddr pa;  // the range checks of every paged entry point
  const int rc = paged_addr(&pa, block_table, table_stride, pool_blocks, "paged_plan");
  if (rc != DSR_OK) return rc;
  DSR_REQUIRE(lengths && new_tokens && held && free_ring && ring_state && cu_tokens && visible && err,
              "paged_plan: null pointer");
  DSR_REQUIRE(batch > 0 && batch <= kPlanMaxBatch, "paged_plan: batch %lld outside [1, %d]", (long long)batch,
              kPlanMaxBatch);
  DSR_REQUIRE(tokens >= 0 && tokens < (int64_t(1) << 31), "paged_plan: tokens %lld outside [0, 2^31)",
              (long long)tokens);
  DSR_REQUIRE(tokens == 0 || (seq && positions && slots), "paged_plan: null token map");
  const size_t smem = 3 * size_t(batch + 1) * sizeof(int32_t);
  const int set = set_max_smem(plan_kernel, 3 * size_t(kPlanMaxBatch + 1) * sizeof(int32_t), "paged_plan");
  if (set != DSR_OK) return set;
  const PlanArgs a{lengths, new_tokens, held,  block_table, table_stride, free_ring, ring_state,  pool_blocks, seq,
                   positions, slots,    cu_tokens, visible, err,          tokens,    int(batch)};
  // a CTA for every four tokens a thread, and for the moves of blocks, whose number is not
  // known here, one for every 32 table entries a thread; up to one per SM
  const int64_t by_tokens = (tokens + kPlanThreads * 4 - 1) / (kPlanThreads * 4);
  const int64_t by_table = (batch * table_stride + kPlanThreads * 32 - 1) / (kPlanThreads * 32);
  int64_t grid = by_tokens > by_table ? by_tokens : by_table;
  if (grid > sm_count()) grid = sm_count();
  plan_kernel<<<unsigned(grid), kPlanThreads, smem, as_stream(stream)>>>(a);
  return launch_status("paged_plan launch");
}
