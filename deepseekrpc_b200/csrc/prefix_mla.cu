// MLA attention of a batch whose requests continue common prompts (sm_100a): what
// tree_mla.cu computes, with the rows that consecutive requests share read and multiplied
// once for all of them.
//
//   request b attends over positions p < S_b = 64 floor(prefix_b / 64) through table row
//   holder_b and over S_b <= p through its own; requests in a row with the same holder and
//   S form a run, whose (node, head) pairs R are one matrix:
//     S = Q K^T,  P = e^{s - m},  O = P V  over the S shared rows, for all R at once,
//   and each request's own rows as there.  Every part leaves (m, l, O) in FP32; a row's
//   parts are joined with its sink:
//     out = sum_p 2^{m_p - M} O_p / (2^{sink - M} + sum_p 2^{m_p - M} l_p).
//
// Three launches without a host read: the plan (one CTA), the attention, the join.  More than
// 64 query rows, or 32 requests: by pairs of CTAs in groups of 128 rows, the runs' and the
// requests' own rows alike.  Fewer: one group has all rows of a run, and the tree attention's
// kernel takes the jobs from a list (two requests of 16 heads over 4096 rows: 21 us; by pairs
// in an earlier form 38, for 27 by the list).
//
// Bound by the tensor cores, and by the power that they may take.  Measured with cold inputs,
// alone and one call after another: 64 requests of 128 heads that share 32768 rows and have up to
// 1500 of their own 385 and 471 us (598 GFLOP: 1.55 PFLOP/s, 93% of a measured BF16 GEMM, and 1.27,
// 91% of a sustained one); 256 of 64 heads over 65472 rows 1640 and 1930 us (1.43 PFLOP/s, 86%, and
// 1.22, 88%); 23 requests of 1 to 6 nodes and 32 heads over 5 prompts 72 and 71 us (60%: the plan
// 3.5 us, 7 until the first tile is there, outputs of 3.5, the join 7.5).  The same by the tree
// attention's groups of 64 rows, alone: 831, 3133 and 122 us.  FP32 queries: 390, 1668 and 82 us
// alone, since the softmax warps convert them before a piece's first product.
#include <type_traits>

#include "common.cuh"
#include "host_common.h"
#include "tree_jobs.cuh"

namespace dsr {
namespace {

constexpr int kPrefixMaxBatch = 16384;
constexpr int kFewBatch = 32, kFewRows = 64;  // what the tree attention's kernel takes
constexpr int kPlanWaves = 4, kPlanTried = kPlanWaves + 1;
// A job's cost beside its tiles, in tiles: first copies, output, its part of the join.
constexpr float kPlanJobTiles = 4.f;
constexpr int kPairRows = 128;
// The same of a piece, added to a group's tiles where the pairs share out the work.  (A change of
// the group takes 9000 cycles, 3.7 tiles, but a pair's last output holds up no other group.  With
// 2, 3 and 4: 256 requests of 64 heads over 65472 rows 1670, 1646 and 1663 us, 64 of 128 heads over 32768 385,
// 385 and 387, 23 of 5 prompts 73.8, 71.8 and 73.7, 9 of 128 heads over 5184 38.9, 35.8 and 35.8;
// 100 of 3 nodes and 32 heads with 4000 rows of their own 195 with 2, 197 with 3.)
constexpr int kPairLead = 3;
static_assert(DSR_BLOCK_TOKENS == 64, "64-row blocks");

// A request: its query rows, where its own parts are, and where those of its run: part +
// segment * rows, or (segments < 0, the pairs') item -1 - segments.
struct alignas(16) PrefixRequest {
  int32_t node0, nodes;
  int32_t own_part, own_segments;
  int32_t run_part, run_rows, run_segments;
  int32_t run_node0;
};
static_assert(sizeof(PrefixRequest) == 32, "two 16-byte words");

// What the pairs of CTAs take.  A run's query rows are cut into groups of 128.  A group has the
// tiles of the shared rows, then, where all of its rows are one request's, those of the request's
// own rows: O stays where it is (137 requests of 128 heads over 752 shared rows: 92 us with every
// request's own rows by themselves, 72 so; the 64 requests above 412 and 393).  The own rows of a
// request whose groups have other requests' rows too, or that has no run, are an item by
// themselves, in groups of its own rows: with weights of zero another request's values would
// still reach a row where they are not finite.  (Taken all the same: 23 requests of 5 prompts 68 us
// for 74, 52 of 32 heads 35 for 39, 100 of 3 nodes and 32 heads with 640 rows of their own 111 for
// 124, 256 of 64 heads over 65472 rows 1642 for 1659.)
// Units are tiles, and kPairLead before each group's first; pair c has the units [c share,
// (c + 1) share) of all runs, then those of all items by themselves, in one piece per group.
// Piece (group g, pair c) leaves its partials at part + 128 (g + c), since g or c rises from
// piece to piece.
struct alignas(16) PairItem {
  int64_t unit0;                 // (of a run: its first group)
  int32_t groups, tiles;         // tiles: of a run's shared rows
  int32_t row0, rows;            // query rows
  int32_t table, part;
  int32_t block0;                // tile i: positions 64 block0 + 128 i and up
  int32_t context, drafts;       // positions from `context` on are drafted, seen as the masks say
  int32_t unused;
  __device__ __forceinline__ int32_t span() const { return tiles + kPairLead; }
};
static_assert(sizeof(PairItem) == 48, "three 16-byte words");
// A run's group, with the request that has its first row; behind the last one its end.
struct alignas(16) PairGroup {
  int64_t unit0;
  int32_t item, request;
};
// A request's own rows, where they are taken with its run: as in an item.
struct alignas(16) PairSegment {
  int32_t block0, context, drafts;
  int32_t unused;
};
static_assert(sizeof(PairSegment) == 16, "a 16-byte word");

// Where the parts of a node's rows are: of its request's own rows, then of its run.  The pairs'
// idle warp finds it, so that a CTA of the join has one load to wait for and not four.
struct alignas(16) PairNode {
  int32_t own_part, own_parts;  // of the node's first row; -1: a row of no request
  int32_t run_part, run_parts;
};

struct PrefixArgs {
  int64_t stride, table_rows;
  const int32_t* context;
  const int32_t* cu_nodes;
  const int32_t* prefix;
  const int32_t* holder;
  const float* sink;
  void* out;
  bool out_wide, zero_unused;
  float* lse;
  int32_t* err;
  int32_t* head;  // {jobs, 1 when no request was refused, 0, 0, groups of runs, share, items of requests, share}
  PrefixRequest* requests;
  PairItem* items;        // [batch] of runs, [batch] of requests
  PairGroup* groups;      // [groups of runs + 1]
  PairSegment* segments;  // [batch]
  int32_t* owner;         // [nodes] the request, where it has a run (see owns_all)
  PairNode* records;      // [nodes]
  TreeJob* jobs;
  float *part_o, *part_m, *part_l;
  int64_t nodes;
  int batch, heads, max_nodes, ctas;
  int rows;              // of a job's group
  int pairs;             // of CTAs (0: the jobs are the tree attention's)
  int32_t own_part;      // where the partials of the requests' own items begin
};

// ---- request b: what it has to itself, and the blocks that it reads through `holder`
struct PrefixSeq {
  int32_t node0, nodes, context, shared, holder;
  bool ok;
};
__device__ __forceinline__ PrefixSeq prefix_seq(const PrefixArgs& a, int b) {
  const int32_t n0 = a.cu_nodes[b], n1 = a.cu_nodes[b + 1], ctx = a.context[b], pre = a.prefix[b];
  PrefixSeq s{n0, n1 - n0, ctx, pre / DSR_BLOCK_TOKENS, a.holder[b], true};
  if (pre < DSR_BLOCK_TOKENS) s.shared = 0, s.holder = -1;
  if (n0 < 0 || n1 < n0 || n1 > a.nodes || n1 - n0 > a.max_nodes || ctx < 0 ||
      int64_t(ctx) + (n1 - n0) > a.stride * DSR_BLOCK_TOKENS ||
      (n1 > n0 && (pre < 0 || pre > ctx || (s.shared > 0 && (s.holder < 0 || s.holder >= a.table_rows)))))
    return PrefixSeq{0, 0, 0, 0, -1, false};
  return s;
}
// A refused request is a run of its own.
__device__ __forceinline__ bool prefix_continues(const PrefixSeq& before, const PrefixSeq& s) {
  return s.ok && before.ok && s.shared == before.shared && s.holder == before.holder;
}

// ---- what is to do for a run, or a request's own rows, in groups of `rows` query rows
__device__ __forceinline__ PairItem own_item(const PrefixArgs& a, int b, const PrefixSeq& s, int rows) {
  PairItem it{};
  const int64_t keys = int64_t(s.context) + s.nodes - s.shared * DSR_BLOCK_TOKENS;
  if (s.nodes == 0 || keys <= 0) return it;
  it.row0 = s.node0 * a.heads, it.rows = s.nodes * a.heads;
  it.groups = (it.rows + rows - 1) / rows;
  it.tiles = int32_t((keys + 127) / 128);
  it.table = b, it.block0 = s.shared;
  it.context = s.context, it.drafts = s.nodes;
  return it;
}
// (Of a run's first and last request.)
__device__ __forceinline__ PairItem run_item(const PrefixArgs& a, const PrefixSeq& s, const PrefixSeq& last, int rows) {
  PairItem it{};
  if (!s.ok || s.shared == 0 || last.node0 + last.nodes == s.node0) return it;
  it.row0 = s.node0 * a.heads, it.rows = (last.node0 + last.nodes - s.node0) * a.heads;
  it.groups = (it.rows + rows - 1) / rows;
  it.tiles = (s.shared + 1) / 2;
  it.table = s.holder;
  it.context = s.shared * DSR_BLOCK_TOKENS;
  return it;
}
// The pair that has a unit: a quotient below 256, for which a 64-bit division would take a
// hundred instructions.
__device__ __forceinline__ int32_t pair_of(int64_t unit, int64_t share) {
  int32_t c = int32_t(float(unit) / float(share));  // off by one at most
  if (c * share > unit) --c;
  if ((c + 1) * share <= unit) ++c;
  return c;
}
__device__ __forceinline__ int64_t pair_units(const PairItem& it) { return int64_t(it.groups) * it.span(); }
__device__ __forceinline__ PairItem load_item(const PairItem* item) {
  const int4* words = reinterpret_cast<const int4*>(item);
  const int4 x = __ldcg(words), y = __ldcg(words + 1), z = __ldcg(words + 2);
  return PairItem{int64_t(uint32_t(x.x)) | int64_t(x.y) << 32, x.z, x.w, y.x, y.y, y.z, y.w, z.x, z.y, z.z, z.w};
}

// Exclusive sums over the CTA's threads, and their total.  `part` is not used by the scan
// before this one.
template <int Threads, typename T>
__device__ __forceinline__ T plan_scan(T mine, T& all, T* part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto inclusive = [&](T x) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const T up = __shfl_up_sync(~0u, x, d);
      if (lane >= d) x += up;
    }
    return x;
  };
  const T sum = inclusive(mine);
  if (lane == 31) part[warp] = sum;
  __syncthreads();
  const T one = lane < Threads / 32 ? part[lane] : T(0), upto = inclusive(one);
  all = __shfl_sync(~0u, upto, 31);
  return sum - mine + __shfl_sync(~0u, upto - one, warp);
}
// Groups (which overflow only in sums that are refused for their rows), rows (64 nodes of 128
// heads each at most) and items in one sum.
constexpr int kItemBits = 16, kRowBits = 28;
static_assert(kPrefixMaxBatch < 1 << kItemBits && int64_t(kPrefixMaxBatch) * 64 * 128 < 1 << kRowBits, "of a call");
__device__ __forceinline__ int64_t pair_counts(const PairItem& it) {
  return int64_t(uint64_t(it.groups) << (kItemBits + kRowBits)) + (int64_t(it.rows) << kItemBits) + (it.groups > 0);
}
__device__ __forceinline__ int32_t items_of(int64_t counts) { return int32_t(counts & ((1 << kItemBits) - 1)); }
__device__ __forceinline__ int32_t rows_of(int64_t counts) {
  return int32_t(counts >> kItemBits & ((1 << kRowBits) - 1));
}
__device__ __forceinline__ int32_t groups_of(int64_t counts) {
  return int32_t(uint64_t(counts) >> (kItemBits + kRowBits));
}

// What the pairs share: false, with nothing to do and a status, when sums in disorder give rows to
// several requests, more than there are partials for, or a pair's share is above 2^31 units (in
// all 2.6e15 pairs of a query row and a key).
__device__ __forceinline__ bool write_pair_head(const PrefixArgs& a, bool writes, bool fine, int64_t run_units,
                                                int64_t run_all, int64_t own_units, int64_t own_all) {
  const int64_t run_share = (run_units + a.pairs - 1) / a.pairs, own_share = (own_units + a.pairs - 1) / a.pairs;
  const int64_t most = a.nodes * a.heads;
  const bool fits = rows_of(run_all) <= most && rows_of(own_all) <= most && run_share <= INT32_MAX &&
                    own_share <= INT32_MAX;
  if (writes) {
    if (!fits) flag(a.err, DSR_ERR_ID);
    int4* head = reinterpret_cast<int4*>(a.head);
    head[0] = make_int4(0, fits ? int(fine) : 1, 0, 0);
    head[1] = fits ? make_int4(groups_of(run_all), int(run_share), items_of(own_all), int(own_share))
                   : make_int4(0, 0, 0, 0);
    if (fits) a.groups[groups_of(run_all)] = PairGroup{run_units, -1, -1};
  }
  return fits;
}
// The groups of its run that a request lies across, and its own tiles in each of them: none where
// they have other requests' rows too.
struct PairShare {
  int32_t first, n, tiles;
};
__device__ __forceinline__ PairShare pair_share(const PairItem& own, int32_t run_groups, int32_t run_row0,
                                                int32_t run_rows) {
  if (run_groups == 0 || own.groups == 0) return PairShare{0, 0, 0};
  const int32_t in = own.row0 - run_row0, end = in + own.rows, first = in / kPairRows;
  const bool whole = in % kPairRows == 0 && (end % kPairRows == 0 || end == run_rows);
  return PairShare{first, (end - 1) / kPairRows - first + 1, whole ? own.tiles : 0};
}
// What the pairs have to know of a request of a run: its segment, the groups that begin in its
// rows, and whose its nodes are.  base: the run's first unit, and the own tiles before the request's.
__device__ __forceinline__ void write_share(const PrefixArgs& a, int b, const PrefixSeq& s, const PairItem& own,
                                            const PairShare& share, int64_t base, int32_t run_item, int32_t run_row0,
                                            int32_t run_group0, int32_t span) {
  a.segments[b] = PairSegment{own.block0, own.context, own.drafts, 0};
  const int32_t from = share.first + (own.row0 - run_row0 > share.first * kPairRows);
  for (int32_t g = from; g < share.first + share.n; ++g)
    a.groups[run_group0 + g] = PairGroup{base + int64_t(g) * span + int64_t(g - share.first) * share.tiles, run_item, b};
  for (int32_t x = 0; x < s.nodes; ++x) a.owner[s.node0 + x] = b;
}
// Sums in disorder may give a node to two runs, whose groups would not be whole then.
__device__ __forceinline__ bool owns_all(const PrefixArgs& a, int b, const PrefixSeq& s) {
  bool all = true;
  for (int32_t x = 0; x < s.nodes; ++x) all &= __ldcg(a.owner + s.node0 + x) == b;
  return all;
}
__device__ __forceinline__ void write_nothing(const PrefixArgs& a) {
  int4* head = reinterpret_cast<int4*>(a.head);
  head[0] = make_int4(0, 1, 0, 0), head[1] = make_int4(0, 0, 0, 0);
}

// The plan of the pairs' work.  Threads: 256 for up to 1024 requests, whose sequences are then
// kept in shared memory.
constexpr int kPlanCached = 1024;
template <int Threads, bool Cached>
__global__ void __launch_bounds__(Threads, 1) prefix_plan_kernel(const __grid_constant__ PrefixArgs a) {
  extern __shared__ int32_t starts[];  // [batch + 1] first request of each run
  __shared__ PrefixSeq cache[Cached ? kPlanCached : 1];
  __shared__ int64_t sums[4][32];
  __shared__ int32_t start_sums[32];
  const int tid = threadIdx.x;
  pdl_launch_dependents();
  const int per = (a.batch + Threads - 1) / Threads;
  const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
  auto seq = [&](int b) {
    if constexpr (Cached) return cache[b];
    else return prefix_seq(a, b);
  };
  if constexpr (Cached) {
    for (int b = tid; b < a.batch; b += Threads) cache[b] = prefix_seq(a, b);
    __syncthreads();
  }
  // ---- the runs
  auto starts_run = [&](int b) { return b == 0 || !prefix_continues(seq(b - 1), seq(b)); };
  int32_t first = 0, runs;
  bool fine = true;
  for (int b = b0; b < b1; ++b) {
    first += starts_run(b);
    if (!seq(b).ok) {
      fine = false;
      flag(a.err, DSR_ERR_ID);
    }
  }
  const int32_t run0 = plan_scan<Threads>(first, runs, start_sums);
  for (int b = b0, r = run0; b < b1; ++b)
    if (starts_run(b)) starts[r++] = b;
  if (tid == 0) starts[runs] = a.batch;
  fine = __syncthreads_and(fine);
  // ---- this thread's requests with their runs: f(b, its sequence, the run, whether it begins
  // there, its own rows, what is taken with the run)
  auto each = [&](auto&& f) {
    PairItem run{};
    for (int b = b0, r = run0 - 1; b < b1; ++b) {
      const bool begins = r + 1 < runs && starts[r + 1] == b;
      if (begins) ++r;
      if (begins || b == b0) run = run_item(a, seq(starts[r]), seq(starts[r + 1] - 1), kPairRows);
      const PrefixSeq s = seq(b);
      const PairItem own = own_item(a, b, s, kPairRows);
      f(b, s, run, begins, own, pair_share(own, run.groups, run.row0, run.rows));
    }
  };
  // ---- units and counts before each
  int64_t unit = 0, at = 0, own_unit = 0, own_at = 0, units, all, own_units, own_all;
  auto add = [&](const PairItem& run, bool begins, const PairItem& own, const PairShare& share) {
    if (begins) unit += pair_units(run), at += pair_counts(run);
    unit += int64_t(share.n) * share.tiles;
    if (share.tiles == 0) own_unit += pair_units(own), own_at += pair_counts(own);
  };
  each([&](int, const PrefixSeq&, const PairItem& run, bool begins, const PairItem& own, const PairShare& share) {
    add(run, begins, own, share);
  });
  unit = plan_scan<Threads>(unit, units, sums[0]);
  at = plan_scan<Threads>(at, all, sums[1]);
  own_unit = plan_scan<Threads>(own_unit, own_units, sums[2]);
  own_at = plan_scan<Threads>(own_at, own_all, sums[3]);
  const bool fits = write_pair_head(a, tid == 0, fine, units, all, own_units, own_all);
  each([&](int b, const PrefixSeq& s, PairItem run, bool begins, PairItem own, const PairShare& share) {
    if (!fits) {
      a.requests[b] = PrefixRequest{};
      return;
    }
    // (behind its first request the sums have the run in them)
    const int64_t base = begins ? unit : unit - pair_units(run), before = begins ? at : at - pair_counts(run);
    const int32_t index = items_of(before), own_index = items_of(own_at);
    const PairItem whole_run = run, whole_own = own;
    if (begins && run.groups > 0) {
      run.unit0 = groups_of(before), run.part = rows_of(before);
      a.items[index] = run;
    }
    if (run.groups > 0 && own.groups > 0)
      write_share(a, b, s, own, share, base, index, run.row0, groups_of(before), run.span());
    const bool alone = own.groups > 0 && share.tiles == 0;
    if (alone) {
      own.unit0 = own_unit, own.part = a.own_part + rows_of(own_at);
      a.items[a.batch + own_index] = own;
    }
    a.requests[b] = PrefixRequest{s.node0, s.nodes, 0, alone ? -1 - (a.batch + own_index) : 0, 0, 0,
                                  run.groups > 0 ? -1 - index : 0, 0};
    add(whole_run, begins, whole_own, share);
  });
  if (fine || !fits) return;
  __syncthreads();
  bool mine = true;
  each([&](int b, const PrefixSeq& s, const PairItem& run, bool, const PairItem&, const PairShare&) {
    if (run.groups > 0) mine &= owns_all(a, b, s);
  });
  if (__syncthreads_and(mine)) return;
  if (tid == 0) write_nothing(a);
  for (int b = b0; b < b1; ++b) a.requests[b] = PrefixRequest{};
}

// Up to 32 requests, without a barrier: lane b of every warp has request b and, if one starts
// there, its run; each warp finds the whole plan and writes its share of the jobs (3 us; the
// scans of the other kernel take 7).
//
// The tree attention's jobs (a.pairs == 0): a run's or a request's tiles are cut into segments
// of at most `length` tiles: one tile each when all units (group x tile) fit the grid, else the
// best of a few lengths by the time that the busiest CTA takes.  Jobs with long segments come
// first in the list, so that a CTA with a long one gets a short one next.
constexpr int kFewThreads = 256;
__global__ void __launch_bounds__(kFewThreads, 1) prefix_plan_few_kernel(const __grid_constant__ PrefixArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_launch_dependents();
  const bool here = lane < a.batch;
  const PrefixSeq s = here ? prefix_seq(a, lane) : PrefixSeq{0, 0, 0, 0, -1, true};
  const bool fine = __all_sync(~0u, s.ok);
  if (!s.ok && warp == 0) flag(a.err, DSR_ERR_ID);
  // ---- the runs: `last` request of the one that starts here, `start` of the one this is in
  const PrefixSeq before{0, 0, 0, __shfl_up_sync(~0u, s.shared, 1), __shfl_up_sync(~0u, s.holder, 1),
                         __shfl_up_sync(~0u, int(s.ok), 1) != 0};
  const bool starts = here && (lane == 0 || !prefix_continues(before, s));
  const unsigned all_starts = __ballot_sync(~0u, starts);
  const unsigned later = lane < 31 ? all_starts >> (lane + 1) : 0u;
  const int last = later != 0 ? lane + __ffs(later) - 1 : a.batch - 1;
  const int start = 31 - __clz(all_starts & (~0u >> (31 - lane)));
  const PrefixSeq end{__shfl_sync(~0u, s.node0, last & 31), __shfl_sync(~0u, s.nodes, last & 31), 0, 0, 0, true};
  PairItem own = own_item(a, lane, s, a.rows), run = starts ? run_item(a, s, end, a.rows) : PairItem{};
  auto before64 = [&](int64_t x, int64_t& all) {  // exclusive sums
    int64_t upto = x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t up = __shfl_up_sync(~0u, upto, d);
      if (lane >= d) upto += up;
    }
    all = __shfl_sync(~0u, upto, 31);
    return upto - x;
  };
  if (a.pairs > 0) {
    if (warp > 0) return;
    const int32_t groups = __shfl_sync(~0u, run.groups, start & 31), row0 = __shfl_sync(~0u, run.row0, start & 31);
    const int32_t span = __shfl_sync(~0u, run.span(), start & 31);
    const PairShare share = pair_share(own, groups, row0, __shfl_sync(~0u, run.rows, start & 31));
    const PairItem alone = share.tiles > 0 ? PairItem{} : own;
    int64_t units, run_all, own_units, own_all;
    const int64_t unit = before64(pair_units(run) + int64_t(share.n) * share.tiles, units);
    const int64_t at = before64(pair_counts(run), run_all), own_unit = before64(pair_units(alone), own_units);
    const int64_t own_at = before64(pair_counts(alone), own_all);
    const bool fits = write_pair_head(a, lane == 0, fine, units, run_all, own_units, own_all);
    const int32_t index = __shfl_sync(~0u, items_of(at), start & 31), own_index = items_of(own_at);
    const int32_t group0 = __shfl_sync(~0u, groups_of(at), start & 31);
    if (fits && run.groups > 0) {
      PairItem it = run;
      it.unit0 = group0, it.part = rows_of(at);
      a.items[index] = it;
    }
    // (behind its first request the sums have the run in them)
    if (fits && groups > 0 && own.groups > 0)
      write_share(a, lane, s, own, share, starts ? unit : unit - int64_t(groups) * span, index, row0, group0, span);
    if (fits && alone.groups > 0) {
      PairItem it = alone;
      it.unit0 = own_unit, it.part = a.own_part + rows_of(own_at);
      a.items[a.batch + own_index] = it;
    }
    bool whole = fits;
    if (!fine) {
      __syncwarp();
      whole = __all_sync(~0u, fits && (groups == 0 || owns_all(a, lane, s)));
      if (!whole && lane == 0) write_nothing(a);
    }
    if (here)
      a.requests[lane] = !whole ? PrefixRequest{}
                                : PrefixRequest{s.node0, s.nodes, 0, alone.groups > 0 ? -1 - (a.batch + own_index) : 0, 0, 0,
                                                groups > 0 ? -1 - index : 0, 0};
    return;
  }
  int64_t run_all, own_all;
  before64(pair_counts(run), run_all), before64(pair_counts(own), own_all);
  const int64_t most = a.nodes * a.heads;
  if (rows_of(run_all) > most || rows_of(own_all) > most) {  // as in write_pair_head
    if (threadIdx.x == 0) a.head[0] = 0, a.head[1] = 1;
    if (warp == 0 && here) a.requests[lane] = PrefixRequest{};
    return;
  }
  // ---- the segments' length
  auto segments = [](int32_t tiles, int32_t length) { return (tiles + length - 1) / length; };
  int64_t units;
  before64(int64_t(own.groups) * own.tiles + int64_t(run.groups) * run.tiles, units);
  int32_t length = 1;
  if (units > a.ctas) {
    const int32_t longest = __reduce_max_sync(~0u, max(own.tiles, run.tiles));
    float best = CUDART_INF_F;
#pragma unroll
    for (int w = 0; w < kPlanTried; ++w) {
      // the even share of so many jobs a CTA, or no cut at all
      const int64_t room = int64_t(w + 1) * a.ctas;
      const int32_t tried = w < kPlanWaves ? int32_t(min((units + room - 1) / room, int64_t(longest))) : longest;
      const int32_t jobs =
          __reduce_add_sync(~0u, own.groups * segments(own.tiles, tried) + run.groups * segments(run.tiles, tried));
      // the longest job, or a CTA's share of all
      const float time = fmaxf(float(tried) + kPlanJobTiles,
                               (float(units) + kPlanJobTiles * float(jobs)) / float(a.ctas));
      if (time < best) best = time, length = tried;
    }
  }
  // ---- jobs and partials before each lane's run and request
  const int32_t run_n = segments(run.tiles, length), own_n = segments(own.tiles, length);
  const int32_t run_jobs = run.groups * run_n, own_jobs = own.groups * own_n;
  int64_t at_all;  // jobs, and (low) rows of partials
  const int64_t at = before64(
      (int64_t(run_jobs + own_jobs) << 32) + int64_t(run.rows) * run_n + int64_t(own.rows) * own_n, at_all);
  const int32_t first = int32_t(at >> 32), run_part = int32_t(at & 0xffffffff), own_part = run_part + run.rows * run_n;
  const int32_t jobs = int32_t(at_all >> 32);
  // and their places in the list, where CTAs take several: long segments first
  int32_t run_place = first, own_place = first + run_jobs;
  if (jobs > a.ctas) {
    const float run_mine = run_n > 0 ? float(run.tiles) / float(run_n) : 0.f;
    const float own_mine = own_n > 0 ? float(own.tiles) / float(own_n) : 0.f;
    run_place = own_place = 0;
    for (int b = 0; b < a.batch; ++b) {  // equal ones: runs before requests, then by their number
      const float r = __shfl_sync(~0u, run_mine, b), o = __shfl_sync(~0u, own_mine, b);
      const int32_t rn = __shfl_sync(~0u, run_jobs, b), on = __shfl_sync(~0u, own_jobs, b);
      run_place += (r > run_mine || (r == run_mine && b < lane) ? rn : 0) + (o > run_mine ? on : 0);
      own_place += (r >= own_mine ? rn : 0) + (o > own_mine || (o == own_mine && b < lane) ? on : 0);
    }
  }
  if (threadIdx.x == 0) a.head[0] = jobs, a.head[1] = fine;
  // ---- the requests' records
  const int32_t of_part = __shfl_sync(~0u, run_part, start & 31), of_rows = __shfl_sync(~0u, run.rows, start & 31);
  const int32_t of_n = __shfl_sync(~0u, run_n, start & 31), of_node0 = __shfl_sync(~0u, s.node0, start & 31);
  if (warp == 0 && here) a.requests[lane] = PrefixRequest{s.node0, s.nodes, own_part, own_n, of_part, of_rows, of_n, of_node0};
  // ---- the jobs: an item's segments one after another, the groups of one side by side
  for (int32_t j0 = warp * 32; j0 < jobs; j0 += kFewThreads) {
    const int32_t j = min(j0 + lane, jobs - 1);
    int b = 0;  // the last lane whose jobs start at or before j
#pragma unroll
    for (int d = 16; d; d >>= 1)
      if (__shfl_sync(~0u, first, (b + d) & 31) <= j && b + d < 32) b += d;
    // (lanes without jobs start where the next one does: the last of those is the one that has j)
    const int32_t in_lane = j - __shfl_sync(~0u, first, b), of_run = __shfl_sync(~0u, run_jobs, b);
    const bool shared = in_lane < of_run;
    auto pick = [&](int32_t r, int32_t o) {
      const int32_t x = __shfl_sync(~0u, r, b), y = __shfl_sync(~0u, o, b);
      return shared ? x : y;
    };
    const int32_t in = shared ? in_lane : in_lane - of_run;
    const int32_t groups = pick(run.groups, own.groups), tiles = pick(run.tiles, own.tiles), n = pick(run_n, own_n);
    const int32_t all_rows = pick(run.rows, own.rows), part = pick(run_part, own_part), place = pick(run_place, own_place);
    const int32_t table = pick(run.table, own.table), block0 = pick(0, own.block0), first_row = pick(run.row0, own.row0);
    const int32_t drafts = pick(0, own.drafts), context = pick(run.context, own.context);
    if (j0 + lane >= jobs) continue;
    const int32_t segment = in / groups, group = in - segment * groups, row0 = group * a.rows;
    const int32_t whole = tiles / n, longer = tiles - whole * n;
    a.jobs[place + in] = TreeJob{table, block0, first_row / a.heads, row0, min(a.rows, all_rows - row0), drafts, context,
                                 segment * whole + min(segment, longer), whole + (segment < longer),
                                 part + segment * all_rows + row0, {}};
  }
}

// ---------------------------------------------------------------------------
// The attention by pairs of CTAs (clusters of two).  A unit is one group of 128 query rows x
// one 128-key tile, 64 rows of it in either CTA; the MMAs are the pair's (cta_group::2,
// M = 128), issued by CTA 0:
//   S[row, key]   = Q[row, :576] K[key, :576]      (N = 128 keys, 64 from either CTA)
//   O[row, dim]  += P[row, key] V[key, dim]        (N = 256 dims x 2, 128 from either CTA)
// so that an SM reads of every operand its own half only: 4 KB of shared memory for an MMA
// of 32 cycles, 6 KB for one of 64 (a CTA alone, with 64 rows: 6 KB for 32).  For S a CTA has
// its 64 keys of the tile with all columns, for O all 128 keys with its half of the value
// columns, which are fetched once more, from L2.  A tile takes some 2450 cycles, its 52 MMAs
// 2209 (measured by themselves: 32.6 and 64.7 cycles); 139 KB arrive in either SM meanwhile, 12
// TB/s in all.  A change of the group takes 9000: output, query, first tile.  What got it there,
// for the 64 requests above: copies of three and two column blocks issued by a converged warp (a
// lane by itself takes some 200 cycles a copy), page ids a tile ahead, and arrivals at the pair's
// barriers without a release to the cluster (1000 cycles).
// Not kept: pages prefetched into L2 a tile ahead (402 to 438 us).
// An accumulator of 64 rows takes tensor memory's lanes twice: lanes 0..63 have the rows and
// the first half of the columns, lanes 64..127 the same rows and the second half.
//   warps 0..7  (FP32 query -> shared memory,) softmax: warp w has rows 32 (w % 2) .. of
//               this CTA and of the keys, value columns in half w / 2 % 2 those in half w / 4;
//               the running maximum of a row is followed only when it grows by more than 2^8
//               (four warps: 2 to 8% slower where pieces are short, 1% faster in the largest)
//   warp 8      tensor memory; in CTA 0 the MMAs: S of the next tile, then O of this one, so
//               that they run through the softmax between
//   warp 9      query, keys and values by TMA; what arrives in either CTA is counted by CTA
//               0's barriers.  Values of a request's last tiles come to a barrier of the CTA's
//               own first: rows that no query sees may hold anything and are cleared, since
//               0 x NaN would reach the output
// ---------------------------------------------------------------------------
constexpr int kPairSoftmax = 256, kPairThreads = kPairSoftmax + 64;
constexpr int kPairKeys = 128;
constexpr int kKStages = 3, kKBlocks = 3;  // 64-column blocks of a copy: the nine of a key,
constexpr int kVBlocks = 2;                // and a CTA's of a pass over 256 value columns
constexpr float kPairSlack = 8.f;  // log2 units a row's maximum may lag behind

struct PairLayout {
  static constexpr int kBlock = 64 * 128;                    // 64 rows x 64 columns
  static constexpr int kQOff = 0;                            // 9 blocks
  static constexpr int kKOff = kQOff + 9 * kBlock;           // 9 blocks
  static constexpr int kVOff = kKOff + 9 * kBlock;           // 2 passes x 2 pages x 2 blocks
  static constexpr int kPOff = kVOff + 8 * kBlock;           // 2 blocks of 64 rows x 64 keys
  static constexpr int kBarOff = kPOff + 2 * kBlock;
  static constexpr int kBars = 2 * kKStages + 2 * 2 + 2 + 6;
  static constexpr int kRedOff = kBarOff + (kBars * 8 + 15) / 16 * 16;  // f32[4][64]
  static constexpr int kMiscOff = kRedOff + 4 * 64 * 4;
  static constexpr int kBytes = kMiscOff + 16;
  static constexpr int kAlloc = kBytes + 1024;
  static constexpr uint32_t kTmemCols = 512;  // O: 256 columns, S: two of 64
  static_assert(kAlloc <= 232448, "shared memory of one CTA");
};

struct PairArgs {
  const void* q;
  bool q_wide;  // fp32 (else bf16)
  const int32_t* table;
  int64_t stride, pool_rows;
  const int64_t* masks;
  float scale_log2;
  float *part_o, *part_m, *part_l;
  const int32_t* head;
  const PairItem* items;
  const PairGroup* groups;
  const PairSegment* segments;
  int32_t* err;
  int batch, heads, pairs;
  const int32_t* cu_nodes;
  const PrefixRequest* requests;
  PairNode* records;
  int32_t nodes;
};

__device__ __forceinline__ PrefixRequest load_request(const PrefixRequest* request) {
  const int4* words = reinterpret_cast<const int4*>(request);
  const int4 x = __ldcg(words), y = __ldcg(words + 1);
  return PrefixRequest{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
}
__device__ __forceinline__ PairGroup load_group(const PairGroup* group) {
  const int4 x = __ldcg(reinterpret_cast<const int4*>(group));
  return PairGroup{int64_t(uint32_t(x.x)) | int64_t(x.y) << 32, x.z, x.w};
}
__device__ __forceinline__ PairSegment load_segment(const PairSegment* segment) {
  const int4 x = __ldcg(reinterpret_cast<const int4*>(segment));
  return PairSegment{x.x, x.y, x.z, 0};
}
__device__ __forceinline__ PairNode find_node(const PairArgs& a, int32_t node) {
  int lo = 0;  // the largest b with cu_nodes[b] <= node
  for (int hi = a.batch; hi - lo > 1;) {
    const int mid = (lo + hi) >> 1;
    if (a.cu_nodes[mid] <= node) lo = mid;
    else hi = mid;
  }
  PrefixRequest s = load_request(a.requests + lo);
  if (node < s.node0 || node >= s.node0 + s.nodes) {
    // a padding row.  Where a request was refused the sums may be in disorder and the search
    // may have missed the request that has the row: every one is asked
    lo = -1;
    if (!__ldcg(a.head + 1)) {
#pragma unroll 8
      for (int b = 0; b < a.batch; ++b) {
        const int2 rows = __ldcg(reinterpret_cast<const int2*>(a.requests + b));  // node0, nodes
        if (node >= rows.x && node < rows.x + rows.y) lo = b;
      }
    }
    if (lo < 0) return PairNode{0, -1, 0, 0};
    s = load_request(a.requests + lo);
  }
  // the parts: those of the pairs that have a tile of the node's group
  auto parts = [&](const PairItem& item, int64_t unit, int64_t end, int share_at, int32_t& part, int32_t& count) {
    const int64_t share = __ldcg(a.head + share_at);
    const int32_t first = pair_of(unit + kPairLead, share), last = pair_of(end - 1, share);
    part = item.part + node * a.heads - item.row0 + kPairRows * first;
    count = last - first + 1;
  };
  PairNode found{0, 0, 0, 0};
  if (s.own_segments < 0) {
    const PairItem item = load_item(a.items - 1 - s.own_segments);
    const int64_t unit = item.unit0 + int64_t((node * a.heads - item.row0) / kPairRows) * item.span();
    parts(item, unit, unit + item.span(), 7, found.own_part, found.own_parts);
  }
  if (s.run_segments < 0) {
    const PairItem item = load_item(a.items - 1 - s.run_segments);
    const PairGroup* group = a.groups + item.unit0 + (node * a.heads - item.row0) / kPairRows;
    parts(item, load_group(group).unit0, load_group(group + 1).unit0, 5, found.run_part, found.run_parts);
  }
  return found;
}

// A pair's pieces, one after another (every warp walks them for itself): of the runs, then of
// the requests by themselves.
struct PairWalk {
  const PairArgs& a;
  int64_t unit, end;
  int32_t at, pair, phase;  // phase: 0 runs (`at` a group), 1 requests (an item)
  PairItem item;
  int64_t group_unit, next_unit;  // of a run's group, and the one behind it
  int32_t item_at, next_item, group;
  int32_t request, next_request;  // of their first rows
  int32_t row0, rows, tile0, count, part;  // of the piece at hand
  // the requests' range and first item, found with the runs'
  int64_t own_unit, own_end;
  int32_t own_at;
  __device__ __forceinline__ PairWalk(const PairArgs& a_, int pair_) : a(a_), pair(pair_), phase(0) {
    const int4 head = __ldcg(reinterpret_cast<const int4*>(a.head) + 1);
    unit = end = int64_t(head.y) * pair;
    own_unit = own_end = int64_t(head.w) * pair;
    at = own_at = 0;
    if (head.x > 0) {
      end = min(unit + head.y, load_group(a.groups + head.x).unit0);
      at = find(&a.groups->unit0, sizeof(PairGroup), head.x, unit);
    }
    if (head.z > 0) {
      const PairItem last = load_item(a.items + a.batch + head.z - 1);
      own_end = min(own_unit + head.w, last.unit0 + int64_t(last.groups) * last.span());
      own_at = find(&a.items[a.batch].unit0, sizeof(PairItem), head.z, own_unit);
    }
    if (unit >= end) return;
    const PairGroup here = load_group(a.groups + at), next = load_group(a.groups + at + 1);
    group_unit = here.unit0, item_at = here.item, request = here.request;
    next_unit = next.unit0, next_item = next.item, next_request = next.request;
    item = load_item(a.items + item_at);
  }
  // The last of n records, their first units `stride` bytes apart, that starts at or before the
  // unit, 32 ways a step.
  __device__ __forceinline__ int32_t find(const int64_t* units, int64_t stride, int32_t n_all, int64_t from) {
    int32_t first = 0;
    const char* base = reinterpret_cast<const char*>(units);
    for (int n = n_all; n > 1;) {
      const int step = (n + 31) / 32, i = int(threadIdx.x & 31) * step;
      const unsigned below =
          __ballot_sync(~0u, i < n && __ldcg(reinterpret_cast<const int64_t*>(base + (first + i) * stride)) <= from);
      const int lead = (31 - __clz(below)) * step;
      first += lead;
      n = min(step, n - lead);
    }
    return first;
  }
  __device__ __forceinline__ bool next() {
    for (;;) {
      if (unit >= end) {
        if (phase == 1 || own_unit >= own_end) return false;
        phase = 1;
        unit = own_unit, end = own_end, at = own_at;
        item = load_item(a.items + a.batch + at);
      }
      int64_t start, stop;  // the group's units
      if (phase == 0) {
        if (unit >= next_unit) {
          group_unit = next_unit, request = next_request;
          if (next_item != item_at) item_at = next_item, item = load_item(a.items + item_at);
          const PairGroup next = load_group(a.groups + ++at + 1);
          next_unit = next.unit0, next_item = next.item, next_request = next.request;
        }
        group = at - int32_t(item.unit0);
        start = group_unit, stop = next_unit;
      } else {
        if (unit >= item.unit0 + int64_t(item.groups) * item.span()) item = load_item(a.items + a.batch + ++at);
        group = int32_t((unit - item.unit0) / item.span());
        start = item.unit0 + int64_t(group) * item.span(), stop = start + item.span();
      }
      const int32_t from = int32_t(unit - start), to = int32_t(min(stop, end) - start);
      unit += to - from;
      tile0 = max(from - kPairLead, 0);
      count = max(to - kPairLead, 0) - tile0;
      row0 = item.row0 + group * kPairRows;
      rows = min(kPairRows, item.rows - group * kPairRows);
      part = item.part + (group + pair) * kPairRows;
      if (count > 0) return true;
    }
  }
  // The group's first tiles, of rows that all of it shares.
  __device__ __forceinline__ int32_t shared() const { return phase == 0 ? item.tiles : 0; }
  // What the tiles behind those are of: a request's own rows, from `position` on.
  struct Own {
    int32_t request, position, context, drafts;
  };
  __device__ __forceinline__ Own own() const {
    if (phase == 1) return Own{item.table, item.block0 * DSR_BLOCK_TOKENS, item.context, item.drafts};
    const PairSegment s = load_segment(a.segments + request);
    return Own{request, s.block0 * DSR_BLOCK_TOKENS, s.context, s.drafts};
  }
  // Whether some query rows of the group do not see all of a tile.
  __device__ __forceinline__ bool masked(int32_t tile) const {
    return item.block0 * DSR_BLOCK_TOKENS - item.context + int64_t(tile) * 128 > -128;  // (of a run: past its shared rows too)
  }
};

// ---- barriers of a pair
__device__ __forceinline__ uint32_t pair_address(const void* p, uint32_t cta) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(cta));
  return r;
}
__device__ __forceinline__ void pair_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Arrives at a barrier of either CTA (an address from pair_address).  At the scope of this
// CTA: no thread of the other one reads what this one's threads write, only the tensor core
// of this SM does, behind a proxy fence.  (A release to the cluster took some 1000 cycles.)
__device__ __forceinline__ void pair_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// mbar_wait whose polls sleep in the barrier unit.
__device__ __forceinline__ bool pair_try(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool pair_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int32_t* err) {
  if (pair_try(bar, parity)) return true;
  const uint64_t start = global_ns();
  for (;;) {
    if (pair_try(bar, parity)) return true;
    if (*abort) return false;
    if (global_ns() - start > kWaitNs) {
      *abort = 1;
      flag(err, DSR_ERR_TIMEOUT);
      return false;
    }
  }
}
// The same for a whole warp, with one answer for all lanes.
__device__ __forceinline__ bool pair_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort, int32_t* err) {
  return __all_sync(~0u, pair_wait(bar, parity, abort, err));
}
// A copy to this CTA that a barrier of CTA 0 (an address from pair_address) counts: 64 rows
// from y on of the 64-column blocks from z on, a block after another.
__device__ __forceinline__ void pair_load(uint32_t dst, const void* tmap, uint32_t bar, int32_t y, int32_t z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(0), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void pair_umma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives on `bar` of both CTAs once all MMAs issued so far are complete.
__device__ __forceinline__ void pair_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"(uint16_t(3))
      : "memory");
}
// The softmax threads of one half of a CTA's rows, four a row: a barrier, and whether every one
// is fine.
__device__ __forceinline__ bool rows_sync(int half, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(uint32_t(ok)), "r"(1 + half)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Two FP32 values an instruction, each rounded as by itself.
__device__ __forceinline__ uint64_t pack2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

__global__ void __launch_bounds__(kPairThreads, 1)
    prefix_pair_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                       const __grid_constant__ CUtensorMap q_map, const __grid_constant__ PairArgs a) {
  using L = PairLayout;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_smem_1024(smem_raw);
  const uint32_t sbase = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  // CTA 0's are waited for
  uint64_t* full_k = bars;                  // [kKStages] in both CTAs (TMA bytes + 1)
  uint64_t* full_v = full_k + kKStages;     // [2] (TMA bytes + 1 of either CTA)
  uint64_t* bar_p = full_v + 2;             // P written in both CTAs (a warp arrives)
  uint64_t* bar_q = bar_p + 1;              // query in place (TMA bytes + 1; FP32: a warp arrives)
  uint64_t* bar_free = bar_p + 2;           // O read by the output (a warp arrives)
  uint64_t* bar_end = bar_p + 3;            // all MMAs complete (commit)
  // each CTA has its own
  uint64_t* empty_k = bar_p + 4;            // [kKStages] read by the S MMAs (commit)
  uint64_t* empty_v = empty_k + kKStages;   // [2] read by the O MMAs (commit)
  uint64_t* bar_s = empty_v + 2;            // [2] S complete (commit)
  uint64_t* bar_o = bar_s + 2;              // the tile's O MMAs complete (commit)
  uint64_t* bar_own = bar_o + 1;            // values of a ragged tile here (TMA bytes + 1)
  static_assert(2 * kKStages + 2 * 2 + 2 + 6 == L::kBars, "");
  float* red = reinterpret_cast<float*>(smem + L::kRedOff);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMiscOff);
  volatile int* abort = reinterpret_cast<volatile int*>(smem + L::kMiscOff + 4);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = int(blockIdx.x & 1), pair = int(blockIdx.x >> 1);  // clusters of two along x

  if (tid == 0) {
    tma_prefetch_desc(&k_map);
    tma_prefetch_desc(&v_map);
    if (!a.q_wide) tma_prefetch_desc(&q_map);
    for (int i = 0; i < kKStages; ++i) mbar_init(full_k + i, 1), mbar_init(empty_k + i, 1);
    for (int i = 0; i < 2; ++i) mbar_init(full_v + i, 2), mbar_init(empty_v + i, 1), mbar_init(bar_s + i, 1);
    constexpr int kWarps = 2 * kPairSoftmax / 32;  // of both CTAs
    mbar_init(bar_p, kWarps);
    mbar_init(bar_q, a.q_wide ? kWarps : 1);
    mbar_init(bar_free, kWarps);
    mbar_init(bar_end, 1);
    mbar_init(bar_o, 1);
    mbar_init(bar_own, 1);
    *abort = 0;
    fence_barrier_init();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(L::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  pair_sync();  // the other CTA's barriers and tensor memory are there
  tc_fence_after();
  const uint32_t tmem_o = *tmem_slot, tmem_s = tmem_o + 256;
  pdl_wait();
  pdl_launch_dependents();
  PairWalk walk(a, pair);

  if (warp < 8) {
    // ------------------------------------------------------------ softmax
    const int pack = warp & 1, r = 32 * pack + lane;            // this thread's row of the CTA's
    const int half = warp >> 1 & 1, side = warp >> 2;           // of the columns, and of that half
    const uint32_t lanes = uint32_t(warp & 3) * 32 << 16;       // this warp's TMEM lanes
    const uint32_t to_p = pair_address(bar_p, 0), to_q = pair_address(bar_q, 0), to_free = pair_address(bar_free, 0);
    int n = 0;
    bool ok = true;
    while (ok && walk.next()) {
      const int count = walk.count, mine = 64 * rank + r;  // the row in its group
      if (a.q_wide) {
        // FP32 query rows -> bf16, K-major, 128-byte swizzle (as in the tree attention).  The
        // S MMAs of the piece before have been waited for with its last tile
        const float* src = static_cast<const float*>(a.q) + int64_t(walk.row0 + 64 * rank) * DSR_KV_DIM;
        constexpr int kVec = 64 * (DSR_KV_DIM / 8);
        for (int i = tid; i < kVec; i += kPairSoftmax) {
          const int row = i / (DSR_KV_DIM / 8), d = (i - row * (DSR_KV_DIM / 8)) * 8;
          uint4 v = make_uint4(0, 0, 0, 0);
          if (64 * rank + row < walk.rows) {
            const float4* at = reinterpret_cast<const float4*>(src + int64_t(row) * DSR_KV_DIM + d);
            const float4 lo = __ldg(at), hi = __ldg(at + 1);
            v = make_uint4(pack_bf16(lo.x, lo.y), pack_bf16(lo.z, lo.w), pack_bf16(hi.x, hi.y), pack_bf16(hi.z, hi.w));
          }
          *reinterpret_cast<uint4*>(smem + L::kQOff + (d >> 6) * L::kBlock + sw128_offset(row, d & 63)) = v;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) pair_arrive(to_q);
      }
      // the drafted positions that this thread's row sees, and where they are behind the first own
      // tile's start
      const PairWalk::Own own = walk.own();
      const int32_t shared = walk.shared(), own_left = own.context - own.position;
      uint64_t word = mine < walk.rows ? uint64_t(a.masks[(walk.row0 + mine) / a.heads]) : 0ull;
      if (own.drafts < 64) word &= (1ull << own.drafts) - 1ull;
      float m = -CUDART_INF_F, l = 0.f;
      for (int i = 0; i < count; ++i, ++n) {
        ok = ok && pair_wait_warp(bar_s + (n & 1), (n >> 1) & 1, abort, a.err);
        float v[32];
        float top = -CUDART_INF_F;
        if (ok) {
          tc_fence_after();
          uint32_t t0[32];
          tmem_ld32(tmem_s + (n & 1) * 64 + 32 * side + lanes, t0);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < 32; ++c) v[c] = __uint_as_float(t0[c]);
          const int32_t tile = walk.tile0 + i;
          if (walk.masked(tile)) {
            // bit c: this thread's key c is seen; key c is drafted position `first` + c.  (None
            // of a run's are drafted)
            const bool common = tile < shared;
            const int32_t first = 64 * half + 32 * side + (common ? int32_t(128u * tile - walk.item.context)
                                                                  : int32_t(128u * (tile - shared) - own_left));
            const uint64_t drafted = common ? 0ull : word;
            const uint32_t shown = first >= 64    ? 0u
                                   : first >= 0   ? uint32_t(drafted >> first)
                                   : first <= -32 ? ~0u
                                                  : uint32_t(drafted) << -first | ((1u << -first) - 1u);
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (!(shown >> c & 1u)) v[c] = -CUDART_INF_F;
          }
#pragma unroll
          for (int c = 0; c < 32; c += 2) top = max3(top, v[c], v[c + 1]);
          top *= a.scale_log2;
        }
        // weights against the running maximum as it stands; their sums are of the weights as
        // formed, for the product with V they are rounded to BF16 (as in the tree attention)
        uint32_t packed[16];
        float sum = 0.f;
        auto weigh = [&] {
          const float base = m == -CUDART_INF_F ? 0.f : m;
          const uint64_t scales = pack2(a.scale_log2, a.scale_log2), bases = pack2(-base, -base);
          uint64_t both = 0;
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            float x, y;
            unpack2(fma2(pack2(v[2 * c], v[2 * c + 1]), scales, bases), x, y);
            x = ex2(x), y = ex2(y);
            both = add2(both, pack2(x, y));
            packed[c] = pack_bf16(x, y);
          }
          float s0, s1;
          unpack2(both, s0, s1);
          sum = s0 + s1;
        };
        bool fits = ok && i > 0 && !(top > m + kPairSlack);
        if (ok && i > 0) weigh();
        // most tiles end here: no row's maximum has to follow
        if (!rows_sync(pack, fits)) {
          ok = rows_sync(pack, ok);
          if (!ok) break;
          red[64 * (2 * half + side) + r] = top;
          rows_sync(pack, true);
#pragma unroll
          for (int x = 0; x < 4; ++x) top = fmaxf(top, red[64 * x + r]);
          float f = 1.f;
          if (top > m + kPairSlack) f = ex2(m - top), l *= f, m = top;  // f: 0 when the row had seen nothing
          if (i > 0) {
            ok = rows_sync(pack, pair_wait_warp(bar_o, (n - 1) & 1, abort, a.err));
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 128 * side; c < 128 * side + 128; c += 32) {
              uint32_t o[32];
              tmem_ld32(tmem_o + c + lanes, o);
              tmem_wait_ld();
#pragma unroll
              for (int x = 0; x < 32; x += 2) {
                float lo, hi;
                unpack2(mul2(pack2(__uint_as_float(o[x]), __uint_as_float(o[x + 1])), pack2(f, f)), lo, hi);
                o[x] = __float_as_uint(lo), o[x + 1] = __float_as_uint(hi);
              }
              tmem_st32(tmem_o + c + lanes, o);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          }
          weigh();
        }
        l += sum;
        // P, once the O MMAs of the tile before have read theirs.  (A warp whose wait gives up
        // says so in the next vote: its rows' other warp must not wait there alone.)
        if (n > 0) ok = pair_wait_warp(bar_o, (n - 1) & 1, abort, a.err);
        if (!ok) continue;
#pragma unroll
        for (int c = 0; c < 4; ++c)
          *reinterpret_cast<uint4*>(smem + L::kPOff + half * L::kBlock + sw128_offset(r, 32 * side + 8 * c)) =
              make_uint4(packed[4 * c], packed[4 * c + 1], packed[4 * c + 2], packed[4 * c + 3]);
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) pair_arrive(to_p);
      }

      // ---- the piece's partials
      ok = ok && pair_wait_warp(bar_o, (n - 1) & 1, abort, a.err);
      red[64 * (2 * half + side) + r] = l;
      ok = rows_sync(pack, ok);
      if (!ok) break;
      const bool valid = mine < walk.rows;
      if (half == 0 && side == 0 && valid) {
        const float total = (red[r] + red[64 + r]) + (red[128 + r] + red[192 + r]);
        if (!(total < CUDART_INF_F)) flag(a.err, DSR_ERR_NONFINITE);
        a.part_m[int64_t(walk.part) + mine] = m;
        a.part_l[int64_t(walk.part) + mine] = total;
      }
      tc_fence_after();
      // four rows side by side: a quad's 4 x 4 values are transposed, so that a thread has
      // one column of its four rows
      const int q = lane & 3;
      float4* dst = reinterpret_cast<float4*>(a.part_o + (int64_t(walk.part) + (mine & ~3)) * DSR_V_DIM);
      const int first = 128 * side;  // of its 256 columns, this thread's
      uint32_t next[32];
      tmem_ld32(tmem_o + first + lanes, next);
#pragma unroll 1
      for (int c0 = first; c0 < first + 128; c0 += 32) {
        uint32_t o[32];
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 32; ++c) o[c] = next[c];
        if (c0 < first + 96) tmem_ld32(tmem_o + c0 + 32 + lanes, next);
        const int d0 = half * 256 + c0;  // a pass has 128 columns of either CTA's 256
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          // exchange with the neighbour, then with the other two
          uint32_t w[4] = {o[c], o[c + 1], o[c + 2], o[c + 3]};
          const uint32_t a0 = __shfl_xor_sync(~0u, q & 1 ? w[0] : w[1], 1), a1 = __shfl_xor_sync(~0u, q & 1 ? w[2] : w[3], 1);
          if (q & 1) w[0] = a0, w[2] = a1;
          else w[1] = a0, w[3] = a1;
          const uint32_t b0 = __shfl_xor_sync(~0u, q & 2 ? w[0] : w[2], 2), b1 = __shfl_xor_sync(~0u, q & 2 ? w[1] : w[3], 2);
          if (q & 2) w[0] = b0, w[1] = b1;
          else w[2] = b0, w[3] = b1;
          if (valid)
            dst[d0 + c + q] = make_float4(__uint_as_float(w[0]), __uint_as_float(w[1]), __uint_as_float(w[2]),
                                          __uint_as_float(w[3]));
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) pair_arrive(to_free);
    }
  } else if (warp == 8) {
    if (rank == 0) {
      // ------------------------------------------------------------ MMA issuer
      // The whole warp runs the loop and one lane issues, on values that are the same in all
      // lanes: descriptors then stay in uniform registers
      constexpr uint32_t idesc_s = umma_idesc_bf16(kPairRows, kPairKeys, false, false);
      constexpr uint32_t idesc_o = umma_idesc_bf16(kPairRows, 256, false, true);
      const uint32_t sb = __shfl_sync(~0u, sbase, 0);
      const uint32_t ts = __shfl_sync(~0u, tmem_s, 0), to = __shfl_sync(~0u, tmem_o, 0);
      const bool leader = elect_one();
      const uint64_t desc_q = umma_desc_sw128(sb + L::kQOff, 16, 1024), desc_k = umma_desc_sw128(sb + L::kKOff, 16, 1024);
      const uint64_t desc_p = umma_desc_sw128(sb + L::kPOff, 16, 1024);
      const uint64_t desc_v = umma_desc_sw128(sb + L::kVOff, L::kBlock, 1024);
      auto wait = [&](uint64_t* bar, uint32_t parity) { return pair_wait_warp(bar, parity, abort, a.err); };
      int n = 0, piece = 0;
      bool ok = true;
      // A descriptor that the compiler takes for a new value, so that it adds the steps below
      // each time and does not keep all 52 sums in registers
      auto anew = [](uint64_t x) {
        asm volatile("" : "+l"(x));
        return x;
      };
      // S of tile k: a step of 16 columns moves both operands by 32 bytes
      auto scores = [&](int k) {
#pragma unroll
        for (int c = 0; c < kKStages; ++c) {
          ok = ok && wait(full_k + c, k & 1);
          if (!ok) return;
          tc_fence_after();
          if (leader) {
            const uint64_t q = anew(desc_q), key = anew(desc_k);
#pragma unroll
            for (int x = 0; x < 4 * kKBlocks; ++x)
              pair_umma(ts + (k & 1) * 64, q + (kKBlocks * c + (x >> 2)) * (L::kBlock / 16) + 2 * (x & 3),
                        key + (kKBlocks * c + (x >> 2)) * (L::kBlock / 16) + 2 * (x & 3), idesc_s,
                        (c | x) != 0 ? 1u : 0u);
            pair_commit(empty_k + c);
          }
        }
        if (leader) pair_commit(bar_s + (k & 1));
      };
      while (ok) {
        if (!walk.next()) break;  // alike in all lanes
        const int count = __shfl_sync(~0u, walk.count, 0);
        ok = wait(bar_q, piece & 1);
        if (ok) scores(n);
        for (int i = 0; i < count && ok; ++i, ++n) {
          if (i + 1 < count) scores(n + 1);
          ok = ok && wait(bar_p, n & 1);
          // the output of the piece before has read O
          if (ok && i == 0 && piece > 0) ok = wait(bar_free, (piece - 1) & 1);
          if (!ok) break;
          const uint32_t accumulate = i > 0;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            ok = ok && wait(full_v + c, n & 1);
            if (!ok) break;
            tc_fence_after();
            if (leader) {
              const uint64_t weights = anew(desc_p), value = anew(desc_v);
#pragma unroll
              for (int ks = 0; ks < kPairKeys / 16; ++ks)
                pair_umma(to + c * 128, weights + (ks >> 2) * (L::kBlock / 16) + 2 * (ks & 3),
                          value + (4 * c + 2 * (ks >> 2)) * (L::kBlock / 16) + (ks & 3) * (2048 / 16), idesc_o,
                          ks > 0 ? 1u : accumulate);
              pair_commit(empty_v + c);
            }
          }
          if (leader && ok) pair_commit(bar_o);
        }
        ++piece;
      }
      // the last MMAs retire before TMEM is released
      if (leader)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                         smem_u32(bar_end))
                     : "memory");
      mbar_drain(bar_end, 0);
    } else {
      // ------------------------------------------------------------ what the join asks for
      for (int32_t node = pair * 32 + lane; node < a.nodes; node += a.pairs * 32) a.records[node] = find_node(a, node);
    }
  } else {
    // ------------------------------------------------------------ copies
    const uint32_t sb = __shfl_sync(~0u, sbase, 0);
    const uint32_t to_k = __shfl_sync(~0u, pair_address(full_k, 0), 0);
    const uint32_t to_v = __shfl_sync(~0u, pair_address(full_v, 0), 0);
    const uint32_t to_q = __shfl_sync(~0u, pair_address(bar_q, 0), 0);
    const uint32_t to_own = __shfl_sync(~0u, pair_address(bar_own, rank), 0);
    const bool leader = elect_one();
    int n = 0, cleared = 0;
    bool ok = true;
    while (ok && walk.next()) {
      // of the own rows, the drafted positions that any of the group's rows sees (8 nodes at most)
      const int32_t shared = walk.shared();
      const PairWalk::Own own = walk.own();
      const uint64_t word = lane * a.heads < walk.rows ? uint64_t(a.masks[walk.row0 / a.heads + lane]) : 0ull;
      const uint64_t seen = uint64_t(__reduce_or_sync(~0u, uint32_t(word))) |
                            uint64_t(__reduce_or_sync(~0u, uint32_t(word >> 32))) << 32;
      const int32_t none = int32_t(a.pool_rows);  // past the pool: reads zeros
      // the tile's two pages; what a block id means is seen when they are used
      auto pages = [&](int32_t tile) {
        int32_t row = walk.item.table, j = 2 * tile, blocks = walk.item.context / DSR_BLOCK_TOKENS;
        if (tile >= shared) {
          row = own.request;
          j = own.position / DSR_BLOCK_TOKENS + 2 * (tile - shared);
          blocks = int32_t((int64_t(own.context) + own.drafts + DSR_BLOCK_TOKENS - 1) / DSR_BLOCK_TOKENS);
        }
        const int32_t* table = a.table + int64_t(row) * a.stride;
        return make_int2(j < blocks ? table[j] : INT32_MIN, j + 1 < blocks ? table[j + 1] : INT32_MIN);
      };
      auto row_of = [&](int32_t blk) {
        if (blk == INT32_MIN) return none;
        if (blk < 0 || blk * int64_t(DSR_BLOCK_TOKENS) >= a.pool_rows) {
          flag(a.err, DSR_ERR_ID);
          return none;
        }
        return int32_t(blk * DSR_BLOCK_TOKENS);
      };
      // The whole warp runs the loop and one lane issues, as the MMAs are: a copy from a
      // one-lane branch takes some 200 cycles to be on its way
      auto wait = [&](uint64_t* bar, uint32_t parity) { return pair_wait_warp(bar, parity, abort, a.err); };
      if (!a.q_wide) {
        // the query, once the last S MMA of the piece before has read the one there
        if (n > 0) ok = wait(bar_s + ((n - 1) & 1), ((n - 1) >> 1) & 1);
        if (!ok) break;
        if (leader) {
          if (rank == 0) mbar_arrive_expect_tx(bar_q, 2 * 9 * L::kBlock);
          for (int c = 0; c < kKStages; ++c)
            pair_load(sb + L::kQOff + kKBlocks * c * L::kBlock, &q_map, to_q, walk.row0 + 64 * rank, kKBlocks * c);
        }
      }
      // keys of tile i from page `rank` of the tile's two, values of both
      auto keys = [&](int k, int32_t y) {
#pragma unroll
        for (int c = 0; c < kKStages; ++c) {
          ok = ok && wait(empty_k + c, (k & 1) ^ 1);
          if (!ok) return;
          if (leader) {
            if (rank == 0) mbar_arrive_expect_tx(full_k + c, 2 * kKBlocks * L::kBlock);
            pair_load(sb + L::kKOff + kKBlocks * c * L::kBlock, &k_map, to_k + 8 * c, y, kKBlocks * c);
          }
        }
      };
      auto values = [&](int k, int32_t tile, int32_t y0, int32_t y1) {
        // a request's rows from its context on: hidden ones are cleared before they count
        int32_t first = -kPairKeys;  // of its drafted positions, where the tile starts
        if (tile >= shared) first = int32_t(128u * (tile - shared) + own.position - own.context);
        const bool clears = first > -kPairKeys;
        if (clears && leader) mbar_arrive_expect_tx(bar_own, 2 * 4 * L::kBlock);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          ok = ok && wait(empty_v + c, (k & 1) ^ 1);
          if (!ok) return;
          if (leader) {
            if (!clears && rank == 0) mbar_arrive_expect_tx(full_v + c, 2 * 4 * L::kBlock);
            const uint32_t bar = clears ? to_own : to_v + 8 * c;
            const int32_t z = 4 * rank + kVBlocks * c;
            pair_load(sb + L::kVOff + 4 * c * L::kBlock, &v_map, bar, y0, z);
            pair_load(sb + L::kVOff + (4 * c + 2) * L::kBlock, &v_map, bar, y1, z);
            if (!clears && rank == 1) pair_arrive(to_v + 8 * c);
          }
        }
        if (!clears) return;
        ok = wait(bar_own, cleared++ & 1);
        if (!ok) return;
        // a lane has 16 bytes of a row: its four blocks' parts are 512 bytes
        uint8_t* mine = smem + L::kVOff + (4 * (lane >> 4) + (lane >> 3 & 1)) * L::kBlock + (lane & 7) * 16;
        auto clear = [&](int x) {
          *reinterpret_cast<uint4*>(mine + 2 * (x >> 6) * L::kBlock + (x & 63) * 128) = make_uint4(0, 0, 0, 0);
        };
        const int past = min(max(own.drafts - first, 0), kPairKeys);
        for (int x = max(-first, 0); x < past; ++x)
          if (!(seen >> (first + x) & 1)) clear(x);
#pragma unroll 4
        for (int x = past; x < kPairKeys; ++x) clear(x);
        fence_proxy_async_smem();
        __syncwarp();
        if (leader) pair_arrive(to_v), pair_arrive(to_v + 8);
      };
      const int count = __shfl_sync(~0u, walk.count, 0);
      int2 now = pages(walk.tile0), next = count > 1 ? pages(walk.tile0 + 1) : now;
      int32_t x0 = __shfl_sync(~0u, row_of(now.x), 0), x1 = __shfl_sync(~0u, row_of(now.y), 0);
      keys(n, rank == 0 ? x0 : x1);
      for (int i = 0; i < count && ok; ++i, ++n) {
        int32_t y0 = none, y1 = none;
        if (i + 1 < count) {
          y0 = __shfl_sync(~0u, row_of(next.x), 0), y1 = __shfl_sync(~0u, row_of(next.y), 0);
          if (i + 2 < count) next = pages(walk.tile0 + i + 2);  // a tile ahead
          keys(n + 1, rank == 0 ? y0 : y1);
        }
        if (ok) values(n, walk.tile0 + i, x0, x1);
        x0 = y0, x1 = y1;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort && tid == 0) {
    // a wait gave up: copies that nobody waits for any more land meanwhile
    const uint64_t start = global_ns();
    while (global_ns() - start < 2000000) __nanosleep(1000);
  }
  __syncthreads();
  pair_sync();  // neither CTA leaves while the other's copies, commits or MMAs may reach it
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_o), "r"(L::kTmemCols) : "memory");
  }
}

// ---------------------------------------------------------------------------
// Joins the parts of a row: one CTA per four query rows (of one node, since heads come in
// sixteens) and 128 Columns value columns, a thread Columns of them of all four and every
// Split-th part.  Few rows of many parts are bound by the latency of one part after another
// (32 rows of 34 parts: 10 us by one thread a column, each after eight others), many rows by
// the partials that come from L2 (17536 rows, 54 MB: 15 us).
// ---------------------------------------------------------------------------
constexpr int kJoinThreads = 128;
constexpr int kJoinMaxParts = kPlanWaves * kTreeMaxCtas + 16;

template <bool kPairs, int Columns, int Split, int kBatch>  // kBatch: parts requested together
__global__ void __launch_bounds__(kJoinThreads * Split) prefix_join_kernel(const __grid_constant__ PrefixArgs a) {
  __shared__ float weight[4][kPairs ? kTreeMaxCtas + 2 : kJoinMaxParts];
  __shared__ float inverse[4], tops[4][Split], sums[4][Split];
  __shared__ float4 others[Split > 1 ? Split - 1 : 1][Columns][kJoinThreads];
  const int64_t row = int64_t(blockIdx.x) * 4;
  const int32_t node = int32_t(row / a.heads);
  const int tid = threadIdx.x, thread = tid % kJoinThreads, turn = tid / kJoinThreads;
  const int d = blockIdx.y * Columns * kJoinThreads + thread;  // the first column
  // ---- where the row's parts are: part p at own0 + p own_rows, then run0 + p run_rows
  int64_t own0, run0;
  int32_t own_rows = kPairRows, run_rows = kPairRows;
  int own = -1, parts = 0;
  if constexpr (kPairs) {
    pdl_wait();  // before any CTA leaves: the join must not end ahead of the attention
    const int4 found = __ldcg(reinterpret_cast<const int4*>(a.records + node));
    const int64_t in = row - int64_t(node) * a.heads;
    own0 = found.x + in, own = found.y;
    run0 = found.z + in, parts = own + found.w;
  } else {
    // the request (of up to 32) that has the node: the last whose first node is not behind it
    const int lane = tid & 31;
    const unsigned below = __ballot_sync(~0u, lane < a.batch && a.cu_nodes[lane] <= node);
    const int last = below == 0 ? 0 : 31 - __clz(below);
    pdl_wait();
    PrefixRequest s = load_request(a.requests + last);
    auto has_node = [&] { return node >= s.node0 && node < s.node0 + s.nodes; };
    bool found = has_node();
    if (!found) {
      // a padding row.  Where a request was refused the sums may be in disorder: all are asked
      s = lane < a.batch ? load_request(a.requests + lane) : PrefixRequest{};
      const unsigned has = __ballot_sync(~0u, has_node());
      found = has != 0;
      if (found) s = load_request(a.requests + 31 - __clz(has));
    }
    if (found) {
      own0 = s.own_part + row - int64_t(s.node0) * a.heads;
      run0 = s.run_part + row - int64_t(s.run_node0) * a.heads;
      own_rows = s.nodes * a.heads;
      run_rows = s.run_rows;
      own = s.own_segments;
      parts = own + s.run_segments;
    }
  }
  if (own < 0) {  // a padding row
    if (!a.zero_unused || turn > 0) return;
    for (int x = 0; x < 4 * Columns; ++x) {
      const int64_t at = (row + x % 4) * DSR_V_DIM + d + x / 4 * kJoinThreads;
      if (a.out_wide) static_cast<float*>(a.out)[at] = 0.f;
      else static_cast<uint16_t*>(a.out)[at] = 0;
    }
    if (a.lse != nullptr && blockIdx.y == 0 && tid < 4) a.lse[row + tid] = -CUDART_INF_F;
    return;
  }
  auto place = [&](int p) { return p < own ? own0 + int64_t(p) * own_rows : run0 + int64_t(p - own) * run_rows; };
  float4 v[kBatch][Columns];
  auto request = [&](int p0) {
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (p0 + j * Split < parts) {
        const float4* from = reinterpret_cast<const float4*>(a.part_o + place(p0 + j * Split) * DSR_V_DIM) + d;
#pragma unroll
        for (int c = 0; c < Columns; ++c) v[j][c] = __ldcg(from + c * kJoinThreads);
      }
  };
  request(turn);
  // ---- the parts' weights: row w by the warps w + 4 k, a lane every (32 Split)-th part
  const int w = (tid >> 5) & 3, p_first = turn + Split * (tid & 31);
  {
    const float m0 = p_first < parts ? __ldcg(a.part_m + place(p_first) + w) : -CUDART_INF_F;
    const float l0 = p_first < parts ? __ldcg(a.part_l + place(p_first) + w) : 0.f;
    float top = m0, sum = 0.f;
    for (int p = p_first + 32 * Split; p < parts; p += 32 * Split) top = fmaxf(top, __ldcg(a.part_m + place(p) + w));
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    if constexpr (Split > 1) {
      if ((tid & 31) == 0) tops[w][turn] = top;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < Split; ++k) top = fmaxf(top, tops[w][k]);
    }
    const float base = top == -CUDART_INF_F ? 0.f : top;
    for (int p = p_first; p < parts; p += 32 * Split) {
      const float e = ex2((p == p_first ? m0 : __ldcg(a.part_m + place(p) + w)) - base);
      weight[w][p] = e;
      sum += e * (p == p_first ? l0 : __ldcg(a.part_l + place(p) + w));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if ((tid & 31) == 0) sums[w][turn] = sum, tops[w][turn] = top;
  }
  __syncthreads();
  if (turn == 0 && (tid & 31) == 0) {
    float total, sum = 0.f;
#pragma unroll
    for (int k = 0; k < Split; ++k) sum += sums[w][k];
    const float lse = tree_total(a.sink, a.err, int((row + w) % a.heads), tops[w][0], sum, total);
    inverse[w] = total > 0.f ? 1.f / total : 0.f;
    if (a.lse != nullptr && blockIdx.y == 0) a.lse[row + w] = lse;
  }
  float4 acc[Columns];
#pragma unroll
  for (int c = 0; c < Columns; ++c) acc[c] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p0 = turn; p0 < parts; p0 += kBatch * Split) {
    if (p0 > turn) request(p0);
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int p = p0 + j * Split;
      if (p < parts)
#pragma unroll
        for (int c = 0; c < Columns; ++c) {
          acc[c].x = fmaf(weight[0][p], v[j][c].x, acc[c].x), acc[c].y = fmaf(weight[1][p], v[j][c].y, acc[c].y);
          acc[c].z = fmaf(weight[2][p], v[j][c].z, acc[c].z), acc[c].w = fmaf(weight[3][p], v[j][c].w, acc[c].w);
        }
    }
  }
  if constexpr (Split > 1) {
    if (turn > 0)
#pragma unroll
      for (int c = 0; c < Columns; ++c) others[turn - 1][c][thread] = acc[c];
  }
  __syncthreads();
  if (turn > 0) return;
  if constexpr (Split > 1) {
#pragma unroll
    for (int k = 0; k < Split - 1; ++k)
#pragma unroll
      for (int c = 0; c < Columns; ++c) {
        const float4 x = others[k][c][thread];
        acc[c].x += x.x, acc[c].y += x.y, acc[c].z += x.z, acc[c].w += x.w;
      }
  }
  float finite = 0.f;  // stays zero
#pragma unroll
  for (int c = 0; c < Columns; ++c) {
    const float out[4] = {acc[c].x * inverse[0], acc[c].y * inverse[1], acc[c].z * inverse[2], acc[c].w * inverse[3]};
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      finite = fmaf(out[y], 0.f, finite);
      const int64_t at = (row + y) * DSR_V_DIM + d + c * kJoinThreads;
      if (a.out_wide) static_cast<float*>(a.out)[at] = out[y];
      else static_cast<uint16_t*>(a.out)[at] = __bfloat16_as_ushort(__float2bfloat16_rn(out[y]));
    }
  }
  if (finite != 0.f) flag(a.err, DSR_ERR_NONFINITE);
}

int launch_pairs(const PairArgs& a, const uint16_t* kv_pool, int64_t rows, cudaStream_t stream) {
  int rc = set_max_smem(prefix_pair_kernel, PairLayout::kAlloc, "prefix_mla_decode");
  if (rc != DSR_OK) return rc;
  CUtensorMap k_map, v_map, q_map;  // 64 rows (a page, a CTA's of a group) of some 64-column blocks
  rc = encode_tmap_bf16_blocks(&k_map, kv_pool, DSR_KV_DIM, uint64_t(a.pool_rows), DSR_BLOCK_TOKENS, kKBlocks);
  if (rc != DSR_OK) return rc;
  rc = encode_tmap_bf16_blocks(&v_map, kv_pool, DSR_KV_DIM, uint64_t(a.pool_rows), DSR_BLOCK_TOKENS, kVBlocks);
  if (rc != DSR_OK) return rc;
  q_map = k_map;
  if (!a.q_wide) {
    rc = encode_tmap_bf16_blocks(&q_map, a.q, DSR_KV_DIM, uint64_t(rows), kPairRows / 2, kKBlocks);
    if (rc != DSR_OK) return rc;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(2 * a.pairs), 1, 1);
  cfg.blockDim = dim3(kPairThreads, 1, 1);
  cfg.dynamicSmemBytes = PairLayout::kAlloc;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, prefix_pair_kernel, k_map, v_map, q_map, a);
  if (e != cudaSuccess) return fail(DSR_ECUDA, "prefix_mla_decode pair launch: %s", cudaGetErrorString(e));
  return DSR_OK;
}

// ---- scratch: the head, the requests' records, the plan's own, the pairs' items or the jobs,
// the partials
size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }

struct PrefixSizes {
  int rows;
  int pairs;
  size_t requests, items, groups, segments, owner, records, jobs;  // bytes
  size_t parts, own_part;                // rows of partials, and where those of the requests' items begin
};
PrefixSizes prefix_sizes(int64_t batch, int64_t nodes, int64_t heads) {
  PrefixSizes s = {};
  const size_t rows = size_t(nodes) * heads;
  s.requests = rounded(size_t(batch) * sizeof(PrefixRequest));
  if (nodes * heads <= kFewRows && batch <= kFewBatch) {
    s.rows = tree_rows(heads, nodes);  // all rows in one group
    // a job per run and request; a cut adds at most kPlanWaves jobs a CTA
    const size_t cut = size_t(kPlanWaves) * tree_ctas();
    s.jobs = rounded((2 * size_t(batch) + cut) * sizeof(TreeJob));
    s.parts = 2 * rows + cut * s.rows;
  } else {
    s.rows = kPairRows;
    s.pairs = tree_ctas() / 2;
    s.items = rounded(2 * size_t(batch) * sizeof(PairItem));
    s.groups = rounded((rows / kPairRows + size_t(batch) + 1) * sizeof(PairGroup));
    s.segments = rounded(size_t(batch) * sizeof(PairSegment));
    s.owner = rounded(size_t(nodes) * sizeof(int32_t));
    s.records = rounded(size_t(nodes) * sizeof(PairNode));
    s.own_part = rows + size_t(kPairRows) * s.pairs;
    s.parts = 2 * s.own_part;
  }
  return s;
}

}  // namespace
}  // namespace dsr

extern "C" size_t dsr_prefix_mla_workspace_bytes(int64_t batch, int64_t nodes, int64_t heads) {
  using namespace dsr;
  if (batch <= 0 || nodes <= 0 || heads <= 0) return 0;
  const PrefixSizes s = prefix_sizes(batch, nodes, heads);
  return 256 + s.requests + s.items + s.groups + s.segments + s.owner + s.records + s.jobs +
         s.parts * (DSR_V_DIM + 2) * 4;
}

extern "C" int dsr_prefix_mla_decode(const void* q, int q_dtype, const uint16_t* kv_pool, int64_t pool_blocks,
                                     const int32_t* block_table, int64_t table_rows, int64_t table_stride,
                                     const int32_t* context, const int32_t* cu_nodes, const int64_t* tree_mask,
                                     int64_t max_nodes, const int32_t* prefix, const int32_t* holder,
                                     const float* sink, float scale, void* out, int out_dtype, float* lse,
                                     void* workspace, size_t workspace_bytes, int32_t* err, int64_t batch,
                                     int64_t nodes, int64_t heads, void* stream) {
  using namespace dsr;
  clear_error();
  PoolAddr pa;
  int rc = paged_addr(&pa, block_table, table_stride, pool_blocks, "prefix_mla_decode");
  if (rc != DSR_OK) return rc;
  DSR_REQUIRE(q && kv_pool && context && cu_nodes && tree_mask && prefix && holder && out && workspace && err,
              "prefix_mla_decode: null pointer");
  const bool zero_unused = (out_dtype & DSR_ZERO_UNUSED) != 0;
  out_dtype &= ~DSR_ZERO_UNUSED;
  DSR_REQUIRE((q_dtype == DSR_BF16 || q_dtype == DSR_F32) && (out_dtype == DSR_BF16 || out_dtype == DSR_F32),
              "prefix_mla_decode: unknown element type");
  DSR_REQUIRE(heads == 16 || heads == 32 || heads == 64 || heads == 128,
              "prefix_mla_decode: heads %lld not in {16,32,64,128}", (long long)heads);
  DSR_REQUIRE(max_nodes > 0 && max_nodes <= 64, "prefix_mla_decode: max nodes %lld outside [1, 64]",
              (long long)max_nodes);
  DSR_REQUIRE(batch > 0 && batch <= kPrefixMaxBatch, "prefix_mla_decode: batch %lld outside [1, %d]",
              (long long)batch, kPrefixMaxBatch);
  DSR_REQUIRE(table_rows >= batch && table_rows < (int64_t(1) << 31),
              "prefix_mla_decode: %lld table rows for a batch of %lld", (long long)table_rows, (long long)batch);
  DSR_REQUIRE(nodes > 0 && nodes * heads <= (int64_t(1) << 24), "prefix_mla_decode: %lld nodes of %lld heads above 2^24",
              (long long)nodes, (long long)heads);
  DSR_REQUIRE(isfinite(scale) && scale > 0.f, "invalid attention scale");
  DSR_REQUIRE(aligned16(q) && aligned16(kv_pool) && aligned16(out),
              "prefix_mla_decode: q, kv_pool and out must be 16-byte aligned");
  DSR_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255u) == 0,
              "prefix_mla_decode: workspace must be 256-byte aligned");
  const size_t need = dsr_prefix_mla_workspace_bytes(batch, nodes, heads);
  DSR_REQUIRE(workspace_bytes >= need, "prefix_mla_decode: workspace %zu < %zu bytes", workspace_bytes, need);
  const PrefixSizes sizes = prefix_sizes(batch, nodes, heads);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  PrefixArgs a = {};
  a.stride = table_stride;
  a.table_rows = table_rows;
  a.context = context;
  a.cu_nodes = cu_nodes;
  a.prefix = prefix;
  a.holder = holder;
  a.sink = sink;
  a.out = out;
  a.out_wide = out_dtype == DSR_F32;
  a.zero_unused = zero_unused;
  a.lse = lse;
  a.err = err;
  a.head = reinterpret_cast<int32_t*>(ws);
  a.requests = reinterpret_cast<PrefixRequest*>(ws + 256);
  uint8_t* at = ws + 256 + sizes.requests;
  auto take = [&](auto*& p, size_t bytes) {
    p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(at);
    at += bytes;
  };
  take(a.items, sizes.items);
  take(a.groups, sizes.groups);
  take(a.segments, sizes.segments);
  take(a.owner, sizes.owner);
  take(a.records, sizes.records);
  a.jobs = reinterpret_cast<TreeJob*>(at);
  a.part_o = reinterpret_cast<float*>(at + sizes.jobs);
  a.part_m = a.part_o + sizes.parts * DSR_V_DIM;
  a.part_l = a.part_m + sizes.parts;
  a.nodes = nodes;
  a.batch = int(batch);
  a.heads = int(heads);
  a.max_nodes = int(max_nodes);
  a.ctas = tree_ctas();
  a.rows = sizes.rows;
  a.pairs = sizes.pairs;
  a.own_part = int32_t(sizes.own_part);
  const size_t smem = size_t(batch + 1) * sizeof(int32_t);
  if (batch <= kFewBatch) {
    prefix_plan_few_kernel<<<1, kFewThreads, 0, as_stream(stream)>>>(a);
  } else if (batch <= kPlanCached) {
    prefix_plan_kernel<256, true><<<1, 256, smem, as_stream(stream)>>>(a);
  } else {
    rc = set_max_smem(prefix_plan_kernel<1024, false>, size_t(kPrefixMaxBatch + 1) * sizeof(int32_t),
                      "prefix_mla_decode");
    if (rc != DSR_OK) return rc;
    prefix_plan_kernel<1024, false><<<1, 1024, smem, as_stream(stream)>>>(a);
  }
  rc = launch_status("prefix_mla_decode launch");
  if (rc != DSR_OK) return rc;
  const float scale_log2 = scale * kTreeLog2e;
  if (a.pairs > 0) {
    rc = launch_pairs(PairArgs{q, q_dtype == DSR_F32, block_table, table_stride, pa.rows, tree_mask, scale_log2,
                               a.part_o, a.part_m, a.part_l, a.head, a.items, a.groups, a.segments, err,
                               a.batch, a.heads, a.pairs, cu_nodes,
                               a.requests, a.records, int32_t(nodes)},
                      kv_pool, nodes * heads, as_stream(stream));
  } else {
    rc = launch_tree_listed(TreeListedCall{q, q_dtype, kv_pool, pa.rows, block_table, table_stride, tree_mask, scale_log2,
                                           nodes, a.heads, a.rows, TreeListed{a.jobs, a.head}, a.part_o, a.part_m,
                                           a.part_l, err},
                            as_stream(stream));
  }
  if (rc != DSR_OK) return rc;
  // The list's few rows and many parts: a column and every fourth part a thread.  The pairs':
  // with a CTA a SM at most, a part is a large share of a row's too, two columns and every fourth
  // part a thread (128 rows of 75 parts: 66 to 42 us in all, 448 rows 75 to 62, 384 rows of three
  // parts 24 to 25.5).  Else a CTA has all columns of its rows (2048 rows: 105 us, 113 the other
  // way); with up to eight CTAs a SM it is bound by latency, and more parts at once pay (2576
  // rows: 14 to 11 us), with more it is not (8192 rows: 17 and 22 us)
  const int64_t quads = nodes * heads / 4;
  auto launch_join = [&](auto* join, int columns, int split) {
    return launch_after(join, dim3(unsigned(quads), DSR_V_DIM / (kJoinThreads * columns)), kJoinThreads * split, 0,
                        as_stream(stream), "prefix_mla_decode join", a);
  };
  return a.pairs == 0              ? launch_join(prefix_join_kernel<false, 1, 4, 8>, 1, 4)
         : quads <= sm_count()     ? launch_join(prefix_join_kernel<true, 2, 4, 4>, 2, 4)
         : quads <= 8 * sm_count() ? launch_join(prefix_join_kernel<true, 4, 1, 4>, 4, 1)
                                   : launch_join(prefix_join_kernel<true, 4, 1, 2>, 4, 1);
}
