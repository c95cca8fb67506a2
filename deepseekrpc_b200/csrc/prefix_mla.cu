// MLA attention of a batch whose requests continue common prompts (sm_100a): what
// tree_mla.cu computes, with the rows that consecutive requests share read and multiplied
// once for all of them.
//
//   request b attends over positions p < S_b = 64 floor(prefix_b / 64) through table row
//   holder_b and over S_b <= p through its own; requests in a row with the same holder and
//   S form a run, whose (node, head) pairs R are one matrix:
//     S^T = K Q^T,  P = e^{s - m},  O = P V  over the S shared rows, for all R at once,
//   and each request's own rows as there.  Every part leaves (m, l, O) in FP32; a row's
//   parts are joined with its sink:
//     out = sum_p 2^{m_p - M} O_p / (2^{sink - M} + sum_p 2^{m_p - M} l_p).
//
// Three launches without a host read: the plan of the jobs (one CTA), the attention over
// them, the join.
#include "common.cuh"
#include "host_common.h"
#include "tree_jobs.cuh"

namespace dsr {
namespace {

constexpr int kPrefixMaxBatch = 16384;
constexpr int kPrefixTileBlocks = 2;  // 128-key tiles of 64-row blocks
constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = 4;
static_assert(DSR_BLOCK_TOKENS == 64, "64-row blocks");

// What the join has to know of a request: its query rows, where its own parts are, and
// where those of its run.
struct alignas(16) PrefixRequest {
  int32_t node0, nodes;
  int32_t own_part, own_segments;              // its rows' parts: own_part + segment * rows
  int32_t run_part, run_rows, run_segments;    // its run's: run_part + segment * run_rows
  int32_t run_node0;
};
static_assert(sizeof(PrefixRequest) == 32, "two 16-byte words");

struct PrefixArgs {
  const int32_t* table;
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
  int32_t* head;  // {jobs, 1 when no request was refused}
  PrefixRequest* requests;
  int32_t* places;  // the plan's own
  TreeJob* jobs;
  float *part_o, *part_m, *part_l;
  int64_t nodes;
  int batch, heads, max_nodes, ctas;
  int rows;  // of a job's group
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
__device__ __forceinline__ bool prefix_starts(const PrefixArgs& a, int b) {
  if (b == 0) return true;
  const PrefixSeq s = prefix_seq(a, b), t = prefix_seq(a, b - 1);
  return !s.ok || !t.ok || s.shared != t.shared || s.holder != t.holder;
}

// ---- an item of the plan: a run's shared rows (items 0 .. runs - 1), then a request's own
struct PrefixItem {
  int32_t table, block0, node0, rows, drafts, context;
  int32_t tiles, groups;
};
__device__ __forceinline__ PrefixItem own_item(const PrefixArgs& a, int b) {
  const PrefixSeq s = prefix_seq(a, b);
  PrefixItem it{b, s.shared, s.node0, s.nodes * a.heads, s.nodes, s.context, 0, 0};
  const int32_t keys = s.context + s.nodes - s.shared * DSR_BLOCK_TOKENS;
  if (s.nodes > 0 && keys > 0) {
    it.tiles = (keys + 127) / 128;
    it.groups = (it.rows + a.rows - 1) / a.rows;
  }
  return it;
}
__device__ __forceinline__ PrefixItem run_item(const PrefixArgs& a, int b0, int b1) {
  const PrefixSeq s = prefix_seq(a, b0);
  PrefixItem it{s.holder, 0, s.node0, 0, 0, s.shared * DSR_BLOCK_TOKENS, 0, 0};
  if (!s.ok || s.shared == 0) return it;
  it.rows = (a.cu_nodes[b1] - s.node0) * a.heads;
  if (it.rows == 0) return it;
  it.tiles = (s.shared + kPrefixTileBlocks - 1) / kPrefixTileBlocks;
  it.groups = (it.rows + a.rows - 1) / a.rows;
  return it;
}

struct PlanPair {
  int64_t x, y;
};
__device__ __forceinline__ PlanPair operator+(const PlanPair& a, const PlanPair& b) {
  return PlanPair{a.x + b.x, a.y + b.y};
}
// Exclusive sums over the CTA's threads; `all` the totals.
__device__ __forceinline__ PlanPair plan_scan(const PlanPair& mine, PlanPair* part, PlanPair& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  PlanPair run = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const PlanPair up{__shfl_up_sync(~0u, run.x, d), __shfl_up_sync(~0u, run.y, d)};
    if (lane >= d) run = run + up;
  }
  if (lane == 31) part[warp] = run;
  __syncthreads();
  PlanPair before{0, 0};
  all = PlanPair{0, 0};
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w < warp) before = before + part[w];
    all = all + part[w];
  }
  __syncthreads();
  return PlanPair{before.x + run.x - mine.x, before.y + run.y - mine.y};
}

// Lays the jobs out.  An item's tiles are cut into segments of at most `length` tiles:
// one tile each when all units (group x tile) fit the grid, else the best of a few lengths by
// the time that the busiest CTA takes.
__global__ void __launch_bounds__(kPlanThreads, 1) prefix_plan_kernel(const __grid_constant__ PrefixArgs a) {
  extern __shared__ int32_t plan_smem[];
  int32_t* starts = plan_smem;               // [batch + 1] first request of each run
  int32_t* cu_jobs = starts + a.batch + 1;   // [2 batch + 1] jobs before each item
  int32_t* parts = a.places;                 // [2 batch] where its partials are
  __shared__ PlanPair part[kPlanThreads / 32];
  __shared__ unsigned long long counted[kPlanWaves];
  __shared__ int longest;
  const int tid = threadIdx.x;
  const int per = (a.batch + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
  if (tid < kPlanWaves) counted[tid] = 0;
  if (tid == 0) longest = 0;
  // ---- the runs
  int first = 0;
  bool fine = true;
  for (int b = b0; b < b1; ++b) {
    first += prefix_starts(a, b);
    if (!prefix_seq(a, b).ok) {
      fine = false;
      flag(a.err, DSR_ERR_ID);
    }
  }
  fine = __syncthreads_and(fine);
  PlanPair all;
  const int run0 = int(plan_scan(PlanPair{first, 0}, part, all).x), runs = int(all.x);
  for (int b = b0, r = run0; b < b1; ++b)
    if (prefix_starts(a, b)) starts[r++] = b;
  if (tid == 0) starts[runs] = a.batch;
  __syncthreads();
  // ---- units and groups of all items
  const int items = runs + a.batch;
  auto item = [&](int i) { return i < runs ? run_item(a, starts[i], starts[i + 1]) : own_item(a, i - runs); };
  const int per_item = (items + kPlanThreads - 1) / kPlanThreads;
  const int i0 = min(tid * per_item, items), i1 = min(i0 + per_item, items);
  PlanPair mine{0, 0};
  int most = 0;
  for (int i = i0; i < i1; ++i) {
    const PrefixItem it = item(i);
    mine = mine + PlanPair{int64_t(it.groups) * it.tiles, it.groups > 0 ? it.rows : 0};
    most = max(most, it.tiles);
  }
  atomicMax(&longest, most);
  plan_scan(mine, part, all);
  const int64_t units = all.x;
  if (all.y > 2 * a.nodes * a.heads) {
    // sums in disorder that give rows to several requests, more than there are partials for
    if (tid == 0) a.head[0] = 0, a.head[1] = 1;
    for (int b = b0; b < b1; ++b) a.requests[b] = PrefixRequest{0, 0, 0, 0, 0, 0, 0, 0};
    return;
  }
  auto segments = [](int32_t tiles, int32_t length) { return (tiles + length - 1) / length; };
  int32_t length = 1;
  if (units > a.ctas) {
    int32_t tried[kPlanWaves];
    int64_t jobs[kPlanWaves] = {};
    for (int w = 0; w < kPlanWaves; ++w) {
      const int64_t room = int64_t(w + 1) * a.ctas, share = (units + room - 1) / room;
      tried[w] = int32_t(min(share, int64_t(1) << 24));  // no item has more tiles
    }
    for (int i = i0; i < i1; ++i) {
      const PrefixItem it = item(i);
      for (int w = 0; w < kPlanWaves; ++w) jobs[w] += int64_t(it.groups) * segments(it.tiles, tried[w]);
    }
    for (int w = 0; w < kPlanWaves; ++w)
      if (jobs[w] > 0) atomicAdd(counted + w, (unsigned long long)jobs[w]);
    __syncthreads();
    float best = CUDART_INF_F;
    for (int w = 0; w < kPlanWaves; ++w) {
      // a job costs some 8 tiles beside its own: first copies, output, its part of the join
      const float rounds = ceilf(float(counted[w]) / float(a.ctas));
      const float time = rounds * (float(min(tried[w], longest)) + 8.f);
      if (time < best) best = time, length = tried[w];
    }
  }
  // ---- jobs and partials before each item
  mine = PlanPair{0, 0};
  for (int i = i0; i < i1; ++i) {
    const PrefixItem it = item(i);
    const int32_t n = segments(it.tiles, length);
    mine = mine + PlanPair{int64_t(it.groups) * n, int64_t(it.rows) * n};
  }
  PlanPair at = plan_scan(mine, part, all);
  for (int i = i0; i < i1; ++i) {
    const PrefixItem it = item(i);
    const int32_t n = segments(it.tiles, length);
    cu_jobs[i] = int32_t(at.x);
    parts[i] = int32_t(at.y);
    at = at + PlanPair{int64_t(it.groups) * n, int64_t(it.rows) * n};
  }
  if (tid == 0) cu_jobs[items] = int32_t(all.x);
  const int32_t jobs = int32_t(all.x);
  if (tid == 0) a.head[0] = jobs, a.head[1] = fine;
  __syncthreads();
  // ---- the requests' records
  for (int b = b0, r = run0 - 1; b < b1; ++b) {
    if (r + 1 < runs && starts[r + 1] == b) ++r;
    const PrefixItem it = own_item(a, b), run = run_item(a, starts[r], starts[r + 1]);
    const PrefixSeq s = prefix_seq(a, b);
    a.requests[b] = PrefixRequest{s.node0, s.nodes, parts[runs + b], segments(it.tiles, length), parts[r], run.rows,
                                  segments(run.tiles, length), run.node0};
  }
  // ---- the jobs: an item's segments one after another, the groups of one side by side
  for (int32_t j = tid; j < jobs; j += kPlanThreads) {
    int lo = 0, hi = items;  // cu_jobs[lo] <= j < cu_jobs[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cu_jobs[mid] <= j) lo = mid;
      else hi = mid;
    }
    const PrefixItem it = item(lo);
    const int32_t n = segments(it.tiles, length), in = j - cu_jobs[lo];
    const int32_t segment = in / it.groups, group = in - segment * it.groups;
    const int32_t whole = it.tiles / n, longer = it.tiles - whole * n, row0 = group * a.rows;
    a.jobs[j] = TreeJob{it.table, it.block0, it.node0, row0, min(a.rows, it.rows - row0), it.drafts, it.context,
                        segment * whole + min(segment, longer), whole + (segment < longer),
                        parts[lo] + segment * it.rows + row0, {}};
  }
}

// ---------------------------------------------------------------------------
// Joins the parts of a row: one CTA per four query rows (of one node, since heads come in
// sixteens) and 128 value columns, a thread one column of all four.
// ---------------------------------------------------------------------------
constexpr int kJoinThreads = 128, kJoinBatch = 8;  // kJoinBatch: parts requested together
constexpr int kJoinMaxParts = kPlanWaves * kTreeMaxCtas + 16;

__global__ void __launch_bounds__(kJoinThreads) prefix_join_kernel(const __grid_constant__ PrefixArgs a) {
  __shared__ float weight[4][kJoinMaxParts];
  __shared__ float inverse[4];
  __shared__ int owner;
  const int64_t row = int64_t(blockIdx.x) * 4;
  const int32_t node = int32_t(row / a.heads);
  const int tid = threadIdx.x, d = blockIdx.y * kJoinThreads + tid;
  // the request of the node: the largest b with cu_nodes[b] <= node, 32 ways a step
  int lo = 0;
  for (int n = a.batch; n > 1;) {
    const int stride = (n + 31) / 32, at = (tid & 31) * stride;
    const unsigned below = __ballot_sync(~0u, at < n && a.cu_nodes[lo + at] <= node);
    const int last = below == 0 ? 0 : (31 - __clz(below)) * stride;
    lo += last;
    n = min(stride, n - last);
  }
  pdl_wait();  // before any CTA leaves: the join must not end ahead of the attention
  auto record = [&](int b) {
    const int4* words = reinterpret_cast<const int4*>(a.requests + b);
    const int4 x = __ldcg(words), y = __ldcg(words + 1);
    return PrefixRequest{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
  };
  PrefixRequest s = record(lo);
  if (node < s.node0 || node >= s.node0 + s.nodes) {
    // a padding row.  Where a request was refused the sums may be in disorder and the search
    // may have missed the request that has the row: every one is asked
    lo = -1;
    if (!__ldcg(a.head + 1)) {
      if (tid == 0) owner = -1;
      __syncthreads();
      for (int b = tid; b < a.batch; b += kJoinThreads) {
        const PrefixRequest other = record(b);
        if (node >= other.node0 && node < other.node0 + other.nodes) atomicMax(&owner, b);
      }
      __syncthreads();
      lo = owner;
    }
    if (lo < 0) {
      if (!a.zero_unused) return;
      for (int y = 0; y < 4; ++y) {
        const int64_t at = (row + y) * DSR_V_DIM + d;
        if (a.out_wide) static_cast<float*>(a.out)[at] = 0.f;
        else static_cast<uint16_t*>(a.out)[at] = 0;
      }
      if (a.lse != nullptr && blockIdx.y == 0 && tid < 4) a.lse[row + tid] = -CUDART_INF_F;
      return;
    }
    s = record(lo);
  }
  const int32_t own_rows = s.nodes * a.heads;
  const int64_t own0 = s.own_part + row - int64_t(s.node0) * a.heads;
  const int64_t run0 = s.run_part + row - int64_t(s.run_node0) * a.heads;
  const int own = s.own_segments, parts = own + s.run_segments;
  auto place = [&](int p) { return p < own ? own0 + int64_t(p) * own_rows : run0 + int64_t(p - own) * s.run_rows; };
  float4 v[kJoinBatch];
  auto request = [&](int p0) {
#pragma unroll
    for (int j = 0; j < kJoinBatch; ++j)
      if (p0 + j < parts) v[j] = __ldcg(reinterpret_cast<const float4*>(a.part_o + place(p0 + j) * DSR_V_DIM) + d);
  };
  request(0);
  {
    const int w = tid >> 5, lane = tid & 31;  // one warp per row
    const float m0 = lane < parts ? __ldcg(a.part_m + place(lane) + w) : -CUDART_INF_F;
    const float l0 = lane < parts ? __ldcg(a.part_l + place(lane) + w) : 0.f;
    float top = m0, sum = 0.f;
    for (int p = lane + 32; p < parts; p += 32) top = fmaxf(top, __ldcg(a.part_m + place(p) + w));
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    const float base = top == -CUDART_INF_F ? 0.f : top;
    for (int p = lane; p < parts; p += 32) {
      const float e = ex2((p < 32 ? m0 : __ldcg(a.part_m + place(p) + w)) - base);
      weight[w][p] = e;
      sum += e * (p < 32 ? l0 : __ldcg(a.part_l + place(p) + w));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (lane == 0) {
      float total;
      const float lse = tree_total(a.sink, a.err, int((row + w) % a.heads), top, sum, total);
      inverse[w] = total > 0.f ? 1.f / total : 0.f;
      if (a.lse != nullptr && blockIdx.y == 0) a.lse[row + w] = lse;
    }
  }
  __syncthreads();
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p0 = 0; p0 < parts; p0 += kJoinBatch) {
    if (p0 > 0) request(p0);
#pragma unroll
    for (int j = 0; j < kJoinBatch; ++j)
      if (p0 + j < parts) {
        acc.x = fmaf(weight[0][p0 + j], v[j].x, acc.x), acc.y = fmaf(weight[1][p0 + j], v[j].y, acc.y);
        acc.z = fmaf(weight[2][p0 + j], v[j].z, acc.z), acc.w = fmaf(weight[3][p0 + j], v[j].w, acc.w);
      }
  }
  const float out[4] = {acc.x * inverse[0], acc.y * inverse[1], acc.z * inverse[2], acc.w * inverse[3]};
#pragma unroll
  for (int y = 0; y < 4; ++y) {
    if (!isfinite(out[y])) flag(a.err, DSR_ERR_NONFINITE);
    const int64_t at = (row + y) * DSR_V_DIM + d;
    if (a.out_wide) static_cast<float*>(a.out)[at] = out[y];
    else static_cast<uint16_t*>(a.out)[at] = __bfloat16_as_ushort(__float2bfloat16_rn(out[y]));
  }
}

// ---- scratch: {jobs, fine}, the requests' records, the jobs, the partials
size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }

struct PrefixSizes {
  int rows;
  size_t requests, places, jobs, parts;  // bytes, and rows
};
PrefixSizes prefix_sizes(int64_t batch, int64_t nodes, int64_t heads, int64_t max_nodes) {
  PrefixSizes s;
  s.rows = tree_rows(heads, max_nodes);
  // a segment or more per group: a cut adds at most kPlanWaves jobs a CTA, and an item's
  // last group may be short of rows
  const size_t groups = 2 * (size_t(nodes) * heads / s.rows + size_t(batch)), cut = size_t(kPlanWaves) * tree_ctas();
  s.requests = rounded(size_t(batch) * sizeof(PrefixRequest));
  s.places = rounded(size_t(batch) * 2 * sizeof(int32_t));
  s.jobs = rounded((groups + cut) * sizeof(TreeJob));
  s.parts = 2 * size_t(nodes) * heads + cut * s.rows;
  return s;
}

size_t plan_smem_bytes(int64_t batch) { return (size_t(batch) * 3 + 2) * sizeof(int32_t); }

}  // namespace
}  // namespace dsr

extern "C" size_t dsr_prefix_mla_workspace_bytes(int64_t batch, int64_t nodes, int64_t heads, int64_t max_nodes) {
  using namespace dsr;
  if (batch <= 0 || nodes <= 0 || heads <= 0 || max_nodes <= 0) return 0;
  const PrefixSizes s = prefix_sizes(batch, nodes, heads, max_nodes);
  return 256 + s.requests + s.places + s.jobs + s.parts * (DSR_V_DIM + 2) * 4;
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
  const size_t need = dsr_prefix_mla_workspace_bytes(batch, nodes, heads, max_nodes);
  DSR_REQUIRE(workspace_bytes >= need, "prefix_mla_decode: workspace %zu < %zu bytes", workspace_bytes, need);
  const PrefixSizes sizes = prefix_sizes(batch, nodes, heads, max_nodes);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  PrefixArgs a = {};
  a.table = block_table;
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
  a.places = reinterpret_cast<int32_t*>(ws + 256 + sizes.requests);
  a.jobs = reinterpret_cast<TreeJob*>(ws + 256 + sizes.requests + sizes.places);
  a.part_o = reinterpret_cast<float*>(ws + 256 + sizes.requests + sizes.places + sizes.jobs);
  a.part_m = a.part_o + sizes.parts * DSR_V_DIM;
  a.part_l = a.part_m + sizes.parts;
  a.nodes = nodes;
  a.batch = int(batch);
  a.heads = int(heads);
  a.max_nodes = int(max_nodes);
  a.ctas = tree_ctas();
  a.rows = sizes.rows;
  rc = set_max_smem(prefix_plan_kernel, plan_smem_bytes(kPrefixMaxBatch), "prefix_mla_decode");
  if (rc != DSR_OK) return rc;
  prefix_plan_kernel<<<1, kPlanThreads, plan_smem_bytes(batch), as_stream(stream)>>>(a);
  rc = launch_status("prefix_mla_decode launch");
  if (rc != DSR_OK) return rc;
  TreeListedCall call = {};
  call.q = q;
  call.q_dtype = q_dtype;
  call.kv_pool = kv_pool;
  call.pool_rows = pa.rows;
  call.table = block_table;
  call.stride = table_stride;
  call.masks = tree_mask;
  call.scale_log2 = scale * kTreeLog2e;
  call.nodes = nodes;
  call.heads = int(heads);
  call.rows = sizes.rows;
  call.list = TreeListed{a.jobs, a.head, true};
  call.part_o = a.part_o;
  call.part_m = a.part_m;
  call.part_l = a.part_l;
  call.err = err;
  rc = launch_tree_listed(call, as_stream(stream));
  if (rc != DSR_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(nodes * heads / 4), DSR_V_DIM / kJoinThreads, 1);
  cfg.blockDim = dim3(kJoinThreads, 1, 1);
  cfg.stream = as_stream(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, prefix_join_kernel, a);
  if (e != cudaSuccess) return fail(DSR_ECUDA, "prefix_mla_decode join launch: %s", cudaGetErrorString(e));
  return DSR_OK;
}
