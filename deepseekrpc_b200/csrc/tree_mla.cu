// MLA attention of drafted tokens over a paged BF16 cache (sm_100a): every node of
// a request's draft tree attends over all cached rows of the request and over the
// drafted rows that its mask names (its branch).
//
//   out[n,h] = sum_j seen(n,j) e^{s_j} v_j / (e^{sink_h} + sum_j seen(n,j) e^{s_j}),
//   s_j = scale q[n,h].k_j,  v_j = the leading 512 columns of the 576-wide row k_j,
//   seen(n,j) = j < context, or bit (j - context) of node n's mask.
//
// The (node, head) pairs of a request are its query rows, N of which (16, 32 or 64)
// form a group.  A work unit is one group x one 128-key tile, as two products:
//   S^T[key, row] = K[key, :576] Q[row, :576]   (M = 128 keys, N rows)
//   O^T[dim, row] += V[key, dim] P[row, key]    (M = 128 dims x 4, N rows)
// so that the key tile, once in shared memory, is the A operand of both (K-major,
// then MN-major) and O^T of 64 rows takes half of the tensor memory.
//
// A job is one group over a segment of consecutive tiles.  Every CTA finds the same
// segment length from the lengths on the device (tree_length, a search; more than
// kTreeSearchBatch requests take an even share); a request's tiles are cut into equal
// segments, and the jobs, in the order (request, segment, group), are dealt to the CTAs
// to and fro: the groups of a segment run side by side and share its rows in L2, and a
// CTA with a long job gets a short one next.  Up to 32 requests go with the longest
// segments first (ragged ones: the busiest CTA has 4 to 6% more than its share in two
// rounds; dealt in the order of requests it had 14% in four), more in their own order
// (counted for ragged requests of 8192 to 65536 rows: 20% for 33, 37% for 128).  (Runs of
// units in the order request, group, tile balance better, but read the rows once per
// group: 1213 us against 1010 us for 32 requests of 3 to 6 groups.)  A group of several
// segments leaves partials (m, l, unnormalised O in FP32) that tree_combine_kernel joins.
//
//   warps 0..7  (FP32 query -> shared memory,) softmax over the tile's keys (running
//               maximum; O is rescaled only when a maximum grows by more than 2^8),
//               output.  Warps 0..3 have the first half of the group's rows, warps
//               4..7 the second; warp w and w + 4 hold the tensor memory's lanes
//               (keys, value columns) 32 w and up
//   warp 8      TMEM and the MMAs
//   warp 9      query and key tiles by TMA: column blocks 0..7 (the value columns) through a
//               ring of block pairs that the O MMA frees pair by pair, block 8 (the
//               rotary columns) in a buffer that P^T takes over once S^T is done
//
// Bound at 64 rows by two things of about equal weight.  An MMA of 128 x 64 x 16 takes 48
// cycles, not 32, to read its operands from shared memory: the 68 of a tile 3264 cycles.  And
// a tile takes nearly 6000: there is one S^T, and the ring holds one tile, so that the MMAs
// wait through every softmax.  Measured: 8 nodes of 64 heads over 131072 rows 186 to 194 us
// (750 to 785 TFLOP/s, 46 to 48% of a measured BF16 GEMM), FP32 queries cost no more; 32
// requests of 6 nodes over up to 65536 rows 0.91 to 1.03 ms (0.72 to 0.82 PFLOP/s), 33 of them
// 1.11 ms, 64 2.07, 128 5.06.  Bound by memory at 16 rows: 32 requests of one node and 16 heads
// over 65536 rows 378 to 406 us from box to box, 6.0 to 6.4 TB/s, 91 to 97% of a plain copy.
// Bound by latency for little: one node over 4096 rows 16.4 to 18.4 us in two launches.
#include <type_traits>

#include "common.cuh"
#include "host_common.h"
#include "tree_jobs.cuh"

namespace dsr {
namespace {

constexpr int kTreeSoftmax = 256;  // warps 0..7
constexpr int kTreeThreads = kTreeSoftmax + 64;
constexpr int kTreeKeys = 128;
constexpr int kTreeD = DSR_KV_DIM, kTreeDv = DSR_V_DIM;
constexpr int kTreeMaxNodes = 64;
constexpr float kTreeSlack = 8.f;  // log2 units a row's maximum may lag behind

template <int N>
struct TreeLayout {
  static constexpr int kPairs = N == 64 ? 4 : 5;        // ring of 32 KB block pairs
  static constexpr int kRingOff = 0;
  static constexpr int kROff = kPairs * 32768;          // rotary block, then P^T
  static constexpr int kQOff = kROff + 16384;           // 9 x N x 128 B
  static constexpr int kBarOff = kQOff + 9 * N * 128;
  static constexpr int kBars = 2 * kPairs + 6;
  static constexpr int kMaskOff = kBarOff + kBars * 8;  // u64[2][N + 1] seen-masks of the rows, their union, per half
  static constexpr int kRedOff = kMaskOff + 2 * (N + 1) * 8;  // f32[4][N] per-warp maxima, then sums
  static constexpr int kStatOff = (kRedOff + 4 * N * 4 + 15) / 16 * 16;  // f32[N] factors / reciprocals
  static constexpr int kChunkOff = kStatOff + N * 4;    // i32[2][kTreeThreads]
  static constexpr int kMiscOff = kChunkOff + 2 * kTreeThreads * 4;
  static constexpr int kScratchOff = kMiscOff + 64;     // the schedule's sums, see tree_mla_kernel
  static constexpr int kBytes = kScratchOff + 2 * (kTreeThreads / 32) * 8 + 2 * 4 * 4;
  static constexpr int kAlloc = kBytes + 1024;
  static constexpr uint32_t kTmemCols = N == 64 ? 512 : (N == 32 ? 256 : 128);  // >= 5 N
  static_assert(2 * N * 128 <= 16384, "P^T fits the rotary block's buffer");
  static_assert(kAlloc <= 232448, "shared memory of one CTA");
  // ordinary accesses and TMA's are not ordered by a barrier alone
  static_assert(kScratchOff >= kQOff + 9 * N * 128 && kScratchOff % 8 == 0, "the scratch is no place that TMA writes");
};

struct TreeArgs {
  const void* q;
  bool q_wide, out_wide;  // fp32 (else bf16)
  bool zero_unused;       // rows of no request: zeros (else left)
  const int32_t* table;
  int64_t stride, pool_rows;
  const int32_t* context;
  const int32_t* cu_nodes;
  const int64_t* masks;
  const float* sink;  // nullable
  float scale_log2;
  void* out;
  float* lse;  // nullable
  int32_t* err;
  int32_t* slot_start;  // [batch + 1] first partial slot of each request; the segment length (negative: a request was refused)
  float* part_o;        // [slots][N / 4][512][4]: value columns of four rows side by side
  float* part_m;        // [slots][N]
  float* part_l;
  int64_t nodes;
  int batch, heads, max_nodes, ctas;
  TreeListed list;  // of a Listed kernel, in place of what its jobs follow from
};

// ---- the work of request b
struct TreeSeq {
  int32_t node0, nodes, context, tiles, groups;
  bool ok;
};
template <int N>
__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs& a, int b) {
  const int32_t n0 = a.cu_nodes[b], n1 = a.cu_nodes[b + 1], ctx = a.context[b];
  TreeSeq s{n0, 0, ctx, 0, 0, true};
  if (n0 < 0 || n1 < n0 || n1 > a.nodes || n1 - n0 > a.max_nodes || ctx < 0 ||
      int64_t(ctx) + (n1 - n0) > a.stride * DSR_BLOCK_TOKENS) {
    s.ok = false;
    s.node0 = s.context = 0;
    return s;
  }
  s.nodes = n1 - n0;
  s.tiles = int32_t((int64_t(ctx) + s.nodes + kTreeKeys - 1) / kTreeKeys);
  s.groups = (s.nodes * a.heads + N - 1) / N;
  if (s.nodes == 0) s.tiles = 0;
  return s;
}

__device__ __forceinline__ int32_t tree_segments(const TreeSeq& s, int32_t length) {
  return (s.tiles + length - 1) / length;
}

// ---- the jobs of a call
// Requests of a search at most.  It reads every request several times, and many requests
// share evenly without it.  Its time over the even share's, mean (and range) over contexts of
// 500 to 32000 rows and 1 to 4 nodes of 16 to 128 heads: 96 requests 0.93 (0.76 to 1.15), 128
// 0.94 (0.79 to 1.06), 160 0.96 (0.80 to 1.03), 200 1.00 (0.92 to 1.10), 300 1.02 (0.86 to 1.10)
constexpr int kTreeSearchBatch = 160;
constexpr int kTreeSlotsPerCta = 4;  // partial slots, per CTA of the grid
// A round's cost beside its tiles, in tiles: first copies, output, its part of the join.
constexpr float kTreeJobCost = 8.f;

// A segment length for `waves` jobs per CTA at most: starts at the even share and
// grows until the jobs (requests' tiles rounded up to whole segments) and the partial
// slots fit.  One warp (`own`: of up to 32 requests, lane b's is request b); estimates the
// time in tiles (infinite when none was found).
template <int N>
__device__ __forceinline__ float tree_length(const TreeArgs& a, const TreeSeq& own, int64_t units, int waves,
                                             int32_t& length) {
  const int64_t room = int64_t(waves) * a.ctas;
  float len = fmaxf(ceilf(float(units) / float(room)), 1.f);
  for (int tries = 0; tries < 8; ++tries) {
    length = int32_t(len);
    int32_t jobs = 0, slots = 0;
    for (int b = threadIdx.x & 31; b < a.batch; b += 32) {
      const TreeSeq s = a.batch <= 32 ? own : tree_seq<N>(a, b);
      const int32_t n = s.groups * tree_segments(s, length);
      jobs += n;
      if (s.tiles > length) slots += n;
    }
    jobs = __reduce_add_sync(~0u, jobs);
    slots = __reduce_add_sync(~0u, slots);
    if (jobs <= room && slots <= int64_t(kTreeSlotsPerCta) * a.ctas) {
      // one round lasts as long as its longest job; several come near the mean
      const float mean = float(units) / float(a.ctas);
      return (waves == 1 ? len : fminf(float(waves) * len, mean + 0.1f * len)) + float(waves) * kTreeJobCost;
    }
    len += fmaxf(floorf(len * (1.f - float(room) / float(jobs))), 1.f);
  }
  return CUDART_INF_F;
}

// ---- a CTA's jobs, one after another (every warp walks them for itself)
// Up to 32 requests: what they are, the jobs and slots before each, in shared memory.
struct TreeEntry {
  TreeSeq s;
  int32_t jobs, count, slots;
};
template <int N>
struct TreeWalk {
  const TreeArgs& a;
  const TreeEntry* entries;                 // [batch <= 32]
  const int32_t *chunk_jobs, *chunk_slots;  // else: [kTreeThreads] before each chunk of `per` requests
  int32_t length, jobs;
  int round, per;
  int b, group, tile0, count, slot;  // slot < 0: the group's only segment
  TreeSeq s;
  __device__ __forceinline__ void at_job(int32_t at, int32_t segments, int32_t slots) {
    const int32_t segment = at / s.groups;
    group = at - segment * s.groups;
    const int32_t whole = s.tiles / segments, longer = s.tiles - whole * segments;
    tile0 = segment * whole + min(segment, longer);
    count = whole + (segment < longer);
    slot = segments > 1 ? slots + at : -1;
  }
  __device__ __forceinline__ bool next() {
    // to and fro: odd rounds from the last CTA to the first
    const int32_t job = round * int(gridDim.x) + (round & 1 ? int(gridDim.x) - 1 - int(blockIdx.x) : int(blockIdx.x));
    if (job >= jobs) return false;
    ++round;
    if (a.batch <= 32) {
      const int lane = threadIdx.x & 31;
      bool has = false;
      if (lane < a.batch) {
        const int32_t at = job - entries[lane].jobs;
        has = at >= 0 && at < entries[lane].count;
      }
      b = __ffs(__ballot_sync(~0u, has)) - 1;
      s = entries[b].s;
      at_job(job - entries[b].jobs, tree_segments(s, length), entries[b].slots);
      return true;
    }
    int lo = 0, hi = kTreeThreads;  // the last chunk that starts at or before the job
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (chunk_jobs[mid] <= job) lo = mid;
      else hi = mid;
    }
    int32_t base = chunk_jobs[lo], slots = chunk_slots[lo], segments;
    for (b = lo * per;; ++b) {
      s = tree_seq<N>(a, b);
      segments = tree_segments(s, length);
      const int32_t n = s.groups * segments;
      if (job < base + n) break;
      base += n;
      if (segments > 1) slots += n;
    }
    at_job(job - base, segments, slots);
    return true;
  }
};

// The jobs of a list, dealt like those of a walk.
struct TreeList {
  const TreeJob* jobs;
  int32_t count;
  int round;
  TreeJob job;
  __device__ __forceinline__ bool next() {
    const int at = round * int(gridDim.x) + (round & 1 ? int(gridDim.x) - 1 - int(blockIdx.x) : int(blockIdx.x));
    if (at >= count) return false;
    ++round;
    const int4* words = reinterpret_cast<const int4*>(jobs + at);
    const int4 x = __ldcg(words), y = __ldcg(words + 1), z = __ldcg(words + 2);
    job = TreeJob{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w, z.x, z.y, {}};
    return true;
  }
};

// What the job at hand is, for all warps.
struct TreeWork {
  int32_t table, block0, node0, row0, rows, drafts, context, tile0, count;
  int32_t part;  // first row of its partials
  bool whole;    // or none: the group's only segment
};
template <int N>
__device__ __forceinline__ TreeWork tree_work(const TreeWalk<N>& w) {
  return TreeWork{w.b,       0,           w.s.node0, w.group * N, min(N, w.s.nodes * w.a.heads - w.group * N),
                  w.s.nodes, w.s.context, w.tile0,   w.count,     w.slot * N,
                  w.slot < 0};
}
__device__ __forceinline__ TreeWork tree_work(const TreeList& l) {
  const TreeJob& j = l.job;
  return TreeWork{j.table, j.block0, j.node0, j.row0, j.rows, j.drafts, j.context, j.tile0, j.count, j.part, false};
}

// mbar_wait whose polls sleep in the barrier unit until the phase completes (or a few
// microseconds pass): the ten warps that wait here would otherwise poll shared memory
// all the time, whose bandwidth the MMAs of 64 columns need to the last byte.
__device__ __forceinline__ bool tree_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int32_t* err) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t start = global_ns();
  for (;;) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)
        : "memory");
    if (ok) return true;
    if (*abort) return false;
    if (global_ns() - start > kWaitNs) {
      *abort = 1;
      flag(err, DSR_ERR_TIMEOUT);
      return false;
    }
  }
}

// The same for a whole warp, with one answer for all lanes: a lane may see the phase
// complete while another gives up, and what follows a wait (tcgen05.ld, votes, shuffles) is
// for all lanes or none.
__device__ __forceinline__ bool tree_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort, int32_t* err) {
  return __all_sync(~0u, tree_wait(bar, parity, abort, err));
}

// 16 TMEM lanes x 8 C columns: thread i holds lanes i/4 and i/4 + 8 (of the 16),
// columns 8c + 2(i%4) and the next: r[4c + 2h + e] is lane i/4 + 8h, column + e.
template <int C>
__device__ __forceinline__ void tmem_ld_16x256(uint32_t taddr, uint32_t (&r)[4 * C]) {
  static_assert(C == 1 || C == 2 || C == 4, "");
  if constexpr (C == 1) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(taddr));
  } else if constexpr (C == 2) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
  } else {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
  }
}
// 32 lanes x W columns, thread i lane i
template <int W>
__device__ __forceinline__ void tmem_ld_lanes(uint32_t taddr, uint32_t (&r)[W]) {
  static_assert(W == 8 || W == 16, "");
  if constexpr (W == 16) {
    tmem_ld16(taddr, r);
  } else {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
  }
}
template <int W>
__device__ __forceinline__ void tmem_st_lanes(uint32_t taddr, const uint32_t (&r)[W]) {
  static_assert(W == 8 || W == 16, "");
  if constexpr (W == 16) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
  } else {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
  }
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Four 8x8 b16 matrices (row i/4, columns 2(i%4).. in thread i's register) stored
// transposed: thread i gives the address of row i%8 of the transposed matrix i/8.
__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(r0), "r"(r1),
               "r"(r2), "r"(r3)
               : "memory");
}

__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// The 128 softmax threads of one half: a barrier, and whether every one is fine.
__device__ __forceinline__ bool softmax_sync(int half, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(uint32_t(ok)), "r"(1 + half)
      : "memory");
  return r != 0;
}

// Listed: the jobs are a list that a kernel before this one wrote, and all leave partials.
template <int N, bool Listed>
__global__ void __launch_bounds__(kTreeThreads, 1)
    tree_mla_kernel(const __grid_constant__ CUtensorMap kv_map, const __grid_constant__ CUtensorMap q_map,
                    const __grid_constant__ TreeArgs a) {
  using L = TreeLayout<N>;
  constexpr int kHalf = N / 2, C = kHalf / 8;  // rows of a half of the softmax warps, in chunks of 8
  constexpr int W = kHalf < 16 ? kHalf : 16;   // rows taken from O^T at a time
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_smem_1024(smem_raw);
  const uint32_t sbase = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* full = bars;                    // [kPairs] block pair loaded (TMA bytes + 1)
  uint64_t* empty = bars + L::kPairs;       // [kPairs] block pair read by the O MMA (commit)
  uint64_t* bar_r = bars + 2 * L::kPairs;   // rotary block loaded
  uint64_t* bar_s = bar_r + 1;              // S^T complete (commit)
  uint64_t* bar_p = bar_r + 2;              // P^T written (kTreeSoftmax arrivals)
  uint64_t* bar_o = bar_r + 3;              // the tile's O MMAs complete (commit)
  uint64_t* bar_q = bar_r + 4;              // query in place (TMA bytes + 1; FP32: kTreeSoftmax arrivals)
  uint64_t* bar_free = bar_r + 5;           // O^T read by the epilogue (kTreeSoftmax arrivals)
  float* red = reinterpret_cast<float*>(smem + L::kRedOff);
  float* stat = reinterpret_cast<float*>(smem + L::kStatOff);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMiscOff);
  volatile int* abort = reinterpret_cast<volatile int*>(smem + L::kMiscOff + 4);
  int* loaded = reinterpret_cast<int*>(smem + L::kMiscOff + 8);     // block pairs requested, for an abort
  int* loaded_r = reinterpret_cast<int*>(smem + L::kMiscOff + 12);  // rotary blocks
  int* loaded_q = reinterpret_cast<int*>(smem + L::kMiscOff + 16);  // queries
  int32_t* chunk_jobs = reinterpret_cast<int32_t*>(smem + L::kChunkOff);
  int32_t* chunk_slots = chunk_jobs + kTreeThreads;
  // [10] sums of the warps (units, groups), [4] estimates and lengths
  int64_t* warp_units = reinterpret_cast<int64_t*>(smem + L::kScratchOff);
  int64_t* warp_groups = warp_units + kTreeThreads / 32;
  float* estimate = reinterpret_cast<float*>(warp_groups + kTreeThreads / 32);
  int32_t* estimated = reinterpret_cast<int32_t*>(estimate + 4);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    tma_prefetch_desc(&kv_map);
    if (!a.q_wide) tma_prefetch_desc(&q_map);
    for (int i = 0; i < L::kPairs; ++i) mbar_init(full + i, 1), mbar_init(empty + i, 1);
    mbar_init(bar_r, 1);
    mbar_init(bar_s, 1);
    mbar_init(bar_p, kTreeSoftmax);
    mbar_init(bar_o, 1);
    mbar_init(bar_q, a.q_wide ? kTreeSoftmax : 1);
    mbar_init(bar_free, kTreeSoftmax);
    *abort = 0;
    *loaded = *loaded_r = *loaded_q = 0;
    fence_barrier_init();
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, L::kTmemCols);
    tmem_relinquish();
  }

  // ---- the work of all requests
  if constexpr (Listed) pdl_wait();
  TreeEntry* entries = reinterpret_cast<TreeEntry*>(smem + L::kChunkOff);  // in the chunks' place
  static_assert(32 * sizeof(TreeEntry) <= 2 * kTreeThreads * 4, "");
  auto walk = [&] {
    if constexpr (Listed) return TreeList{a.list.jobs, __ldcg(a.list.count), 0, {}};
    else return TreeWalk<N>{a, entries, chunk_jobs, chunk_slots, 1, 0, 0, 1};
  }();
  if constexpr (!Listed) {
    TreeSeq own_seq{};
    const bool small = a.batch <= 32;
    const int per = (a.batch + kTreeThreads - 1) / kTreeThreads;  // else: requests of a thread's chunk
    const int r0 = small ? lane : min(tid * per, a.batch), r1 = small ? min(lane + 1, a.batch) : min(r0 + per, a.batch);
    walk.per = per;
    int64_t units = 0;
    int32_t groups = 0;
    bool fine = true;  // no request is refused: the node sums rise
    for (int b = r0; b < r1; ++b) {
      const TreeSeq s = tree_seq<N>(a, b);
      if (!s.ok && blockIdx.x == 0) flag(a.err, DSR_ERR_ID);
      fine = fine && s.ok;
      units += int64_t(s.groups) * s.tiles;
      groups += s.groups;
      own_seq = s;
    }
    // sums over the warp: low and high parts of the units by themselves
    units = (int64_t(__reduce_add_sync(~0u, uint32_t(units >> 24))) << 24) +
            __reduce_add_sync(~0u, uint32_t(units) & 0xffffffu);
    groups = __reduce_add_sync(~0u, groups);
    fine = __all_sync(~0u, fine);
    tc_fence_before();
    if (!small) {
      if (lane == 0) warp_units[warp] = units, warp_groups[warp] = groups;
      fine = __syncthreads_and(fine);
      units = groups = 0;
      for (int w = 0; w < kTreeThreads / 32; ++w) units += warp_units[w], groups += warp_groups[w];
    }
    // ---- the segment length: one tile when that fills no more than the grid, else the
    // best of four wave counts
    int32_t length = units <= a.ctas ? 1 : 0;
    if (length == 0 && a.batch <= kTreeSearchBatch) {
      if (warp < 4) {
        int32_t len = 1;
        const float e = tree_length<N>(a, own_seq, units, (groups + a.ctas - 1) / a.ctas + warp, len);
        if (lane == 0) estimate[warp] = e, estimated[warp] = len;
      }
      __syncthreads();
      float best = CUDART_INF_F;
      for (int w = 0; w < 4; ++w)
        if (estimate[w] < best) best = estimate[w], length = estimated[w];
    }
    // or the even share of two jobs per CTA, whose partials always fit: a cut request's
    // groups have at most 2 U / length of them.  Batches beyond the search's take that, as do
    // those without a find
    if (length == 0) length = max(int32_t((units + 2 * a.ctas - 1) / (2 * a.ctas)), 1);
    // ---- jobs and partial slots before each lane's request, or each thread's chunk
    int32_t jobs = 0, slots = 0;
    for (int b = r0; b < r1; ++b) {
      const TreeSeq s = small ? own_seq : tree_seq<N>(a, b);
      const int32_t n = s.groups * tree_segments(s, length);
      jobs += n;
      if (s.tiles > length) slots += n;
    }
    walk.length = length;
    int32_t jobs_before = 0, slots_before = 0;
    if (small) {
      // those of the requests with longer segments come first
      const float mine = jobs > 0 ? float(own_seq.tiles) / float(tree_segments(own_seq, length)) : 0.f;
      for (int b = 0; b < a.batch; ++b) {
        const float other = __shfl_sync(~0u, mine, b);
        const int32_t n = __shfl_sync(~0u, jobs, b), m = __shfl_sync(~0u, slots, b);
        if (other > mine || (other == mine && b < lane)) jobs_before += n, slots_before += m;
        walk.jobs += n;
      }
      if (warp == 0 && lane < a.batch) entries[lane] = TreeEntry{own_seq, jobs_before, jobs, slots_before};
    } else {
      int32_t jobs_upto = jobs, slots_upto = slots;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int32_t u = __shfl_up_sync(~0u, jobs_upto, d), v = __shfl_up_sync(~0u, slots_upto, d);
        if (lane >= d) jobs_upto += u, slots_upto += v;
      }
      jobs_before = jobs_upto - jobs;
      slots_before = slots_upto - slots;
      __syncthreads();  // the sums above have been read
      if (lane == 31) warp_units[warp] = jobs_upto, warp_groups[warp] = slots_upto;
      __syncthreads();
      for (int w = 0; w < kTreeThreads / 32; ++w) {
        if (w < warp) jobs_before += int32_t(warp_units[w]), slots_before += int32_t(warp_groups[w]);
        walk.jobs += int32_t(warp_units[w]);
      }
      chunk_jobs[tid] = jobs_before;
      chunk_slots[tid] = slots_before;
    }
    if (blockIdx.x == 0 && (!small || warp == 0)) {
      for (int b = r0; b < r1; ++b) {
        const TreeSeq s = small ? own_seq : tree_seq<N>(a, b);
        a.slot_start[b] = slots_before;
        if (s.tiles > length) slots_before += s.groups * tree_segments(s, length);
      }
      if (tid == 0) a.slot_start[a.batch] = fine ? length : -length;
    }
  } else {
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_o = *tmem_slot, tmem_s = tmem_o + 4 * N;
  pdl_launch_dependents();

  if (warp < 8) {
    // ------------------------------------------------------------ softmax
    const int half = warp >> 2, row_h = half * kHalf, t = tid & 127;  // t: key, or value column
    uint64_t* masks = reinterpret_cast<uint64_t*>(smem + L::kMaskOff) + half * (N + 1);
    const uint32_t lanes = uint32_t(warp & 3) * 32 << 16;             // this warp's TMEM lanes
    const int quad = lane >> 2, mine = row_h + 2 * (lane & 3);        // key of a fragment, first of its two rows
    int n = 0;
    bool ok = true;
    bool more = walk.next();
    while (ok && more) {
      const TreeWork s = tree_work(walk);
      const int count = s.count, rows = s.rows;
      const int64_t qrow = int64_t(s.node0) * a.heads + s.row0;
      if (a.q_wide) {
        // ---- FP32 query rows -> bf16, K-major, 128-byte swizzle (BF16 ones come by TMA).  As
        // in the sparse attention: the keys are BF16, and one product takes one type.  It moves
        // the output by 1.8e-3 to 2.7e-3 of its norm (60000 to 500 rows); FP32 in and out saves
        // the caller a cast, no more
        constexpr int kVec = N * (kTreeD / 8), kBatch = 3;
        for (int i0 = tid; i0 < kVec; i0 += kTreeSoftmax * kBatch) {
          uint4 v[kBatch];
#pragma unroll
          for (int j = 0; j < kBatch; ++j) {
            const int i = i0 + kTreeSoftmax * j, r = i / (kTreeD / 8);
            v[j] = make_uint4(0, 0, 0, 0);
            if (i < kVec && r < rows) {
              const float4* src = reinterpret_cast<const float4*>(
                  static_cast<const float*>(a.q) + (qrow + r) * kTreeD + (i - r * (kTreeD / 8)) * 8);
              const float4 lo = __ldg(src), hi = __ldg(src + 1);
              v[j] = make_uint4(bf16x2(lo.x, lo.y), bf16x2(lo.z, lo.w), bf16x2(hi.x, hi.y), bf16x2(hi.z, hi.w));
            }
          }
#pragma unroll
          for (int j = 0; j < kBatch; ++j) {
            const int i = i0 + kTreeSoftmax * j, r = i / (kTreeD / 8), d = (i - r * (kTreeD / 8)) * 8;
            if (i < kVec)
              *reinterpret_cast<uint4*>(smem + L::kQOff + (d >> 6) * (N * 128) + sw128_offset(r, d & 63)) = v[j];
          }
        }
        fence_proxy_async_smem();
        mbar_arrive(bar_q);
      }
      if ((warp & 3) == 0) {  // the rows' masks, and what any of them sees
        uint64_t any = 0;
        for (int r = lane; r < N; r += 32) {
          const uint64_t word = r < rows ? uint64_t(a.masks[s.node0 + (s.row0 + r) / a.heads]) : 0ull;
          masks[r] = word;
          any |= word;
        }
        const uint32_t low = __reduce_or_sync(~0u, uint32_t(any)), high = __reduce_or_sync(~0u, uint32_t(any >> 32));
        if (lane == 0) masks[N] = uint64_t(high) << 32 | low;
      }
      // a half has its own, since it leaves alone when one of its waits gives up: a barrier
      // of both would then never be complete
      softmax_sync(half, true);

      // a maximum follows when a score passes it by more than the slack (or is the first)
      auto limit = [](float m) { return m + kTreeSlack; };
      float m[C][2], l[C][2];
#pragma unroll
      for (int c = 0; c < C; ++c) m[c][0] = m[c][1] = -CUDART_INF_F, l[c][0] = l[c][1] = 0.f;
      for (int i = 0; i < count; ++i, ++n) {
        const int32_t p0 = s.block0 * DSR_BLOCK_TOKENS + (s.tile0 + i) * kTreeKeys;
        ok = tree_wait_warp(bar_s, n & 1, abort, a.err);
        // ---- scores of keys 32 (warp % 4) + quad + 8j, rows row_h + 8c + 2 (lane % 4) + e
        float v[C][4][2];
        if (ok) {
          tc_fence_after();
          uint32_t t0[4 * C], t1[4 * C];
          tmem_ld_16x256<C>(tmem_s + row_h + lanes, t0);
          tmem_ld_16x256<C>(tmem_s + row_h + lanes + (16u << 16), t1);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              v[c][0][e] = __uint_as_float(t0[4 * c + e]);
              v[c][1][e] = __uint_as_float(t0[4 * c + 2 + e]);
              v[c][2][e] = __uint_as_float(t1[4 * c + e]);
              v[c][3][e] = __uint_as_float(t1[4 * c + 2 + e]);
            }
          if (s.context - p0 < kTreeKeys) {  // drafted rows, or past the end
            const int32_t drafted = p0 - s.context;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const uint64_t word = masks[8 * c + mine + e];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const int32_t d = drafted + (warp & 3) * 32 + quad + 8 * j;
                  if (d >= 0 && (d >= s.drafts || !(word >> d & 1))) v[c][j][e] = -CUDART_INF_F;
                }
              }
            // a row that no node of the group sees may hold anything: it is cleared, since
            // 0 x NaN would reach the output.  Eight lanes a row: a thread per row would
            // send the 32 lanes of a store to the same banks (4.7 us for one such tile)
            const uint64_t any = masks[N];
            const int32_t d = drafted + t;
            const uint32_t hidden = __ballot_sync(~0u, d >= 0 && (d >= s.drafts || !(any >> d & 1)));
            if (hidden != 0) {
#pragma unroll 1
              for (int c = 4 * half; c < 4 * half + 4; ++c) {
                const int pair = (4 * n + (c >> 1)) % L::kPairs;
                uint8_t* block = smem + L::kRingOff + pair * 32768 + (c & 1) * 16384 + (warp & 3) * 32 * 128;
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                  const int r = 4 * x + (lane >> 3);
                  if (hidden >> r & 1)
                    *reinterpret_cast<uint4*>(block + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
              }
            }
          }
        }
        // ---- weights against the running maxima as they stand, their sums, P^T.  The sums are
        // of the weights as formed; for the product with V they are rounded to BF16, the type
        // the tensor cores take beside V's (by 2^-8 of a weight at most: measured over 500 to
        // 60000 rows 4e-4 to 9e-4 of an output's norm, where an output in BF16 rounds by 1.7e-3)
        float sum[C][2];
        bool fits = ok && i > 0;
        auto weigh = [&] {
#pragma unroll
          for (int c = 0; c < C; ++c) {
            uint32_t packed[4];
            const float b0 = m[c][0] == -CUDART_INF_F ? 0.f : m[c][0], b1 = m[c][1] == -CUDART_INF_F ? 0.f : m[c][1];
            sum[c][0] = sum[c][1] = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float x = ex2(fmaf(v[c][j][0], a.scale_log2, -b0)), y = ex2(fmaf(v[c][j][1], a.scale_log2, -b1));
              sum[c][0] += x;
              sum[c][1] += y;
              packed[j] = bf16x2(x, y);
            }
            const int r = row_h + 8 * c + (lane & 7), key = (warp & 3) * 32 + 8 * (lane >> 3);
            stmatrix_x4_trans(sbase + L::kROff + (key >> 6) * (N * 128) + sw128_offset(r, key & 63), packed[0],
                              packed[1], packed[2], packed[3]);
          }
        };
        auto top_of = [&](int c, int e) {
          return fmaxf(fmaxf(v[c][0][e], v[c][1][e]), fmaxf(v[c][2][e], v[c][3][e])) * a.scale_log2;
        };
        if (fits) {
#pragma unroll
          for (int c = 0; c < C; ++c) fits = fits && !(top_of(c, 0) > limit(m[c][0])) && !(top_of(c, 1) > limit(m[c][1]));
          weigh();
        }
        // most tiles end here: no maximum has to follow, no row needs the others' maxima
        if (!softmax_sync(half, fits)) {
          ok = softmax_sync(half, ok);
          if (!ok) break;
          // ---- the maximum of each row over the tile's keys; a thread follows its rows, all alike
#pragma unroll
          for (int c = 0; c < C; ++c) {
            float x[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              x[e] = top_of(c, e);
              x[e] = fmaxf(x[e], __shfl_xor_sync(~0u, x[e], 4));
              x[e] = fmaxf(x[e], __shfl_xor_sync(~0u, x[e], 8));
              x[e] = fmaxf(x[e], __shfl_xor_sync(~0u, x[e], 16));
            }
            if (quad == 0) *reinterpret_cast<float2*>(red + (warp & 3) * N + 8 * c + mine) = make_float2(x[0], x[1]);
          }
          softmax_sync(half, true);
#pragma unroll
          for (int c = 0; c < C; ++c) {
            float2 x = *reinterpret_cast<const float2*>(red + 8 * c + mine);
#pragma unroll
            for (int w = 1; w < 4; ++w) {
              const float2 y = *reinterpret_cast<const float2*>(red + w * N + 8 * c + mine);
              x.x = fmaxf(x.x, y.x), x.y = fmaxf(x.y, y.y);
            }
            const float top[2] = {x.x, x.y};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float f = 1.f;
              if (top[e] > limit(m[c][e])) {
                f = ex2(m[c][e] - top[e]);  // 0 when the row had seen nothing
                l[c][e] *= f;
                m[c][e] = top[e];
              }
              if (quad == 0 && (warp & 3) == 0) stat[8 * c + mine + e] = f;
            }
          }
          if (i > 0) {
            softmax_sync(half, true);
#pragma unroll 1
            for (int r = 0; r < 4 * kHalf; r += W) {
              uint32_t o[W];
              const int col = (r / kHalf) * N + row_h + r % kHalf;
              tmem_ld_lanes<W>(tmem_o + col + lanes, o);
              tmem_wait_ld();
#pragma unroll
              for (int x = 0; x < W; ++x)
                o[x] = __float_as_uint(__uint_as_float(o[x]) * stat[row_h + r % kHalf + x]);
              tmem_st_lanes<W>(tmem_o + col + lanes, o);
            }
            tmem_wait_st();
          }
          weigh();
        }
#pragma unroll
        for (int c = 0; c < C; ++c) l[c][0] += sum[c][0], l[c][1] += sum[c][1];
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(bar_p);
      }
      if (!ok) break;

      // ---- output of the segment: sums over the keys' threads, then O^T.  The last O
      // MMA follows every thread's last use of red and stat
      more = walk.next();  // while they run
      ok = tree_wait_warp(bar_o, (n - 1) & 1, abort, a.err);
      const bool whole = s.whole;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = l[c][e];
          x += __shfl_xor_sync(~0u, x, 4);
          x += __shfl_xor_sync(~0u, x, 8);
          x += __shfl_xor_sync(~0u, x, 16);
          if (quad == 0) {
            red[(warp & 3) * N + 8 * c + mine + e] = x;
            if ((warp & 3) == 0) stat[8 * c + mine + e] = m[c][e];
          }
        }
      ok = softmax_sync(half, ok);
      if (!ok) break;
      if (t < kHalf) {
        const int r = row_h + t;
        const float sum = (red[r] + red[N + r]) + (red[2 * N + r] + red[3 * N + r]), top = stat[r];
        if (r < rows && !(sum < CUDART_INF_F)) flag(a.err, DSR_ERR_NONFINITE);
        if (whole) {
          float total;
          const float lse = tree_total(a.sink, a.err, (s.row0 + r) % a.heads, top, sum, total);
          stat[r] = total > 0.f ? 1.f / total : 0.f;
          if (a.lse != nullptr && r < rows) a.lse[qrow + r] = lse;
        } else {
          if (!Listed || r < rows) {
            a.part_m[int64_t(s.part) + r] = top;
            a.part_l[int64_t(s.part) + r] = sum;
          }
          stat[r] = 1.f;
        }
      }
      softmax_sync(half, true);
      tc_fence_after();
      float finite = 0.f;  // stays zero
#pragma unroll 1
      for (int x0 = 0; x0 < 4 * kHalf; x0 += W) {
        uint32_t o[W];
        const int r = row_h + x0 % kHalf, d = (x0 / kHalf) * 128 + t;
        tmem_ld_lanes<W>(tmem_o + (x0 / kHalf) * N + r + lanes, o);
        tmem_wait_ld();
        float x[W];
#pragma unroll
        for (int y = 0; y < W; y += 4) {
          const float4 f = *reinterpret_cast<const float4*>(stat + r + y);
          x[y] = __uint_as_float(o[y]) * f.x, x[y + 1] = __uint_as_float(o[y + 1]) * f.y;
          x[y + 2] = __uint_as_float(o[y + 2]) * f.z, x[y + 3] = __uint_as_float(o[y + 3]) * f.w;
        }
        if (!whole) {
          float4* dst = reinterpret_cast<float4*>(a.part_o + (int64_t(s.part) + r) * kTreeDv) + d;
#pragma unroll
          for (int y = 0; y < W; y += 4)
            if (r + y < rows) dst[y / 4 * kTreeDv] = make_float4(x[y], x[y + 1], x[y + 2], x[y + 3]);
        } else if (a.out_wide) {
          float* dst = static_cast<float*>(a.out) + (qrow + r) * kTreeDv + d;
#pragma unroll
          for (int y = 0; y < W; ++y)
            if (r + y < rows) dst[y * kTreeDv] = x[y], finite = fmaf(x[y], 0.f, finite);
        } else {
          uint16_t* dst = static_cast<uint16_t*>(a.out) + (qrow + r) * kTreeDv + d;
#pragma unroll
          for (int y = 0; y < W; ++y)
            if (r + y < rows) {
              dst[y * kTreeDv] = __bfloat16_as_ushort(__float2bfloat16_rn(x[y]));
              finite = fmaf(x[y], 0.f, finite);
            }
        }
      }
      if (finite != 0.f) flag(a.err, DSR_ERR_NONFINITE);
      tc_fence_before();
      mbar_arrive(bar_free);
    }
  } else if (warp == 8) {
    // ------------------------------------------------------------ MMA issuer
    // The whole warp runs the loop and one lane issues, on values that are the same in
    // all lanes: descriptors then stay in uniform registers.  Issued from a one-lane
    // branch each MMA waited some 80 to 120 cycles for its operands to get there
    // (measured; the MMA itself takes 48).
    constexpr uint32_t idesc_s = umma_idesc_bf16(128, N, false, false);
    constexpr uint32_t idesc_o = umma_idesc_bf16(128, N, true, false);
    const uint32_t sb = __shfl_sync(~0u, sbase, 0);
    const uint32_t ts = __shfl_sync(~0u, tmem_s, 0), to = __shfl_sync(~0u, tmem_o, 0);
    const bool leader = elect_one();
    const uint64_t desc_s = umma_desc_sw128(sb, 16, 1024), desc_q = umma_desc_sw128(sb + L::kQOff, 16, 1024);
    const uint64_t desc_v = umma_desc_sw128(sb + L::kRingOff, 16384, 1024);
    const uint64_t desc_p = umma_desc_sw128(sb + L::kROff, 16, 1024);
    int n = 0, segment = 0, pair = 0;  // pair: ring position of the tile's first block pair
    uint32_t lap = 0;                  // the ring's phase there
    bool ok = true, committed = false;  // committed: the tile's S MMAs
    auto wait = [&](uint64_t* bar, uint32_t parity) { return tree_wait_warp(bar, parity, abort, a.err); };
    while (ok) {
      if (!walk.next()) break;  // alike in all lanes
      const int count = __shfl_sync(~0u, tree_work(walk).count, 0);
      committed = false;
      ok = wait(bar_q, segment & 1);
      for (int i = 0; i < count && ok; ++i, ++n) {
        // S^T: column blocks 0..7 pair by pair, then the rotary block.  A step of 16
        // columns moves both operands by 32 bytes, a block by its size: constants added
        // to a descriptor's address field (units of 16 bytes)
        int at = pair;
        uint32_t phase = lap;
        committed = false;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          ok = ok && wait(full + at, phase);
          if (ok) {
            tc_fence_after();
            const uint64_t ad = desc_s + (L::kRingOff + at * 32768) / 16, bd = desc_q + 2 * c * (N * 128 / 16);
            if (leader) {
#pragma unroll
              for (int x = 0; x < 8; ++x)
                umma_bf16(ts, ad + (x >> 2) * 1024 + 2 * (x & 3), bd + (x >> 2) * (N * 128 / 16) + 2 * (x & 3), idesc_s,
                          (c | x) != 0 ? 1u : 0u);
            }
          }
          if (++at == L::kPairs) at = 0, phase ^= 1;
        }
        ok = ok && wait(bar_r, n & 1);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            umma_bf16(ts, desc_s + L::kROff / 16 + 2 * x, desc_q + 8 * (N * 128 / 16) + 2 * x, idesc_s, 1u);
          umma_commit(bar_s);
        }
        committed = true;
        ok = wait(bar_p, n & 1);
        // the previous segment's O^T has been read
        if (ok && i == 0 && segment > 0) ok = wait(bar_free, (segment - 1) & 1);
        if (!ok) break;
        tc_fence_after();
        // O^T, 128 value columns after another, so that their block pair is free early
        at = pair;
        const uint32_t accumulate = i > 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint64_t ad = desc_v + at * (32768 / 16);
          if (leader) {
#pragma unroll
            for (int ks = 0; ks < kTreeKeys / 16; ++ks)
              umma_bf16(to + c * N, ad + ks * (2048 / 16), desc_p + (ks >> 2) * (N * 128 / 16) + 2 * (ks & 3), idesc_o,
                        ks > 0 ? 1u : accumulate);
            umma_commit(empty + at);
          }
          if (++at == L::kPairs) at = 0;
        }
        if (leader) umma_commit(bar_o);
        lap = pair + 4 >= L::kPairs ? lap ^ 1 : lap;
        pair = at;
      }
      ++segment;
    }
    // the last MMAs retire before TMEM is released (commits cover all before them)
    if (n > 0) mbar_drain(bar_o, (n - 1) & 1);
    if (!ok) {  // a wait gave up: nor may S MMAs of the tile it was in outlive TMEM
      if (!committed && leader) umma_commit(bar_s);
      mbar_drain(bar_s, n & 1);
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------ key tiles
    int n = 0;
    bool ok = true;
    while (ok && walk.next()) {
      const TreeWork s = tree_work(walk);
      const int32_t* table = a.table + int64_t(s.table) * a.stride;
      const int32_t blocks = int32_t((int64_t(s.context) + s.drafts + DSR_BLOCK_TOKENS - 1) / DSR_BLOCK_TOKENS);
      auto row_of = [&](int32_t j) -> int32_t {  // first pool row of block j; past the pool: reads zeros
        if (j >= blocks || lane != 0) return int32_t(a.pool_rows);
        const int64_t blk = table[j];
        if (blk < 0 || blk * DSR_BLOCK_TOKENS >= a.pool_rows) {
          flag(a.err, DSR_ERR_ID);
          return int32_t(a.pool_rows);
        }
        return int32_t(blk * DSR_BLOCK_TOKENS);
      };
      if (!a.q_wide) {
        // the query, once the last S MMA of the job before has read the one there
        if (n > 0) ok = tree_wait_warp(bar_s, (n - 1) & 1, abort, a.err);
        if (!ok) break;
        if (lane == 0) {
          const int32_t qrow = s.node0 * a.heads + s.row0;
          mbar_arrive_expect_tx(bar_q, 9 * N * 128);
          for (int c = 0; c < 9; ++c) tma_load_2d(sbase + L::kQOff + c * (N * 128), &q_map, bar_q, c * 64, qrow);
          ++*loaded_q;
        }
      }
      const int32_t block0 = s.block0 + 2 * s.tile0;
      int32_t y0 = row_of(block0), y1 = row_of(block0 + 1);
      for (int i = 0; lane == 0 && i < s.count && ok; ++i, ++n) {
        const int32_t x0 = y0, x1 = y1;
        if (i + 1 < s.count) y0 = row_of(block0 + 2 * i + 2), y1 = row_of(block0 + 2 * i + 3);
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          const int k = 4 * n + c, pair = k % L::kPairs;
          ok = tree_wait(empty + pair, ((k / L::kPairs) & 1) ^ 1, abort, a.err);
          if (!ok) break;
          mbar_arrive_expect_tx(full + pair, 32768);
          const uint32_t dst = sbase + L::kRingOff + pair * 32768;
          for (int h = 0; h < 2; ++h) {
            tma_load_2d(dst + h * 16384, &kv_map, full + pair, (2 * c + h) * 64, x0);
            tma_load_2d(dst + h * 16384 + 8192, &kv_map, full + pair, (2 * c + h) * 64, x1);
          }
          *loaded = k + 1;
        }
        // P^T of the tile before sits in the rotary buffer until its O MMAs are done
        if (ok && n > 0) ok = tree_wait(bar_o, (n - 1) & 1, abort, a.err);
        if (!ok) break;
        mbar_arrive_expect_tx(bar_r, 16384);
        tma_load_2d(sbase + L::kROff, &kv_map, bar_r, 512, x0);
        tma_load_2d(sbase + L::kROff + 8192, &kv_map, bar_r, 512, x1);
        *loaded_r = n + 1;
        if (i + 1 < s.count)  // the next tile's rows into L2 (209 to 199 us for 8 nodes over 131072 rows)
          for (int c = 0; c < 9; ++c) {
            tma_prefetch_2d(&kv_map, c * 64, y0);
            tma_prefetch_2d(&kv_map, c * 64, y1);
          }
      }
      n = __shfl_sync(~0u, n, 0);
      ok = __shfl_sync(~0u, int(ok), 0) != 0;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort && tid == 0) {
    // a wait gave up: let the copies in flight land before exit
    for (int k = max(0, *loaded - L::kPairs); k < *loaded; ++k) mbar_drain(full + k % L::kPairs, (k / L::kPairs) & 1);
    if (*loaded_r > 0) mbar_drain(bar_r, (*loaded_r - 1) & 1);
    if (*loaded_q > 0) mbar_drain(bar_q, (*loaded_q - 1) & 1);
  }
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem_o, L::kTmemCols);
  }
}

// ---------------------------------------------------------------------------
// Joins the partials of a group of several segments: one CTA per four query rows
// (of one node, since heads come in sixteens) and 128 value columns, a thread one
// column of all four.
//   out = sum_p 2^(m_p - M) O_p / (2^(sink - M) + sum_p 2^(m_p - M) l_p)
// The statistics and a thread's first values are requested together, so that few
// parts take one memory round trip.
// ---------------------------------------------------------------------------
constexpr int kTreeMaxParts = kTreeSlotsPerCta * kTreeMaxCtas;  // of one row
constexpr int kJoinThreads = 128, kJoinBatch = 8;  // kJoinBatch: parts requested together

template <int N>
__global__ void __launch_bounds__(kJoinThreads) tree_combine_kernel(const __grid_constant__ TreeArgs a) {
  __shared__ float weight[4][kTreeMaxParts];
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
  TreeSeq s = tree_seq<N>(a, lo);
  pdl_wait();  // before any CTA leaves: the join must not end ahead of the attention
  const int32_t length = __ldcg(a.slot_start + a.batch);
  if (node < s.node0 || node >= s.node0 + s.nodes) {
    // a padding row.  Where a request was refused the sums may be in disorder and the search
    // may have missed the request that has the row: every one is asked
    lo = -1;
    if (length < 0) {
      if (tid == 0) owner = -1;
      __syncthreads();
      for (int b = tid; b < a.batch; b += kJoinThreads) {
        const TreeSeq other = tree_seq<N>(a, b);
        if (node >= other.node0 && node < other.node0 + other.nodes) atomicMax(&owner, b);
      }
      __syncthreads();
      lo = owner;
    }
    if (lo < 0) {
      if (!a.zero_unused) return;
      for (int y = 0; y < 4; ++y) {
        const int64_t at = (row + y) * kTreeDv + d;
        if (a.out_wide) static_cast<float*>(a.out)[at] = 0.f;
        else static_cast<uint16_t*>(a.out)[at] = 0;
      }
      if (a.lse != nullptr && blockIdx.y == 0 && tid < 4) a.lse[row + tid] = -CUDART_INF_F;
      return;
    }
    s = tree_seq<N>(a, lo);
  }
  const int parts = tree_segments(s, abs(length));
  if (parts <= 1) return;  // written by its job
  const int in = int(row - int64_t(s.node0) * a.heads), group = in / N, r = in % N;
  const int64_t first = int64_t(__ldcg(a.slot_start + lo)) + group;
  auto slot = [&](int p) { return (first + int64_t(p) * s.groups) * N + r; };
  float4 v[kJoinBatch];
  auto request = [&](int p0) {
#pragma unroll
    for (int j = 0; j < kJoinBatch; ++j)
      if (p0 + j < parts) v[j] = __ldcg(reinterpret_cast<const float4*>(a.part_o + slot(p0 + j) * kTreeDv) + d);
  };
  request(0);
  {
    const int w = tid >> 5, lane = tid & 31;  // one warp per row
    const float m0 = lane < parts ? __ldcg(a.part_m + slot(lane) + w) : -CUDART_INF_F;
    const float l0 = lane < parts ? __ldcg(a.part_l + slot(lane) + w) : 0.f;
    float top = m0, sum = 0.f;
    for (int p = lane + 32; p < parts; p += 32) top = fmaxf(top, __ldcg(a.part_m + slot(p) + w));
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    const float base = top == -CUDART_INF_F ? 0.f : top;
    for (int p = lane; p < parts; p += 32) {
      const float e = ex2((p < 32 ? m0 : __ldcg(a.part_m + slot(p) + w)) - base);
      weight[w][p] = e;
      sum += e * (p < 32 ? l0 : __ldcg(a.part_l + slot(p) + w));
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
    const int64_t at = (row + y) * kTreeDv + d;
    if (a.out_wide) static_cast<float*>(a.out)[at] = out[y];
    else static_cast<uint16_t*>(a.out)[at] = __bfloat16_as_ushort(__float2bfloat16_rn(out[y]));
  }
}

// Rows per group: all of a request's rows in one group when that fits, since a
// group reads every key tile once, and no more, since the MMAs of empty rows cost as much
// (16 rows over 131072: 64 us in groups of 16, 88 of 32, 92 of 64).
}  // namespace
int tree_rows(int64_t heads, int64_t max_nodes) {
  const int64_t rows = heads * max_nodes;
  return rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
}

int tree_ctas() { return sm_count() < kTreeMaxCtas ? sm_count() : kTreeMaxCtas; }
namespace {

size_t tree_start_bytes(int64_t batch) { return (size_t(batch + 1) * 4 + 255) / 256 * 256; }

// The tensor maps: one page by 64 columns, and a group's queries (FP32 ones are converted, not copied).
template <int N>
int tree_maps(const TreeArgs& a, const uint16_t* kv_pool, CUtensorMap& map, CUtensorMap& q_map) {
  const int rc = encode_tmap_bf16_2d(&map, kv_pool, kTreeD, uint64_t(a.pool_rows), 64, DSR_BLOCK_TOKENS);
  if (rc != DSR_OK) return rc;
  q_map = map;
  return a.q_wide ? DSR_OK : encode_tmap_bf16_2d(&q_map, a.q, kTreeD, uint64_t(a.nodes) * a.heads, 64, N);
}

template <int N>
int launch_tree(TreeArgs& a, const uint16_t* kv_pool, void* workspace, cudaStream_t stream) {
  using L = TreeLayout<N>;
  int rc = set_max_smem(tree_mla_kernel<N, false>, L::kAlloc, "tree_mla_decode");
  if (rc != DSR_OK) return rc;
  CUtensorMap map, q_map;
  rc = tree_maps<N>(a, kv_pool, map, q_map);
  if (rc != DSR_OK) return rc;
  a.slot_start = static_cast<int32_t*>(workspace);
  a.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + tree_start_bytes(a.batch));
  a.part_m = a.part_o + size_t(kTreeSlotsPerCta) * a.ctas * N * kTreeDv;
  a.part_l = a.part_m + size_t(kTreeSlotsPerCta) * a.ctas * N;
  tree_mla_kernel<N, false><<<unsigned(a.ctas), kTreeThreads, L::kAlloc, stream>>>(map, q_map, a);
  rc = launch_status("tree_mla_decode launch");
  if (rc != DSR_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(a.nodes * a.heads / 4), kTreeDv / kJoinThreads, 1);
  cfg.blockDim = dim3(kJoinThreads, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, tree_combine_kernel<N>, a);
  if (e != cudaSuccess) return fail(DSR_ECUDA, "tree_mla_decode combine launch: %s", cudaGetErrorString(e));
  return DSR_OK;
}

template <int N>
int launch_listed(const TreeArgs& a, const uint16_t* kv_pool, cudaStream_t stream) {
  using L = TreeLayout<N>;
  int rc = set_max_smem(tree_mla_kernel<N, true>, L::kAlloc, "prefix_mla_decode");
  if (rc != DSR_OK) return rc;
  CUtensorMap map, q_map;
  rc = tree_maps<N>(a, kv_pool, map, q_map);
  if (rc != DSR_OK) return rc;
  return launch_after(tree_mla_kernel<N, true>, dim3(unsigned(a.ctas)), kTreeThreads, L::kAlloc, stream,
                      "prefix_mla_decode", map, q_map, a);
}

}  // namespace

int launch_tree_listed(const TreeListedCall& c, cudaStream_t stream) {
  TreeArgs a = {};
  a.q = c.q;
  a.q_wide = c.q_dtype == DSR_F32;
  a.table = c.table;
  a.stride = c.stride;
  a.pool_rows = c.pool_rows;
  a.masks = c.masks;
  a.scale_log2 = c.scale_log2;
  a.err = c.err;
  a.part_o = c.part_o;
  a.part_m = c.part_m;
  a.part_l = c.part_l;
  a.nodes = c.nodes;
  a.heads = c.heads;
  a.ctas = tree_ctas();
  a.list = c.list;
  switch (c.rows) {
    case 16:
      return launch_listed<16>(a, c.kv_pool, stream);
    case 32:
      return launch_listed<32>(a, c.kv_pool, stream);
    default:
      return launch_listed<64>(a, c.kv_pool, stream);
  }
}

}  // namespace dsr

extern "C" size_t dsr_tree_mla_workspace_bytes(int64_t batch, int64_t heads, int64_t max_nodes) {
  using namespace dsr;
  if (batch <= 0 || heads <= 0 || max_nodes <= 0) return 0;
  const size_t rows = size_t(kTreeSlotsPerCta) * tree_ctas() * tree_rows(heads, max_nodes);
  return tree_start_bytes(batch) + rows * (kTreeDv + 2) * 4;
}

extern "C" int dsr_tree_mla_decode(const void* q, int q_dtype, const uint16_t* kv_pool, int64_t pool_blocks,
                                   const int32_t* block_table, int64_t table_stride, const int32_t* context,
                                   const int32_t* cu_nodes, const int64_t* tree_mask, int64_t max_nodes,
                                   const float* sink, float scale, void* out, int out_dtype, float* lse,
                                   void* workspace, size_t workspace_bytes, int32_t* err, int64_t batch,
                                   int64_t nodes, int64_t heads, void* stream) {
  using namespace dsr;
  clear_error();
  PoolAddr pa;
  const int rc = paged_addr(&pa, block_table, table_stride, pool_blocks, "tree_mla_decode");
  if (rc != DSR_OK) return rc;
  DSR_REQUIRE(q && kv_pool && context && cu_nodes && tree_mask && out && workspace && err,
              "tree_mla_decode: null pointer");
  const bool zero_unused = (out_dtype & DSR_ZERO_UNUSED) != 0;
  out_dtype &= ~DSR_ZERO_UNUSED;
  DSR_REQUIRE((q_dtype == DSR_BF16 || q_dtype == DSR_F32) && (out_dtype == DSR_BF16 || out_dtype == DSR_F32),
              "tree_mla_decode: unknown element type");
  DSR_REQUIRE(heads == 16 || heads == 32 || heads == 64 || heads == 128,
              "tree_mla_decode: heads %lld not in {16,32,64,128}", (long long)heads);
  DSR_REQUIRE(max_nodes > 0 && max_nodes <= kTreeMaxNodes, "tree_mla_decode: max nodes %lld outside [1, %d]",
              (long long)max_nodes, kTreeMaxNodes);
  DSR_REQUIRE(batch > 0 && batch <= 65535, "tree_mla_decode: batch %lld outside [1, 65535]", (long long)batch);
  DSR_REQUIRE(nodes > 0 && nodes <= int64_t(65535) * kTreeMaxNodes, "tree_mla_decode: nodes %lld outside [1, %d]",
              (long long)nodes, 65535 * kTreeMaxNodes);
  DSR_REQUIRE(isfinite(scale) && scale > 0.f, "invalid attention scale");
  DSR_REQUIRE(aligned16(q) && aligned16(kv_pool) && aligned16(out),
              "tree_mla_decode: q, kv_pool and out must be 16-byte aligned");
  DSR_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255u) == 0, "tree_mla_decode: workspace must be 256-byte aligned");
  const size_t need = dsr_tree_mla_workspace_bytes(batch, heads, max_nodes);
  DSR_REQUIRE(workspace_bytes >= need, "tree_mla_decode: workspace %zu < %zu bytes", workspace_bytes, need);
  TreeArgs a = {};
  a.q = q;
  a.q_wide = q_dtype == DSR_F32;
  a.out_wide = out_dtype == DSR_F32;
  a.zero_unused = zero_unused;
  a.table = block_table;
  a.stride = table_stride;
  a.pool_rows = pa.rows;
  a.context = context;
  a.cu_nodes = cu_nodes;
  a.masks = tree_mask;
  a.sink = sink;
  a.scale_log2 = scale * kTreeLog2e;
  a.out = out;
  a.lse = lse;
  a.err = err;
  a.nodes = nodes;
  a.batch = int(batch);
  a.heads = int(heads);
  a.max_nodes = int(max_nodes);
  a.ctas = tree_ctas();
  switch (tree_rows(heads, max_nodes)) {
    case 16:
      return launch_tree<16>(a, kv_pool, workspace, as_stream(stream));
    case 32:
      return launch_tree<32>(a, kv_pool, workspace, as_stream(stream));
    default:
      return launch_tree<64>(a, kv_pool, workspace, as_stream(stream));
  }
}
