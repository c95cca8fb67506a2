// What the tree attention and the attention over shared prefixes have in common: jobs that
// a plan lays out, the partials they leave, and a row's total.
#pragma once

#include <math_constants.h>

#include "common.cuh"

namespace dsr {

constexpr float kTreeLog2e = 1.4426950408889634f;
constexpr int kTreeMaxCtas = 256;

// One group of query rows over a run of 128-key tiles.  Tile i holds positions
// 64 block0 + 128 i and up of the table row; positions from `context` on are the `drafts`
// drafted ones, seen as the masks say.
struct alignas(16) TreeJob {
  int32_t table, block0;
  int32_t node0, row0, rows;  // query rows node0 * heads + row0 ..
  int32_t drafts, context;
  int32_t tile0, count;
  int32_t part;               // where the rows' partials go
  int32_t unused[2];
};
static_assert(sizeof(TreeJob) == 48, "three 16-byte words");

// Partials (m in log2 units, l, unnormalised O) of `row`, a multiple of 4 and up:
// part_o [rows / 4][512][4], part_m and part_l [rows].
struct TreeListed {
  const TreeJob* jobs;
  const int32_t* count;
};

// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A row's total with its head's sink (in units of 2^top), and the logarithm of its sum.
__device__ __forceinline__ float tree_total(const float* sinks, int32_t* err, int head, float top, float sum,
                                            float& total) {
  total = sum;
  if (sinks == nullptr) return top == -CUDART_INF_F ? top : (top + log2f(sum)) / kTreeLog2e;
  float sink = sinks[head];
  if (!isfinite(sink)) {
    flag(err, DSR_ERR_NONFINITE);
    sink = 0.f;
  }
  if (top == -CUDART_INF_F) return sink;
  const float over = sink * kTreeLog2e - top;  // the sink's weight, log2
  total = sum + ex2(over);
  return over > 100.f ? sink : (top + log2f(total)) / kTreeLog2e;
}

// The tree attention over listed jobs (tree_mla.cu): every group leaves partials.
struct TreeListedCall {
  const void* q;
  int q_dtype;
  const uint16_t* kv_pool;
  int64_t pool_rows;
  const int32_t* table;
  int64_t stride;
  const int64_t* masks;
  float scale_log2;
  int64_t nodes;
  int heads, rows;  // rows: of a group (16, 32 or 64)
  TreeListed list;
  float *part_o, *part_m, *part_l;
  int32_t* err;
};
int tree_rows(int64_t heads, int64_t max_nodes);
int tree_ctas();
int launch_tree_listed(const TreeListedCall& call, cudaStream_t stream);

}  // namespace dsr
