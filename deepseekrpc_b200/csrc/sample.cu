// Sampling of one token per row of logits with temperature, top-k, top-p and
// min-p, from given uniform numbers.
//
//   w_i = exp((x_i - max x) / T).  In the order of (value descending, index
//   ascending) the filters keep prefixes: the first k; of those the shortest whose
//   mass reaches p times theirs; of those the ones with w_i >= min_p.  The token is
//   the first kept index, in vocabulary order, whose cumulative weight exceeds
//   u times the kept weight.  T = 0 is the arg max (lowest index).
//
// Weights are formed in 64-bit floating point and summed as 2^-44 fixed point, so
// that every sum is the same in any order (a 32-bit sum of 10^5 weights moves the
// borders between tokens by up to a few percent of a token).
//
// A cluster of 1 to 8 CTAs takes a row and holds it in shared memory, so that it is
// read from memory once.  Prefixes are found from a histogram over 2048 equal steps of
// the value below the maximum, of which each CTA sums up its share for the cluster:
//   up to 100 by rank   the histogram is that of the threads' maxima, 512 a CTA, instead
//                       of all entries: at least k entries lie in the steps down to the
//                       one that holds the k-th maximum, and hardly any more
//   by rank             the counts of all entries say which step holds entry k
//   by mass             the steps' exact masses say which one p lies in
// Entries in question go to a list in the first CTA, which ranks them on the unique
// 64-bit rank (order-preserving value, inverted index) with exact weights: by comparing
// all with all where there are few, after a finer histogram where there are more.  Where
// a list overflows (equal logits, masks), the prefix comes from a radix descent over the
// ranks, 11 bits a level.
//
// Bound by the passes over the row in shared memory, and for a few rows by the 7 to 14
// barriers of a cluster (some 0.6 us each).  By mass every entry's weight is formed at least
// twice, ten 64-bit operations each, and costs four shared atomics; 48 rows so (76 to 84 us)
// are 384 CTAs on 296 places: a second wave, one third full, is near half of that.
// Measured, FP32, T = 0.8: 1 row of 128000, top_k 50 and top_p 0.95, 16.4 us; 148 rows 80
// us; 511 rows 244 us = 1.1 TB/s; 148 rows by top_p alone 188 us.  T = 0, 1, 48 and 511
// (BF16) rows of 128K: 12.3, 24.6 and 79.9 us.
#include <cooperative_groups.h>
#include <math_constants.h>

#include <cfloat>
#include <climits>
#include <type_traits>
#include <utility>

#include "common.cuh"
#include "host_common.h"

namespace dsr {
namespace {

namespace cg = cooperative_groups;

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleBins = 2048, kSamplePer = kSampleBins / kSampleThreads;
constexpr int kSampleMaxCluster = 8;
constexpr int kSampleList = 1984;  // entries of a list
constexpr int kSampleFew = 128;    // entries compared with one another
constexpr int kSampleMaxVocab = 1 << 18;
constexpr int kWeightBits = 44;  // 2^18 weights of at most 2^44 fit 62 bits
constexpr double kLog2eD = 1.4426950408889634074;

struct SampleArgs {
  const void* logits;
  int64_t stride;
  int vocab, slice;  // slice: entries of one CTA
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* uniform;
  int32_t* tokens;
  float* chances;
  int32_t* err;
};

// exp((x - high) / heat) for x <= high in 64 bits, as 2^(n/16 + r/16): 2^(n/16) from a
// table and an exponent, 2^(r/16), |r| <= 1/2, by the Taylor series of e^(r ln2/16),
// whose first dropped term is below 2^-42 of it.  (16 entries: a warp's lookups then
// meet no shared-memory bank twice, as they do some eight times among 64.)
struct Weight {
  const double* table;  // [16] 2^(j/16)
  double high, scale;   // scale: 16 log2(e) / heat
  float floor;          // below: no weight (less than 2^-60 of the largest, or -inf)
  // The weight plus 2^(52 - kWeightBits), whose lowest bit is a step of the fixed point.
  __device__ __forceinline__ double shifted(float x) const {
    const double t = (double(fmaxf(x, floor)) - high) * scale;
    constexpr double kRound = 6755399441055744.0, c = 0.043321698784996582;  // 1.5 * 2^52; ln(2) / 16
    const double n = t + kRound, r = t - (n - kRound);
    double p = fma(r, c * c * c * c * c / 120, c * c * c * c / 24);
    p = fma(p, r, c * c * c / 6);
    p = fma(p, r, c * c / 2);
    p = fma(p, r, c);
    p = fma(p, r, 1.0);
    const int m = __double2loint(n);
    const double e = table[m & 15];
    return fma(p, __hiloint2double(__double2hiint(e) + (m >> 4) * (1 << 20), __double2loint(e)), kMagic);
  }
  static constexpr double kMagic = double(1ull << (52 - kWeightBits));
  // What a weight is in steps of 2^-44, rounded.  At the floor that is zero by itself, but
  // in a row whose finite values end there (a maximum near the lowest number).
  __device__ __forceinline__ unsigned long long operator()(float x) const {
    const unsigned long long w =
        (unsigned long long)__double_as_longlong(shifted(x)) - (unsigned long long)__double_as_longlong(kMagic);
    return x >= floor ? w : 0;
  }
};

__device__ __forceinline__ unsigned long long rank_of(float x, int i) {
  return (static_cast<unsigned long long>(score_key(x)) << 32) | (0xffffffffu - uint32_t(i));
}
__device__ __forceinline__ float rank_value(unsigned long long r) { return key_score(uint32_t(r >> 32)); }

struct alignas(16) SampleSmem {
  double table[16];
  unsigned long long list[kSampleList];  // ranks of the entries to sort
  uint32_t wide[3][kSampleBins];         // exact sums of weights (words of 15 bits) or counts, per step or digit
  uint32_t hist[kSampleBins];            // this CTA's counts
  unsigned long long part[kSampleWarps];
  float extremes[kSampleWarps];
  // written by every CTA of the cluster for all
  ulonglong2 counts[2][kSampleMaxCluster];  // of a scan, and of the one before
  unsigned long long kept[kSampleMaxCluster];
  float tops[kSampleMaxCluster], lows[kSampleMaxCluster];
  int firsts[kSampleMaxCluster];
  // written by one CTA for all
  unsigned long long cut, step_before;
  int step_bin, step_ahead, step_in;
  // this CTA's own
  unsigned long long found_before, found_through;
  int found_bin, found_last, listed;
};

template <bool W>
struct SampleRow {
  using T = typename std::conditional<W, float, uint16_t>::type;
  static constexpr int kVec = 16 / sizeof(T);
  __device__ static __forceinline__ float value(T v) {
    if constexpr (W) return v;
    else return bf16_to_float(v);
  }
};

// The block's exclusive sum of x, and the total.
__device__ __forceinline__ unsigned long long block_scan(SampleSmem& s, unsigned long long x, unsigned long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long run = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const unsigned long long up = __shfl_up_sync(~0u, run, d);
    if (lane >= d) run += up;
  }
  __syncthreads();
  if (lane == 31) s.part[warp] = run;
  __syncthreads();
  unsigned long long before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSampleWarps; ++w) {
    const unsigned long long v = s.part[w];
    if (w < warp) before += v;
    total += v;
  }
  return before + run - x;
}
__device__ __forceinline__ unsigned long long warp_sum(unsigned long long v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// The word at p's place in CTA c of the cluster.  (By instruction: the addresses of eight
// CTAs, kept over loops by the compiler, would not leave registers for anything else.)
__device__ __forceinline__ uint32_t cluster_word(const uint32_t* p, int c) {
  uint32_t v;
  asm volatile(
      "{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.u32 %0, [a];\n\t}"
      : "=r"(v)
      : "r"(smem_u32(p)), "r"(c)
      : "memory");
  return v;
}

// Bitonic sort of list[0, n) in descending order; list has room for the next power of two.
__device__ __forceinline__ void block_sort(unsigned long long* list, int n) {
  int all = 2;
  while (all < n) all <<= 1;
  for (int i = n + threadIdx.x; i < all; i += kSampleThreads) list[i] = 0;
  for (int size = 2; size <= all; size <<= 1)
    for (int gap = size >> 1; gap > 0; gap >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < all / 2; i += kSampleThreads) {
        const int lo = (i & ~(gap - 1)) * 2 + (i & (gap - 1)), hi = lo + gap;
        const unsigned long long x = list[lo], y = list[hi];
        if (((lo & size) == 0) == (x < y)) list[lo] = y, list[hi] = x;
      }
    }
  __syncthreads();
}

template <bool W>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(const SampleArgs a) {
  using Row = SampleRow<W>;
  using T = typename Row::T;
  constexpr int kVec = Row::kVec;
  extern __shared__ uint4 sample_smem[];
  SampleSmem& s = *reinterpret_cast<SampleSmem*>(sample_smem);
  T* held = reinterpret_cast<T*>(&s + 1);  // this CTA's slice of the row
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = int(cluster.block_rank()), ctas = int(cluster.num_blocks());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x / ctas;
  // Entry i of the row is at place i + shift, places being counted from a 16-byte
  // boundary; this CTA holds the places [first, first + slice).
  const T* x = static_cast<const T*>(a.logits) + row * a.stride;
  const int shift = int(reinterpret_cast<uintptr_t>(x) / sizeof(T) % kVec);
  const int first = rank * a.slice, base = first - shift;  // base: entry of place `first`
  const int end = a.vocab + shift;

  auto started = cluster.barrier_arrive();  // every CTA is there before one writes to another
  const float heat = a.temperature[row], p = a.top_p[row], least = a.min_p[row], u = a.uniform[row];
  const int k = a.top_k[row];
  const double scale = 16.0 * kLog2eD / double(heat);  // a division in 64 bits: while the row is on its way
  if (tid < 16) s.table[tid] = exp2(tid / 16.0);
  if (tid == 0) s.listed = 0;
  for (int b = tid; b < kSampleBins; b += kSampleThreads) s.hist[b] = 0;

  // ---- the slice into shared memory (places off the row: -inf); extremes, non-finite values
  const float nothing = -CUDART_INF_F;
  float most = nothing;  // NaN when there is one
  constexpr int kAhead = 4;  // pieces requested together
  for (int v0 = tid * kVec; v0 < a.slice; v0 += kAhead * kSampleThreads * kVec) {
    uint4 raw[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const int v = v0 + q * kSampleThreads * kVec, place = first + v;
      if (v < a.slice && place >= shift && place + kVec <= end)
        raw[q] = __ldg(reinterpret_cast<const uint4*>(x + (place - shift)));
    }
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const int v = v0 + q * kSampleThreads * kVec, place = first + v;
      if (v >= a.slice) break;
      T* t = reinterpret_cast<T*>(&raw[q]);
      if (place < shift || place + kVec > end) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          const int e = place + j;
          if constexpr (W) t[j] = e >= shift && e < end ? x[e - shift] : nothing;
          else t[j] = e >= shift && e < end ? x[e - shift] : uint16_t(0xff80);
        }
      }
      *reinterpret_cast<uint4*>(held + v) = raw[q];
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const float f = Row::value(t[j]);
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(most) : "f"(f));
      }
    }
  }
  float top = most;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float other = __shfl_xor_sync(~0u, top, o);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(other));
  }
  if (lane == 0) s.extremes[warp] = top;
  __syncthreads();
  cluster.barrier_wait(std::move(started));
  if (tid < ctas) {  // thread c tells CTA c
    for (int w = 0; w < kSampleWarps; ++w) {
      const float other = s.extremes[w];
      asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(other));
    }
    cluster.map_shared_rank(&s, tid)->tops[rank] = top;
  }
  cluster.sync();
  for (int c = 0; c < ctas; ++c) {
    const float other = s.tops[c];
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(other));
  }
  const bool bad = !(top < CUDART_INF_F);
  const bool valid = heat >= 0.f && heat < CUDART_INF_F && p >= 0.f && p <= 1.f && least >= 0.f && least <= 1.f &&
                     u >= 0.f && u < 1.f && k >= 0;
  if (bad || !valid || top == nothing) {  // alike in all CTAs
    if (rank == 0 && tid == 0) {
      if (bad) flag(a.err, DSR_ERR_NONFINITE);
      else if (!valid) flag(a.err, DSR_ERR_ID);
      a.tokens[row] = -1;
      a.chances[row] = 0.f;
    }
    return;
  }
  // 2^-60 is exp(-41.6); -inf stays out also where that lies below all finite numbers
  const Weight weight{s.table, double(top), scale, fmaxf(top - 41.6f * heat, -FLT_MAX)};

  // Weights are formed four at a time, without branches: a 64-bit operation has tens of
  // cycles of latency.
  constexpr int kFour = 4;
  // each_four(f): f(values, first entry) for this CTA's entries (places off the row: -inf)
  auto each_four = [&](auto&& f) {
    for (int v = tid * kVec; v < a.slice; v += kSampleThreads * kVec) {
      const uint4 raw = *reinterpret_cast<const uint4*>(held + v);
      const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int j = 0; j < kVec; j += kFour) {
        const float g[kFour] = {Row::value(t[j]), Row::value(t[j + 1]), Row::value(t[j + 2]), Row::value(t[j + 3])};
        f(g, base + v + j);
      }
    }
  };
  // each(f): f(value, entry) one by one
  auto each = [&](auto&& f) {
    each_four([&](const float (&g)[kFour], int i) {
#pragma unroll
      for (int j = 0; j < kFour; ++j) f(g[j], i + j);
    });
  };

  if (heat == 0.f) {  // the lowest index of the maximum
    int index = INT_MAX;
    each([&](float f, int i) { index = f == top ? min(index, i) : index; });
    index = __reduce_min_sync(~0u, index);
    if (lane == 0) s.part[warp] = unsigned(index);
    __syncthreads();
    if (tid == 0) {
      for (int w = 0; w < kSampleWarps; ++w) index = min(index, int(s.part[w]));
      cluster.map_shared_rank(&s, 0)->firsts[rank] = index;
    }
    cluster.sync();
    if (rank == 0 && tid == 0) {
      for (int c = 0; c < ctas; ++c) index = min(index, s.firsts[c]);
      a.tokens[row] = index;
      a.chances[row] = 1.f;
    }
    return;
  }

  // Exact sums of weights by step or digit: words of 15 bits, which hold the 2^17 entries
  // that a slice has at most.  Three 32-bit shared atomics take 7 cycles a warp, one of 64
  // bits 20 to 34.
  auto clear_wide = [&] {
    for (int b = tid; b < kSampleBins; b += kSampleThreads) s.wide[0][b] = s.wide[1][b] = s.wide[2][b] = 0;
    __syncthreads();
  };
  auto add_wide = [&](int b, unsigned long long w) {
    atomicAdd(&s.wide[0][b], uint32_t(w) & 0x7fffu);
    atomicAdd(&s.wide[1][b], uint32_t(w >> 15) & 0x7fffu);
    atomicAdd(&s.wide[2][b], uint32_t(w >> 30));
  };
  // This CTA's share of the steps: `share` of them from first_step on, thread t those from
  // first_step + t * per on (threads with t * per >= share: none).
  const int share = kSampleBins / ctas, first_step = rank * share;
  const int per = share > kSampleThreads ? share / kSampleThreads : 1, my_step = first_step + tid * per;
  const bool mine_any = tid * per < share;
  // Adds the cluster's sums of this thread's steps, shifted.  After a cluster barrier;
  // `words` must not change until the next.
  auto gather_words = [&](const uint32_t* words, unsigned long long (&sum)[kSamplePer], int bits) {
    if (!mine_any) return;
#pragma unroll
    for (int j = 0; j < kSamplePer; ++j) {
      if (j >= per) break;
      uint32_t h[kSampleMaxCluster];  // requested together
#pragma unroll
      for (int c = 0; c < kSampleMaxCluster; ++c)
        h[c] = c < ctas ? cluster_word(words + my_step + j, c) : 0;
#pragma unroll
      for (int c = 0; c < kSampleMaxCluster; ++c) sum[j] += static_cast<unsigned long long>(h[c]) << bits;
    }
  };
  // Sums over the cluster's steps before this thread's, and over all.  A cluster barrier.
  struct Sum {
    unsigned long long v, n;  // a measure (mass, count), entries
  };
  int scans = 0;
  auto cluster_scan = [&](Sum own, bool counts_alone, Sum& total) {
    Sum sum, at;
    at.n = block_scan(s, own.n, sum.n);
    at.v = at.n, sum.v = sum.n;
    if (!counts_alone) at.v = block_scan(s, own.v, sum.v);
    scans ^= 1;
    if (tid < ctas) cluster.map_shared_rank(&s, tid)->counts[scans][rank] = make_ulonglong2(sum.v, sum.n);
    cluster.sync();
    total = Sum{0, 0};
    for (int c = 0; c < ctas; ++c) {
      const ulonglong2 other = s.counts[scans][c];
      if (c < rank) at.v += other.x, at.n += other.y;
      total.v += other.x, total.n += other.y;
    }
    return at;
  };
  // The step in which the measure reaches target, what lies before it, the entries before
  // it and in it: the thread that has it tells everybody.  A cluster barrier.
  auto find_step = [&](Sum at, const unsigned long long (&v)[kSamplePer], const unsigned long long (&n)[kSamplePer],
                       unsigned long long target) {
#pragma unroll
    for (int j = 0; j < kSamplePer; ++j) {
      if (at.v < target && at.v + v[j] >= target)
        for (int c = 0; c < ctas; ++c) {
          SampleSmem* other = cluster.map_shared_rank(&s, c);
          other->step_bin = my_step + j;
          other->step_before = at.v;
          other->step_ahead = int(at.n);
          other->step_in = int(n[j]);
        }
      at.v += v[j], at.n += n[j];
    }
    cluster.sync();
  };

  // The rank of the last entry of the shortest prefix, among ranks >= cut, whose count
  // or mass reaches target: radix descent, every CTA alike.
  auto descend = [&](bool mass, unsigned long long target, unsigned long long cut) {
    unsigned long long known = 0, before = 0;  // leading bits of the rank; what lies above them
    for (int level = 55; level >= 0; level -= 11) {
      clear_wide();
      each([&](float f, int i) {
        const unsigned long long r = rank_of(f, i);
        if (f == nothing || r < cut || (level != 55 && (r >> (level + 11)) != known)) return;
        const int b = kSampleBins - 1 - (int(r >> level) & (kSampleBins - 1));  // from the top
        if (mass) add_wide(b, weight(f));
        else atomicAdd(&s.wide[0][b], 1u);
      });
      cluster.sync();
      unsigned long long digit[kSamplePer] = {0, 0, 0, 0};
      gather_words(s.wide[0], digit, 0);
      if (mass) gather_words(s.wide[1], digit, 15), gather_words(s.wide[2], digit, 30);
      const unsigned long long own = (digit[0] + digit[1]) + (digit[2] + digit[3]);
      Sum total, at = cluster_scan(Sum{own, own}, true, total);
      at.v += before;
      find_step(at, digit, digit, target);
      known = (known << 11) | unsigned(kSampleBins - 1 - s.step_bin);
      before = s.step_before;
      __syncthreads();
    }
    return known;
  };

  // ---- lists: entries gathered in each CTA, then brought together in the first one
  auto keep = [&](float f, int i) {
    const int at = atomicAdd(&s.listed, 1);
    if (at < kSampleList) s.list[at] = rank_of(f, i);
  };
  // After a cluster barrier: the first CTA's list becomes everybody's; their number.
  auto bring = [&] {
    int from[kSampleMaxCluster + 1];
    from[0] = 0;
#pragma unroll
    for (int c = 0; c < kSampleMaxCluster; ++c)
      from[c + 1] = from[c] + (c < ctas ? cluster.map_shared_rank(&s, c)->listed : 0);
    if (rank == 0 && from[kSampleMaxCluster] <= kSampleList)
      for (int i = from[1] + tid; i < from[kSampleMaxCluster]; i += kSampleThreads) {
        int c = 1, at = i - from[1];
#pragma unroll
        for (int q = 2; q < kSampleMaxCluster; ++q)
          if (i >= from[q]) c = q, at = i - from[q];
        s.list[i] = cluster.map_shared_rank(&s, c)->list[at];
      }
    return from[kSampleMaxCluster];
  };
  auto mass_target = [&](unsigned long long mass) {
    const unsigned long long t = (unsigned long long)(ceil(double(p) * double(mass)));
    return t < 1 ? 1ull : (t > mass ? mass : t);
  };
  // weights that pass min-p, in steps of 2^-44
  const unsigned long long enough = (unsigned long long)ceil(double(least) * double(1ull << kWeightBits));

  const bool by_rank = k > 0 && k < a.vocab, by_mass = p < 1.f;
  auto draw = [&](int i, unsigned long long w, unsigned long long all) {
    a.tokens[row] = i;
    a.chances[row] = float(double(w) / double(all));
  };
  auto border_of = [&](unsigned long long all) { return (unsigned long long)(double(u) * double(all)); };
  // The first CTA, with every entry that may be kept (at most kSampleFew) in its list: the
  // rest of the filters and the draw.  `limit` entries by rank; `mass`: what p refers to, or 0 for theirs.
  auto finish = [&](int n, int limit, unsigned long long mass) {
    constexpr int kShare = kSampleThreads / kSampleFew;
    // four threads per entry compare it with all: how many and how much lie above it
    const int e = tid / kShare, part = tid % kShare;
    __syncthreads();
    const unsigned long long r = e < n ? s.list[e] : 0;
    const unsigned long long w = e < n ? weight(rank_value(r)) : 0;
    unsigned long long* weights = s.list + kSampleFew;
    if (part == 0) weights[e] = w;
    __syncthreads();
    int ahead = 0;
    unsigned long long above = 0;
    for (int j = part; j < n; j += kShare) {
      const bool more = s.list[j] > r;
      ahead += more;
      above += more ? weights[j] : 0;
    }
#pragma unroll
    for (int o = 1; o < kShare; o <<= 1) {
      ahead += __shfl_xor_sync(~0u, ahead, o);
      above += __shfl_xor_sync(~0u, above, o);
    }
    const bool in = e < n && ahead < limit;
    unsigned long long all;
    block_scan(s, in && part == 0 ? w : 0, all);  // also: the weights have been read
    const unsigned long long target = by_mass ? mass_target(mass == 0 ? all : mass) : ~0ull;
    const unsigned long long stays = in && above < target && w >= enough ? w : 0;
    if (part == 0) weights[e] = stays;
    __syncthreads();
    unsigned long long before = 0;
    all = 0;
    for (int j = part; j < n; j += kShare) {
      const unsigned long long v = weights[j];
      all += v;
      before += uint32_t(s.list[j]) > uint32_t(r) ? v : 0;  // a lower index
    }
#pragma unroll
    for (int o = 1; o < kShare; o <<= 1) {
      all += __shfl_xor_sync(~0u, all, o);
      before += __shfl_xor_sync(~0u, before, o);
    }
    const unsigned long long border = border_of(all);
    if (part == 0 && before <= border && before + stays > border) draw(int(0xffffffffu - uint32_t(r)), stays, all);
  };
  // Every CTA, after a barrier behind its list: once the first one has read the lists they
  // may leave; it draws.  False (alike in all) when there are too many entries.
  auto finish_alone = [&](int limit, unsigned long long mass) {
    const int n = bring();
    if (n > kSampleFew) return false;
    auto read = cluster.barrier_arrive();
    if (rank == 0) finish(n, limit, mass);
    cluster.barrier_wait(std::move(read));
    return true;
  };
  // The first CTA, with n entries of step `bin` in its list: the rank of the one at which
  // their count, or mass, reaches target.  A finer histogram of the step, then the entries
  // of one of its parts.
  auto rank_listed = [&](int n, bool mass, unsigned long long target, auto&& part_of) {
    for (int b = tid; b < kSampleBins; b += kSampleThreads) s.hist[b] = 0;
    if (mass)
      for (int b = tid; b < kSampleBins; b += kSampleThreads) s.wide[0][b] = s.wide[1][b] = s.wide[2][b] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kSampleThreads) {
      const float f = rank_value(s.list[i]);
      const int b = part_of(f);
      atomicAdd(&s.hist[b], 1u);
      if (mass) add_wide(b, weight(f));
    }
    __syncthreads();
    unsigned long long v[kSamplePer], own = 0, all;
#pragma unroll
    for (int j = 0; j < kSamplePer; ++j) {
      const int b = tid * kSamplePer + j;
      v[j] = !mass ? s.hist[b]
                   : s.wide[0][b] + (static_cast<unsigned long long>(s.wide[1][b]) << 15) +
                         (static_cast<unsigned long long>(s.wide[2][b]) << 30);
      own += v[j];
    }
    unsigned long long at = block_scan(s, own, all);
#pragma unroll
    for (int j = 0; j < kSamplePer; ++j) {
      if (at < target && at + v[j] >= target) s.found_bin = tid * kSamplePer + j, s.found_before = at;
      at += v[j];
    }
    if (tid == 0) s.found_last = 0;
    __syncthreads();
    const int part = s.found_bin;
    const unsigned long long before = s.found_before;
    unsigned long long* some = reinterpret_cast<unsigned long long*>(s.wide);  // 24 KB: every entry fits
    for (int i = tid; i < n; i += kSampleThreads) {
      const unsigned long long r = s.list[i];
      if (part_of(rank_value(r)) == part) some[atomicAdd(&s.found_last, 1)] = r;
    }
    __syncthreads();
    const int m = s.found_last;
    if (m > 1) block_sort(some, m);
    // entry by entry from the top (a part holds one entry as a rule; many when they are equal)
    unsigned long long cut = some[0];
    if (!mass) {
      cut = some[target - before - 1];
    } else if (m > 1) {
      const int each_has = (m + kSampleThreads - 1) / kSampleThreads, i0 = min(tid * each_has, m),
                i1 = min(i0 + each_has, m);
      own = 0;
      for (int i = i0; i < i1; ++i) own += weight(rank_value(some[i]));
      unsigned long long run = before + block_scan(s, own, all);
      for (int i = i0; i < i1; ++i) {
        const unsigned long long w = weight(rank_value(some[i]));
        if (run < target && run + w >= target) s.found_through = some[i];
        run += w;
      }
      __syncthreads();
      cut = s.found_through;
    }
    if (tid < ctas) cluster.map_shared_rank(&s, tid)->cut = cut;
  };

  // ---- filters: the prefix of ranks >= cut
  unsigned long long cut = 0;
  if (by_rank || by_mass) {
    // steps below the maximum: as far as weights count (2^-44), or the row reaches
    float reach = heat * 30.6f;
    if (heat > 1.5f) {  // the row may end long before: steps of such a temperature would be too wide
      float low = CUDART_INF_F;
      each([&](float f, int) { low = fminf(low, f > nothing ? f : low); });
#pragma unroll
      for (int o = 16; o; o >>= 1) low = fminf(low, __shfl_xor_sync(~0u, low, o));
      if (lane == 0) s.extremes[warp] = low;
      __syncthreads();
      if (tid < ctas) {
        for (int w = 0; w < kSampleWarps; ++w) low = fminf(low, s.extremes[w]);
        cluster.map_shared_rank(&s, tid)->lows[rank] = low;
      }
      cluster.sync();
      for (int c = 0; c < ctas; ++c) low = fminf(low, s.lows[c]);
      reach = fminf(reach, top - low);
    }
    const float per_step = reach > 0.f ? float(kSampleBins) / reach : 0.f;
    // one value only, or a temperature whose steps are no normal numbers: all in step 0
    const bool binned = per_step > 0.f && per_step < CUDART_INF_F && heat > 1e-30f;
    // where f lies among the steps; its step; whether that is at most b, or below it
    auto place_of = [&](float f) { return binned ? (top - f) * per_step : 0.f; };
    auto bin_of = [&](float f) { return int(fminf(place_of(f), float(kSampleBins - 1))); };
    // up_to(place, bound_after(b)): step <= b.  Places may be infinite (a mask's lowest value
    // over a small step), and all of them are in the last step: no bound, as a NaN
    auto bound_after = [&](int b) { return b < kSampleBins - 1 ? float(b + 1) : CUDART_NAN_F; };
    auto up_to = [](float place, float bound) { return !(place >= bound); };
    auto part_of = [&](int bin) {  // of step `bin`, in kSampleBins parts
      return [=](float f) {
        return int(fminf(fmaxf((place_of(f) - float(bin)) * float(kSampleBins), 0.f), float(kSampleBins - 1)));
      };
    };
    unsigned long long count[kSamplePer] = {0, 0, 0, 0};
    Sum total;

    if (by_rank && k <= 100) {  // hardly ever more than kSampleFew entries then
      // the steps of the threads' maxima (148 rows of 128000: 82 us; k = 101, counted, 125)
      if (most != nothing) atomicAdd(&s.hist[bin_of(most)], 1u);
      cluster.sync();
      gather_words(s.hist, count, 0);
      const unsigned long long own = (count[0] + count[1]) + (count[2] + count[3]);
      const Sum at = cluster_scan(Sum{own, own}, true, total);
      if (unsigned(k) <= total.n) {
        find_step(at, count, count, unsigned(k));
        const float bound = bound_after(s.step_bin);
        each([&](float f, int i) {
          if (up_to(place_of(f), bound) && f != nothing) keep(f, i);
        });
        cluster.sync();
        if (finish_alone(k, 0)) return;
      }
      // too many of them: the ordinary way, from the start
      cluster.sync();
      if (tid == 0) s.listed = 0;
      for (int b = tid; b < kSampleBins; b += kSampleThreads) s.hist[b] = 0;
#pragma unroll
      for (int j = 0; j < kSamplePer; ++j) count[j] = 0;
      __syncthreads();
    }
    if (by_rank) {
      // the last step holds all that is far below (a mask's low value): counted by thread
      uint32_t tail = 0;
      each([&](float f, int) {
        const float at = place_of(f);
        const bool counts = f != nothing;  // -inf is never drawn, and all that lies off the row
        if (at >= float(kSampleBins - 1) || !binned) tail += counts;
        else if (counts) atomicAdd(&s.hist[int(at)], 1u);
      });
      tail = __reduce_add_sync(~0u, tail);
      if (lane == 0 && tail > 0) atomicAdd(&s.hist[binned ? kSampleBins - 1 : 0], tail);
      cluster.sync();
      gather_words(s.hist, count, 0);
      const unsigned long long own = (count[0] + count[1]) + (count[2] + count[3]);
      const Sum at = cluster_scan(Sum{own, own}, true, total);
      if (unsigned(k) < total.n) {
        find_step(at, count, count, unsigned(k));
        const int bin = s.step_bin, before = s.step_ahead, in = s.step_in;
        if (in <= kSampleList) {
          const float from = float(bin), bound = bound_after(bin);
          each([&](float f, int i) {
            const float at = place_of(f);
            if (at >= from && up_to(at, bound) && f != nothing) keep(f, i);
          });
          cluster.sync();
          const int n = bring();
          if (rank == 0) rank_listed(n, false, unsigned(k - before), part_of(bin));
          cluster.sync();
          cut = s.cut;
        } else {
          cut = descend(false, unsigned(k), 0);
        }
      }
    }
    if (by_mass) {
      // the exact masses of the steps' entries in the prefix, and their number
      __syncthreads();
      if (tid == 0) s.listed = 0;
      for (int b = tid; b < kSampleBins; b += kSampleThreads) s.hist[b] = 0;
      clear_wide();
      const float cut_at = cut == 0 ? nothing : rank_value(cut);
      each_four([&](const float (&f)[kFour], int i) {
        if (cut != 0) {
          bool any = false;
#pragma unroll
          for (int j = 0; j < kFour; ++j) any |= f[j] >= cut_at;
          if (!any) return;
        }
        unsigned long long w[kFour];
#pragma unroll
        for (int j = 0; j < kFour; ++j) w[j] = weight(f[j]);
#pragma unroll
        for (int j = 0; j < kFour; ++j) {
          if (w[j] == 0 || (cut != 0 && (f[j] < cut_at || rank_of(f[j], i + j) < cut))) continue;
          const int b = bin_of(f[j]);
          atomicAdd(&s.hist[b], 1u);
          add_wide(b, w[j]);
        }
      });
      cluster.sync();
      unsigned long long mass[kSamplePer] = {0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < kSamplePer; ++j) count[j] = 0;
      gather_words(s.hist, count, 0);
      gather_words(s.wide[0], mass, 0);
      gather_words(s.wide[1], mass, 15);
      gather_words(s.wide[2], mass, 30);
      const Sum at = cluster_scan(Sum{(mass[0] + mass[1]) + (mass[2] + mass[3]), (count[0] + count[1]) + (count[2] + count[3])},
                                  false, total);
      const unsigned long long target = mass_target(total.v);
      // the step that the target lies in, and its entries (with all above them, if they are few)
      find_step(at, mass, count, target);
      const int bin = s.step_bin, ahead = s.step_ahead, in = s.step_in;
      const unsigned long long over = s.step_before;
      const bool whole = cut == 0 && ahead + in <= kSampleFew;
      if (in <= kSampleList) {
        const float from = whole ? 0.f : float(bin), bound = bound_after(bin);
        each([&](float f, int i) {
          const float at = place_of(f);
          // what the steps counted, and nothing else: the list has room for that
          if (at >= from && up_to(at, bound) && (cut == 0 || rank_of(f, i) >= cut) && weight(f) != 0) keep(f, i);
        });
        cluster.sync();
        if (whole && finish_alone(kSampleFew, total.v)) return;
        const int n = bring();
        if (rank == 0) rank_listed(n, true, target - over, part_of(bin));
        cluster.sync();
        cut = s.cut;
      } else {
        cut = descend(true, target, cut);
      }
    }
  }

  // ---- the kept weights, warp by warp in vocabulary order, four consecutive places a lane
  const float cut_at = cut == 0 ? nothing : rank_value(cut);
  // below it no weight passes min-p (the margin covers the rounding of all three terms)
  const float lowest =
      least > 0.f ? fmaxf(weight.floor, top + heat * logf(least) - 1e-6f * (fabsf(top) + heat * 120.f)) : weight.floor;
  auto values = [&](int v, float (&f)[kFour]) {  // of places first + v ..
#pragma unroll
    for (int j = 0; j < kFour; ++j) f[j] = nothing;
    if (v < a.slice) {  // a multiple of four
      if constexpr (W) {
        const float4 g = *reinterpret_cast<const float4*>(held + v);
        f[0] = g.x, f[1] = g.y, f[2] = g.z, f[3] = g.w;
      } else {
        const uint2 g = *reinterpret_cast<const uint2*>(held + v);
        f[0] = __uint_as_float(g.x << 16), f[1] = __uint_as_float(g.x & 0xffff0000u);
        f[2] = __uint_as_float(g.y << 16), f[3] = __uint_as_float(g.y & 0xffff0000u);
      }
    }
  };
  auto kept = [&](int v, unsigned long long (&w)[kFour]) {
    float f[kFour];
    values(v, f);
    bool any = false;
#pragma unroll
    for (int j = 0; j < kFour; ++j) any |= f[j] >= cut_at && f[j] >= lowest, w[j] = 0;
    if (!__any_sync(~0u, any)) return;
#pragma unroll
    for (int j = 0; j < kFour; ++j) w[j] = weight(f[j]);
    if (cut != 0) {
#pragma unroll
      for (int j = 0; j < kFour; ++j)
        if (f[j] < cut_at || (f[j] == cut_at && rank_of(f[j], base + v + j) < cut)) w[j] = 0;
    }
    if (least > 0.f) {
#pragma unroll
      for (int j = 0; j < kFour; ++j)
        if (w[j] < enough) w[j] = 0;
    }
  };
  constexpr int kTurn = 32 * kFour;  // places of a warp at a time
  const int seg = ((a.slice + kSampleWarps - 1) / kSampleWarps + kTurn - 1) / kTurn * kTurn, start = warp * seg;
  unsigned long long own = 0, all = 0;
  if (cut == 0 && least == 0.f) {
    for (int v = start + lane * kFour; v < start + seg; v += kTurn) {
      unsigned long long w[kFour];
      kept(v, w);
      own += (w[0] + w[1]) + (w[2] + w[3]);
    }
  } else {
    // the kept values side by side first, so that weights are formed of them alone
    constexpr int kRoom = kSampleList * 8 / 4 / kSampleWarps / 4 * 4;  // 248 of a warp
    static_assert(kRoom >= kTurn - 8 + 64, "two rows of 32 fit behind what is not formed yet");
    float* side = reinterpret_cast<float*>(s.list) + warp * kRoom;
    int n = 0;
    auto form = [&](int m) {  // the first m <= kTurn
#pragma unroll
      for (int j = 0; j < kFour; ++j) {
        const float f = j * 32 + lane < m ? side[j * 32 + lane] : nothing;
        const unsigned long long w = weight(f);
        own += w >= enough ? w : 0;
      }
    };
    __syncthreads();
    for (int v = start + lane * kFour; v - lane * kFour < start + seg; v += kTurn) {
      float f[kFour];
      values(v, f);
#pragma unroll
      for (int j = 0; j < kFour; ++j) {
        const bool stays = f[j] >= lowest && f[j] >= cut_at &&
                           (f[j] > cut_at || rank_of(f[j], base + v + j) >= cut);
        const unsigned who = __ballot_sync(~0u, stays);
        if (stays) side[n + __popc(who & ((1u << lane) - 1))] = f[j];
        n += __popc(who);
        if (j % 2 == 1 && n >= kTurn - 8) {  // at most 64 more come before the next look
          __syncwarp();
          form(min(n, kTurn));
          __syncwarp();
          const int rest = n - min(n, kTurn);
          const float moved = lane < rest ? side[kTurn + lane] : 0.f, moved2 = lane + 32 < rest ? side[kTurn + 32 + lane] : 0.f;
          __syncwarp();
          if (lane < rest) side[lane] = moved;
          if (lane + 32 < rest) side[32 + lane] = moved2;
          n = rest;
          __syncwarp();
        }
      }
    }
    __syncwarp();
    form(n);
  }
  own = warp_sum(own);
  __syncthreads();
  if (lane == 0) s.part[warp] = own;
  __syncthreads();
  if (tid < ctas) {
    for (int w = 0; w < kSampleWarps; ++w) all += s.part[w];
    cluster.map_shared_rank(&s, tid)->kept[rank] = all;
  }
  cluster.sync();
  unsigned long long at = 0;
  all = 0;
  for (int c = 0; c < ctas; ++c) {
    if (c < rank) at += s.kept[c];
    all += s.kept[c];
  }
  for (int w = 0; w < warp; ++w) at += s.part[w];
  const unsigned long long border = border_of(all);  // the sum that has to be exceeded
  if (at <= border && at + own > border) {
    for (int v = start + lane * kFour; v - lane * kFour < start + seg; v += kTurn) {
      unsigned long long w[kFour];
      kept(v, w);
      const unsigned long long mine = (w[0] + w[1]) + (w[2] + w[3]);
      unsigned long long run = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const unsigned long long up = __shfl_up_sync(~0u, run, d);
        if (lane >= d) run += up;
      }
      const unsigned hit = __ballot_sync(~0u, at + run > border);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          unsigned long long upto = at + run - mine;
#pragma unroll
          for (int j = 0; j < kFour; ++j) {
            if (upto <= border && upto + w[j] > border) draw(base + v + j, w[j], all);
            upto += w[j];
          }
        }
        break;
      }
      at += __shfl_sync(~0u, run, 31);
    }
  }
}

static_assert(sizeof(SampleSmem) <= 50160, "two CTAs with 65,552 bytes of a row each share an SM");

template <bool W>
int launch_sample(SampleArgs& a, int64_t rows, cudaStream_t stream) {
  constexpr int64_t kVec = SampleRow<W>::kVec;
  // CTAs per row: enough that two slices fit an SM, and as many as fill the GPU where rows
  // are few and slices stay above 2048 entries.  One row of 32000: 14.4 us with 8, 18.5 with
  // 1; 300 rows of 8000: 28.7 with 1, 104 with 8.  148 rows of 128000 need 8 for two slices
  // an SM, or 4 for one: 188 against 217 us by top_p alone, 80 against 78 with top_k 50 (511
  // rows: 244 against 223); the settings are not known here
  int ctas = 1;
  while (ctas < kSampleMaxCluster &&
         (int64_t(a.vocab) * int64_t(16 / kVec) > int64_t(ctas) * 66000 ||
          (rows * ctas < sm_count() && a.vocab > 2 * ctas * 2048)))
    ctas *= 2;
  a.slice = int(((a.vocab + kVec - 1 + ctas - 1) / ctas + kVec - 1) / kVec * kVec);
  const size_t smem = sizeof(SampleSmem) + size_t(a.slice) * (16 / kVec);
  const int rc = set_max_smem(sample_kernel<W>, 232448, "sample");
  if (rc != DSR_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(rows * ctas), 1, 1);
  cfg.blockDim = dim3(kSampleThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(ctas);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel<W>, a);
  if (e != cudaSuccess) return fail(DSR_ECUDA, "sample launch: %s", cudaGetErrorString(e));
  return DSR_OK;
}

}  // namespace
}  // namespace dsr

extern "C" int dsr_sample(const void* logits, int dtype, int64_t row_stride, int64_t vocab, const float* temperature,
                          const int32_t* top_k, const float* top_p, const float* min_p, const float* uniform,
                          int32_t* tokens, float* chances, int32_t* err, int64_t rows, void* stream) {
  using namespace dsr;
  clear_error();
  DSR_REQUIRE(logits && temperature && top_k && top_p && min_p && uniform && tokens && chances && err,
              "sample: null pointer");
  DSR_REQUIRE(dtype == DSR_BF16 || dtype == DSR_F32, "sample: unknown element type %d", dtype);
  DSR_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (dtype == DSR_F32 ? 4 : 2) == 0, "sample: misaligned logits");
  DSR_REQUIRE(vocab > 0 && vocab <= kSampleMaxVocab, "sample: vocabulary %lld outside [1, %d]", (long long)vocab,
              kSampleMaxVocab);
  DSR_REQUIRE(rows > 0 && rows <= 65535, "sample: rows %lld outside [1, 65535]", (long long)rows);
  DSR_REQUIRE(row_stride >= 0, "sample: negative row stride");
  SampleArgs a{logits, row_stride, int(vocab), 0, temperature, top_k, top_p, min_p, uniform, tokens, chances, err};
  return dtype == DSR_F32 ? launch_sample<true>(a, rows, as_stream(stream))
                          : launch_sample<false>(a, rows, as_stream(stream));
}
