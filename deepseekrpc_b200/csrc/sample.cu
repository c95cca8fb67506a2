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
// read from memory once.  Prefixes are found from a histogram of counts over 2048 equal
// steps of the value below the maximum: it says exactly which step holds rank k, and,
// since the weights of a step are known to within its width, between which two steps
// the mass p lies (where those hold too many entries, their exact masses say which).
// Only the entries there are ranked, in the first CTA, on the unique 64-bit rank
// (order-preserving value, inverted index) with exact weights.  Where the steps hold too many entries (equal logits, masks), the prefix comes from a
// radix descent over the ranks instead, 11 bits a level.
#include <cooperative_groups.h>
#include <math_constants.h>

#include <cfloat>
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
constexpr int kSampleList = 2048;  // entries ranked by the sort
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
  float floor;          // below: no weight (2^-60 of the largest, or -inf)
  // The weight in the fixed point's steps, plus the bits of 2^(52 - kWeightBits).
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
  // what a weight is in steps of 2^-44, rounded
  __device__ __forceinline__ unsigned long long operator()(float x) const {
    const double w = shifted(x);
    const unsigned long long bits = (unsigned long long)__double_as_longlong(w) - (unsigned long long)__double_as_longlong(kMagic);
    return x >= floor ? bits : 0;
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
  unsigned long long part[kSampleWarps], part2[kSampleWarps];
  float2 bounds[kSampleWarps];
  // written by every CTA of the cluster for all
  unsigned long long best[kSampleMaxCluster], sums[kSampleMaxCluster], above[kSampleMaxCluster],
      kept[kSampleMaxCluster];
  float low[kSampleMaxCluster];
  int bad[kSampleMaxCluster];
  // written by the first CTA for all
  unsigned long long cut;
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

// Bitonic sort of list[0, n), n <= kSampleThreads * Q, in descending (or ascending)
// order; thread t holds the entries t, t + kSampleThreads, ..: exchanges over less than
// a warp go by shuffles, over a warp or more through the list itself.
template <int Q, bool Descending>
__device__ __forceinline__ void block_sort(unsigned long long* list, int n) {
  const int tid = threadIdx.x;
  unsigned long long v[Q];
  __syncthreads();
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int e = q * kSampleThreads + tid;
    v[q] = e < n ? list[e] : (Descending ? 0 : ~0ull);
  }
  for (int size = 2; size < 2 * n; size <<= 1)
    for (int gap = size >> 1; gap > 0; gap >>= 1) {
      unsigned long long other[Q];
      if (gap >= kSampleThreads) {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          other[q] = v[q ^ 1];
          if (Q > 2 && gap == 2 * kSampleThreads) other[q] = v[(q ^ 2) % Q];
        }
      } else if (gap >= 32) {
        __syncthreads();
#pragma unroll
        for (int q = 0; q < Q; ++q) list[q * kSampleThreads + tid] = v[q];
        __syncthreads();
#pragma unroll
        for (int q = 0; q < Q; ++q) other[q] = list[(q * kSampleThreads + tid) ^ gap];
      } else {
#pragma unroll
        for (int q = 0; q < Q; ++q) other[q] = __shfl_xor_sync(~0u, v[q], gap);
      }
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int e = q * kSampleThreads + tid;
        const bool ascends = ((e & size) == 0) != Descending, smaller = ((e & gap) == 0) == ascends;
        if (smaller == (other[q] < v[q])) v[q] = other[q];
      }
    }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < Q; ++q) list[q * kSampleThreads + tid] = v[q];
  __syncthreads();
}
template <bool Descending>
__device__ __forceinline__ void block_sort_any(unsigned long long* list, int n) {
  static_assert(kSampleList == 4 * kSampleThreads, "");
  if (n <= kSampleThreads) block_sort<1, Descending>(list, n);
  else block_sort<4, Descending>(list, n);
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
  if (tid < 16) s.table[tid] = exp2(tid / 16.0);
  if (tid == 0) s.listed = 0;
  for (int b = tid; b < kSampleBins; b += kSampleThreads) s.hist[b] = 0;

  // ---- the slice into shared memory (places off the row: -inf); extremes, non-finite values
  const float nothing = -CUDART_INF_F;
  float most = nothing, low = CUDART_INF_F;
  int at_most = 0;
  int bad = 0;
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
        bad |= !(f < CUDART_INF_F);
        if (f > most) most = f, at_most = base + v + j;  // the first of equal ones
        low = fminf(low, f > nothing ? f : low);
      }
    }
  }
  unsigned long long best = rank_of(most, at_most);
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const unsigned long long r = __shfl_xor_sync(~0u, best, o);
    best = r > best ? r : best;
    low = fminf(low, __shfl_xor_sync(~0u, low, o));
  }
  if (lane == 0) s.part[warp] = best, s.bounds[warp].x = low;
  bad = __syncthreads_or(bad);
  cluster.barrier_wait(std::move(started));
  if (tid < ctas) {  // thread c tells CTA c
    for (int w = 0; w < kSampleWarps; ++w) {
      best = s.part[w] > best ? s.part[w] : best;
      low = fminf(low, s.bounds[w].x);
    }
    SampleSmem* other = cluster.map_shared_rank(&s, tid);
    other->best[rank] = best;
    other->low[rank] = low;
    other->bad[rank] = bad;
  }
  cluster.sync();
  bad = 0;
  for (int c = 0; c < ctas; ++c) {
    best = s.best[c] > best ? s.best[c] : best;
    low = fminf(low, s.low[c]);
    bad |= s.bad[c];
  }
  const float top = rank_value(best);
  const bool valid = heat >= 0.f && heat < CUDART_INF_F && p >= 0.f && p <= 1.f && least >= 0.f && least <= 1.f &&
                     u >= 0.f && u < 1.f && k >= 0;
  if (bad || !valid || top == nothing || heat == 0.f) {  // alike in all CTAs
    if (rank == 0 && tid == 0) {
      if (bad) flag(a.err, DSR_ERR_NONFINITE);
      else if (!valid) flag(a.err, DSR_ERR_ID);
      const bool greedy = !bad && valid && top != nothing;
      a.tokens[row] = greedy ? int32_t(0xffffffffu - uint32_t(best)) : -1;
      a.chances[row] = greedy ? 1.f : 0.f;
    }
    return;
  }
  // 2^-60 is exp(-41.6); -inf stays out also where that lies below all finite numbers
  const Weight weight{s.table, double(top), 16.0 * kLog2eD / double(heat), fmaxf(top - 41.6f * heat, -FLT_MAX)};

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
  // Adds the cluster's sums of four consecutive words, shifted.
  static_assert(kSamplePer == 4, "a thread's steps are one 16-byte piece");
  auto cluster_words = [&](const uint32_t* words, unsigned long long (&sum)[kSamplePer], int bits) {
    const uint32_t* mine = words + tid * kSamplePer;
    constexpr int kTogether = 4;
#pragma unroll
    for (int c0 = 0; c0 < kSampleMaxCluster; c0 += kTogether) {
      uint4 h[kTogether];
#pragma unroll
      for (int c = 0; c < kTogether; ++c)
        h[c] = c0 + c < ctas ? *reinterpret_cast<const uint4*>(cluster.map_shared_rank(mine, c0 + c))
                             : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int c = 0; c < kTogether; ++c) {
        sum[0] += static_cast<unsigned long long>(h[c].x) << bits, sum[1] += static_cast<unsigned long long>(h[c].y) << bits;
        sum[2] += static_cast<unsigned long long>(h[c].z) << bits, sum[3] += static_cast<unsigned long long>(h[c].w) << bits;
      }
    }
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
      unsigned long long digit[kSamplePer] = {0, 0, 0, 0}, total;
      cluster_words(s.wide[0], digit, 0);
      if (mass) cluster_words(s.wide[1], digit, 15), cluster_words(s.wide[2], digit, 30);
      const unsigned long long own = (digit[0] + digit[1]) + (digit[2] + digit[3]);
      unsigned long long at = before + block_scan(s, own, total);
#pragma unroll
      for (int j = 0; j < kSamplePer; ++j) {
        if (at < target && at + digit[j] >= target) {
          s.found_bin = kSampleBins - 1 - (tid * kSamplePer + j);
          s.found_before = at;
        }
        at += digit[j];
      }
      cluster.sync();  // before the sums are cleared again
      known = (known << 11) | unsigned(s.found_bin);
      before = s.found_before;
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
  // whether a weight passes min-p (compared in steps of 2^-44)
  auto enough = [&](float f) { return least == 0.f || weight.shifted(f) - Weight::kMagic >= double(least); };

  const bool by_rank = k > 0 && k < a.vocab, by_mass = p < 1.f;
  auto draw = [&](int i, unsigned long long w, unsigned long long all) {
    a.tokens[row] = i;
    a.chances[row] = float(double(w) / double(all));
  };
  auto border_of = [&](unsigned long long all) { return (unsigned long long)(double(u) * double(all)); };
  // The first CTA, with every entry that may be kept in its list: the rest of the
  // filters and the draw.  `limit` entries by rank; `mass`: what p refers to, or 0 for theirs.
  auto finish = [&](int n, int limit, unsigned long long mass) {
    constexpr int kFew = 128, kShare = kSampleThreads / kFew;
    if (n <= kFew) {
      // four threads per entry compare it with all: how many and how much lie above it
      const int e = tid / kShare, part = tid % kShare;
      __syncthreads();
      const unsigned long long r = e < n ? s.list[e] : 0;
      const unsigned long long w = e < n ? weight(rank_value(r)) : 0;
      unsigned long long* weights = s.list + kFew;
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
      const unsigned long long stays = in && above < target && enough(rank_value(r)) ? w : 0;
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
      return;
    }
    block_sort_any<true>(s.list, n);
    n = min(n, limit);
    unsigned long long w[kSamplePer], own = 0, all;
    static_assert(kSampleList == kSamplePer * kSampleThreads, "");
#pragma unroll
    for (int j = 0; j < kSamplePer; ++j) {
      const int i = tid * kSamplePer + j;
      w[j] = weight(i < n ? rank_value(s.list[i]) : nothing);
      own += w[j];
    }
    unsigned long long run = block_scan(s, own, all);
    const unsigned long long target = by_mass ? mass_target(mass == 0 ? all : mass) : ~0ull;
    // kept: what is above has not reached the target, and the weight is large enough
    int mine = 0;
    unsigned long long stays[kSamplePer];
#pragma unroll
    for (int j = 0; j < kSamplePer; ++j) {
      const int i = tid * kSamplePer + j;
      stays[j] = 0;
      if (i < n && run < target && w[j] > 0) {
        const unsigned long long r = s.list[i];
        if (enough(rank_value(r))) {
          stays[j] = (static_cast<unsigned long long>(0xffffffffu - uint32_t(r)) << (kWeightBits + 1)) | w[j];
          ++mine;
        }
      }
      run += w[j];
    }
    unsigned long long m;
    int to = int(block_scan(s, unsigned(mine), m));  // also: the list has been read
#pragma unroll
    for (int j = 0; j < kSamplePer; ++j)
      if (stays[j] != 0) s.list[to++] = stays[j];
    block_sort_any<false>(s.list, int(m));  // vocabulary order
    constexpr unsigned long long kMask = (1ull << (kWeightBits + 1)) - 1;
    own = 0;
#pragma unroll
    for (int j = 0; j < kSamplePer; ++j) {
      const int i = tid * kSamplePer + j;
      w[j] = i < int(m) ? s.list[i] & kMask : 0;
      own += w[j];
    }
    run = block_scan(s, own, all);
    const unsigned long long border = border_of(all);
#pragma unroll
    for (int j = 0; j < kSamplePer; ++j) {
      if (run <= border && run + w[j] > border) draw(int(s.list[tid * kSamplePer + j] >> (kWeightBits + 1)), w[j], all);
      run += w[j];
    }
  };
  // Every CTA: after the first one has read their lists they may leave; it draws.
  auto finish_alone = [&](int limit, unsigned long long mass) {
    cluster.sync();
    const int n = bring();
    auto read = cluster.barrier_arrive();
    if (rank == 0) finish(n, limit, mass);
    cluster.barrier_wait(std::move(read));
  };

  // ---- filters: the prefix of ranks >= cut
  unsigned long long cut = 0;
  if (by_rank || by_mass) {
    // steps below the maximum: as far as weights count (2^-44), or the row reaches
    const float reach = fminf(heat * 30.6f, top - low), per_step = reach > 0.f ? float(kSampleBins) / reach : 0.f;
    const float step = reach / float(kSampleBins);  // inverse of per_step
    // one value only, or a temperature whose steps are no normal numbers: all in step 0
    const bool binned = per_step > 0.f && per_step < CUDART_INF_F && heat > 1e-30f;
    auto bin_of = [&](float f) {
      return binned ? int(fminf((top - f) * per_step, float(kSampleBins - 1))) : 0;
    };
    // the last step holds all that is far below (a mask's low value): counted by thread
    uint32_t tail = 0;
    each([&](float f, int) {
      const int b = bin_of(f);
      const bool counts = f != nothing;  // -inf is never drawn, and all that lies off the row
      if (b == kSampleBins - 1 || !binned) tail += counts;
      else if (counts) atomicAdd(&s.hist[b], 1u);
    });
    tail = __reduce_add_sync(~0u, tail);
    if (lane == 0 && tail > 0) atomicAdd(&s.hist[binned ? kSampleBins - 1 : 0], tail);
    cluster.sync();
    // thread t: the counts of steps kSamplePer t .., over all CTAs
    unsigned long long count[kSamplePer] = {0, 0, 0, 0}, total;
    cluster_words(s.hist, count, 0);
    const unsigned long long own = (count[0] + count[1]) + (count[2] + count[3]);
    unsigned long long at = block_scan(s, own, total);

    if (by_rank && unsigned(k) < total) {
#pragma unroll
      for (int j = 0; j < kSamplePer; ++j) {
        if (at < unsigned(k) && at + count[j] >= unsigned(k)) {
          s.found_bin = tid * kSamplePer + j;
          s.found_before = at;
          s.found_last = int(count[j]);
        }
        at += count[j];
      }
      __syncthreads();
      const int bin = s.found_bin, before = int(s.found_before), in = s.found_last;
      if (before + in <= kSampleList) {  // every kept entry fits the list
        each([&](float f, int i) {
          if (bin_of(f) <= bin && f != nothing) keep(f, i);
        });
        finish_alone(k, 0);
        return;
      }
      if (in <= kSampleList) {
        each([&](float f, int i) {
          if (bin_of(f) == bin && f != nothing) keep(f, i);
        });
        cluster.sync();
        const int n = bring();
        if (rank == 0) {
          block_sort_any<true>(s.list, n);
          if (tid < ctas) cluster.map_shared_rank(&s, tid)->cut = s.list[k - before - 1];
        }
        cluster.sync();
        cut = s.cut;
        if (tid == 0) s.listed = 0;
        __syncthreads();
      } else {
        cut = descend(false, unsigned(k), 0);
      }
      // the counts of the prefix, for the mass below
#pragma unroll
      for (int j = 0; j < kSamplePer; ++j) {
        const int b = tid * kSamplePer + j;
        if (b == bin) count[j] = unsigned(k - before);
        else if (b > bin) count[j] = 0;
      }
    }
    if (by_mass) {
      // bounds of the mass up to and including each step, from its counts
      const float fall = step / heat;
      float lo[kSamplePer], hi[kSamplePer], lo_own = 0.f, hi_own = 0.f;
#pragma unroll
      for (int j = 0; j < kSamplePer; ++j) {
        const int b = tid * kSamplePer + j;
        // a hundredth of a step covers the rounding of the step's number
        hi_own += float(count[j]) * expf(-fmaxf(float(b) - 0.01f, 0.f) * fall) * 1.0001f;
        if (b < kSampleBins - 1) lo_own += float(count[j]) * expf(-(float(b) + 1.01f) * fall) * 0.9999f;
        lo[j] = lo_own, hi[j] = hi_own;
      }
      float lo_run = lo_own, hi_run = hi_own;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const float l = __shfl_up_sync(~0u, lo_run, d), h = __shfl_up_sync(~0u, hi_run, d);
        if (lane >= d) lo_run += l, hi_run += h;
      }
      __syncthreads();
      if (lane == 31) s.bounds[warp] = make_float2(lo_run, hi_run);
      if (tid == 0) s.found_bin = kSampleBins, s.found_last = kSampleBins - 1;
      __syncthreads();
      float lo_at = lo_run - lo_own, hi_at = hi_run - hi_own, lo_all = 0.f, hi_all = 0.f;
#pragma unroll
      for (int w = 0; w < kSampleWarps; ++w) {
        const float2 v = s.bounds[w];
        if (w < warp) lo_at += v.x, hi_at += v.y;
        lo_all += v.x, hi_all += v.y;
      }
      // the cut lies past every step whose upper bound is below p times the total's
      // lower one, and no later than the first whose lower bound reaches p times the
      // total's upper one (the sums' own rounding: below 10^-4)
      const float below = p * lo_all * 0.999f, reached = p * hi_all * 1.001f;
      int first_bin = kSampleBins, last_bin = kSampleBins;
#pragma unroll
      for (int j = kSamplePer - 1; j >= 0; --j) {
        const int b = tid * kSamplePer + j;
        if (hi_at + hi[j] >= below) first_bin = b;
        if (lo_at + lo[j] >= reached) last_bin = b;
      }
      first_bin = __reduce_min_sync(~0u, first_bin), last_bin = __reduce_min_sync(~0u, last_bin);
      if (lane == 0) atomicMin(&s.found_bin, first_bin), atomicMin(&s.found_last, last_bin);
      __syncthreads();
      const int from = binned ? s.found_bin : 0, to = binned ? s.found_last : kSampleBins - 1;
      // counts before the one and through the other
      unsigned long long total2;
      unsigned long long upto = block_scan(s, (count[0] + count[1]) + (count[2] + count[3]), total2);
#pragma unroll
      for (int j = 0; j < kSamplePer; ++j) {
        const int b = tid * kSamplePer + j;
        if (b == from) s.found_before = upto;
        upto += count[j];
        if (b == to) s.found_through = upto;
      }
      __syncthreads();
      const unsigned long long before = s.found_before, through = s.found_through;
      const bool whole = cut == 0 && through <= kSampleList, some = whole || through - before <= kSampleList;
      const int list_from = whole ? 0 : from;
      // one pass: the exact mass of the prefix and of its part before step `from`, and the
      // entries of the steps between, where they fit the list, else the steps' exact masses
      if (!some) clear_wide();
      unsigned long long z = 0, over = 0;
      const float cut_at = cut == 0 ? nothing : rank_value(cut);
      each_four([&](const float (&f)[kFour], int i) {
        unsigned long long w[kFour];
#pragma unroll
        for (int j = 0; j < kFour; ++j) w[j] = weight(f[j]);
#pragma unroll
        for (int j = 0; j < kFour; ++j) {
          const bool in = f[j] > cut_at || (f[j] == cut_at && rank_of(f[j], i + j) >= cut);
          w[j] = in ? w[j] : 0;
          z += w[j];
          const int b = bin_of(f[j]);
          over += b < from ? w[j] : 0;
          if (in && b >= list_from && b <= to && f[j] != nothing) {
            if (some) keep(f[j], i + j);
            else add_wide(b, w[j]);
          }
        }
      });
      z = warp_sum(z), over = warp_sum(over);
      if (lane == 0) s.part[warp] = z, s.part2[warp] = over;
      __syncthreads();
      if (tid < ctas) {
        z = over = 0;
        for (int w = 0; w < kSampleWarps; ++w) z += s.part[w], over += s.part2[w];
        SampleSmem* other = cluster.map_shared_rank(&s, tid);
        other->sums[rank] = z;
        other->above[rank] = over;
      }
      cluster.sync();
      z = over = 0;
      for (int c = 0; c < ctas; ++c) z += s.sums[c], over += s.above[c];
      if (whole) {
        finish_alone(kSampleList, z);
        return;
      }
      const unsigned long long target = mass_target(z);
      bool fits = some;
      if (!some) {
        // the step that the target lies in; its entries
        unsigned long long mass[kSamplePer] = {0, 0, 0, 0};
        cluster_words(s.wide[0], mass, 0);
        cluster_words(s.wide[1], mass, 15);
        cluster_words(s.wide[2], mass, 30);
        unsigned long long run = over + block_scan(s, (mass[0] + mass[1]) + (mass[2] + mass[3]), total2);
#pragma unroll
        for (int j = 0; j < kSamplePer; ++j) {
          if (run < target && run + mass[j] >= target) {
            s.found_bin = tid * kSamplePer + j;
            s.found_before = run;
            s.found_last = int(count[j]);
          }
          run += mass[j];
        }
        __syncthreads();
        const int bin = s.found_bin;
        fits = s.found_last <= kSampleList;
        over = s.found_before;
        if (fits) each([&](float f, int i) {
            if (bin_of(f) == bin && f != nothing && rank_of(f, i) >= cut) keep(f, i);
          });
        cluster.sync();
      }
      if (fits) {
        const int n = bring();
        if (rank == 0) {
          block_sort_any<true>(s.list, n);
          unsigned long long w[kSamplePer], own = 0, all;
#pragma unroll
          for (int j = 0; j < kSamplePer; ++j) {
            const int i = tid * kSamplePer + j;
            w[j] = weight(i < n ? rank_value(s.list[i]) : nothing);
            own += w[j];
          }
          unsigned long long run = over + block_scan(s, own, all);
#pragma unroll
          for (int j = 0; j < kSamplePer; ++j) {
            if (run < target && run + w[j] >= target) {
              const unsigned long long r = s.list[tid * kSamplePer + j];
              for (int c = 0; c < ctas; ++c) cluster.map_shared_rank(&s, c)->cut = r;
            }
            run += w[j];
          }
        }
        cluster.sync();
        cut = s.cut;
      } else {
        cut = descend(true, target, cut);
      }
    }
  }

  // ---- the kept weights, warp by warp in vocabulary order, four consecutive places a lane
  const float cut_at = cut == 0 ? nothing : rank_value(cut);
  auto kept = [&](int v, unsigned long long (&w)[kFour]) {  // of places first + v ..
    float f[kFour] = {nothing, nothing, nothing, nothing};
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
    bool any = false;
#pragma unroll
    for (int j = 0; j < kFour; ++j) any |= f[j] >= cut_at && f[j] >= weight.floor, w[j] = 0;
    if (!__any_sync(~0u, any)) return;
#pragma unroll
    for (int j = 0; j < kFour; ++j) w[j] = weight(f[j]);
#pragma unroll
    for (int j = 0; j < kFour; ++j)
      if (f[j] < cut_at || (f[j] == cut_at && rank_of(f[j], base + v + j) < cut)) w[j] = 0;
    if (least > 0.f) {
#pragma unroll
      for (int j = 0; j < kFour; ++j)
        if (!enough(f[j])) w[j] = 0;
    }
  };
  constexpr int kTurn = 32 * kFour;  // places of a warp at a time
  const int seg = ((a.slice + kSampleWarps - 1) / kSampleWarps + kTurn - 1) / kTurn * kTurn, start = warp * seg;
  unsigned long long own = 0, all = 0;
  for (int v = start + lane * kFour; v < start + seg; v += kTurn) {
    unsigned long long w[kFour];
    kept(v, w);
    own += (w[0] + w[1]) + (w[2] + w[3]);
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

template <bool W>
int launch_sample(SampleArgs& a, int64_t rows, cudaStream_t stream) {
  constexpr int64_t kVec = SampleRow<W>::kVec;
  // CTAs per row: enough that a slice leaves room for two more on the SM, and as many
  // as fill the GPU where rows are few and slices stay above 2048 entries
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
