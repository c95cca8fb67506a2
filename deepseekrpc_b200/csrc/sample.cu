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
// Only the entries there are ranked, by a sort in the first CTA on the unique 64-bit rank (order-preserving value, inverted index) with exact weights.
// Where the steps hold too many entries (equal logits, masks), the prefix comes from a
// radix descent over the ranks instead, 11 bits a level.
#include <cooperative_groups.h>
#include <math_constants.h>

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

// exp((x - high) / heat) for x <= high in 64 bits, as 2^(n/64 + r/64): 2^(n/64) from a
// table and an exponent, 2^(r/64), |r| <= 1/2, by the Taylor series of e^(r ln2/64),
// whose first dropped term is below 2^-44 of it.
struct Weight {
  const double* table;  // [64] 2^(j/64)
  double high, scale;   // scale: 64 log2(e) / heat
  __device__ __forceinline__ double operator()(float x) const {
    const double t = (double(x) - high) * scale;
    if (!(t > -64.0 * 60.0)) return 0.0;  // far below half a step of the fixed point
    constexpr double kRound = 6755399441055744.0, c = 0.010830424696249145;  // 1.5 * 2^52; ln(2) / 64
    const double shifted = t + kRound, r = t - (shifted - kRound);
    const int n = __double2loint(shifted);
    double p = fma(r, c * c * c * c / 24, c * c * c / 6);
    p = fma(p, r, c * c / 2);
    p = fma(p, r, c);
    p = fma(p, r, 1.0);
    const double e = table[n & 63];
    return p * __hiloint2double(__double2hiint(e) + (n >> 6) * (1 << 20), __double2loint(e));
  }
};

__device__ __forceinline__ unsigned long long to_fixed(double w) {  // w in [0, 1]
  constexpr double kMagic = double(1ull << (52 - kWeightBits));
  return (unsigned long long)(__double_as_longlong(w + kMagic) - __double_as_longlong(kMagic));
}

__device__ __forceinline__ unsigned long long rank_of(float x, int i) {
  return (static_cast<unsigned long long>(score_key(x)) << 32) | (0xffffffffu - uint32_t(i));
}

struct alignas(16) SampleSmem {
  double table[64];
  unsigned long long list[kSampleList];  // ranks of the entries to sort
  unsigned long long wide[kSampleBins];  // exact masses of steps; radix descent: sums of the digits
  uint32_t hist[kSampleBins];                // this CTA's counts
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

// The block's inclusive sum of x, the exclusive one, and the total.
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

// Sorts v[0, n), n a power of two, in descending (or ascending) order.
template <bool Descending>
__device__ __forceinline__ void block_sort(unsigned long long* v, int n) {
  for (int size = 2; size <= n; size <<= 1)
    for (int gap = size >> 1; gap > 0; gap >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < n / 2; i += kSampleThreads) {
        const int lo = (i & ~(gap - 1)) * 2 + (i & (gap - 1)), hi = lo + gap;
        const bool up = ((lo & size) == 0) != Descending;  // this run ascends
        const unsigned long long x = v[lo], y = v[hi];
        if ((x > y) == up) v[lo] = y, v[hi] = x;
      }
    }
  __syncthreads();
}

template <bool W>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const SampleArgs a) {
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
  const int first = rank * a.slice, base = first - shift;  // entry of place `first`
  const int end = a.vocab + shift;

  const float heat = a.temperature[row], p = a.top_p[row], least = a.min_p[row], u = a.uniform[row];
  const int k = a.top_k[row];
  auto started = cluster.barrier_arrive();  // every CTA is there before one writes to another
  if (tid < 64) s.table[tid] = exp2(tid / 64.0);
  if (tid == 0) s.listed = 0;
  for (int b = tid; b < kSampleBins; b += kSampleThreads) s.hist[b] = 0;

  // ---- the slice into shared memory (places off the row: -inf); extremes, non-finite values
  const float nothing = -CUDART_INF_F;
  float most = nothing, low = CUDART_INF_F;
  int at_most = 0;
  int bad = 0;
  for (int v = tid * kVec; v < a.slice; v += kSampleThreads * kVec) {
    const int place = first + v;
    uint4 raw;
    T* t = reinterpret_cast<T*>(&raw);
    if (place >= shift && place + kVec <= end) {
      raw = __ldg(reinterpret_cast<const uint4*>(x + (place - shift)));
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const int q = place + j;
        if constexpr (W) t[j] = q >= shift && q < end ? x[q - shift] : nothing;
        else t[j] = q >= shift && q < end ? x[q - shift] : uint16_t(0xff80);
      }
    }
    *reinterpret_cast<uint4*>(held + v) = raw;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const float f = Row::value(t[j]);
      bad |= !(f < CUDART_INF_F);
      if (f > most) most = f, at_most = base + v + j;  // the first of equal ones
      if (f > nothing) low = fminf(low, f);
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
  const float top = key_score(uint32_t(best >> 32));
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
  const Weight weight{s.table, double(top), 64.0 * kLog2eD / double(heat)};

  // each(f): f(value, entry) for this CTA's entries (and places off the row, as -inf)
  auto each = [&](auto&& f) {
    for (int v = tid * kVec; v < a.slice; v += kSampleThreads * kVec) {
      const uint4 raw = *reinterpret_cast<const uint4*>(held + v);
      const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int j = 0; j < kVec; ++j) f(Row::value(t[j]), base + v + j);
    }
  };

  // The rank of the last entry of the shortest prefix, among ranks >= cut, whose count
  // or mass reaches target: radix descent, every CTA alike.
  auto descend = [&](bool mass, unsigned long long target, unsigned long long cut) {
    unsigned long long known = 0, before = 0;  // leading bits of the rank; what lies above them
    for (int level = 55; level >= 0; level -= 11) {
      for (int b = tid; b < kSampleBins; b += kSampleThreads) s.wide[b] = 0;
      __syncthreads();
      each([&](float f, int i) {
        const unsigned long long r = rank_of(f, i);
        if (f != nothing && r >= cut && (level == 55 || (r >> (level + 11)) == known))
          atomicAdd(&s.wide[(r >> level) & (kSampleBins - 1)], mass ? to_fixed(weight(f)) : 1ull);
      });
      cluster.sync();
      // thread t holds the digits from the top, kSamplePer each, over all CTAs
      unsigned long long digit[kSamplePer], own = 0, total;
#pragma unroll
      for (int j = 0; j < kSamplePer; ++j) {
        const int b = kSampleBins - 1 - (tid * kSamplePer + j);
        digit[j] = 0;
        for (int c = 0; c < ctas; ++c) digit[j] += cluster.map_shared_rank(&s, c)->wide[b];
        own += digit[j];
      }
      unsigned long long at = before + block_scan(s, own, total);
      if (at < target && at + own >= target) {
        int j = 0;
#pragma unroll
        for (int q = 0; q < kSamplePer - 1; ++q)
          if (j == q && at + digit[q] < target) at += digit[q], ++j;
        s.found_bin = kSampleBins - 1 - (tid * kSamplePer + j);
        s.found_before = at;
      }
      cluster.sync();  // before the masses are cleared again
      known = (known << 11) | unsigned(s.found_bin);
      before = s.found_before;
      __syncthreads();
    }
    return known;
  };

  // ---- filters: the prefix of ranks >= cut
  unsigned long long cut = 0;
  const bool by_rank = k > 0 && k < a.vocab, by_mass = p < 1.f;
  if (by_rank || by_mass) {
    // steps below the maximum: as far as weights count (2^-44), or the row reaches
    const float reach = fminf(heat * 30.6f, top - low), per_step = reach > 0.f ? float(kSampleBins) / reach : 0.f;
    const float step = reach / float(kSampleBins);  // inverse of per_step
    auto bin_of = [&](float f) { return int(fminf((top - f) * per_step, float(kSampleBins - 1))); };
    // one value only, or a temperature whose steps are no normal numbers: all in step 0
    const bool binned = per_step > 0.f && per_step < CUDART_INF_F && heat > 1e-30f;
    // the last step holds all that is far below (a mask's low value): counted by thread
    uint32_t tail = 0;
    each([&](float f, int) {
      if (f == nothing) return;  // never drawn, and all that lies off the row
      const int b = binned ? bin_of(f) : 0;
      if (b == kSampleBins - 1 || !binned) ++tail;
      else atomicAdd(&s.hist[b], 1u);
    });
    tail = __reduce_add_sync(~0u, tail);
    if (lane == 0 && tail > 0) atomicAdd(&s.hist[binned ? kSampleBins - 1 : 0], tail);
    cluster.sync();
    // thread t: the counts of steps kSamplePer t .., over all CTAs
    uint32_t count[kSamplePer];
    unsigned long long own = 0, total;
#pragma unroll
    for (int j = 0; j < kSamplePer; ++j) count[j] = 0;
    for (int c = 0; c < ctas; ++c) {
      const uint4 h = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(&s, c)->hist + tid * kSamplePer);
      count[0] += h.x, count[1] += h.y, count[2] += h.z, count[3] += h.w;
    }
    static_assert(kSamplePer == 4, "a thread's counts are one 16-byte piece");
#pragma unroll
    for (int j = 0; j < kSamplePer; ++j) own += count[j];
    unsigned long long at = block_scan(s, own, total);

    // entries of the steps [from, to] into the first CTA's list; whether they fit is known before
    auto gather = [&](float f, int i, int from, int to) {
      const int b = binned ? bin_of(f) : 0;
      if (b >= from && b <= to && f != nothing) {
        SampleSmem* leader = cluster.map_shared_rank(&s, 0);
        leader->list[atomicAdd(&leader->listed, 1)] = rank_of(f, i);
      }
    };
    // the first CTA: its list, sorted from the top, padded with zeros to a power of two
    auto sorted = [&](int n) {
      int size = 2;
      while (size < n) size <<= 1;
      for (int i = n + tid; i < size; i += kSampleThreads) s.list[i] = 0;
      block_sort<true>(s.list, size);
    };
    auto listed_weight = [&](unsigned long long r) { return weight(key_score(uint32_t(r >> 32))); };
    // The first CTA, with every entry that may be kept in its list: the rest of the
    // filters and the draw.  `limit` entries by rank; `mass`: what p refers to, or 0 for theirs.
    auto finish = [&](int n, int limit, unsigned long long mass) {
      sorted(n);
      n = min(n, limit);
      constexpr int kPer = kSampleList / kSampleThreads;
      unsigned long long w[kPer], own = 0, all;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int i = tid * kPer + j;
        w[j] = 0;
        if (i < n) w[j] = to_fixed(listed_weight(s.list[i]));
        own += w[j];
      }
      unsigned long long run = block_scan(s, own, all);
      if (mass == 0) mass = all;
      unsigned long long target = ~0ull;
      if (by_mass) {
        target = (unsigned long long)(ceil(double(p) * double(mass)));
        target = target < 1 ? 1 : (target > mass ? mass : target);
      }
      // kept: what is above has not reached the target, and the weight is large enough
      int mine = 0;
      unsigned long long kept[kPer];
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int i = tid * kPer + j;
        kept[j] = 0;
        if (i < n && run < target && w[j] > 0) {
          const unsigned long long r = s.list[i];
          if (listed_weight(r) >= double(least)) {
            kept[j] = (static_cast<unsigned long long>(0xffffffffu - uint32_t(r)) << (kWeightBits + 1)) | w[j];
            ++mine;
          }
        }
        run += w[j];
      }
      unsigned long long m;
      int to = int(block_scan(s, unsigned(mine), m));  // also: the list has been read
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int i = tid * kPer + j;
        if (i < n && kept[j] != 0) s.list[to++] = kept[j];
      }
      __syncthreads();
      int size = 2;
      while (size < int(m)) size <<= 1;
      for (int i = int(m) + tid; i < size; i += kSampleThreads) s.list[i] = ~0ull;
      block_sort<false>(s.list, size);  // vocabulary order
      constexpr unsigned long long kMask = (1ull << (kWeightBits + 1)) - 1;
      own = 0;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int i = tid * kPer + j;
        w[j] = i < int(m) ? s.list[i] & kMask : 0;
        own += w[j];
      }
      run = block_scan(s, own, all);
      const unsigned long long border = (unsigned long long)(double(u) * double(all));
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if (run <= border && run + w[j] > border) {
          a.tokens[row] = int32_t(s.list[tid * kPer + j] >> (kWeightBits + 1));
          a.chances[row] = float(double(w[j]) / double(all));
        }
        run += w[j];
      }
    };

    if (by_rank && unsigned(k) < total) {
      if (at < unsigned(k) && at + own >= unsigned(k)) {
        unsigned long long run = at;
        int j = 0;
#pragma unroll
        for (int q = 0; q < kSamplePer - 1; ++q)
          if (j == q && run + count[q] < unsigned(k)) run += count[q], ++j;
        s.found_bin = tid * kSamplePer + j;
        s.found_before = run;
        s.found_last = int(j == 0 ? count[0] : j == 1 ? count[1] : j == 2 ? count[2] : count[3]);
      }
      __syncthreads();
      const int bin = s.found_bin, before = int(s.found_before), in = s.found_last;
      if (before + in <= kSampleList) {  // every kept entry fits the list
        each([&](float f, int i) { gather(f, i, 0, bin); });
        cluster.sync();
        if (rank == 0) finish(s.listed, k, 0);
        return;
      }
      if (in <= kSampleList) {
        each([&](float f, int i) { gather(f, i, bin, bin); });
        cluster.sync();
        if (rank == 0) {
          sorted(in);
          if (tid < ctas) cluster.map_shared_rank(&s, tid)->cut = s.list[k - before - 1];
        }
        cluster.sync();
        cut = s.cut;
        if (tid == 0) s.listed = 0;
      } else {
        cut = descend(false, unsigned(k), 0);
      }
      // the counts of the prefix, for the mass below
#pragma unroll
      for (int j = 0; j < kSamplePer; ++j) {
        const int b = tid * kSamplePer + j;
        if (b == bin) count[j] = uint32_t(k - before);
        else if (b > bin) count[j] = 0;
      }
      cluster.sync();  // no list is written before every one is empty
    }
    if (by_mass) {
      // bounds of the mass up to and including each step, from its counts
      const float fall = 1.f / heat;
      float lo[kSamplePer], hi[kSamplePer], lo_own = 0.f, hi_own = 0.f;
#pragma unroll
      for (int j = 0; j < kSamplePer; ++j) {
        const int b = tid * kSamplePer + j;
        // a hundredth of a step covers the rounding of the step's number
        hi_own += float(count[j]) * expf(-fmaxf(float(b) - 0.01f, 0.f) * step * fall) * 1.0001f;
        if (b < kSampleBins - 1) lo_own += float(count[j]) * expf(-(float(b) + 1.01f) * step * fall) * 0.9999f;
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
#pragma unroll
      for (int j = 0; j < kSamplePer; ++j) {
        const int b = tid * kSamplePer + j;
        if (hi_at + hi[j] >= below) atomicMin(&s.found_bin, b);
        if (lo_at + lo[j] >= reached) atomicMin(&s.found_last, b);
      }
      __syncthreads();
      const int from = binned ? s.found_bin : 0, to = binned ? s.found_last : kSampleBins - 1;
      // counts up to each of them
      unsigned long long own2 = 0, total2;
#pragma unroll
      for (int j = 0; j < kSamplePer; ++j) own2 += count[j];
      const unsigned long long at2 = block_scan(s, own2, total2);
      if (tid == 0) s.found_before = 0;
      __syncthreads();
      unsigned long long upto = at2;
#pragma unroll
      for (int j = 0; j < kSamplePer; ++j) {
        const int b = tid * kSamplePer + j;
        if (b == from) s.found_before = upto;  // before step `from`
        upto += count[j];
        if (b == to) s.found_through = upto;   // through step `to`
      }
      __syncthreads();
      const unsigned long long before = s.found_before, through = s.found_through;
      __syncthreads();
      const bool whole = cut == 0 && through <= kSampleList, some = through - before <= kSampleList;
      // one pass: the exact mass of the prefix and of its part before step `from`, and the
      // entries of the steps between, where they fit the list, else the steps' exact masses
      if (!some && !whole) {
        for (int b = tid; b < kSampleBins; b += kSampleThreads) s.wide[b] = 0;
        __syncthreads();
      }
      unsigned long long z = 0, over = 0;
      each([&](float f, int i) {
        const unsigned long long r = rank_of(f, i);
        if (r < cut) return;
        const unsigned long long w = to_fixed(weight(f));
        z += w;
        const int b = binned ? bin_of(f) : 0;
        if (b < from) over += w;
        if (whole || some) gather(f, i, whole ? 0 : from, to);
        else if (b >= from && b <= to && w > 0) atomicAdd(&s.wide[b], w);
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
        if (rank == 0) finish(s.listed, kSampleList, z);
        return;
      }
      unsigned long long target = (unsigned long long)(ceil(double(p) * double(z)));
      target = target < 1 ? 1 : (target > z ? z : target);
      bool fits = some;
      if (!some) {
        // the step that the target lies in; its entries
        unsigned long long mass[kSamplePer], own = 0, total;
#pragma unroll
        for (int j = 0; j < kSamplePer; ++j) mass[j] = 0;
        for (int c = 0; c < ctas; ++c)
#pragma unroll
          for (int j = 0; j < kSamplePer; ++j) mass[j] += cluster.map_shared_rank(&s, c)->wide[tid * kSamplePer + j];
#pragma unroll
        for (int j = 0; j < kSamplePer; ++j) own += mass[j];
        unsigned long long run = over + block_scan(s, own, total);
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
            if (rank_of(f, i) >= cut) gather(f, i, bin, bin);
          });
        cluster.sync();
      }
      if (fits) {
        if (rank == 0) {
          const int n = s.listed;
          sorted(n);
          constexpr int kPer = kSampleList / kSampleThreads;
          unsigned long long w[kPer], own = 0, all;
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            const int i = tid * kPer + j;
            w[j] = i < n ? to_fixed(listed_weight(s.list[i])) : 0;
            own += w[j];
          }
          unsigned long long run = over + block_scan(s, own, all);
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            if (run < target && run + w[j] >= target) {
              const unsigned long long r = s.list[tid * kPer + j];
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

  // ---- the kept weights, warp by warp in vocabulary order
  auto kept = [&](int v) -> unsigned long long {  // of place first + v
    if (v >= a.slice) return 0;
    const float f = Row::value(held[v]);
    if (rank_of(f, base + v) < cut) return 0;
    const double w = weight(f);
    return w >= double(least) ? to_fixed(w) : 0;
  };
  const int seg = ((a.slice + kSampleWarps - 1) / kSampleWarps + 31) / 32 * 32, start = warp * seg;
  unsigned long long own = 0, all = 0;
  for (int v = start + lane; v < start + seg; v += 32) own += kept(v);
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
  const unsigned long long border = (unsigned long long)(double(u) * double(all));  // the sum that has to be exceeded
  if (at <= border && at + own > border) {
    for (int v = start; v < start + seg; v += 32) {
      const unsigned long long w = kept(v + lane);
      unsigned long long run = w;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const unsigned long long up = __shfl_up_sync(~0u, run, d);
        if (lane >= d) run += up;
      }
      const unsigned hit = __ballot_sync(~0u, at + run > border);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          a.tokens[row] = base + v + lane;
          a.chances[row] = float(double(w) / double(all));
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
