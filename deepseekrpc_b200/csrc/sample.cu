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
// borders between tokens by up to a few percent of a token).  A prefix is found
// by radix descent over the unique 64-bit rank (order-preserving value, inverted
// index), 11 bits a level, on a histogram of counts or of weights.
//
// One CTA per row, which reads the row once per level.
#include <math_constants.h>

#include "common.cuh"
#include "host_common.h"

namespace dsr {
namespace {

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleBins = 2048;
constexpr int kSampleMaxVocab = 1 << 18;
constexpr int kWeightBits = 44;  // 2^18 weights of at most 2^44 fit 62 bits
constexpr double kLog2eD = 1.4426950408889634074;

struct SampleArgs {
  const void* logits;
  int64_t stride;
  int vocab;
  bool wide;  // fp32 (else bf16)
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* uniform;
  int32_t* tokens;
  float* chances;
  int32_t* err;
};

// 2^t for t <= 0 in 64 bits: 2^(n/64) from a table, the rest |r| <= 1/128 by the
// Taylor series of e^(r ln 2), whose first dropped term is below 2^-52.
struct Exp2 {
  const double* table;  // [64] 2^(j/64)
  __device__ __forceinline__ double operator()(double t) const {
    if (!(t > -60.0)) return 0.0;  // below half a step of the fixed point
    const double n = rint(t * 64.0);
    const double r = fma(n, -1.0 / 64.0, t) * 0.69314718055994530942;
    double p = fma(r, 1.0 / 120, 1.0 / 24);
    p = fma(p, r, 1.0 / 6);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    const int m = int(n);
    return p * table[m & 63] * __hiloint2double((1023 + (m >> 6)) << 20, 0);
  }
};

__device__ __forceinline__ uint64_t to_fixed(double w) {  // w in [0, 1]
  constexpr double kMagic = double(1ull << (52 - kWeightBits));
  return uint64_t(__double_as_longlong(w + kMagic) - __double_as_longlong(kMagic));
}

__device__ __forceinline__ uint64_t rank_of(float x, int i) {
  return (uint64_t(score_key(x)) << 32) | (0xffffffffu - uint32_t(i));
}

template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

struct SampleSmem {
  double table[64];
  unsigned long long hist[kSampleBins];
  unsigned long long part[kSampleWarps];
  unsigned long long found_before;
  int found_bin;
  int token;
  float chance;
};

__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const SampleArgs a) {
  __shared__ SampleSmem s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x;
  const float* x32 = static_cast<const float*>(a.logits) + row * a.stride;
  const uint16_t* x16 = static_cast<const uint16_t*>(a.logits) + row * a.stride;
  auto value = [&](int i) { return a.wide ? x32[i] : bf16_to_float(x16[i]); };

  // ---- largest rank; non-finite values
  unsigned long long best = 0;
  int bad = 0;
  for (int i = tid; i < a.vocab; i += kSampleThreads) {
    const float x = value(i);
    if (!(x < CUDART_INF_F)) bad = 1;
    const unsigned long long r = rank_of(x, i);
    best = r > best ? r : best;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const unsigned long long r = __shfl_xor_sync(~0u, best, o);
    best = r > best ? r : best;
  }
  if (lane == 0) s.part[warp] = best;
  if (tid < 64) s.table[tid] = exp2(tid / 64.0);
  bad = __syncthreads_or(bad);
  for (int w = 0; w < kSampleWarps; ++w) best = s.part[w] > best ? s.part[w] : best;
  const float top = key_score(uint32_t(best >> 32));
  const float heat = a.temperature[row], p = a.top_p[row], least = a.min_p[row], u = a.uniform[row];
  const int k = a.top_k[row];
  const bool valid = heat >= 0.f && heat < CUDART_INF_F && p >= 0.f && p <= 1.f && least >= 0.f && least <= 1.f &&
                     u >= 0.f && u < 1.f && k >= 0;
  if (bad || !valid || top == -CUDART_INF_F || heat == 0.f) {
    if (tid == 0) {
      if (bad) flag(a.err, DSR_ERR_NONFINITE);
      else if (!valid) flag(a.err, DSR_ERR_ID);
      const bool greedy = !bad && valid && top != -CUDART_INF_F;
      a.tokens[row] = greedy ? int32_t(0xffffffffu - uint32_t(best)) : -1;
      a.chances[row] = greedy ? 1.f : 0.f;
    }
    return;
  }
  const Exp2 pow2{s.table};
  const double scale = kLog2eD / double(heat), high = top;
  auto weight = [&](float x) { return pow2((double(x) - high) * scale); };
  auto block_sum = [&](unsigned long long v) {
    v = warp_sum(v);
    __syncthreads();
    if (lane == 0) s.part[warp] = v;
    __syncthreads();
    unsigned long long all = 0;
    for (int w = 0; w < kSampleWarps; ++w) all += s.part[w];
    return all;
  };

  // The rank of the last entry of the shortest prefix, among ranks >= cut, whose
  // count or mass reaches target.
  auto prefix = [&](bool mass, unsigned long long target, unsigned long long cut) {
    unsigned long long known = 0, before = 0;  // leading bits of the rank; what lies above them
    for (int shift = 55; shift >= 0; shift -= 11) {
      for (int b = tid; b < kSampleBins; b += kSampleThreads) s.hist[b] = 0;
      __syncthreads();
      for (int i = tid; i < a.vocab; i += kSampleThreads) {
        const float x = value(i);
        const unsigned long long r = rank_of(x, i);
        if (r >= cut && (shift == 55 || (r >> (shift + 11)) == known))
          atomicAdd(&s.hist[(r >> shift) & (kSampleBins - 1)], mass ? to_fixed(weight(x)) : 1ull);
      }
      __syncthreads();
      // thread t holds the bins from the top, 4 each
      constexpr int kPer = kSampleBins / kSampleThreads;
      unsigned long long own = 0;
      for (int j = 0; j < kPer; ++j) own += s.hist[kSampleBins - 1 - (tid * kPer + j)];
      unsigned long long run = own;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const unsigned long long up = __shfl_up_sync(~0u, run, d);
        if (lane >= d) run += up;
      }
      if (lane == 31) s.part[warp] = run;
      __syncthreads();
      unsigned long long at = before + run - own;
      for (int w = 0; w < warp; ++w) at += s.part[w];
      if (at < target && at + own >= target) {
        int b = kSampleBins - 1 - tid * kPer;
        while (at + s.hist[b] < target) at += s.hist[b--];
        s.found_bin = b;
        s.found_before = at;
      }
      __syncthreads();
      known = (known << 11) | unsigned(s.found_bin);
      before = s.found_before;
      __syncthreads();
    }
    return known;
  };

  unsigned long long cut = 0;
  if (k > 0 && k < a.vocab) cut = prefix(false, unsigned(k), 0);
  if (p < 1.f) {
    unsigned long long z = 0;
    for (int i = tid; i < a.vocab; i += kSampleThreads) {
      const float x = value(i);
      if (rank_of(x, i) >= cut) z += to_fixed(weight(x));
    }
    z = block_sum(z);
    unsigned long long target = (unsigned long long)(ceil(double(p) * double(z)));
    target = target < 1 ? 1 : (target > z ? z : target);
    cut = prefix(true, target, cut);
  }

  // ---- the kept weights, warp by warp in vocabulary order
  auto kept = [&](int i) -> unsigned long long {
    if (i >= a.vocab) return 0;
    const float x = value(i);
    if (rank_of(x, i) < cut) return 0;
    const double w = weight(x);
    return w >= double(least) ? to_fixed(w) : 0;
  };
  const int seg = ((a.vocab + kSampleWarps - 1) / kSampleWarps + 31) / 32 * 32, first = warp * seg;
  unsigned long long own = 0;
  for (int i = first + lane; i < first + seg; i += 32) own += kept(i);
  own = warp_sum(own);
  __syncthreads();
  if (lane == 0) s.part[warp] = own;
  __syncthreads();
  unsigned long long all = 0, at = 0;
  for (int w = 0; w < kSampleWarps; ++w) {
    if (w < warp) at += s.part[w];
    all += s.part[w];
  }
  const unsigned long long border = (unsigned long long)(double(u) * double(all));  // the sum that has to be exceeded
  if (at <= border && at + own > border) {
    for (int i = first; i < first + seg; i += 32) {
      const unsigned long long w = kept(i + lane);
      unsigned long long run = w;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const unsigned long long up = __shfl_up_sync(~0u, run, d);
        if (lane >= d) run += up;
      }
      const unsigned hit = __ballot_sync(~0u, at + run > border);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          a.tokens[row] = i + lane;
          a.chances[row] = float(double(w) / double(all));
        }
        break;
      }
      at += __shfl_sync(~0u, run, 31);
    }
  }
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
  const SampleArgs a{logits, row_stride, int(vocab), dtype == DSR_F32, temperature, top_k,
                     top_p,  min_p,      uniform,    tokens,           chances,     err};
  sample_kernel<<<unsigned(rows), kSampleThreads, 0, as_stream(stream)>>>(a);
  return launch_status("sample launch");
}
