// Rotary positions: rotates column pairs of up to four tensors (MLA query, index
// query, KV row, index key, say) by their tokens' positions, in one launch.
//
//   (y_a, y_b) = m (x_a cos t - x_b sin t, x_b cos t + x_a sin t),  t = position * frequency[i]
//
// for pair i of the rotated columns [offset, offset + 2 pairs): (a, b) = (2i, 2i+1)
// interleaved, (i, i + pairs) in halves.  The inverse rotation (sin -> -sin) is the
// transpose, hence the gradient.  Frequencies are 64-bit numbers from the caller,
// which holds any long-context scaling; the amplitude m multiplies the rotated
// columns alone.  The other columns are copied unless the rotation is in place.
//
// The angle is formed in 64 bits and reduced to a fraction of a turn before it is
// rounded to 32: at position 10^6 a 32-bit angle would be off by 0.06.  Each CTA
// takes one token (or a share of one: few tokens have to fill the GPU too) and
// forms its cosines once for all heads of all tensors.  Every value is read and written
// once, in 16-byte pieces wherever pointers, strides and columns allow (one tensor of 64
// heads, 64 of 576 columns rotated in place, 8192 tokens: 41 us; off the 16-byte grid,
// column by column, 90).  Bound by instructions as much as by memory: 173 warp
// instructions for 32 items of one or two pieces, mostly the way from an item to its
// tensor, head and column, which every token walks anew; issue slots are 62% busy, DRAM
// 51%.  Measured: 8192 tokens of four tensors in BF16, 560 MB, 127 us = 4.4 TB/s, 67% of a
// plain copy, in FP32, 1.1 GB, 207 us = 5.3 TB/s; 999 tokens, 44 MB, 14.5 us = 3.0 TB/s; 1
// token 5.8 us, a launch.  Two to four pieces a thread ahead, streaming hints, loops per
// tensor and several tokens a CTA were all slower (129 to 186 us of the first).
#include "common.cuh"
#include "host_common.h"
#include "strided.h"

namespace dsr {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxPairs = 256;
constexpr int kRopeMaxTensors = 4;

struct RopeTensor {
  const uint8_t* x;
  uint8_t* out;
  int64_t x_token, x_head, out_token, out_head;  // elements
  int offset;      // first rotated column
  int per_head;    // work items of one head: rotated, then copied
  int rotated;     // of them rotated ones
  int items;       // of one token
  bool interleaved, wide, vec;  // wide: fp32 (else bf16); vec: 16-byte pieces
};
struct RopeArgs {
  RopeTensor t[kRopeMaxTensors];
  const int32_t* positions;
  const double* frequencies;
  int32_t* err;
  int64_t tokens;
  int count, pairs, items;
  float mscale;
  bool inverse;
};

__device__ __forceinline__ float2 rotate(float a, float b, float2 cs) {
  return make_float2(a * cs.x - b * cs.y, b * cs.x + a * cs.y);
}

// 16 bytes as floats (4 fp32 or 8 bf16) and back
template <bool W>
__device__ __forceinline__ void unpack(const uint4& v, float* f) {
  if constexpr (W) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  } else {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
template <bool W>
__device__ __forceinline__ uint4 pack(const float* f) {
  if constexpr (W) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = __bfloat16_as_ushort(__float2bfloat16_rn(f[2 * i])) |
             (uint32_t(__bfloat16_as_ushort(__float2bfloat16_rn(f[2 * i + 1]))) << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Item k of one head: rotated items first, then copied ones.
template <bool W>
__device__ __forceinline__ void rope_vector(const RopeTensor& t, const uint8_t* x, uint8_t* y, int k, int pairs,
                                            const float2* cs) {
  constexpr int kSize = W ? 4 : 2, kV = 16 / kSize;
  if (k >= t.rotated) {
    int c = (k - t.rotated) * kV;  // column among the copied ones
    if (c >= t.offset) c += 2 * pairs;
    *reinterpret_cast<uint4*>(y + int64_t(c) * kSize) = *reinterpret_cast<const uint4*>(x + int64_t(c) * kSize);
  } else if (t.interleaved) {
    const int64_t at = int64_t(t.offset + k * kV) * kSize;
    float f[kV];
    unpack<W>(*reinterpret_cast<const uint4*>(x + at), f);
#pragma unroll
    for (int i = 0; i < kV; i += 2) {
      const float2 r = rotate(f[i], f[i + 1], cs[(k * kV + i) >> 1]);
      f[i] = r.x, f[i + 1] = r.y;
    }
    *reinterpret_cast<uint4*>(y + at) = pack<W>(f);
  } else {
    const int64_t at = int64_t(t.offset + k * kV) * kSize, half = int64_t(pairs) * kSize;
    float f[kV], g[kV];
    unpack<W>(*reinterpret_cast<const uint4*>(x + at), f);
    unpack<W>(*reinterpret_cast<const uint4*>(x + at + half), g);
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      const float2 r = rotate(f[i], g[i], cs[k * kV + i]);
      f[i] = r.x, g[i] = r.y;
    }
    *reinterpret_cast<uint4*>(y + at) = pack<W>(f);
    *reinterpret_cast<uint4*>(y + at + half) = pack<W>(g);
  }
}

template <bool W>
__device__ __forceinline__ float rope_get(const uint8_t* x, int c) {
  return W ? reinterpret_cast<const float*>(x)[c] : bf16_to_float(reinterpret_cast<const uint16_t*>(x)[c]);
}
template <bool W>
__device__ __forceinline__ void rope_put(uint8_t* y, int c, float v) {
  if (W) reinterpret_cast<float*>(y)[c] = v;
  else reinterpret_cast<uint16_t*>(y)[c] = __bfloat16_as_ushort(__float2bfloat16_rn(v));
}

// The same for pointers, strides or columns off the 16-byte grid: a pair, or one column.
template <bool W>
__device__ __forceinline__ void rope_scalar(const RopeTensor& t, const uint8_t* x, uint8_t* y, int k, int pairs,
                                            const float2* cs) {
  if (k >= t.rotated) {
    int c = k - t.rotated;
    if (c >= t.offset) c += 2 * pairs;
    if (W) reinterpret_cast<uint32_t*>(y)[c] = reinterpret_cast<const uint32_t*>(x)[c];
    else reinterpret_cast<uint16_t*>(y)[c] = reinterpret_cast<const uint16_t*>(x)[c];
  } else {
    const int a = t.offset + (t.interleaved ? 2 * k : k), b = a + (t.interleaved ? 1 : pairs);
    const float2 r = rotate(rope_get<W>(x, a), rope_get<W>(x, b), cs[k]);
    rope_put<W>(y, a, r.x);
    rope_put<W>(y, b, r.y);
  }
}

__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const __grid_constant__ RopeArgs a) {
  __shared__ float2 cs[kRopeMaxPairs];
  for (int64_t token = blockIdx.x; token < a.tokens; token += gridDim.x) {
    const int32_t position = a.positions[token];
    if (position < 0) {  // -1: a padding row, left as it is
      if (position < -1 && threadIdx.x == 0) flag(a.err, DSR_ERR_ID);
      continue;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.pairs; i += kRopeThreads) {
      const double turns = position * (a.frequencies[i] * 0.15915494309189533577);  // 1 / (2 pi)
      float s, c;
      sincospif(2.0f * float(turns - rint(turns)), &s, &c);
      cs[i] = make_float2(c * a.mscale, (a.inverse ? -s : s) * a.mscale);
    }
    __syncthreads();
    for (int item = blockIdx.y * kRopeThreads + threadIdx.x; item < a.items; item += gridDim.y * kRopeThreads) {
      int n = 0, k = item;
      while (k >= a.t[n].items) k -= a.t[n++].items;
      const RopeTensor& t = a.t[n];
      const int head = k / t.per_head;
      k -= head * t.per_head;
      const int size = t.wide ? 4 : 2;
      const uint8_t* x = t.x + (token * t.x_token + head * t.x_head) * size;
      uint8_t* y = t.out + (token * t.out_token + head * t.out_head) * size;
      if (t.vec) {
        if (t.wide) rope_vector<true>(t, x, y, k, a.pairs, cs);
        else rope_vector<false>(t, x, y, k, a.pairs, cs);
      } else {
        if (t.wide) rope_scalar<true>(t, x, y, k, a.pairs, cs);
        else rope_scalar<false>(t, x, y, k, a.pairs, cs);
      }
    }
  }
}

}  // namespace
}  // namespace dsr

extern "C" int dsr_rope(const dsr_rope_tensor* tensors, int64_t count, const int32_t* positions,
                        const double* frequencies, int64_t pairs, float mscale, int inverse, int32_t* err,
                        int64_t tokens, void* stream) {
  using namespace dsr;
  clear_error();
  DSR_REQUIRE(tensors && positions && frequencies && err, "rope: null pointer");
  DSR_REQUIRE(count > 0 && count <= kRopeMaxTensors, "rope: tensors %lld outside [1, %d]", (long long)count,
              kRopeMaxTensors);
  DSR_REQUIRE(pairs > 0 && pairs <= kRopeMaxPairs, "rope: pairs %lld outside [1, %d]", (long long)pairs,
              kRopeMaxPairs);
  DSR_REQUIRE(tokens > 0 && tokens < (int64_t(1) << 31), "rope: tokens %lld outside [1, 2^31)", (long long)tokens);
  DSR_REQUIRE(isfinite(mscale) && mscale > 0.f, "rope: invalid amplitude");
  RopeArgs a = {};
  int64_t items = 0;
  for (int n = 0; n < count; ++n) {
    const dsr_rope_tensor& s = tensors[n];
    DSR_REQUIRE(s.x && s.out, "rope: null pointer");
    DSR_REQUIRE(s.dtype == DSR_BF16 || s.dtype == DSR_F32, "rope: unknown element type %d", int(s.dtype));
    DSR_REQUIRE(s.heads > 0 && s.heads <= 65536 && s.width > 0 && s.width <= 65536, "rope: invalid heads or width");
    DSR_REQUIRE(s.offset >= 0 && s.offset + 2 * pairs <= s.width, "rope: rotated columns [%d, %lld) outside the row",
                int(s.offset), (long long)(s.offset + 2 * pairs));
    const bool in_place = s.x == s.out;
    DSR_REQUIRE(!in_place || (s.x_token == s.out_token && s.x_head == s.out_head),
                "rope: an in-place rotation needs equal strides");
    DSR_REQUIRE((s.out_token != 0 || tokens == 1) && (s.out_head != 0 || s.heads == 1),
                "rope: rows of an output overlap");
    for (int m = 0; m < count; ++m)
      DSR_REQUIRE(m == n || (s.out != tensors[m].out && s.out != tensors[m].x),
                  "rope: tensor %d's output is tensor %d's input or output", n, m);
    const int size = s.dtype == DSR_F32 ? 4 : 2, v = 16 / size;
    DSR_REQUIRE((reinterpret_cast<uintptr_t>(s.x) | reinterpret_cast<uintptr_t>(s.out)) % size == 0,
                "rope: misaligned tensor");
    auto on_grid = [v](int64_t e) { return e % v == 0; };
    RopeTensor& t = a.t[n];
    t.x = static_cast<const uint8_t*>(s.x);
    t.out = static_cast<uint8_t*>(s.out);
    t.x_token = s.x_token, t.x_head = s.x_head, t.out_token = s.out_token, t.out_head = s.out_head;
    t.offset = s.offset;
    t.interleaved = s.interleaved != 0;
    t.wide = s.dtype == DSR_F32;
    t.vec = aligned16(s.x) && aligned16(s.out) && on_grid(s.x_token) && on_grid(s.x_head) && on_grid(s.out_token) &&
            on_grid(s.out_head) && on_grid(s.offset) && on_grid(t.interleaved ? 2 * pairs : pairs) &&
            (in_place || on_grid(s.width));
    const int piece = t.vec ? v : 1;
    t.rotated = int(t.vec ? (t.interleaved ? 2 * pairs : pairs) / v : pairs);
    t.per_head = t.rotated + (in_place ? 0 : int(s.width - 2 * pairs) / piece);
    const int64_t own = int64_t(t.per_head) * s.heads;
    items += own;
    DSR_REQUIRE(items < (int64_t(1) << 30), "rope: too many columns for one call");
    t.items = int(own);
  }
  // CTAs of different tokens, and threads of different tensors, run in no order: what one
  // writes no other may read or write.  In place only the rotated columns are touched.
  StridedBytes in[kRopeMaxTensors], out[kRopeMaxTensors];
  for (int n = 0; n < count; ++n) {
    const dsr_rope_tensor& s = tensors[n];
    const int size = s.dtype == DSR_F32 ? 4 : 2;
    const bool in_place = s.x == s.out;
    const int64_t first = in_place ? int64_t(s.offset) * size : 0, width = in_place ? 2 * pairs : s.width;
    out[n] = StridedBytes(static_cast<const uint8_t*>(s.out) + first, width, tokens, s.out_token, s.heads, s.out_head,
                          size);
    in[n] = in_place ? out[n] : StridedBytes(s.x, width, tokens, s.x_token, s.heads, s.x_head, size);
    DSR_REQUIRE(!out[n].folds(), "rope: rows of an output overlap");
  }
  for (int n = 0; n < count; ++n)
    for (int m = 0; m < count; ++m) {
      if (m != n || tensors[n].x != tensors[n].out)
        DSR_REQUIRE(!StridedBytes::meet(out[n], in[m]), "rope: tensor %d's output overlaps tensor %d's input", n, m);
      if (m > n)
        DSR_REQUIRE(!StridedBytes::meet(out[n], out[m]), "rope: tensor %d's output overlaps tensor %d's output", n, m);
    }
  a.positions = positions;
  a.frequencies = frequencies;
  a.err = err;
  a.tokens = tokens;
  a.count = int(count);
  a.pairs = int(pairs);
  a.items = int(items);
  a.mscale = mscale;
  a.inverse = inverse != 0;
  // few tokens: several CTAs share one, so that the grid covers the GPU twice
  const int64_t shares = (items + kRopeThreads - 1) / kRopeThreads, want = (2 * sm_count() + tokens - 1) / tokens;
  const dim3 grid(unsigned(tokens < 65536 * 8 ? tokens : 65536 * 8), unsigned(want < shares ? want : shares), 1);
  rope_kernel<<<grid, kRopeThreads, 0, as_stream(stream)>>>(a);
  return launch_status("rope launch");
}
