// prefix_attn.cuh -- what the two kernels of prefix_attention share: the workspace's parts, fp16 operand
// conversion, bounded barrier waits.
#pragma once

#include "serving.cuh"

namespace needle {

constexpr float kLn2 = 0.6931471805599453f;
// The reference maximum of a head covers the value scales too: a weight is 2^(s - M) vs, s and M base 2.  M is
// raised, and what was summed rescaled, only when a block could bring weights of 2^15 (fp16 ends at 65504);
// a raised M leaves them below 2^7.
constexpr float kRaise = 7.0f;

// Parts of the softmax: M and l of every (part, row, head), and the weighted values.  A part is 2^M times
// its l and values; an empty one has M = -inf and l = 0, and its values are not read (part_of).
struct Parts {
  float2* ml;
  float* o;
  int64_t per_part;  // rows * heads
};

// A part's M and l as they are stored.  Maxima pass over NaN: a part whose scores are all NaN has M = -inf too, and its
// l, which is NaN, says that it is not an empty one.
__device__ __forceinline__ float2 part_of(float M, float l) { return make_float2(l == l ? M : 0.0f, l); }

// The prefix on the tensor cores (prefix_attn_tc.cu): parts 0 .. parts - 1 of `out`, `part_len` positions each.
// part_len is a multiple of prefix_tile().
int prefix_tile();
int prefix_rows();  // packed rows (rows * heads of a KV head) a CTA takes
cudaError_t launch_attend_prefix(const needle_prefix_attention& a, const Parts& out, int parts, int part_len, float scale,
                                 uint32_t* wait_words, cudaStream_t s);

__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }

// Two codes of `w` (biased by 128 with w ^ 0x80808080) as fp16: 0x6400 | byte is 1024 + byte.
__device__ __forceinline__ uint32_t codes_f16(uint32_t w, uint32_t selector) {
  const uint32_t h = __byte_perm(w, 0x64646464u, selector);
  return half2_bits(__hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x6480))));
}

// fp16 head and tail of two binary32 values.
__device__ __forceinline__ void split_f16(float a, float b, uint32_t& head, uint32_t& tail) {
  const __half2 h = __floats2half2_rn(a, b);
  head = half2_bits(h);
  tail = half2_bits(__floats2half2_rn(a - __low2float(h), b - __high2float(h)));
}

// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float power2(int e) { return __int_as_float((e + 127) << 23); }
// Exponent of |v| (0 and subnormals -127, infinities and NaN 128).
__device__ __forceinline__ int exponent_of(float v) { return (int)((__float_as_uint(v) >> 23) & 255u) - 127; }

// What a block whose largest value scale is `top` adds to the reference maximum.  Scales below 2^-60 (rope_append's
// smallest is 2^-47) count as that: a block of values that are all zero keeps a reference 2^-65 below its scores', near
// enough for its weights not to be flushed beside a block with large values, nor to sum up to infinity.
__device__ __forceinline__ float value_reach(float top) { return (float)(min(max(exponent_of(top), -60), 100) - 6); }

// The next kernel of the stream may be started (when it was launched to overlap) / the kernel before has ended
// and its writes are visible.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_prior() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

}  // namespace needle
