// prefix_attn.cu -- decode attention of a batch whose sequences share a prompt prefix: every row
// attends over the prefix's int8 keys and values, held once, and over its own int8 cache
// (#attention, packages/needle.js/src/model/runtime.ts:719-786, with the prefix taken out of the
// per-sequence caches; any head layout, binary32 arithmetic).
//
//   s_j = scale * (q . code_j) * ks_j,  o = sum_j e^(s_j - m) vs_j code_j / sum_j e^(s_j - m),
//   j over the prefix and the row's own positions;  lse = m + log sum_j e^(s_j - m)
//
// k_attend_stream.  The query heads of one KV head (up to 8) meet 16 positions at a time on the tensor
// cores (mma.sync m16n8k16, fp16 x fp16 -> fp32).  M is only the heads of one row, so the products are thin
// and the kernel lives on its loads: a position costs 2 D + 8 bytes.  Codes are exact in fp16; queries and
// weights, binary32, are split into an fp16 head (MMA rows 0-7) and tail (rows 8-15), which the
// accumulator's two row halves add up again, so results have binary32 accuracy for every element type.
// The order of k inside a product is free, so lanes load K and V from global memory straight into
// operand order, 16 (8) consecutive codes at a time, with no shared memory:
//   K: lane (n, c) = (lane / 4, lane % 4) loads D / 4 codes of position n; k-step t takes 4 of them;
//   V: the lane loads D / 8 codes of the positions 2c, 2c + 1, 2c + 8, 2c + 9, which are the ones whose
//      weights the score product left in its registers; output tile j takes code j of each.
// The softmax keeps a reference maximum per head that is only raised when a score exceeds it by 2^8 (the
// weights stay below 2^8, inside fp16), so that accumulators are rarely rescaled; value scales are
// brought to at most 2^7 by a power of two in the same lazy way.
// `warps` warps share a unit (row, KV head, 8 heads, split of the positions) and are merged in shared
// memory; splits and the prefix's parts are merged from the workspace.
#include <algorithm>
#include <cmath>

#include "serving.cuh"

namespace needle {

namespace {

constexpr int kStreamWarps = 8;
constexpr int kStreamThreads = kStreamWarps * 32;
constexpr int kGroupHeads = 8;  // query heads of one KV head taken together
constexpr int kBlock = 16;      // positions of a step
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLazy = 8.0f;   // powers of two a score may exceed the reference maximum by

// Parts of the softmax: m (base 2) and l of every (part, row, head), and the weighted values.
struct Parts {
  float2* ml;
  float* o;
  int64_t per_part;  // rows * heads
};

// How a call is laid out (plan_for).
struct StreamPlan {
  int groups;      // 8-head groups of a KV head
  int warps;       // warps per unit: 1, 2, 4 or 8
  int splits;      // splits of the positions
  int split_len;   // positions of a split
  int parts;       // prefix parts in the workspace, in front of the splits; 0: the stream reads the prefix
  int part_len;    // prefix positions of a part
};

__device__ __forceinline__ void mma_f16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

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

// One segment of positions: the prefix, or a row's own cache, of one KV head.
struct Segment {
  const int8_t *k, *v;
  const float *ks, *vs;
};

template <int D>
struct Block {
  uint4 k[2][D / 64];       // tile (8 positions), 64-dimension half
  uint2 v[4][D / 64];       // positions 2c, 2c + 1, 2c + 8, 2c + 9
  float ks[4], vs[4];       // of the same positions
};

// Loads positions [j, min(j + 16, end)) of a segment; what lies behind `end` becomes zeros.
template <int D>
__device__ __forceinline__ void load_block(Block<D>& b, const Segment& s, int j, int end, int lane) {
  const int n = lane >> 2, c = lane & 3;
#pragma unroll
  for (int t = 0; t < 2; t++) {
    const int p = j + 8 * t + n;
#pragma unroll
    for (int h = 0; h < D / 64; h++)
      b.k[t][h] = p < end ? __ldg(reinterpret_cast<const uint4*>(s.k + (int64_t)p * D + h * 64 + c * 16))
                          : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int p = j + 2 * c + (i & 1) + (i >> 1) * 8;
    const bool in = p < end;
    if constexpr (D == 64) {
      b.v[i][0] = in ? __ldg(reinterpret_cast<const uint2*>(s.v + (int64_t)p * D + n * 8)) : make_uint2(0, 0);
    } else {
      const uint4 w = in ? __ldg(reinterpret_cast<const uint4*>(s.v + (int64_t)p * D + n * 16)) : make_uint4(0, 0, 0, 0);
      b.v[i][0] = make_uint2(w.x, w.y);
      b.v[i][1] = make_uint2(w.z, w.w);
    }
    b.ks[i] = in ? __ldg(s.ks + p) : 0.0f;
    b.vs[i] = in ? __ldg(s.vs + p) : 0.0f;
  }
}

// A warp's state of up to 8 heads: lane (g, c) keeps head g's maximum, its own share of the sum, and
// D / 4 consecutive output dimensions from c * D / 4 on.
template <int D>
struct Rows {
  static constexpr int kTiles = D / 8;
  uint32_t q[D / 16][4];    // A operand of each k-step: head and tail of the scaled query
  float inverse;            // undoes the query's power of two
  float m, l;               // reference maximum (base 2), sum of the lane's weights
  int ev;                   // values are kept as value * 2^-ev
  float o[kTiles][4];
};

template <int D>
__device__ __forceinline__ void attend_block(Rows<D>& r, const Block<D>& b, int j, int end, int lane) {
  const int c = lane & 3;
  float s[4];
#pragma unroll
  for (int t = 0; t < 2; t++) {
    float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int h = 0; h < D / 64; h++) {
      const uint32_t w[4] = {b.k[t][h].x, b.k[t][h].y, b.k[t][h].z, b.k[t][h].w};
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const uint32_t u = w[k] ^ 0x80808080u;
        mma_f16(d, r.q[h * 4 + k], codes_f16(u, 0x4140), codes_f16(u, 0x4342));
      }
    }
    s[2 * t] = d[0] + d[2];
    s[2 * t + 1] = d[1] + d[3];
  }
  float top = -INFINITY;
  float vtop = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int p = j + 2 * c + (i & 1) + (i >> 1) * 8;
    s[i] = p < end ? s[i] * (b.ks[i] * r.inverse) : -INFINITY;
    top = fmaxf(top, s[i]);
    vtop = fmaxf(vtop, fabsf(b.vs[i]));
  }
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, 1));
  vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, 2));
  const int e = min(max(exponent_of(vtop), -100), 100) - 6;  // scaled values below 2^7
  if (__any_sync(0xffffffffu, top > r.m + kLazy || e > r.ev)) {
    const float mn = top > r.m + kLazy ? top : r.m;
    const int en = max(e, r.ev);
    const float fm = r.m == -INFINITY ? 0.0f : exp2f(r.m - mn);
    const float fo = fm * power2(max(r.ev - en, -126));
    r.l *= fm;
#pragma unroll
    for (int t = 0; t < Rows<D>::kTiles; t++)
#pragma unroll
      for (int i = 0; i < 4; i++) r.o[t][i] *= fo;
    r.m = mn;
    r.ev = en;
  }
  const float base = r.m == -INFINITY ? 0.0f : r.m;
  const float unit = power2(-r.ev);
  float w[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float p = exp2f(s[i] - base);
    r.l += p;
    w[i] = p * (b.vs[i] * unit);
  }
  uint32_t a[4];  // rows 0-7: heads of the weights, rows 8-15: tails
  split_f16(w[0], w[1], a[0], a[1]);
  split_f16(w[2], w[3], a[2], a[3]);
#pragma unroll
  for (int h = 0; h < D / 64; h++)
#pragma unroll
    for (int half = 0; half < 2; half++) {
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; i++) u[i] = (half ? b.v[i][h].y : b.v[i][h].x) ^ 0x80808080u;
#pragma unroll
      for (int k = 0; k < 2; k++) {  // code pairs 2k, 2k + 1 of the word
        const uint32_t sel = k ? 0x7362 : 0x5140;
        const uint32_t lo = __byte_perm(u[0], u[1], sel), hi = __byte_perm(u[2], u[3], sel);
        const int t = h * 8 + half * 4 + 2 * k;
        mma_f16(r.o[t], a, codes_f16(lo, 0x4140), codes_f16(hi, 0x4140));
        mma_f16(r.o[t + 1], a, codes_f16(lo, 0x4342), codes_f16(hi, 0x4342));
      }
    }
}

// Reads the unit's queries into MMA operand order, scaled by `scale` * log2(e) and, per head, to a
// largest magnitude in [2^10, 2^11).
template <class T, int D>
__device__ __forceinline__ void load_queries(Rows<D>& r, const T* q, int heads, float scale, int lane) {
  const int g = lane >> 2, c = lane & 3;
  float x[D / 4];
  float top = 0.0f;
#pragma unroll
  for (int h = 0; h < D / 64; h++)
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const float v = g < heads ? to_f32(q[g * D + h * 64 + c * 16 + i]) * (scale * kLog2e) : 0.0f;
      x[h * 16 + i] = v;
      top = fmaxf(top, fabsf(v));
    }
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const int e = min(max(exponent_of(top), -110), 110);
  const float f = power2(10 - e);
  r.inverse = power2(e - 10);
#pragma unroll
  for (int k = 0; k < D / 16; k++) {
    split_f16(x[4 * k] * f, x[4 * k + 1] * f, r.q[k][0], r.q[k][1]);
    split_f16(x[4 * k + 2] * f, x[4 * k + 3] * f, r.q[k][2], r.q[k][3]);
  }
  r.m = -INFINITY;
  r.l = 0.0f;
  r.ev = -127;
#pragma unroll
  for (int t = 0; t < Rows<D>::kTiles; t++)
#pragma unroll
    for (int i = 0; i < 4; i++) r.o[t][i] = 0.0f;
}

template <class T, int N>
__device__ __forceinline__ void store_out(T* p, const float* x, bool vec) {
  constexpr int V = 16 / sizeof(T);
  if (vec) {
#pragma unroll
    for (int k = 0; k < N / V; k++) {
      Vec<T, V> v;
#pragma unroll
      for (int i = 0; i < V; i++) v.v[i] = from_f32<T>(x[k * V + i]);
      reinterpret_cast<Vec<T, V>*>(p)[k] = v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) p[i] = from_f32<T>(x[i]);
  }
}

template <class T, int D>
__global__ void __launch_bounds__(kStreamThreads, D == 64 ? 2 : 1)
    k_attend_stream(const __grid_constant__ needle_prefix_attention a, const StreamPlan plan, const Parts parts, float scale) {
  constexpr int N = D / 4;  // output dimensions of a lane
  __shared__ float merge_m[kStreamWarps][kGroupHeads], merge_l[kStreamWarps][kGroupHeads];
  extern __shared__ __align__(16) float merge_o[];  // [warps][8][D], when warps share a unit
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  const int share = plan.warps, member = warp & (share - 1);
  const int64_t units = (int64_t)a.rows * a.kv_heads * plan.groups;
  const int64_t unit = (int64_t)blockIdx.x * (kStreamWarps / share) + warp / share;
  const int split = blockIdx.y, group = a.heads / a.kv_heads;
  bool live = unit < units;
  const int64_t row = live ? unit / (a.kv_heads * plan.groups) : 0;
  const int rest = live ? (int)(unit - row * (a.kv_heads * plan.groups)) : 0;
  const int h = rest / plan.groups, g0 = (rest - h * plan.groups) * kGroupHeads;
  const int heads = min(kGroupHeads, group - g0);
  const int slot = live ? (a.slots ? a.slots[row] : (int)min(row, (int64_t)0x7fffffff)) : -1;
  live = live && slot >= 0 && slot < a.slot_count;
  const int64_t head = (int64_t)h * group + g0;  // the unit's first query head
  Rows<D> r;
  if (live) {
    load_queries<T, D>(r, static_cast<const T*>(a.q) + row * a.q_stride + head * D, heads, scale, lane);
    const int count = min(max(a.counts[row], 0), a.capacity);
    const int64_t own = ((int64_t)slot * a.kv_heads + h) * a.capacity;
    const int64_t shared = (int64_t)h * a.prefix_capacity;
    const int prefix = plan.parts ? 0 : a.prefix_length;
    // positions [from, to) of prefix ++ own cache, one segment after the other
    const int64_t from = (int64_t)split * plan.split_len;
    const int64_t to = min(from + plan.split_len, (int64_t)prefix + count);
#pragma unroll 1
    for (int seg = 0; seg < 2; seg++) {
      const int64_t base = seg ? own : shared;
      const int begin = (int)max(from - (seg ? prefix : 0), (int64_t)0);
      const int end = (int)min(to - (seg ? prefix : 0), (int64_t)(seg ? count : prefix));
      const Segment s = {(seg ? a.key_codes : a.prefix_key_codes) + base * D,
                         (seg ? a.value_codes : a.prefix_value_codes) + base * D,
                         (seg ? a.key_scales : a.prefix_key_scales) + base,
                         (seg ? a.value_scales : a.prefix_value_scales) + base};
      int j = begin + member * kBlock;
      if (j >= end) continue;
      Block<D> now;
      load_block<D>(now, s, j, end, lane);
#pragma unroll 1
      for (; j < end; j += share * kBlock) {
        Block<D> next;
        load_block<D>(next, s, j + share * kBlock, end, lane);
        attend_block<D>(r, now, j, end, lane);
        now = next;
      }
    }
    r.l += __shfl_xor_sync(0xffffffffu, r.l, 1);
    r.l += __shfl_xor_sync(0xffffffffu, r.l, 2);
  }
  // the lane's output dimensions in order, the two row halves of the accumulators added
  float o[N];
  if (live) {
    const float back = power2(r.ev);
#pragma unroll
    for (int t = 0; t < Rows<D>::kTiles; t++) {
      o[t] = (r.o[t][0] + r.o[t][2]) * back;
      o[N / 2 + t] = (r.o[t][1] + r.o[t][3]) * back;
    }
  }
  if (share > 1) {
    if (live) {
      if (c == 0) {
        merge_m[warp][g] = r.m;
        merge_l[warp][g] = r.l;
      }
#pragma unroll
      for (int i = 0; i < N; i += 4)
        *reinterpret_cast<float4*>(&merge_o[(warp * kGroupHeads + g) * D + c * N + i]) =
            make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
    }
    __syncthreads();
    if (!live || member != 0) return;
    float M = -INFINITY, L = 0.0f;
    for (int w = 0; w < share; w++) M = fmaxf(M, merge_m[warp + w][g]);
#pragma unroll
    for (int i = 0; i < N; i++) o[i] = 0.0f;
    for (int w = 0; w < share; w++) {
      const float m = merge_m[warp + w][g], f = m == -INFINITY ? 0.0f : exp2f(m - M);
      L = fmaf(merge_l[warp + w][g], f, L);
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(&merge_o[((warp + w) * kGroupHeads + g) * D + c * N + i]);
        o[i] = fmaf(v.x, f, o[i]);
        o[i + 1] = fmaf(v.y, f, o[i + 1]);
        o[i + 2] = fmaf(v.z, f, o[i + 2]);
        o[i + 3] = fmaf(v.w, f, o[i + 3]);
      }
    }
    r.m = M;
    r.l = L;
  }
  if (!live || g >= heads) return;
  const int64_t at = row * a.heads + head + g;
  if (plan.splits > 1) {
    const int64_t part = (int64_t)(plan.parts + split) * parts.per_part + at;
    if (c == 0) parts.ml[part] = make_float2(r.m, r.l);
    if (r.m == -INFINITY) return;  // an empty split: its values are never read
#pragma unroll
    for (int i = 0; i < N; i += 4)
      *reinterpret_cast<float4*>(parts.o + part * D + c * N + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
    return;
  }
  for (int p = 0; p < plan.parts; p++) {
    const int64_t part = p * parts.per_part + at;
    const float2 ml = parts.ml[part];
    if (ml.x == -INFINITY) continue;
    const float M = fmaxf(r.m, ml.x), f0 = r.m == -INFINITY ? 0.0f : exp2f(r.m - M), f1 = exp2f(ml.x - M);
    r.l = fmaf(r.l, f0, ml.y * f1);
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(parts.o + part * D + c * N + i);
      o[i] = fmaf(o[i], f0, v.x * f1);
      o[i + 1] = fmaf(o[i + 1], f0, v.y * f1);
      o[i + 2] = fmaf(o[i + 2], f0, v.z * f1);
      o[i + 3] = fmaf(o[i + 3], f0, v.w * f1);
    }
    r.m = M;
  }
  const float over = r.l > 0.0f ? 1.0f / r.l : r.l == 0.0f ? 0.0f : r.l;
#pragma unroll
  for (int i = 0; i < N; i++) o[i] *= over;
  T* out = static_cast<T*>(a.out) + row * a.out_stride + (head + g) * D + c * N;
  store_out<T, N>(out, o, (reinterpret_cast<uintptr_t>(out) & 15) == 0);
  if (c == 0 && a.lse) a.lse[at] = r.l == 0.0f ? -INFINITY : (r.m + log2f(r.l)) * kLn2;
}

// Merges the parts of every (row, head): one warp each.
template <class T, int D>
__global__ void __launch_bounds__(kStreamThreads) k_attend_merge(const __grid_constant__ needle_prefix_attention a, int count,
                                                                 const Parts parts) {
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t at = (int64_t)blockIdx.x * kStreamWarps + (threadIdx.x >> 5);
  if (at >= parts.per_part) return;
  const int64_t row = at / a.heads;
  const int slot = a.slots ? a.slots[row] : (int)min(row, (int64_t)0x7fffffff);
  if (slot < 0 || slot >= a.slot_count) return;
  float M = -INFINITY, L = 0.0f, o[N];
#pragma unroll
  for (int i = 0; i < N; i++) o[i] = 0.0f;
  for (int p = 0; p < count; p++) M = fmaxf(M, parts.ml[p * parts.per_part + at].x);
#pragma unroll 4
  for (int p = 0; p < count; p++) {
    const int64_t part = p * parts.per_part + at;
    const float2 ml = parts.ml[part];
    if (ml.x == -INFINITY) continue;
    const float f = exp2f(ml.x - M);
    L = fmaf(ml.y, f, L);
    const Vec<float, N> v = *reinterpret_cast<const Vec<float, N>*>(parts.o + part * D + lane * N);
#pragma unroll
    for (int i = 0; i < N; i++) o[i] = fmaf(v.v[i], f, o[i]);
  }
  const float over = L > 0.0f ? 1.0f / L : L == 0.0f ? 0.0f : L;
  T* out = static_cast<T*>(a.out) + row * a.out_stride + (at - row * a.heads) * D + lane * N;
#pragma unroll
  for (int i = 0; i < N; i++) out[i] = from_f32<T>(o[i] * over);
  if (lane == 0 && a.lse) a.lse[at] = L == 0.0f ? -INFINITY : (M + log2f(L)) * kLn2;
}

// ------------------------------------------------------------------ the prefix on the tensor cores
//
// k_attend_prefix.  With many rows the prefix is a dense product: the heads of a KV head of all rows are
// packed into M (packed row i = row i / group, head i % group), 256 to a CTA as two tiles of 128, and
// the CTA walks its part of the prefix in tiles of kNT positions:
//   loader warps    read int8 codes, turn them into fp16 (exact) and write K and V tiles, in the same
//                   layout [position][64 dimensions, 128-byte swizzle], into rings in shared memory; V is
//                   the B operand with its N dimension contiguous, so nothing is transposed
//   MMA warp        S_t = Q_t K^T (tcgen05.mma, both from shared memory) and O_t += P_t V (P from
//                   tensor memory), for the two tiles t in turn, so that one tile's products run while
//                   the other's softmax does
//   softmax warps   two warpgroups, one thread per packed row: S from tensor memory twice (maximum,
//                   then exponentials), P back to it as fp16; O stays in tensor memory and is only
//                   rescaled when a tile exceeds the reference maximum by 2^7
// The reference M of a row covers the value scale too: a weight is 2^(s - M) vs <= 2^15, inside fp16, and
// sums and outputs share the factor, which cancels.  16-bit queries are exact in fp16 after their row's
// power of two (the score scale comes after the product), and their weights are rounded to fp16 once (2^-12 each, averaged over the positions; the
// output's own rounding is 2^-12 or more).  Binary32 queries (kSplit) and their weights are split into fp16
// heads and tails, two MMAs each, in tiles of 64 positions (tensor memory holds the tails).
// What bounds it: 128 x 128 exponentials of a tile take 1024 cycles of the SM's 16 a cycle, its two
// products at D = 128 another 1024 on the tensor pipe.
// Every wait is bounded (2 s): a wait that runs out is reported through the wait-status words, and the
// rows' parts become NaN.
constexpr int kPrefixSoftmaxWarps = 8, kPrefixLoaderWarps = 4;
constexpr int kPrefixMmaWarp = kPrefixSoftmaxWarps + kPrefixLoaderWarps;
constexpr int kPrefixThreads = (kPrefixMmaWarp + 1) * 32;
constexpr int kPrefixRows = 256;  // packed rows of a CTA
constexpr uint64_t kPrefixWaitNs = 2000000000ull;
constexpr float kRaise = 7.0f;

template <int D, bool SPLIT>
struct PrefixShape {
  static constexpr int kNT = SPLIT ? 64 : 128;       // positions of a tile
  static constexpr int kHalves = D / 64;
  static constexpr int kParts = SPLIT ? 2 : 1;       // fp16 parts of a query or weight
  static constexpr int kStages = D == 64 ? 3 : 2;
  static constexpr uint32_t kQHalf = 128 * 128;                       // bytes of 128 rows x 64 dimensions
  static constexpr uint32_t kQTile = kQHalf * kHalves * kParts;       // [part][half]
  static constexpr uint32_t kKvHalf = kNT * 128;
  static constexpr uint32_t kKvTile = kKvHalf * kHalves;
  static constexpr uint32_t kK = 2 * kQTile, kV = kK + kStages * kKvTile;
  static constexpr uint32_t kScales = kV + kStages * kKvTile;         // per stage: kNT key, kNT value scales
  static constexpr uint32_t kSmem = kScales + kStages * kNT * 8 + 1024;
  // tensor memory columns
  static constexpr uint32_t kS = 0;                                    // two tiles of kNT
  static constexpr bool kOverlay = D == 128 && !SPLIT;                 // P takes the place of S
  static constexpr uint32_t kP = kOverlay ? 0 : (SPLIT ? 128 : 384);
  static constexpr uint32_t kPStep = kOverlay ? kNT : 64;              // from one tile's P to the other's
  static constexpr uint32_t kO = 256;
};

__device__ __forceinline__ uint32_t shared_address(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void barrier_init(uint64_t* b, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared_address(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(shared_address(b)) : "memory");
}
__device__ __forceinline__ bool barrier_try(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(shared_address(b)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Waits for the phase of the given parity; false once kPrefixWaitNs has passed without it.
__device__ __forceinline__ bool barrier_wait(uint64_t* b, uint32_t parity) {
  if (barrier_try(b, parity)) return true;
  uint64_t start, now;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(start));
  for (;;) {
    for (int i = 0; i < 64; i++)
      if (barrier_try(b, parity)) return true;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
    if (now - start > kPrefixWaitNs) return false;
  }
}

// Byte offset of 16-byte unit `unit` (0..7) of row `row` in a [rows][64 x fp16] tile, 128-byte swizzle.
__device__ __forceinline__ uint32_t swizzled(int row, int unit) {
  return (uint32_t)(row * 128 + ((unit ^ (row & 7)) << 4));
}
// Shared-memory matrix descriptors, 128-byte swizzle, 8-row groups 1024 bytes apart.  K contiguous: the rows
// are M or N.  N contiguous: the rows are K, and 64-wide blocks of N lie `block` bytes apart.
__device__ __forceinline__ uint64_t descriptor(uint32_t address, uint32_t block) {
  return (uint64_t)((address >> 4) & 0x3FFF) | ((uint64_t)((block >> 4) & 0x3FFF) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// fp16 x fp16 -> fp32, M = 128, N = n; B with N contiguous when `b_n`.
__device__ __forceinline__ uint32_t instruction(int n, bool b_n) {
  return (1u << 4) | (b_n ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void mma_shared(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u)
      : "memory");
}
__device__ __forceinline__ void mma_tensor(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u)
      : "memory");
}
// Arrives on `b` once every MMA this thread has issued is complete.
__device__ __forceinline__ void mma_commit_to(uint64_t* b) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(shared_address(b))
               : "memory");
}

// 32 (16) consecutive columns of this thread's lane of tensor memory.
__device__ __forceinline__ void tensor_load32(uint32_t at, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(at));
}
__device__ __forceinline__ void tensor_store16(uint32_t at, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(at),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tensor_wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tensor_wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tensor_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tensor_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Shared-memory writes of this thread before reads of the tensor cores.
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Two binary32 values at once.
struct Two {
  uint64_t v;
};
__device__ __forceinline__ Two two(float a, float b) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void apart(Two t, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(t.v)); }
__device__ __forceinline__ Two mul2(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ float power2f(float v) {  // 2^v, relative error 2^-22, 0 below 2^-126
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Scores from position `valid` on of a 32-position chunk become -inf.
__device__ __forceinline__ void hide(uint32_t* x, int valid) {
#pragma unroll
  for (int j = 0; j < 32; j++)
    if (j >= valid) x[j] = 0xff800000u;
}

template <class T, int D, bool SPLIT>
__global__ void __launch_bounds__(kPrefixThreads, 1)
    k_attend_prefix(const __grid_constant__ needle_prefix_attention a, const Parts parts, int part_len, float scale,
                    uint32_t* wait_words) {
  using P = PrefixShape<D, SPLIT>;
  constexpr int NT = P::kNT;
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ __align__(8) uint64_t q_full, s_full[2], p_full[2], o_full;
  __shared__ __align__(8) uint64_t k_full[P::kStages], k_empty[P::kStages], v_full[P::kStages], v_empty[P::kStages];
  __shared__ uint32_t tensor_base;
  __shared__ int failed;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int h = blockIdx.y, group = a.heads / a.kv_heads;
  const int64_t packed = (int64_t)a.rows * group, first = (int64_t)blockIdx.x * kPrefixRows;
  const int tiles_m = packed - first > 128 ? 2 : 1;
  const int begin = blockIdx.z * part_len, end = min(begin + part_len, a.prefix_length);
  const int n = (end - begin + NT - 1) / NT;
  const uint32_t sm = (shared_address(raw) + 1023u) & ~1023u;
  unsigned char* smem = raw + (sm - shared_address(raw));

  if (tid == 0) {
    barrier_init(&q_full, 4 * tiles_m);
    for (int t = 0; t < 2; t++) {
      barrier_init(&s_full[t], 1);
      barrier_init(&p_full[t], 4);
    }
    barrier_init(&o_full, 1);
    for (int i = 0; i < P::kStages; i++) {
      barrier_init(&k_full[i], kPrefixLoaderWarps);
      barrier_init(&v_full[i], kPrefixLoaderWarps);
      barrier_init(&k_empty[i], 1);
      barrier_init(&v_empty[i], 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    failed = 0;
  }
  if (warp == kPrefixMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_address(&tensor_base)),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tensor_fence_before();
  __syncthreads();
  tensor_fence_after();
  const uint32_t tm = tensor_base;

  if (warp == kPrefixMmaWarp) {
    const uint32_t qk = instruction(NT, false), pv = instruction(D, true);
    bool ok = true;
    auto wait = [&](uint64_t* b, uint32_t parity) {  // one lane polls, the warp stays together
      ok = ok && __all_sync(0xffffffffu, lane != 0 || barrier_wait(b, parity));
      __syncwarp();
    };
    auto scores = [&](int t, int i) {  // S_t = Q_t K_i^T
      const uint32_t q = sm + t * P::kQTile, k = sm + P::kK + (i % P::kStages) * P::kKvTile;
#pragma unroll
      for (int part = 0; part < P::kParts; part++)
#pragma unroll
        for (int half = 0; half < P::kHalves; half++)
#pragma unroll
          for (int s = 0; s < 4; s++)
            mma_shared(tm + P::kS + t * NT, descriptor(q + (part * P::kHalves + half) * P::kQHalf + s * 32, 16),
                       descriptor(k + half * P::kKvHalf + s * 32, 16), qk, part + half + s > 0);
      mma_commit_to(&s_full[t]);
    };
    auto values = [&](int t, int i) {  // O_t += P_t V_i
      const uint32_t v = sm + P::kV + (i % P::kStages) * P::kKvTile;
#pragma unroll
      for (int part = 0; part < P::kParts; part++)
#pragma unroll
        for (int s = 0; s < NT / 16; s++)
          mma_tensor(tm + P::kO + t * D, tm + P::kP + t * P::kPStep + part * (NT / 2) + s * 8,
                     descriptor(v + s * 2048, P::kKvHalf), pv, i > 0 || part + s > 0);
    };
    wait(&q_full, 0);
    wait(&k_full[0], 0);
    if (ok && lane == 0) {
      tensor_fence_after();
      for (int t = 0; t < tiles_m; t++) scores(t, 0);
      mma_commit_to(&k_empty[0]);
    }
    __syncwarp();
    for (int i = 0; i < n && ok; i++) {
      for (int t = 0; t < tiles_m && ok; t++) {
        if (t == 0) wait(&v_full[i % P::kStages], (i / P::kStages) & 1);
        wait(&p_full[t], i & 1);
        if (ok && lane == 0) {
          tensor_fence_after();
          values(t, i);
          if (t == tiles_m - 1) mma_commit_to(&v_empty[i % P::kStages]);
        }
        __syncwarp();
        if (i + 1 < n) {
          const int st = (i + 1) % P::kStages;
          if (t == 0) wait(&k_full[st], ((i + 1) / P::kStages) & 1);
          if (ok && lane == 0) {
            tensor_fence_after();
            scores(t, i + 1);
            if (t == tiles_m - 1) mma_commit_to(&k_empty[st]);
          }
          __syncwarp();
        }
      }
    }
    if (lane == 0) {
      if (!ok) atomicExch(&failed, 1);
      mma_commit_to(&o_full);
    }
    __syncwarp();
  } else if (warp >= kPrefixSoftmaxWarps) {
    // ---- loaders: K and V tiles in turn, the next tile's codes in registers while this one is written
    constexpr int kUnits = NT * D / 16 / (kPrefixLoaderWarps * 32);  // 16-code units of a thread
    constexpr int kRowUnits = D / 16;
    const int lt = tid - kPrefixSoftmaxWarps * 32;
    const int64_t base = (int64_t)h * a.prefix_capacity;
    uint4 code[kUnits];
    float key_scale = 0.0f, value_scale = 0.0f;
    auto fetch = [&](int item) {  // item 2 i: K of tile i, 2 i + 1: V
      const int8_t* src = (item & 1) ? a.prefix_value_codes : a.prefix_key_codes;
      const int j = begin + (item >> 1) * NT;
#pragma unroll
      for (int u = 0; u < kUnits; u++) {
        const int unit = u * kPrefixLoaderWarps * 32 + lt, p = j + unit / kRowUnits;
        code[u] = p < end ? __ldg(reinterpret_cast<const uint4*>(src + (base + p) * D) + unit % kRowUnits) : make_uint4(0, 0, 0, 0);
      }
      if ((item & 1) && lt < NT) {
        key_scale = j + lt < end ? __ldg(a.prefix_key_scales + base + j + lt) : 1.0f;  // -inf stays -inf
        value_scale = j + lt < end ? __ldg(a.prefix_value_scales + base + j + lt) : 0.0f;
      }
    };
    bool ok = true;
    fetch(0);
    for (int item = 0; item < 2 * n; item++) {
      const int i = item >> 1, st = i % P::kStages;
      const bool value = item & 1;
      if (i >= P::kStages) {
        ok = __all_sync(0xffffffffu, lane != 0 || barrier_wait(value ? &v_empty[st] : &k_empty[st], (i / P::kStages - 1) & 1));
        if (!ok) break;
      }
      unsigned char* to = smem + (value ? P::kV : P::kK) + st * P::kKvTile;
#pragma unroll
      for (int u = 0; u < kUnits; u++) {
        const int unit = u * kPrefixLoaderWarps * 32 + lt, row = unit / kRowUnits, cc = unit % kRowUnits;
        const uint32_t w[4] = {code[u].x ^ 0x80808080u, code[u].y ^ 0x80808080u, code[u].z ^ 0x80808080u, code[u].w ^ 0x80808080u};
        const uint4 lo = make_uint4(codes_f16(w[0], 0x4140), codes_f16(w[0], 0x4342), codes_f16(w[1], 0x4140), codes_f16(w[1], 0x4342));
        const uint4 hi = make_uint4(codes_f16(w[2], 0x4140), codes_f16(w[2], 0x4342), codes_f16(w[3], 0x4140), codes_f16(w[3], 0x4342));
        unsigned char* tile = to + (cc >> 2) * P::kKvHalf;
        // the two 64-dimension halves of a row share banks: they write their two units in opposite order
        const int flip = (cc >> 2) & 1, at = (cc & 3) * 2;
        *reinterpret_cast<uint4*>(tile + swizzled(row, at + flip)) = flip ? hi : lo;
        *reinterpret_cast<uint4*>(tile + swizzled(row, at + 1 - flip)) = flip ? lo : hi;
      }
      if (value && lt < NT) {
        float* s = reinterpret_cast<float*>(smem + P::kScales + st * NT * 8);
        s[lt] = key_scale;
        s[NT + lt] = value_scale;
      }
      if (item + 1 < 2 * n) fetch(item + 1);
      fence_async_proxy();
      __syncwarp();
      if (lane == 0) barrier_arrive(value ? &v_full[st] : &k_full[st]);
    }
    if (!ok) atomicExch(&failed, 1);
  } else {
    // ---- softmax: thread = packed row
    const int t = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    if (t < tiles_m) {
      const int64_t i = first + t * 128 + r;
      const int64_t row = i / group, head = (int64_t)h * group + i % group;
      const int slot = i < packed ? (a.slots ? a.slots[row] : (int)min(row, (int64_t)0x7fffffff)) : -1;
      const bool live = slot >= 0 && slot < a.slot_count;
      // the row's query, scaled to a largest magnitude in [2^10, 2^11), as fp16 part(s) in shared memory
      const T* q = static_cast<const T*>(a.q) + (live ? row * a.q_stride + head * D : 0);
      constexpr int V = 16 / sizeof(T);
      const bool vec = live && (reinterpret_cast<uintptr_t>(q) & 15) == 0;
      auto query = [&](int d, float* x) {  // 8 dimensions from d on
#pragma unroll
        for (int k = 0; k < 8 / V; k++) {
          if (vec) {
            const Vec<T, V> v = *reinterpret_cast<const Vec<T, V>*>(q + d + k * V);
#pragma unroll
            for (int e = 0; e < V; e++) x[k * V + e] = to_f32(v.v[e]);
          } else {
#pragma unroll
            for (int e = 0; e < V; e++) x[k * V + e] = live ? to_f32(q[d + k * V + e]) : 0.0f;
          }
        }
      };
      float top = 0.0f;
#pragma unroll 4
      for (int d = 0; d < D; d += 8) {
        float x[8];
        query(d, x);
#pragma unroll
        for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[e]));
      }
      const int e10 = min(max(exponent_of(top), -110), 110);
      const float up = power2(10 - e10), inverse = power2(e10 - 10) * (scale * kLog2e);
#pragma unroll 2
      for (int d = 0; d < D; d += 8) {
        float x[8];
        uint32_t head4[4], tail4[4];
        query(d, x);
#pragma unroll
        for (int e = 0; e < 4; e++) split_f16(x[2 * e] * up, x[2 * e + 1] * up, head4[e], tail4[e]);
        unsigned char* to = smem + t * P::kQTile + (d >> 6) * P::kQHalf + swizzled(r, (d & 63) >> 3);
        *reinterpret_cast<uint4*>(to) = make_uint4(head4[0], head4[1], head4[2], head4[3]);
        if constexpr (SPLIT)
          *reinterpret_cast<uint4*>(to + P::kHalves * P::kQHalf) = make_uint4(tail4[0], tail4[1], tail4[2], tail4[3]);
      }
      fence_async_proxy();
      __syncwarp();
      if (lane == 0) barrier_arrive(&q_full);

      const uint32_t mine = tm + ((uint32_t)(quarter * 32) << 16);
      const uint32_t s_at = mine + P::kS + t * NT, p_at = mine + P::kP + t * P::kPStep, o_at = mine + P::kO + t * D;
      float M = -INFINITY, l = 0.0f;
      bool ok = true;
      for (int k = 0; k < n; k++) {
        const int st = k % P::kStages;
        ok = __all_sync(0xffffffffu, lane != 0 || (barrier_wait(&v_full[st], (k / P::kStages) & 1) && barrier_wait(&s_full[t], k & 1)));
        if (!ok) break;
        __syncwarp();
        tensor_fence_after();
        const ulonglong2* ks = reinterpret_cast<const ulonglong2*>(smem + P::kScales + st * NT * 8);
        const ulonglong2* vs = ks + NT / 4;
        const int valid = min(NT, end - (begin + k * NT));
        // maximum of the scores, and the largest value scale of the tile
        float most = -INFINITY;
#pragma unroll
        for (int c = 0; c < NT; c += 32) {
          uint32_t x[32];
          tensor_load32(s_at + c, x);
          tensor_wait_loads();
          if (c + 32 > valid) hide(x, valid - c);
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const ulonglong2 s2 = ks[(c + j) / 4];
            float v[4];
            apart(mul2(two(__uint_as_float(x[j]), __uint_as_float(x[j + 1])), Two{s2.x}), v[0], v[1]);
            apart(mul2(two(__uint_as_float(x[j + 2]), __uint_as_float(x[j + 3])), Two{s2.y}), v[2], v[3]);
            most = fmaxf(fmaxf(most, fmaxf(v[0], v[1])), fmaxf(v[2], v[3]));
          }
        }
        const float* v1 = reinterpret_cast<const float*>(vs);
        uint32_t vtop = 0;
#pragma unroll
        for (int c = 0; c < NT; c += 32) vtop = max(vtop, __float_as_uint(v1[c + lane]) & 0x7fffffffu);
        vtop = __reduce_max_sync(0xffffffffu, vtop);
        const int ev = min(max(exponent_of(__uint_as_float(vtop)), -100), 100) - 6;
        const float reach = most * inverse + (float)ev;  // weights are below 2^(reach - M + 7)
        const bool raise = reach > M + kRaise;
        if (__any_sync(0xffffffffu, raise)) {
          const float Mn = raise ? reach + 1.0f : M;
          const float f = M == -INFINITY ? 0.0f : power2f(M - Mn);
          l *= f;
          M = Mn;
          if (k > 0) {
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t x[32];
              tensor_load32(o_at + c, x);
              tensor_wait_loads();
#pragma unroll
              for (int j = 0; j < 32; j++) x[j] = __float_as_uint(__uint_as_float(x[j]) * f);
              tensor_store16(o_at + c, x);
              tensor_store16(o_at + c + 16, x + 16);
            }
          }
        }
        const Two inverse2 = two(inverse, inverse), minus = two(-M, -M);
        Two sum = two(0.0f, 0.0f);
#pragma unroll
        for (int c = 0; c < NT; c += 32) {
          uint32_t x[32], head16[16], tail16[16];
          tensor_load32(s_at + c, x);
          tensor_wait_loads();
          if (c + 32 > valid) hide(x, valid - c);
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const ulonglong2 s2 = ks[(c + j) / 4], v2 = vs[(c + j) / 4];
#pragma unroll
            for (int o = 0; o < 4; o += 2) {
              const Two x2 = two(__uint_as_float(x[j + o]), __uint_as_float(x[j + o + 1]));
              float e0, e1;
              apart(fma2(mul2(x2, Two{o ? s2.y : s2.x}), inverse2, minus), e0, e1);
              e0 = power2f(e0);
              e1 = power2f(e1);
              const Two p2 = two(e0, e1);
              sum = add2(sum, p2);
              float w0, w1;
              apart(mul2(p2, Two{o ? v2.y : v2.x}), w0, w1);
              if constexpr (SPLIT) split_f16(w0, w1, head16[(j + o) / 2], tail16[(j + o) / 2]);
              else head16[(j + o) / 2] = half2_bits(__floats2half2_rn(w0, w1));
            }
          }
          tensor_store16(p_at + c / 2, head16);
          if constexpr (SPLIT) tensor_store16(p_at + NT / 2 + c / 2, tail16);
        }
        float s0, s1;
        apart(sum, s0, s1);
        l += s0 + s1;
        tensor_wait_stores();
        tensor_fence_before();
        __syncwarp();
        if (lane == 0) barrier_arrive(&p_full[t]);
      }
      if (!ok) atomicExch(&failed, 1);
      const bool done = __all_sync(0xffffffffu, lane != 0 || barrier_wait(&o_full, 0));
      tensor_fence_after();
      const bool bad = !ok || !done || *(volatile int*)&failed != 0;
      if (bad && lane == 0) report_wait_timeout(wait_words, kWaitAttention);
      const int64_t part = blockIdx.z * parts.per_part + row * a.heads + head;
      if (live) parts.ml[part] = bad ? make_float2(0.0f, NAN) : make_float2(M, l);
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t x[32];
        tensor_load32(o_at + c, x);
        tensor_wait_loads();
        if (live) {
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<uint4*>(parts.o + part * D + c + j) = make_uint4(x[j], x[j + 1], x[j + 2], x[j + 3]);
        }
      }
    }
  }
  tensor_fence_before();
  __syncthreads();
  if (warp == kPrefixMmaWarp) {
    tensor_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(512u) : "memory");
  }
}

// Warps that fill the GPU, at 16 an SM.
constexpr int kFullWarps = 148 * 16;
// Positions below which a warp's share is not worth a further split.
constexpr int kLeastSplit = 256;

// Rows (times heads of a KV head) and prefix positions from which the prefix goes to k_attend_prefix.
constexpr int64_t kPrefixLeastRows = 64, kPrefixLeastPositions = 128;

StreamPlan plan_for(const needle_prefix_attention& a) {
  StreamPlan p{};
  const int group = a.heads / a.kv_heads;
  p.groups = (group + kGroupHeads - 1) / kGroupHeads;
  const int64_t packed = int64_t(a.rows) * group;
  if (packed >= kPrefixLeastRows && a.prefix_length >= kPrefixLeastPositions) {
    // parts of the prefix: as many as keep the waves of CTAs short, each costing about 3 tiles on top
    const int nt = a.type == NEEDLE_TYPE_F32 ? 64 : 128;
    const int tiles = (a.prefix_length + nt - 1) / nt;
    const int64_t units = (packed + kPrefixRows - 1) / kPrefixRows * a.kv_heads;
    int64_t best = 0;
    int parts = 1;
    for (int c = 1; c <= std::min(tiles, 64); c++) {
      const int64_t cost = (units * c + 147) / 148 * ((tiles + c - 1) / c + 3);
      if (c == 1 || cost < best) {
        best = cost;
        parts = c;
      }
    }
    p.part_len = (tiles + parts - 1) / parts * nt;
    p.parts = (a.prefix_length + p.part_len - 1) / p.part_len;
  }
  const int64_t units = int64_t(a.rows) * a.kv_heads * p.groups;
  const int64_t positions = int64_t(p.parts ? 0 : a.prefix_length) + a.capacity;
  p.warps = 1;
  while (p.warps < kStreamWarps && units * p.warps < kFullWarps && positions > int64_t(p.warps) * kBlock) p.warps *= 2;
  // the longest splits that still give every SM its warps
  int64_t splits = 1;
  if (p.warps == kStreamWarps) splits = std::max<int64_t>(1, std::min(kFullWarps / (units * p.warps), positions / kLeastSplit));
  p.split_len = int(std::min<int64_t>((positions + splits - 1) / splits, 0x40000000));
  p.split_len = std::max(kBlock, (p.split_len + kBlock - 1) / kBlock * kBlock);
  p.splits = int(std::max<int64_t>(1, (positions + p.split_len - 1) / p.split_len));
  return p;
}

// Parts in the workspace: those of the prefix and, when there are several, the splits.
int part_count(const StreamPlan& p) { return p.parts + (p.splits > 1 ? p.splits : 0); }

size_t workspace_bytes_for(const needle_prefix_attention& a, const StreamPlan& p) {
  const size_t each = size_t(a.rows) * a.heads;
  return (part_count(p) * each * (8 + size_t(a.head_dim) * 4) + 15) / 16 * 16;
}

template <class T, int D>
cudaError_t launch_attention(const needle_prefix_attention& a, const StreamPlan& p, void* workspace, float scale, uint32_t* wait_words,
                             cudaStream_t s) {
  Parts parts{};
  parts.per_part = int64_t(a.rows) * a.heads;
  parts.o = static_cast<float*>(workspace);
  parts.ml = reinterpret_cast<float2*>(parts.o + part_count(p) * parts.per_part * D);
  if (p.parts > 0) {
    constexpr bool kSplit = sizeof(T) == 4;
    using Shape = PrefixShape<D, kSplit>;
    cudaError_t e = cudaFuncSetAttribute(k_attend_prefix<T, D, kSplit>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape::kSmem);
    if (e != cudaSuccess) return e;
    const int64_t packed = int64_t(a.rows) * (a.heads / a.kv_heads);
    k_attend_prefix<T, D, kSplit><<<dim3((unsigned)((packed + kPrefixRows - 1) / kPrefixRows), a.kv_heads, p.parts), kPrefixThreads, Shape::kSmem, s>>>(a, parts, p.part_len, scale, wait_words);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  const int64_t units = int64_t(a.rows) * a.kv_heads * p.groups;
  const int per_cta = kStreamWarps / p.warps;
  const size_t smem = p.warps > 1 ? size_t(kStreamWarps) * kGroupHeads * D * 4 : 0;
  k_attend_stream<T, D><<<dim3((unsigned)((units + per_cta - 1) / per_cta), p.splits), kStreamThreads, smem, s>>>(a, p, parts, scale);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || p.splits == 1) return e;
  k_attend_merge<T, D><<<(unsigned)((parts.per_part + kStreamWarps - 1) / kStreamWarps), kStreamThreads, 0, s>>>(a, part_count(p), parts);
  return cudaGetLastError();
}

int check_attention(const needle_prefix_attention* a) {
  if (!a) return refuse("null argument");
  if (a->type < NEEDLE_TYPE_F32 || a->type > NEEDLE_TYPE_BF16) return refuse("unknown element type");
  if (a->head_dim != 64 && a->head_dim != 128) return refuse("head dimensions of 64 and 128 only");
  if (a->kv_heads < 1 || a->heads < 1 || a->heads % a->kv_heads != 0 || a->heads > 4096)
    return refuse("heads must be a multiple of kv_heads, at most 4096");
  if (a->rows < 0 || a->prefix_length < 0 || a->slot_count < 0 || a->capacity < 0)
    return refuse("bad row, position or slot count");
  if (a->prefix_length > a->prefix_capacity) return refuse("the prefix is longer than its capacity");
  if (!(std::isfinite(a->scale) && a->scale >= 0.0f)) return refuse("the score scale must be positive, or 0 for its default");
  return NEEDLE_OK;
}

}  // namespace
}  // namespace needle

using namespace needle;

extern "C" int needle_cuda_prefix_attention_workspace(const needle_prefix_attention* a, size_t* bytes) {
  return entry([&] {
    if (int rc = check_attention(a)) return rc;
    if (!bytes) return refuse("null argument");
    *bytes = workspace_bytes_for(*a, plan_for(*a));
    return int(NEEDLE_OK);
  });
}

extern "C" int needle_cuda_prefix_attention_dev(const needle_prefix_attention* a, void* workspace,
                                                size_t workspace_bytes, void* stream) {
  return entry([&] {
    if (int rc = check_attention(a)) return rc;
    if (a->rows == 0) return int(NEEDLE_OK);
    if (!a->q || !a->out) return refuse("null argument");
    if (a->prefix_length > 0 && (!a->prefix_key_codes || !a->prefix_key_scales || !a->prefix_value_codes || !a->prefix_value_scales))
      return refuse("null argument");
    if (!a->counts) return refuse("null argument");
    if (a->capacity > 0 && a->slot_count > 0 && (!a->key_codes || !a->key_scales || !a->value_codes || !a->value_scales))
      return refuse("null argument");
    const int64_t width = int64_t(a->heads) * a->head_dim;
    if (a->rows > 1 && (a->q_stride < width || a->out_stride < width))
      return refuse("a row stride is shorter than its row");
    const size_t element = type_bytes(a->type);
    if (!aligned_to(a->q, element) || !aligned_to(a->out, element))
      return refuse("a buffer is not aligned to its element type");
    for (const void* p : {a->prefix_key_codes, a->prefix_value_codes, a->key_codes, a->value_codes})
      if (!aligned_to(p, 16)) return refuse("key/value codes must be 16-byte aligned");
    const StreamPlan plan = plan_for(*a);
    const size_t need = workspace_bytes_for(*a, plan);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned_to(workspace, 16)))
      return refuse("the workspace must be 16-byte aligned and hold " + std::to_string(need) + " bytes");
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return refuse_cuda("prefix_attention", e);
    if (int rc = check_buffer(a->out, "out", device)) return rc;
    if (int rc = check_buffer(a->q, "q", device)) return rc;
    if (plan.parts > 0 && check_wait_status(device) != NEEDLE_OK) return int(NEEDLE_BACKEND_UNAVAILABLE);
    uint32_t* words = plan.parts > 0 ? wait_status_words(device) : nullptr;
    const float scale = a->scale > 0.0f ? a->scale : 1.0f / std::sqrt(float(a->head_dim));
    e = with_type(a->type, [&](auto zero) {
      using T = decltype(zero);
      return a->head_dim == 64 ? launch_attention<T, 64>(*a, plan, workspace, scale, words, static_cast<cudaStream_t>(stream))
                               : launch_attention<T, 128>(*a, plan, workspace, scale, words, static_cast<cudaStream_t>(stream));
    });
    return e == cudaSuccess ? int(NEEDLE_OK) : refuse_cuda("prefix_attention", e);
  });
}
