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
  int parts;       // prefix parts in the workspace, in front of the splits
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

// Warps that fill the GPU, at 16 an SM.
constexpr int kFullWarps = 148 * 16;
// Positions below which a warp's share is not worth a further split.
constexpr int kLeastSplit = 256;

StreamPlan plan_for(const needle_prefix_attention& a) {
  StreamPlan p{};
  p.groups = (a.heads / a.kv_heads + kGroupHeads - 1) / kGroupHeads;
  const int64_t units = int64_t(a.rows) * a.kv_heads * p.groups;
  const int64_t positions = int64_t(a.prefix_length) + a.capacity;
  p.warps = 1;
  while (p.warps < kStreamWarps && units * p.warps < kFullWarps && positions > int64_t(p.warps) * kBlock) p.warps *= 2;
  // the longest splits that still give every SM its warps
  int64_t splits = 1;
  if (p.warps == kStreamWarps) splits = std::max<int64_t>(1, std::min(kFullWarps / (units * p.warps), positions / kLeastSplit));
  p.split_len = int(std::min<int64_t>((positions + splits - 1) / splits, 0x40000000));
  p.split_len = std::max(kBlock, (p.split_len + kBlock - 1) / kBlock * kBlock);
  p.splits = int(std::max<int64_t>(1, (positions + p.split_len - 1) / p.split_len));
  p.parts = 0;
  return p;
}

// Parts in the workspace: those of the prefix and, when there are several, the splits.
int part_count(const StreamPlan& p) { return p.parts + (p.splits > 1 ? p.splits : 0); }

size_t workspace_bytes_for(const needle_prefix_attention& a, const StreamPlan& p) {
  const size_t each = size_t(a.rows) * a.heads;
  return (part_count(p) * each * (8 + size_t(a.head_dim) * 4) + 15) / 16 * 16;
}

template <class T, int D>
cudaError_t launch_attention(const needle_prefix_attention& a, const StreamPlan& p, void* workspace, float scale, cudaStream_t s) {
  Parts parts{};
  parts.per_part = int64_t(a.rows) * a.heads;
  parts.o = static_cast<float*>(workspace);
  parts.ml = reinterpret_cast<float2*>(parts.o + part_count(p) * parts.per_part * D);
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
    const float scale = a->scale > 0.0f ? a->scale : 1.0f / std::sqrt(float(a->head_dim));
    e = with_type(a->type, [&](auto zero) {
      using T = decltype(zero);
      return a->head_dim == 64 ? launch_attention<T, 64>(*a, plan, workspace, scale, static_cast<cudaStream_t>(stream))
                               : launch_attention<T, 128>(*a, plan, workspace, scale, static_cast<cudaStream_t>(stream));
    });
    return e == cudaSuccess ? int(NEEDLE_OK) : refuse_cuda("prefix_attention", e);
  });
}
