// prefix_attn.cu -- decode attention of a batch whose sequences share a prompt prefix: every row
// attends over the prefix's int8 keys and values, held once, and over its own int8 cache
// (#attention, packages/needle.js/src/model/runtime.ts:719-786, with the prefix taken out of the
// per-sequence caches; any head layout, binary32 arithmetic).
//
//   s_j = scale * (q . code_j) * ks_j,  o = sum_j e^(s_j - m) vs_j code_j / sum_j e^(s_j - m),
//   j over the prefix and the row's own positions;  lse = m + log sum_j e^(s_j - m)
//
// k_attend_stream.  The query heads of one KV head (up to 8) meet 32 positions at a time on the tensor
// cores (mma.sync m16n8k16, fp16 x fp16 -> fp32).  One row has few heads, so the products are thin and the
// kernel lives on its loads, 2 D + 8 bytes a position, and on its instruction count.  Every warp streams
// its positions through a ring of its own in shared memory, filled by bulk copies, so no warp waits for
// another.  Codes are exact in fp16; queries and weights, binary32, are split into fp16 heads and tails
// that sit in neighbouring columns of N (4 query heads fill its 8), whose products a lane adds up again:
// results have binary32 accuracy for every element type.  Positions and output dimensions are the M side:
//   S^T (positions x heads) = K Q^T: lane (g, c) = (lane / 4, lane % 4) reads codes of the positions g and
//     g + 8 straight into operand order (the order of k inside a product is free) and gets their scores of
//     head c;
//   O^T (dimensions x heads) = V^T P^T: the lane reads D / 8 codes of the positions 2c, 2c + 1, 2c + 8,
//     2c + 9 and pairs them byte by byte; the weights, packed as (head, tail), are brought to the lanes that
//     need them by one 8 x 8 transposition (movmatrix) for 8 positions.
// Groups of more than 4 heads (NG 2) use every converted code twice.  With heads on the M side, where 2 of
// 16 rows were of use for 2 heads, the kernel took 1.6 times the instructions.
// A unit (row, KV head, 8 heads, split of the positions) has a CTA of 2 to 8 warps, merged in shared memory, or,
// where units are many, one warp, beside those of the row's other KV heads: caches of one age end together.
// Splits and the prefix's parts are merged from the workspace.
// Measured: 4096 rows x 4 KV heads of 64, 0..256 own positions (302 MB) beside a prefix of 160: 77 us, 70 us of them the
// stream's: 4.3 TB/s, bound by its instructions (67% issued).  333 rows x 8 KV heads of 128, 0..500 (176 MB): 50 us,
// 3.5 TB/s, bound by latency at the 13 warps whose rings an SM holds.  One row of 160 + 256: 4.2 us.
#include <algorithm>
#include <cmath>

#include "prefix_attn.cuh"

namespace needle {

namespace {

constexpr int kStreamWarps = 8;
constexpr int kStreamThreads = kStreamWarps * 32;
constexpr int kStreamStages = 2;
constexpr int kGroupHeads = 8;  // query heads of one KV head taken together
constexpr int kBlock = 32;      // positions of a step

// How a call is laid out (plan_for).
struct StreamPlan {
  int groups;      // 8-head groups of a KV head
  int group;       // query heads of a KV head
  int warps, warps_log2;  // warps per unit: 1, 2, 4 or 8
  int together;    // units of a row in a CTA, where a unit is one warp
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

// 32 positions of a warp's ring.
template <int D>
struct Stage {
  int8_t k[kBlock * D], v[kBlock * D];
  float ks[kBlock], vs[kBlock];  // zeros behind the last position
};

// A warp's state of up to 4 NG heads: lane (g, c) keeps the heads c, 4 + c: their reference maximum, the sum of
// its own weights, and the output dimensions g * D / 8 .. + D / 8 - 1.
template <int D, int NG>
struct Rows {
  uint32_t q[NG][D / 16][2];  // B operand of each k-step: column g is head g / 2, its head or tail by g % 2
  float inverse[NG];          // undoes the query's power of two
  float M[NG], l[NG];         // reference maximum (base 2), sum of the lane's weights
  float o[NG][D / 16][4];
};

__device__ __forceinline__ uint32_t transpose8(uint32_t v) {  // 8 x 8 of 16 bits, a row's pair per lane
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// The n positions of a stage.
template <int D, int NG>
__device__ __forceinline__ void attend_block(Rows<D, NG>& r, const Stage<D>& b, int n, int lane) {
  const int g = lane >> 2, c = lane & 3;
  float s[NG][4], vs[4];  // positions g, g + 8, g + 16, g + 24
  float vtop = 0.0f;
#pragma unroll
  for (int u = 0; u < 2; u++) {
    float d[NG][4];
#pragma unroll
    for (int q = 0; q < NG; q++)
#pragma unroll
      for (int i = 0; i < 4; i++) d[q][i] = 0.0f;
#pragma unroll
    for (int h = 0; h < D / 64; h++) {
      const uint4 k0 = *reinterpret_cast<const uint4*>(b.k + (u * 16 + g) * D + h * 64 + c * 16);
      const uint4 k1 = *reinterpret_cast<const uint4*>(b.k + (u * 16 + 8 + g) * D + h * 64 + c * 16);
      const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const uint32_t x0 = w0[k] ^ 0x80808080u, x1 = w1[k] ^ 0x80808080u;
        const uint32_t a[4] = {codes_f16(x0, 0x4140), codes_f16(x1, 0x4140), codes_f16(x0, 0x4342), codes_f16(x1, 0x4342)};
#pragma unroll
        for (int q = 0; q < NG; q++) mma_f16(d[q], a, r.q[q][h * 4 + k][0], r.q[q][h * 4 + k][1]);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const float ks = b.ks[u * 16 + i * 8 + g];
      vs[2 * u + i] = b.vs[u * 16 + i * 8 + g];
      vtop = fmaxf(vtop, fabsf(vs[2 * u + i]));
#pragma unroll
      for (int q = 0; q < NG; q++) s[q][2 * u + i] = (d[q][2 * i] + d[q][2 * i + 1]) * (ks * r.inverse[q]);
    }
  }
  if (n < kBlock) {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (i * 8 + g >= n) {
#pragma unroll
        for (int q = 0; q < NG; q++) s[q][i] = -INFINITY;
      }
  }
  vtop = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(vtop)));
  const float ev = value_reach(vtop);
  float reach[NG];
  bool raise = false;
#pragma unroll
  for (int q = 0; q < NG; q++) {
    float top = fmaxf(fmaxf(s[q][0], s[q][1]), fmaxf(s[q][2], s[q][3]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
    reach[q] = top + ev;
    raise = raise || reach[q] > r.M[q] + kRaise;
  }
  if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
    for (int q = 0; q < NG; q++) {
      const float Mn = reach[q] > r.M[q] + kRaise ? reach[q] + 1.0f : r.M[q];
      const float f = r.M[q] == -INFINITY ? 0.0f : power2f(r.M[q] - Mn);
      r.l[q] *= f;
#pragma unroll
      for (int t = 0; t < D / 16; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) r.o[q][t][i] *= f;
      r.M[q] = Mn;
    }
  }
  uint32_t p[NG][4];  // weights of 8 positions each, as B operand
#pragma unroll
  for (int q = 0; q < NG; q++) {
    const float base = r.M[q] == -INFINITY ? 0.0f : r.M[q];
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const float e0 = power2f(s[q][i] - base), e1 = power2f(s[q][i + 1] - base);
      r.l[q] += e0 + e1;
      uint32_t heads, tails;
      split_f16(e0 * vs[i], e1 * vs[i + 1], heads, tails);
      p[q][i] = transpose8(__byte_perm(heads, tails, 0x5410));
      p[q][i + 1] = transpose8(__byte_perm(heads, tails, 0x7632));
    }
  }
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const int8_t* v = b.v + (u * 16 + 2 * c) * D + g * (D / 8);
#pragma unroll
    for (int h = 0; h < D / 64; h++) {
      uint2 v2[4];
#pragma unroll
      for (int i = 0; i < 4; i++) v2[i] = *reinterpret_cast<const uint2*>(v + ((i & 1) + (i >> 1) * 8) * D + h * 8);
#pragma unroll
      for (int word = 0; word < 2; word++) {
        uint32_t x[4];
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = (word ? v2[i].y : v2[i].x) ^ 0x80808080u;
#pragma unroll
        for (int k = 0; k < 2; k++) {  // codes 2k, 2k + 1 of the word: two neighbouring dimensions
          const uint32_t sel = k ? 0x7362 : 0x5140;
          const uint32_t lo = __byte_perm(x[0], x[1], sel), hi = __byte_perm(x[2], x[3], sel);
          const uint32_t a[4] = {codes_f16(lo, 0x4140), codes_f16(lo, 0x4342), codes_f16(hi, 0x4140), codes_f16(hi, 0x4342)};
#pragma unroll
          for (int q = 0; q < NG; q++) mma_f16(r.o[q][h * 4 + word * 2 + k], a, p[q][2 * u], p[q][2 * u + 1]);
        }
      }
    }
  }
}

// The unit's queries as they are in memory: lane (g, c) takes its share of head g / 2 (and 4 + g / 2).
template <class T, int D, int NG>
struct RawQueries {
  Vec<T, 16 / sizeof(T)> v[NG][D / 64][sizeof(T)];
};

template <class T, int D, int NG>
__device__ __forceinline__ void load_queries(RawQueries<T, D, NG>& raw, const T* q, int heads, int lane) {
  constexpr int V = 16 / sizeof(T);
  const int g = lane >> 2, c = lane & 3;
  const bool vec = (reinterpret_cast<uintptr_t>(q) & 15) == 0;
#pragma unroll
  for (int n = 0; n < NG; n++) {
    const int head = 4 * n + (g >> 1);
#pragma unroll
    for (int h = 0; h < D / 64; h++)
#pragma unroll
      for (int i = 0; i < (int)sizeof(T); i++) {
        const T* p = q + head * D + h * 64 + c * 16 + i * V;
        raw.v[n][h][i] = Vec<T, V>{};
        if (head < heads) {
          if (vec) {
            raw.v[n][h][i] = *reinterpret_cast<const Vec<T, V>*>(p);
          } else {
#pragma unroll
            for (int e = 0; e < V; e++) raw.v[n][h][i].v[e] = p[e];
          }
        }
      }
  }
}

// The queries in operand order, scaled by `scale` * log2(e) and, per head, to a largest magnitude in
// [2^10, 2^11); the rest of the warp's state at its beginning.
template <class T, int D, int NG>
__device__ __forceinline__ void begin_rows(Rows<D, NG>& r, const RawQueries<T, D, NG>& raw, float scale, int lane) {
  constexpr int V = 16 / sizeof(T);
  const int g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int n = 0; n < NG; n++) {
    float x[D / 4];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 4; i++) {
      x[i] = to_f32(raw.v[n][i / 16][i % 16 / V].v[i % V]);
      top = fmaxf(top, fabsf(x[i]));
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = min(max(exponent_of(top), -110), 110);
    const float f = power2(10 - e);
    // of head c, whose columns are 2c and 2c + 1
    r.inverse[n] = __shfl_sync(0xffffffffu, power2(e - 10), 8 * c) * (scale * kLog2e);
#pragma unroll
    for (int k = 0; k < D / 16; k++)
#pragma unroll
      for (int i = 0; i < 2; i++) {
        uint32_t head2, tail2;
        split_f16(x[4 * k + 2 * i] * f, x[4 * k + 2 * i + 1] * f, head2, tail2);
        r.q[n][k][i] = g & 1 ? tail2 : head2;
      }
    r.M[n] = -INFINITY;
    r.l[n] = 0.0f;
#pragma unroll
    for (int t = 0; t < D / 16; t++)
#pragma unroll
      for (int i = 0; i < 4; i++) r.o[n][t][i] = 0.0f;
  }
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

// What becomes of N output dimensions of a head, from g * N on, held by lane g of its eight.
template <int N>
__device__ __forceinline__ void store_part(const Parts& parts, int64_t part, float m, float l, const float* o, int g) {
  if (g == 0) parts.ml[part] = part_of(m, l);
  if (l == 0.0f) return;  // an empty part: its values are never read
#pragma unroll
  for (int i = 0; i < N; i += 4)
    *reinterpret_cast<float4*>(parts.o + part * (8 * N) + g * N + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
}

template <int N>
__device__ __forceinline__ void add_part(const Parts& parts, int64_t part, float& m, float& l, float* o, int g) {
  const float2 ml = parts.ml[part];
  if (ml.x == -INFINITY) return;
  const float M = fmaxf(m, ml.x), f0 = m == -INFINITY ? 0.0f : power2f(m - M), f1 = power2f(ml.x - M);
  l = fmaf(l, f0, ml.y * f1);
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const float4 v = *reinterpret_cast<const float4*>(parts.o + part * (8 * N) + g * N + i);
    o[i] = fmaf(o[i], f0, v.x * f1);
    o[i + 1] = fmaf(o[i + 1], f0, v.y * f1);
    o[i + 2] = fmaf(o[i + 2], f0, v.z * f1);
    o[i + 3] = fmaf(o[i + 3], f0, v.w * f1);
  }
  m = M;
}

template <class T, int N>
__device__ __forceinline__ void finish(const needle_prefix_attention& a, int row, int64_t head, int64_t at, float m, float l,
                                       float* o, int g) {
  const float over = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
#pragma unroll
  for (int i = 0; i < N; i++) o[i] *= over;
  T* out = static_cast<T*>(a.out) + row * a.out_stride + head * (8 * N) + g * N;
  store_out<T, N>(out, o, (reinterpret_cast<uintptr_t>(out) & 15) == 0);
  if (g == 0 && a.lse) a.lse[at] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
}

template <class T, int D, int NG>
__global__ void __maxnreg__(D == 64 ? (NG == 1 ? 80 : 112) : (NG == 1 ? 144 : 168))
    k_attend_stream(const __grid_constant__ needle_prefix_attention a, const StreamPlan plan, const Parts parts, float scale,
                    uint32_t* wait_words) {
  constexpr int N = D / 8;  // output dimensions of a lane
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ __align__(8) uint64_t full[kStreamWarps][kStreamStages];
  __shared__ float merge_m[kStreamWarps][kGroupHeads], merge_l[kStreamWarps][kGroupHeads];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  const int share = plan.warps, member = share > 1 ? warp : 0;
  const int row = blockIdx.x, split = blockIdx.z, group = plan.group;
  const int unit = blockIdx.y * plan.together + (share > 1 ? 0 : warp);  // of the row: KV head, 8-head group of it
  const int h = plan.groups == 1 ? unit : unit / plan.groups, g0 = (unit - h * plan.groups) * 4 * NG;
  const int heads = min(4 * NG, group - g0);
  const int64_t head = (int64_t)h * group + g0;  // the unit's first query head
  RawQueries<T, D, NG> queries;  // ahead of everything that waits for memory
  load_queries<T, D, NG>(queries, static_cast<const T*>(a.q) + row * a.q_stride + head * D, heads, lane);
  const int slot = a.slots ? __ldg(a.slots + row) : row, count = min(max(__ldg(a.counts + row), 0), a.capacity);
  if (slot < 0 || slot >= a.slot_count) {
    if (plan.parts > 0) wait_for_prior();  // no CTA, so not this kernel either, ends before the prefix kernel
    return;
  }
  Rows<D, NG> r;
  bool ok = true;
  Stage<D>* ring = reinterpret_cast<Stage<D>*>(raw) + warp * kStreamStages;
  uint64_t* bars = full[warp];
  if (lane == 0) {
    for (int s = 0; s < kStreamStages; s++) barrier_init(&bars[s], 33);  // each lane's scale copies, and the codes
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  const int64_t own = ((int64_t)slot * a.kv_heads + h) * a.capacity, shared = (int64_t)h * a.prefix_capacity;
  const int prefix = plan.parts ? 0 : a.prefix_length;
  // positions [from, to) of prefix ++ own cache, in blocks that do not straddle the two
  const int64_t from = (int64_t)split * plan.split_len, to = min(from + plan.split_len, (int64_t)prefix + count);
  const int begin0 = (int)min(from, (int64_t)prefix), end0 = (int)min(max(to, (int64_t)0), (int64_t)prefix);
  const int begin1 = (int)max(from - prefix, (int64_t)0), end1 = (int)max(to - prefix, (int64_t)begin1);
  const int blocks0 = max(end0 - begin0 + kBlock - 1, 0) / kBlock, blocks1 = (end1 - begin1 + kBlock - 1) / kBlock;
  const int mine = (blocks0 + blocks1 - member + share - 1) >> plan.warps_log2;  // blocks member, member + share, ...
  // the next block to be issued: its number, what is left of its segment, and where it is
  int next = member, left = 0;
  const int8_t *kp = nullptr, *vp = nullptr;
  const float *ksp = nullptr, *vsp = nullptr;
  auto point = [&](bool pre) {
    const int b = pre ? next : next - blocks0;
    const int64_t at = (pre ? shared + begin0 : own + begin1) + b * kBlock;
    left = (pre ? end0 - begin0 : end1 - begin1) - b * kBlock;
    kp = (pre ? a.prefix_key_codes : a.key_codes) + at * D;
    vp = (pre ? a.prefix_value_codes : a.value_codes) + at * D;
    ksp = (pre ? a.prefix_key_scales : a.key_scales) + at + lane;
    vsp = (pre ? a.prefix_value_scales : a.value_scales) + at + lane;
  };
  int lengths[kStreamStages];
  auto issue = [&](int st) {
    if (next == member || (next >= blocks0 && next - share < blocks0)) point(next < blocks0);
    const int n = min(kBlock, left);
    lengths[st] = n;
    Stage<D>& s = ring[st];
    uint64_t* bar = &bars[st];
    if (lane == 0) {
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(shared_address(bar)), "r"((uint32_t)(2 * n * D))
                   : "memory");
      copy_bulk(s.k, kp, n * D, bar);
      copy_bulk(s.v, vp, n * D, bar);
    }
    const bool in = lane < n;  // zeros behind the last position
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(shared_address(&s.ks[lane])),
                 "l"(in ? ksp : ksp - lane), "r"(in ? 4 : 0)
                 : "memory");
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(shared_address(&s.vs[lane])),
                 "l"(in ? vsp : vsp - lane), "r"(in ? 4 : 0)
                 : "memory");
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(shared_address(bar)) : "memory");
    next += share;
    left -= share * kBlock;
    kp += share * kBlock * D;
    vp += share * kBlock * D;
    ksp += share * kBlock;
    vsp += share * kBlock;
  };
#pragma unroll
  for (int st = 0; st < kStreamStages; st++)
    if (st < mine) issue(st);
  begin_rows<T, D, NG>(r, queries, scale, lane);
  int i = 0;
#pragma unroll 1
  for (uint32_t parity = 0; i < mine; parity ^= 1) {
#pragma unroll
    for (int st = 0; st < kStreamStages; st++) {
      if (i >= mine) break;
      ok = barrier_wait_warp(&bars[st], parity);
      if (!ok) break;
      attend_block<D, NG>(r, ring[st], lengths[st], lane);
      __syncwarp();  // every lane has read the stage
      if (i + kStreamStages < mine) issue(st);
      i++;
    }
    if (!ok) break;
  }
  if (!ok) {  // copies may still be landing: give them their time before the memory is let go
    for (int k = i; k < min(mine, i + kStreamStages); k++) barrier_wait(&bars[k % kStreamStages], (uint32_t)(k / kStreamStages) & 1);
    if (lane == 0) report_wait_timeout(wait_words, kWaitAttention);
  }
  if (plan.parts > 0) wait_for_prior();  // k_attend_prefix, beside which this kernel was started
  float* merge_o = reinterpret_cast<float*>(raw);  // [warps][4 NG][D], where the rings were
  const int64_t first = (int64_t)row * a.heads + head;
  if (share > 1) __syncthreads();
#pragma unroll
  for (int q = 0; q < NG; q++) {
    const int hh = 4 * q + c;  // the lane's head
    const int64_t at = first + hh;
    float m = ok ? r.M[q] : 0.0f, l = ok ? r.l[q] : NAN;
    l += __shfl_xor_sync(0xffffffffu, l, 4);
    l += __shfl_xor_sync(0xffffffffu, l, 8);
    l += __shfl_xor_sync(0xffffffffu, l, 16);
    // the products of heads and tails added
    float o[N];
#pragma unroll
    for (int t = 0; t < D / 16; t++) {
      o[2 * t] = r.o[q][t][0] + r.o[q][t][1];
      o[2 * t + 1] = r.o[q][t][2] + r.o[q][t][3];
    }
    if (plan.splits > 1 && share == 1) {
      if (hh < heads) store_part<N>(parts, (int64_t)(plan.parts + split) * parts.per_part + at, m, l, o, g);
      continue;
    }
    // the prefix's parts, where no split waits for the merge kernel: each warp of the unit takes some
#pragma unroll 2
    for (int p = plan.splits == 1 && hh < heads ? member : plan.parts; p < plan.parts; p += share)
      add_part<N>(parts, p * parts.per_part + at, m, l, o, g);
    if (share > 1) {
      if (g == 0) {
        merge_m[warp][hh] = m;
        merge_l[warp][hh] = l;
      }
#pragma unroll
      for (int i = 0; i < N; i += 4)
        *reinterpret_cast<float4*>(&merge_o[(warp * 4 * NG + hh) * D + g * N + i]) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
    } else if (hh < heads) {
      finish<T, N>(a, row, head + hh, at, m, l, o, g);
    }
  }
  if (share == 1) return;
  __syncthreads();
  if (member != 0) return;
#pragma unroll
  for (int q = 0; q < NG; q++) {
    const int hh = 4 * q + c;
    if (hh >= heads) continue;
    const int64_t at = first + hh;
    float M = -INFINITY, L = 0.0f, o[N];
    for (int w = 0; w < share; w++) M = fmaxf(M, merge_m[w][hh]);
#pragma unroll
    for (int i = 0; i < N; i++) o[i] = 0.0f;
    for (int w = 0; w < share; w++) {
      const float m = merge_m[w][hh], f = m == -INFINITY ? 0.0f : power2f(m - M);
      L = fmaf(merge_l[w][hh], f, L);
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(&merge_o[(w * 4 * NG + hh) * D + g * N + i]);
        o[i] = fmaf(v.x, f, o[i]);
        o[i + 1] = fmaf(v.y, f, o[i + 1]);
        o[i + 2] = fmaf(v.z, f, o[i + 2]);
        o[i + 3] = fmaf(v.w, f, o[i + 3]);
      }
    }
    if (plan.splits > 1) store_part<N>(parts, (int64_t)(plan.parts + split) * parts.per_part + at, M, L, o, g);
    else finish<T, N>(a, row, head + hh, at, M, L, o, g);
  }
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
  const int slot = a.slots ? a.slots[row] : (int)row;
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

// Warps that fill the GPU, 16 an SM: below them a unit gets more warps.  300 rows x 4 KV heads of 64, 64 + up to 700
// positions: 22.3 us, 27.8 us with 8 an SM, 20.7 us with 32; 600 rows x 64 + 300: 21.1, 21.4, 22.7 us.
constexpr int kFullWarps = 148 * 16;
// Positions below which a split is not worth its merge (a launch, about 3 us), and the warps that splits are made
// for.  One row of 4 KV heads over 8448 positions: 11.9 us with splits of 512, 12.5 us of 1024, 15.8 us of 2048;
// over 1280: 9.0 us in two splits, 7.8 us in one.  Over 64000: 21.8 us with 8 warps an SM, 24.3 us with 4, 28 us with
// 16 (twice the parts to merge).
constexpr int kLeastSplit = 768;
constexpr int kSplitWarps = 148 * 8;

// When the prefix goes to k_attend_prefix, whose launch, partial results and merge take about 4 us (packed rows = rows
// times heads of a KV head).  By scores, packed rows x positions, heads of 64, 4 KV heads (stream, prefix kernel):
// 128 x 256: 7.3, 9.8 us; 64 x 1024: 11.4, 10.6 us; 128 x 1024: 12.1, 12.5 us; 128 x 4096: 29.7, 16.0 us; heads of 128,
// 8 KV heads: 256 x 128: 22.7, 32 us; 64 x 1024: 19.2, 18.4 us; 256 x 4096: 114, 44.4 us.  By positions, 8192 packed
// rows: x 64: 79, 75 us; 2048: x 64: 28.1, 31.2 us, x 127: 34.0, 31.5 us.  By rows: 16 x 4096: 11.5, 12.5 us; 32 x
// 4096: 14.6, 14.4 us.
constexpr int64_t kPrefixLeastRows = 32, kPrefixLeastPositions = 96, kPrefixLeastScores = 65536;

StreamPlan plan_for(const needle_prefix_attention& a) {
  StreamPlan p{};
  const int group = a.heads / a.kv_heads;
  p.groups = (group + kGroupHeads - 1) / kGroupHeads;
  const int64_t packed = int64_t(a.rows) * group;
  if (packed >= kPrefixLeastRows && a.prefix_length >= kPrefixLeastPositions &&
      packed * a.prefix_length >= kPrefixLeastScores) {
    // parts of the prefix: as many as keep the waves of CTAs short, each costing about 6 tiles on top
    const int nt = prefix_tile();
    const int tiles = (a.prefix_length + nt - 1) / nt;
    const int64_t units = (packed + prefix_rows() - 1) / prefix_rows() * a.kv_heads;
    int64_t best = 0;
    int parts = 1;
    for (int c = 1; c <= std::min(tiles, 64); c++) {
      const int64_t cost = (units * c + 147) / 148 * ((tiles + c - 1) / c + 6);
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
  p.group = group;
  p.warps = 1;
  while (p.warps < kStreamWarps && units * p.warps < kFullWarps && positions > int64_t(p.warps) * kBlock) {
    p.warps *= 2;
    p.warps_log2++;
  }
  p.together = 1;  // 4096 rows x 4 KV heads, 160 + 256 positions: 76.7 us with a row's four units in a CTA, 80.1 us apart
  if (p.warps == 1)
    for (int k = 2; k <= kStreamWarps; k++)
      if (a.kv_heads * p.groups % k == 0 && units / k >= kFullWarps) p.together = k;
  // the longest splits that still give every SM its warps
  int64_t splits = 1;
  if (p.warps == kStreamWarps) splits = std::max<int64_t>(1, std::min(kSplitWarps / (units * p.warps), positions / kLeastSplit));
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
    const cudaError_t e = launch_attend_prefix(a, parts, p.parts, p.part_len, scale, wait_words, s);
    if (e != cudaSuccess) return e;
  }
  const int warps = p.warps * p.together;
  const size_t smem = sizeof(Stage<D>) * kStreamStages * warps;
  const dim3 grid(a.rows, a.kv_heads * p.groups / p.together, p.splits);
  static_assert(sizeof(Stage<D>) * kStreamStages >= size_t(kGroupHeads) * D * 4, "the merge takes the rings' place");
  auto go = [&](auto kernel) {
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 int(sizeof(Stage<D>) * kStreamStages * kStreamWarps));
    if (err != cudaSuccess) return err;
    // beside the prefix kernel, whose results are waited for at the end
    cudaLaunchAttribute overlap{};
    overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    overlap.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(warps * 32);
    config.dynamicSmemBytes = smem;
    config.stream = s;
    config.attrs = &overlap;
    config.numAttrs = p.parts > 0 ? 1 : 0;
    return cudaLaunchKernelEx(&config, kernel, a, p, parts, scale, wait_words);
  };
  cudaError_t e = a.heads / a.kv_heads <= 4 ? go(k_attend_stream<T, D, 1>) : go(k_attend_stream<T, D, 2>);
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
  if (int64_t(a->rows) * a->heads > 0x7fffffff) return refuse("rows times heads must stay below 2^31");
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
    *bytes = a->rows == 0 ? 0 : workspace_bytes_for(*a, plan_for(*a));  // (an empty batch has no plan)
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
    const StreamPlan plan = plan_for(*a);
    const size_t need = workspace_bytes_for(*a, plan);
    const bool prefix = a->prefix_length > 0, own = a->capacity > 0 && a->slot_count > 0;  // else never read
    const Buffers buffers = {{a->q, "q", element}, {a->out, "out", element}, {a->lse, "lse", 4}, {a->slots, "slots", 4},
                             {a->counts, "counts", 4}, {need > 0 ? workspace : nullptr, "workspace", 1},
                             {prefix ? a->prefix_key_codes : nullptr, "prefix_key_codes", 1},
                             {prefix ? a->prefix_key_scales : nullptr, "prefix_key_scales", 4},
                             {prefix ? a->prefix_value_codes : nullptr, "prefix_value_codes", 1},
                             {prefix ? a->prefix_value_scales : nullptr, "prefix_value_scales", 4},
                             {own ? a->key_codes : nullptr, "key_codes", 1}, {own ? a->key_scales : nullptr, "key_scales", 4},
                             {own ? a->value_codes : nullptr, "value_codes", 1},
                             {own ? a->value_scales : nullptr, "value_scales", 4}};
    if (int rc = check_alignment(buffers)) return rc;
    for (const void* p : {a->prefix_key_codes, a->prefix_value_codes, a->key_codes, a->value_codes})
      if (!aligned_to(p, 16)) return refuse("key/value codes must be 16-byte aligned");
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned_to(workspace, 16)))
      return refuse("the workspace must be 16-byte aligned and hold " + std::to_string(need) + " bytes");
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return refuse_cuda("prefix_attention", e);
    if (int rc = check_buffers(buffers, device)) return rc;
    if (check_wait_status(device) != NEEDLE_OK) return int(NEEDLE_BACKEND_UNAVAILABLE);
    uint32_t* words = wait_status_words(device);
    const float scale = a->scale > 0.0f ? a->scale : 1.0f / std::sqrt(float(a->head_dim));
    e = with_type(a->type, [&](auto zero) {
      using T = decltype(zero);
      return a->head_dim == 64 ? launch_attention<T, 64>(*a, plan, workspace, scale, words, static_cast<cudaStream_t>(stream))
                               : launch_attention<T, 128>(*a, plan, workspace, scale, words, static_cast<cudaStream_t>(stream));
    });
    return e == cudaSuccess ? int(NEEDLE_OK) : refuse_cuda("prefix_attention", e);
  });
}
