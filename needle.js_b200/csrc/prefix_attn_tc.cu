// prefix_attn_tc.cu -- the shared prefix of a batch on the tensor cores (tcgen05).
//
// k_attend_prefix.  With many rows the prefix is a dense product: the heads of a KV head of all rows are
// packed into M (packed row i = row i / group, head i % group), 256 to a CTA as two tiles of 128, and
// the CTA walks its part of the prefix in tiles of 64 positions:
//   loader warps    read int8 codes, turn them into fp16 (exact) and write K and V tiles, in the same
//                   layout [position][64 dimensions, 128-byte swizzle], into rings in shared memory; V is
//                   the B operand with its N dimension contiguous, so nothing is transposed
//   MMA warp        S_t = Q_t K^T (tcgen05.mma, both from shared memory), two tiles of positions ahead, and
//                   O_t += P_t V (P from tensor memory, where S was), for the two tiles t in turn
//   softmax warps   four for each tile, one thread a packed row: 64 scores into registers, maximum,
//                   exponentials, P back to tensor memory as fp16; O stays in tensor memory and is only
//                   rescaled when a tile could bring weights past 2^15
// S is double-buffered, so the softmax warps never wait for the products of their own scores: with one buffer
// of 128 positions a tile went through softmax (3700 cycles) and products (1900) in turn, 91 us for
// 333 rows x 32 heads x 8191 positions of 128 dimensions.
// Two ahead, a pair of tiles took the softmax warps 2080 cycles (weights in one fp16 part): 70 us.  With heads and tails
// of the weights 84 us, the merge of its parts and the start of the stream included (520 TFLOP/s of useful products, 32%
// of the measured rate; tensor pipe 43% busy, issue slots 46%): the softmax warps' exponentials and conversions, and
// the products behind them, which the tails make half as many again.  64 rows x 2 heads x 2048 positions of 64:
// 15.4 us with the stream and the merge.
// The reference M of a row covers the value scale too: a weight is 2^(s - M) vs <= 2^15, inside fp16, and
// sums and outputs share the factor, which cancels.  16-bit queries are exact in fp16 after their row's
// power of two (the score scale comes after the product); binary32 queries (SPLIT) are split into fp16 heads and
// tails, two MMAs each.  So are the weights, for every type: rounded to fp16 once (2^-12 each) they would show in fp16
// outputs where one position dominates, and a row's result would depend on which kernel its batch reaches; it costs
// 333 rows x 32 heads x 8191 positions 130.6 us a call, 123.3 us without the tails.
// Every wait is bounded (2 s): a wait that runs out is reported through the wait-status words, and the
// rows' parts become NaN.
#include "prefix_attn.cuh"

namespace needle {

namespace {

constexpr int kTileWarps = 4;  // softmax warps of a tile
constexpr int kPrefixSoftmaxWarps = 2 * kTileWarps, kPrefixLoaderWarps = 3;
constexpr int kPrefixMmaWarp = kPrefixSoftmaxWarps + kPrefixLoaderWarps;
constexpr int kPrefixThreads = (kPrefixMmaWarp + 1) * 32;
constexpr int kPrefixRows = 256;  // packed rows of a CTA
constexpr int kNT = 64;           // positions of a tile
constexpr int kTurnRow = 36;      // floats of a row in the epilogue's transposition

template <int D, bool SPLIT>
struct PrefixShape {
  static constexpr int kHalves = D / 64;
  static constexpr int kParts = SPLIT ? 2 : 1;       // fp16 parts of a query
  static constexpr int kStages = D == 128 && SPLIT ? 3 : 4;  // of K and V tiles: two ahead in scores, one in values
  static constexpr uint32_t kQHalf = 128 * 128;                       // bytes of 128 rows x 64 dimensions
  static constexpr uint32_t kQTile = kQHalf * kHalves * kParts;       // [part][half]
  static constexpr uint32_t kKvHalf = kNT * 128;
  static constexpr uint32_t kKvTile = kKvHalf * kHalves;
  static constexpr uint32_t kK = 2 * kQTile, kV = kK + kStages * kKvTile;
  static constexpr uint32_t kScales = kV + kStages * kKvTile;
  static constexpr uint32_t kScaleStage = kNT * 8 + 16;  // key scales, value scales, the largest value scales
  static_assert(kScales >= kPrefixSoftmaxWarps * 32 * kTurnRow * 4, "the epilogue takes the operands' place");
  static constexpr uint32_t kSmem = kScales + kStages * kScaleStage + 1024;
};
// Tensor memory columns: S of tile t, buffer b, and P in its place (heads, then tails); O of tile t.
__device__ __forceinline__ uint32_t s_column(int t, int b) { return t * 128 + b * kNT; }
__device__ __forceinline__ uint32_t o_column(int t, int d) { return 256 + t * d; }

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
// True in one lane of the converged warp.  A whole group of MMAs is issued inside one such branch: per MMA of
// 128 x 64 x 16 that measured 57 cycles, a predicate of each MMA's own (lane == 0) 105.
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(e));
  return e != 0;
}
__device__ __forceinline__ void mma_shared(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_tensor(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives on `b` once every MMA this lane has issued is complete.
__device__ __forceinline__ void mma_commit_to(uint64_t* b) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(shared_address(b))
               : "memory");
}

// 32 (16) consecutive columns of this thread's lane of tensor memory.
__device__ __forceinline__ void tensor_load32(uint32_t at, float2* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
               : "=f"(v[0].x), "=f"(v[0].y), "=f"(v[1].x), "=f"(v[1].y), "=f"(v[2].x), "=f"(v[2].y), "=f"(v[3].x), "=f"(v[3].y), "=f"(v[4].x), "=f"(v[4].y), "=f"(v[5].x), "=f"(v[5].y), "=f"(v[6].x), "=f"(v[6].y), "=f"(v[7].x), "=f"(v[7].y), "=f"(v[8].x), "=f"(v[8].y), "=f"(v[9].x), "=f"(v[9].y), "=f"(v[10].x), "=f"(v[10].y), "=f"(v[11].x), "=f"(v[11].y), "=f"(v[12].x), "=f"(v[12].y), "=f"(v[13].x), "=f"(v[13].y), "=f"(v[14].x), "=f"(v[14].y), "=f"(v[15].x), "=f"(v[15].y)
               : "r"(at));
}
__device__ __forceinline__ void tensor_load16(uint32_t at, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
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

// Scores from position `valid` on become -inf.
template <int N>
__device__ __forceinline__ void hide(float2* x, int valid) {
#pragma unroll
  for (int j = 0; j < N / 2; j++) {
    if (2 * j >= valid) x[j].x = -INFINITY;
    if (2 * j + 1 >= valid) x[j].y = -INFINITY;
  }
}

template <class T, int D, bool SPLIT>
__global__ void __launch_bounds__(kPrefixThreads, 1)
    k_attend_prefix(const __grid_constant__ needle_prefix_attention a, const Parts parts, int part_len, float scale,
                    uint32_t* wait_words) {
  using P = PrefixShape<D, SPLIT>;
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ __align__(8) uint64_t q_full, s_full[2][2], p_full[2][2], rest[2], o_full;
  __shared__ __align__(8) uint64_t full[P::kStages], empty[P::kStages];
  __shared__ uint32_t tensor_base;
  __shared__ int failed;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int h = blockIdx.y, group = a.heads / a.kv_heads;
  const int64_t packed = (int64_t)a.rows * group, first = (int64_t)blockIdx.x * kPrefixRows;
  const int tiles_m = packed - first > 128 ? 2 : 1;
  const int begin = blockIdx.z * part_len, end = min(begin + part_len, a.prefix_length);
  const int n = (end - begin + kNT - 1) / kNT;
  const uint32_t sm = (shared_address(raw) + 1023u) & ~1023u;
  unsigned char* smem = raw + (sm - shared_address(raw));

  launch_dependents();
  // the softmax warps' rows (thread = packed row) and, before anything is waited for, their queries: kLanes
  // lanes take a row, 8 dimensions each
  constexpr int V = 16 / sizeof(T), kLanes = D / 8, kAtOnce = 32 / kLanes, kSteps = 32 / kAtOnce, kBatch = 8;
  const int t = warp / kTileWarps, quarter = warp & 3;
  const uint32_t i_row = (uint32_t)first + t * 128 + quarter * 32 + lane;
  const uint32_t row = i_row / (uint32_t)group, head = (uint32_t)(h * group) + (i_row - row * group);
  const int d0 = lane % kLanes * 8;
  bool live = false;
  int64_t offset = -1;
  Vec<T, V> in[kBatch][8 / V];
  float inverse = 0.0f;
  const bool vec = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 && (a.q_stride * (int64_t)sizeof(T) & 15) == 0;
  auto load = [&](int b) {
#pragma unroll
    for (int k = 0; k < kBatch; k++) {
      const int64_t at = __shfl_sync(0xffffffffu, offset, (b + k) * kAtOnce + lane / kLanes);
      const T* q = static_cast<const T*>(a.q) + at + d0;
#pragma unroll
      for (int p = 0; p < 8 / V; p++) {
        in[k][p] = Vec<T, V>{};
        if (at >= 0) {
          if (vec) {
            in[k][p] = *reinterpret_cast<const Vec<T, V>*>(q + p * V);
          } else {
#pragma unroll
            for (int e = 0; e < V; e++) in[k][p].v[e] = q[p * V + e];
          }
        }
      }
    }
  };
  if (warp < kPrefixSoftmaxWarps && t < tiles_m) {
    const int slot = i_row < (uint32_t)packed ? (a.slots ? __ldg(a.slots + row) : (int)row) : -1;
    live = slot >= 0 && slot < a.slot_count;
    // rows of other slots than the call's are read too (they are in the buffer), and left out at the end
    offset = i_row < (uint32_t)packed ? row * a.q_stride + head * D : -1;
    load(0);
  }
  if (tid == 0) {
    barrier_init(&q_full, kTileWarps * tiles_m);
    for (int t = 0; t < 2; t++) {
      for (int b = 0; b < 2; b++) {
        barrier_init(&s_full[t][b], 1);
        barrier_init(&p_full[t][b], kTileWarps);
      }
      barrier_init(&rest[t], 1);
    }
    barrier_init(&o_full, 1);
    for (int i = 0; i < P::kStages; i++) {
      barrier_init(&full[i], kPrefixLoaderWarps);
      barrier_init(&empty[i], 1);
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
  // All 512 columns are this CTA's, so they begin at address 0; as a constant it leaves the MMAs' operands in
  // uniform registers.
  constexpr uint32_t tm = 0;
  if (tensor_base != tm && tid == 0) failed = 1;

  if (warp == kPrefixMmaWarp) {
    const uint32_t qk = instruction(kNT, false), pv = instruction(D, true);
    bool ok = true;
    auto wait = [&](uint64_t* b, uint32_t parity) {
      ok = ok && barrier_wait_warp(b, parity);
      tensor_fence_after();
    };
    auto scores = [&](int t, int i) {  // S_t = Q_t K_i^T
      const uint64_t q = descriptor(sm + t * P::kQTile, 16), k = descriptor(sm + P::kK + (i % P::kStages) * P::kKvTile, 16);
#pragma unroll
      for (int part = 0; part < P::kParts; part++)
#pragma unroll
        for (int half = 0; half < P::kHalves; half++)
#pragma unroll
          for (int s = 0; s < 4; s++)
            mma_shared(tm + s_column(t, i & 1), q + (((part * P::kHalves + half) * P::kQHalf + s * 32) >> 4),
                       k + ((half * P::kKvHalf + s * 32) >> 4), qk, part + half + s > 0);
      mma_commit_to(&s_full[t][i & 1]);
    };
    auto values = [&](int t, int i) {  // O_t += P_t V_i
      const uint64_t v = descriptor(sm + P::kV + (i % P::kStages) * P::kKvTile, P::kKvHalf);
#pragma unroll
      for (int part = 0; part < 2; part++)  // heads, tails
#pragma unroll
        for (int s = 0; s < kNT / 16; s++)
          mma_tensor(tm + o_column(t, D), tm + s_column(t, i & 1) + part * (kNT / 2) + s * 8, v + ((s * 2048) >> 4), pv,
                     i > 0 || part + s > 0);
    };
    wait(&q_full, 0);
    for (int i = 0; i < min(n, 2) && ok; i++) {
      wait(&full[i], 0);
      if (!ok) break;
      if (elect_one())
        for (int t = 0; t < tiles_m; t++) scores(t, i);
      __syncwarp();
    }
    for (int i = 0; i < n && ok; i++) {
      const bool more = i + 2 < n;
      if (more) wait(&full[(i + 2) % P::kStages], ((i + 2) / P::kStages) & 1);
#pragma unroll
      for (int t = 0; t < 2; t++) {
        if (t >= tiles_m) break;
        wait(&p_full[t][i & 1], (i >> 1) & 1);
        if (!ok) break;
        if (elect_one()) {
          values(t, i);
          if (t == tiles_m - 1) mma_commit_to(&empty[i % P::kStages]);
          if (i == n - 2) mma_commit_to(&rest[t]);
          if (more) scores(t, i + 2);  // behind P_t V_i in the tensor pipe, which reads P from where S goes
        }
        __syncwarp();
      }
    }
    if (elect_one()) {
      if (!ok) atomicExch(&failed, 1);
      mma_commit_to(&o_full);
    }
    __syncwarp();
  } else if (warp >= kPrefixSoftmaxWarps) {
    // ---- loaders: K and V tiles in turn, the next two tiles' codes in registers while one is written.  Eight
    // neighbouring threads write two rows of one 64-dimension half: every bank once.
    constexpr int kLoaders = kPrefixLoaderWarps * 32, kRowUnits = D / 16;  // 16-code units of a row
    constexpr int kStep = kLoaders / kRowUnits;                            // rows that all loaders take at once
    constexpr int kUnits = (kNT + kStep - 1) / kStep;
    const int lt = tid - kPrefixSoftmaxWarps * 32;
    const int half = D == 128 ? (lt >> 3) & 1 : 0, cc = lt & 3;
    const int row0 = D == 128 ? (lt >> 4) * 2 + ((lt >> 2) & 1) : lt >> 2;
    const uint32_t at = half * P::kKvHalf + swizzled(row0, 2 * cc);
    const int64_t base = (int64_t)h * a.prefix_capacity + begin;
    const int64_t code_at = (base + row0) * D + half * 64 + cc * 16;
    uint4 codes[2][kUnits];  // of K, of V
    float key_scale = 1.0f, value_scale = 0.0f;
    auto fetch = [&](int i, bool value) {
      if (i >= n) return;
      uint4(&code)[kUnits] = codes[value];
      const int j = i * kNT, left = end - begin - j;
      const int8_t* src = (value ? a.prefix_value_codes : a.prefix_key_codes) + code_at + (int64_t)j * D;
#pragma unroll
      for (int u = 0; u < kUnits; u++)
        code[u] = row0 + u * kStep < min(left, kNT) ? __ldg(reinterpret_cast<const uint4*>(src + u * kStep * D)) : make_uint4(0, 0, 0, 0);
      if (value && lt < kNT) {
        key_scale = lt < left ? __ldg(a.prefix_key_scales + base + j + lt) : 1.0f;  // -inf stays -inf
        value_scale = lt < left ? __ldg(a.prefix_value_scales + base + j + lt) : 0.0f;
      }
    };
    auto write = [&](int i, bool value) {
      const uint4(&code)[kUnits] = codes[value];
      const int st = i % P::kStages;
      unsigned char* to = smem + (value ? P::kV : P::kK) + st * P::kKvTile;
#pragma unroll
      for (int u = 0; u < kUnits; u++) {
        if (row0 + u * kStep >= kNT) break;
        const uint32_t w[4] = {code[u].x ^ 0x80808080u, code[u].y ^ 0x80808080u, code[u].z ^ 0x80808080u, code[u].w ^ 0x80808080u};
        // kStep is 12 or 24: four rows on, bit 2 of the swizzle flips
        const uint32_t o = (at ^ ((u * kStep & 4) << 4)) + u * kStep * 128;
        *reinterpret_cast<uint4*>(to + o) =
            make_uint4(codes_f16(w[0], 0x4140), codes_f16(w[0], 0x4342), codes_f16(w[1], 0x4140), codes_f16(w[1], 0x4342));
        *reinterpret_cast<uint4*>(to + (o ^ 16)) =
            make_uint4(codes_f16(w[2], 0x4140), codes_f16(w[2], 0x4342), codes_f16(w[3], 0x4140), codes_f16(w[3], 0x4342));
      }
      if (value && lt < kNT) {
        float* s = reinterpret_cast<float*>(smem + P::kScales + st * P::kScaleStage);
        s[lt] = key_scale;
        s[kNT + lt] = value_scale;
        const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(value_scale) & 0x7fffffffu);
        if (lane == 0) s[2 * kNT + (lt >> 5)] = __uint_as_float(top);
      }
    };
    bool ok = true;
    fetch(0, false);
    fetch(0, true);
#pragma unroll 1
    for (int i = 0; i < n; i++) {
      const int st = i % P::kStages;
      ok = i < P::kStages || barrier_wait_warp(&empty[st], (i / P::kStages - 1) & 1);
      if (!ok) break;
      write(i, false);
      write(i, true);
      fence_async_proxy();  // before the next loads: it waits for every access in flight
      __syncwarp();
      if (lane == 0) barrier_arrive(&full[st]);
      fetch(i + 1, false);
      fetch(i + 1, true);
    }
    if (!ok) atomicExch(&failed, 1);
  } else {
    // ---- softmax: thread = packed row
    if (t < tiles_m) {
      // the warp's 32 queries, each scaled to a largest magnitude in [2^10, 2^11), as fp16 part(s) in shared memory
#pragma unroll
      for (int b = 0; b < kSteps; b += kBatch) {
        if (b > 0) load(b);
#pragma unroll
        for (int k = 0; k < kBatch; k++) {
          const int r0 = (b + k) * kAtOnce, rr = r0 + lane / kLanes;
          float x[8], top = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; e++) {
            x[e] = to_f32(in[k][e / V].v[e % V]);
            top = fmaxf(top, fabsf(x[e]));
          }
#pragma unroll
          for (int o = kLanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const int e10 = min(max(exponent_of(top), -110), 110);
          const float up = power2(10 - e10);
          uint32_t heads[4], tails[4];
#pragma unroll
          for (int e = 0; e < 4; e++) split_f16(x[2 * e] * up, x[2 * e + 1] * up, heads[e], tails[e]);
          unsigned char* to = smem + t * P::kQTile + (d0 >> 6) * P::kQHalf + swizzled(quarter * 32 + rr, (d0 & 63) >> 3);
          *reinterpret_cast<uint4*>(to) = make_uint4(heads[0], heads[1], heads[2], heads[3]);
          if constexpr (SPLIT)
            *reinterpret_cast<uint4*>(to + P::kHalves * P::kQHalf) = make_uint4(tails[0], tails[1], tails[2], tails[3]);
          // the row's own lane keeps what undoes the scaling
          const float back = __shfl_sync(0xffffffffu, power2(e10 - 10) * (scale * kLog2e), (lane - r0) * kLanes & 31);
          if (lane >= r0 && lane < r0 + kAtOnce) inverse = back;
        }
      }
      fence_async_proxy();
      __syncwarp();
      if (lane == 0) barrier_arrive(&q_full);

      const uint32_t mine = tm + ((uint32_t)(quarter * 32) << 16), o_at = mine + o_column(t, D);
      float M = -INFINITY, l = 0.0f;
      bool ok = true;
#pragma unroll 1
      for (int k = 0; k < n; k++) {
        const int st = k % P::kStages;
        const uint32_t s_at = mine + s_column(t, k & 1);
        ok = barrier_wait_warp(&full[st], (k / P::kStages) & 1) && barrier_wait_warp(&s_full[t][k & 1], (k >> 1) & 1);
        if (!ok) break;
        tensor_fence_after();
        const float4* ks = reinterpret_cast<const float4*>(smem + P::kScales + st * P::kScaleStage);
        const float4* vs = ks + kNT / 4;
        const float2 vtop = *reinterpret_cast<const float2*>(vs + kNT / 4);
        const int valid = end - (begin + k * kNT);
        // the row's scores, once from tensor memory, and their maximum
        float2 x[kNT / 2];
#pragma unroll
        for (int c = 0; c < kNT; c += 32) tensor_load32(s_at + c, x + c / 2);
        tensor_wait_loads();
        if (valid < kNT) hide<kNT>(x, valid);
        float most4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < kNT / 2; j += 2) {
          const float4 s4 = ks[j / 2];
          x[j] = __fmul2_rn(x[j], make_float2(s4.x, s4.y));
          x[j + 1] = __fmul2_rn(x[j + 1], make_float2(s4.z, s4.w));
          most4[j & 2] = max3(most4[j & 2], x[j].x, x[j].y);
          most4[1 + (j & 2)] = max3(most4[1 + (j & 2)], x[j + 1].x, x[j + 1].y);
        }
        const float most = fmaxf(fmaxf(most4[0], most4[1]), fmaxf(most4[2], most4[3]));
        const float reach = most * inverse + value_reach(fmaxf(vtop.x, vtop.y));  // weights are below 2^(reach - M + 7)
        const bool raise = reach > M + kRaise;
        if (__any_sync(0xffffffffu, raise)) {
          const float Mn = raise ? reach + 1.0f : M;
          const float f = M == -INFINITY ? 0.0f : power2f(M - Mn);
          l *= f;
          M = Mn;
          if (k > 0) {
            // O must be at rest: this tile's products have not begun, and those of the tile before are done when
            // the next tile's scores, issued behind them, are there
            ok = k + 1 < n ? barrier_wait_warp(&s_full[t][(k + 1) & 1], ((k + 1) >> 1) & 1) : barrier_wait_warp(&rest[t], 0);
            if (!ok) break;
            tensor_fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              uint32_t y[16];
              tensor_load16(o_at + c, y);
              tensor_wait_loads();
#pragma unroll
              for (int j = 0; j < 16; j++) y[j] = __float_as_uint(__uint_as_float(y[j]) * f);
              tensor_store16(o_at + c, y);
            }
          }
        }
        const float base = M == -INFINITY ? 0.0f : M;  // (no score above -inf yet)
        // A weight is 2^(x inverse - M) of an unrounded product.  Where steps of M reach 1/8, and may be far above 1,
        // the product is rounded first, as M's was: else no position would meet M, whose weight has to be near 1.
        float times = inverse;
        const bool far = fabsf(base) > 1048576.0f;
        if (__any_sync(0xffffffffu, far)) {
          const float2 round = make_float2(far ? inverse : 1.0f, far ? inverse : 1.0f);
#pragma unroll
          for (int j = 0; j < kNT / 2; j++) x[j] = __fmul2_rn(x[j], round);
          times = far ? 1.0f : inverse;
        }
        const float2 inverse2 = make_float2(times, times), minus = make_float2(-base, -base);
        float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int c = 0; c < kNT; c += 32) {
          uint32_t heads[16], tails[16];
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            const float4 v4 = vs[(c + 2 * j) / 4];
#pragma unroll
            for (int o = 0; o < 2; o++) {
              float2 p = __ffma2_rn(x[c / 2 + j + o], inverse2, minus);
              p.x = power2f(p.x);
              p.y = power2f(p.y);
              sum = __fadd2_rn(sum, p);
              const float2 w = __fmul2_rn(p, o ? make_float2(v4.z, v4.w) : make_float2(v4.x, v4.y));
              split_f16(w.x, w.y, heads[j + o], tails[j + o]);
            }
          }
          tensor_store16(s_at + c / 2, heads);
          tensor_store16(s_at + kNT / 2 + c / 2, tails);
        }
        l += sum.x + sum.y;
        tensor_wait_stores();
        tensor_fence_before();
        __syncwarp();
        if (lane == 0) barrier_arrive(&p_full[t][k & 1]);
      }
      if (!ok) atomicExch(&failed, 1);
      const bool done = barrier_wait_warp(&o_full, 0);
      tensor_fence_after();
      const bool bad = !ok || !done || *(volatile int*)&failed != 0;
      if (bad && lane == 0) report_wait_timeout(wait_words, kWaitAttention);
      const int64_t part = blockIdx.z * parts.per_part + (int64_t)row * a.heads + head;
      if (live) parts.ml[part] = part_of(M, bad ? NAN : l);
      // 32 columns at a time through shared memory (the operands are done with), so that rows are written
      // 128 bytes at once
      float* turn = reinterpret_cast<float*>(smem) + warp * 32 * kTurnRow;
      const int64_t to = live ? part * D : -1;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        float2 x[16];
        tensor_load32(o_at + c, x);
        tensor_wait_loads();
#pragma unroll
        for (int j = 0; j < 16; j += 2)
          *reinterpret_cast<float4*>(turn + lane * kTurnRow + 2 * j) = make_float4(x[j].x, x[j].y, x[j + 1].x, x[j + 1].y);
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 8; k++) {
          const int rr = k * 4 + (lane >> 3);
          const int64_t at = __shfl_sync(0xffffffffu, to, rr);
          const float4 v = *reinterpret_cast<const float4*>(turn + rr * kTurnRow + (lane & 7) * 4);
          if (at >= 0) *reinterpret_cast<float4*>(parts.o + at + c + (lane & 7) * 4) = v;
        }
        __syncwarp();
      }
    }
  }
  tensor_fence_before();
  __syncthreads();
  if (warp == kPrefixMmaWarp) {
    tensor_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tensor_base), "r"(512u) : "memory");
  }
}

}  // namespace

int prefix_tile() { return kNT; }
int prefix_rows() { return kPrefixRows; }

cudaError_t launch_attend_prefix(const needle_prefix_attention& a, const Parts& out, int parts, int part_len, float scale,
                                 uint32_t* wait_words, cudaStream_t s) {
  return with_type(a.type, [&](auto zero) {
    using T = decltype(zero);
    constexpr bool kSplit = sizeof(T) == 4;
    const int64_t packed = int64_t(a.rows) * (a.heads / a.kv_heads);
    const dim3 grid((unsigned)((packed + kPrefixRows - 1) / kPrefixRows), a.kv_heads, parts);
    auto go = [&](auto kernel, size_t smem) {
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
      if (e != cudaSuccess) return e;
      kernel<<<grid, kPrefixThreads, smem, s>>>(a, out, part_len, scale, wait_words);
      return cudaGetLastError();
    };
    return a.head_dim == 64 ? go(k_attend_prefix<T, 64, kSplit>, PrefixShape<64, kSplit>::kSmem)
                            : go(k_attend_prefix<T, 128, kSplit>, PrefixShape<128, kSplit>::kSmem);
  });
}

}  // namespace needle
