// logits.cu -- the rules between the vocabulary projection and the choice of a token, and the choice:
// penalties for repeated ids, biases, grammar masks, then (logits_select) the argmax and log
// probability of selectToken (packages/needle.js/src/model/runtime.ts:880-899).
//
//   x = raw logit l;  seen ids:  x = l > 0 ? l / repetition : l * repetition
//   x = x - frequency * c;  c > 0: x = x - presence       (c: times the id was answered)
//   x = x + bias;  ids the mask leaves out: x = -inf       (every step rounded to binary32)
//   id = argmax x, the lowest on ties;  log p = l[id] - max l - log sum exp(l - max l)
//
// A CTA takes a chunk of 16 ids per thread of one row, its logits held in registers from first to last,
// so a row is read once.  What the rules touch is sparse: per chunk, bitmaps in shared memory say which
// ids are seen, biased and allowed, and a table has counts and bias positions, its entries cleared one by
// one for the ids that occur.  The stream over the chunk knows only the mask; ids with a rule are left to
// the threads that hold them in their lists, which fetch those logits again.  All loads that depend on nothing but the row (logits, lengths, the first ids of the
// lists) are issued before the first barrier.
#include <cooperative_groups.h>

#include "serving.cuh"

namespace needle {

namespace {

namespace cg = cooperative_groups;

constexpr int kPerThread = 16;
constexpr int kRulesThreads = 256;   // chunks of 4096: eight CTAs an SM
constexpr int kSelectThreads = 512;  // chunks of 8192: the engine's vocabulary in one CTA
constexpr int kListIds = 4;          // history ids of a thread kept in registers

// A chunk's tables; count and bias (of THREADS * kPerThread entries each) only where a rule needs them.
template <int THREADS>
struct Tables {
  static constexpr int kChunk = THREADS * kPerThread, kWords = kChunk / 32, kWarps = THREADS / 32;
  uint32_t seen[kWords], biased[kWords], allowed[kWords];
  // one entry per warp, then the CTA's
  float top[kWarps], sum[kWarps];
  uint32_t key[kWarps], id[kWarps], lowest[kWarps];
  float cta_top, cta_sum;
  uint32_t cta_key, cta_id, cta_lowest;
};

template <int THREADS>
__host__ __device__ constexpr size_t tables_bytes() {
  return (sizeof(Tables<THREADS>) + 15) / 16 * 16;
}

template <int THREADS>
size_t smem_bytes(const needle_logits_rules& a) {
  const size_t each = size_t(THREADS) * kPerThread * 4;
  return tables_bytes<THREADS>() + (a.history ? each : 0) + (a.bias_ids ? each : 0);
}

// Order-preserving key of a binary32 value that is not NaN (-0 as +0); 0 is below every key.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// First id (possibly below 0) of 16-byte unit 0 of the row: rows that do not start on a 16-byte
// boundary are taken from the boundary before them, with the ids outside the row left out.
template <class T>
__device__ __forceinline__ int row_offset(const T* row) {
  return (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
}

// Loads the unit at id e (VEC ids); ids outside [0, vocab) become -inf.
template <class T, int VEC>
__device__ __forceinline__ void load_unit(const T* row, int64_t e, int vocab, float* x) {
  if (e >= 0 && e + VEC <= vocab) {
    const Vec<T, VEC> v = *reinterpret_cast<const Vec<T, VEC>*>(row + e);
#pragma unroll
    for (int i = 0; i < VEC; i++) x[i] = to_f32(v.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i++) x[i] = e + i >= 0 && e + i < vocab ? to_f32(row[e + i]) : -INFINITY;
  }
}

// What the rules of a row need from memory, loaded ahead.
struct RowRules {
  float repetition, frequency, presence;
  int64_t length, prompt, biases;
  const int32_t *history, *bias_ids;
  const float* bias_values;
  const uint32_t* mask;  // NULL: every id is allowed, or none (`none`)
  bool none;
};

__device__ __forceinline__ RowRules row_rules(const needle_logits_rules& a, int64_t row) {
  RowRules r;
  r.repetition = a.history && a.repetition ? __ldg(a.repetition + row) : 1.0f;
  r.frequency = a.history && a.frequency ? __ldg(a.frequency + row) : 0.0f;
  r.presence = a.history && a.presence ? __ldg(a.presence + row) : 0.0f;
  r.length = a.history ? min((int64_t)max(__ldg(a.history_lengths + row), 0), a.history_stride) : 0;
  r.prompt = a.history && a.prompt_lengths ? __ldg(a.prompt_lengths + row) : 0;
  r.biases = a.bias_ids ? min((int64_t)max(__ldg(a.bias_counts + row), 0), a.bias_stride) : 0;
  r.history = a.history + row * a.history_stride;
  r.bias_ids = a.bias_ids + row * a.bias_stride;
  r.bias_values = a.bias_values + row * a.bias_stride;
  const int slot = a.masks ? __ldg(a.mask_slots + row) : -1;
  r.none = slot >= a.mask_count && a.masks;  // a slot that does not exist
  r.mask = slot >= 0 && !r.none ? a.masks + (int64_t)slot * ((a.vocab + 31) >> 5) : nullptr;
  return r;
}

// A thread's list entries: places in the chunk (or -1) of its first history ids and its first bias.
struct ListPlaces {
  int history[kListIds], bias;
};

// Place of an id in the chunk from `low` on, or -1.
template <int THREADS>
__device__ __forceinline__ int place_of(int32_t id, int vocab, int64_t low) {
  const int64_t p = (int64_t)id - low;
  return id >= 0 && id < vocab && p >= 0 && p < Tables<THREADS>::kChunk ? (int)p : -1;
}

// Fills the bitmaps and tables of ids [low, low + kChunk).  Begins before and ends with a barrier; gives the
// first id of the chunk that the thread found allowed, 0xffffffff for none.
template <int THREADS>
__device__ __forceinline__ uint32_t build_tables(const RowRules& r, int vocab, int64_t low, Tables<THREADS>& t,
                                                 uint32_t* count, uint32_t* bias, ListPlaces& mine) {
  using S = Tables<THREADS>;
  const int tid = threadIdx.x, words = (vocab + 31) >> 5;
  uint32_t lowest = 0xffffffffu;
  auto place = [&](int32_t id) { return place_of<THREADS>(id, vocab, low); };
  int (&at)[kListIds] = mine.history;
#pragma unroll
  for (int k = 0; k < kListIds; k++) {
    const int64_t i = tid + k * THREADS;
    at[k] = i < r.length ? __ldg(r.history + i) : -1;
  }
  const int32_t first_bias = tid < r.biases ? __ldg(r.bias_ids + tid) : -1;
  for (int w = tid; w < S::kWords; w += THREADS) {
    t.seen[w] = 0;
    t.biased[w] = 0;
    // ids low + 32 w .. + 31: two words of the mask, and none outside the vocabulary
    const int64_t first = low + 32 * w;
    uint32_t bits = r.none ? 0u : 0xffffffffu;
    if (r.mask) {
      const int64_t word = first >> 5;  // floor
      const uint32_t a0 = word >= 0 && word < words ? __ldg(r.mask + word) : 0;
      const uint32_t a1 = word + 1 >= 0 && word + 1 < words ? __ldg(r.mask + word + 1) : 0;
      bits = __funnelshift_r(a0, a1, (uint32_t)(first & 31));
    }
    if (first < 0) bits &= first <= -32 ? 0u : 0xffffffffu << (int)(-first);
    const int64_t left = (int64_t)vocab - first;
    if (left < 32) bits &= left <= 0 ? 0u : 0xffffffffu >> (32 - (int)left);
    t.allowed[w] = bits;
    if (bits) lowest = min(lowest, (uint32_t)(first + __ffs(bits) - 1));
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kListIds; k++) at[k] = place(at[k]);
  mine.bias = place(first_bias);
  if (r.length == 0 && r.biases == 0) return lowest;
  auto see = [&](int p) {
    if (p >= 0) {
      count[p] = 0;
      atomicOr(&t.seen[p >> 5], 1u << (p & 31));
    }
  };
  auto weigh = [&](int p) {
    if (p >= 0) {
      bias[p] = 0;
      atomicOr(&t.biased[p >> 5], 1u << (p & 31));
    }
  };
#pragma unroll
  for (int k = 0; k < kListIds; k++) see(at[k]);
  for (int64_t i = tid + kListIds * THREADS; i < r.length; i += THREADS) see(place(__ldg(r.history + i)));
  weigh(mine.bias);
  for (int64_t i = tid + THREADS; i < r.biases; i += THREADS) weigh(place(__ldg(r.bias_ids + i)));
  __syncthreads();
  auto answer = [&](int64_t i, int p) {
    if (p >= 0 && i >= r.prompt) atomicAdd(&count[p], 1u);
  };
#pragma unroll
  for (int k = 0; k < kListIds; k++) answer(tid + k * THREADS, at[k]);
  for (int64_t i = tid + kListIds * THREADS; i < r.length; i += THREADS) answer(i, place(__ldg(r.history + i)));
  for (int64_t i = tid; i < r.biases; i += THREADS) {
    const int p = i < THREADS ? mine.bias : place(__ldg(r.bias_ids + i));
    if (p >= 0) atomicMax(&bias[p], (uint32_t)i + 1u);
  }
  __syncthreads();
  return lowest;
}

// Calls f(place) for the thread's share of the chunk's ids with a rule, some perhaps more than once.
template <int THREADS, class F>
__device__ __forceinline__ void for_ruled(const RowRules& r, int vocab, int64_t low, const ListPlaces& mine, F f) {
  const int tid = threadIdx.x;
#pragma unroll
  for (int k = 0; k < kListIds; k++)
    if (mine.history[k] >= 0) f(mine.history[k]);
  if (mine.bias >= 0) f(mine.bias);
  for (int64_t i = tid + kListIds * THREADS; i < r.length; i += THREADS) {
    const int p = place_of<THREADS>(__ldg(r.history + i), vocab, low);
    if (p >= 0) f(p);
  }
  for (int64_t i = tid + THREADS; i < r.biases; i += THREADS) {
    const int p = place_of<THREADS>(__ldg(r.bias_ids + i), vocab, low);
    if (p >= 0) f(p);
  }
}

__device__ __forceinline__ bool bit_of(const uint32_t* bits, int p) { return (bits[p >> 5] >> (p & 31)) & 1u; }

// Ruled value (not the mask) of the id at place p, raw logit l.
template <int THREADS>
__device__ __forceinline__ float ruled(float l, int p, const RowRules& r, const Tables<THREADS>& t, const uint32_t* count,
                                       const uint32_t* bias) {
  float x = l;
  if (bit_of(t.seen, p)) {
    x = x > 0.0f ? __fdiv_rn(x, r.repetition) : __fmul_rn(x, r.repetition);
    const uint32_t c = count[p];
    if (c) {
      x = __fsub_rn(x, __fmul_rn(r.frequency, (float)c));
      x = __fsub_rn(x, r.presence);
    }
  }
  if (bit_of(t.biased, p)) x = __fadd_rn(x, __ldg(r.bias_values + bias[p] - 1));
  return x;
}

// exp(v), v <= 0: relative error 2^-22 + |v| 2^-23.
__device__ __forceinline__ float exp_below(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v * 1.4426950408889634f));
  return r;
}

template <class T>
__global__ void __launch_bounds__(kRulesThreads, 6) k_logits_rules(const __grid_constant__ needle_logits_rules a, T* out,
                                                                int64_t out_stride) {
  constexpr int THREADS = kRulesThreads, VEC = 16 / sizeof(T), UNITS = kPerThread / VEC;
  using S = Tables<THREADS>;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  S& t = *reinterpret_cast<S*>(smem_raw);
  uint32_t* count = reinterpret_cast<uint32_t*>(smem_raw + tables_bytes<THREADS>());
  uint32_t* bias = count + (a.history ? S::kChunk : 0);
  const int64_t row = blockIdx.y;
  const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride;
  T* to = out + row * out_stride;
  const int tid = threadIdx.x, off = row_offset(in);
  const int64_t low = (int64_t)blockIdx.x * S::kChunk - off;
  if (low >= a.vocab) return;
  const RowRules r = row_rules(a, row);
  float x[UNITS][VEC];
#pragma unroll
  for (int u = 0; u < UNITS; u++) load_unit<T, VEC>(in, low + (int64_t)(u * THREADS + tid) * VEC, a.vocab, x[u]);
  ListPlaces mine;
  build_tables<THREADS>(r, a.vocab, low, t, count, bias, mine);
  const bool same = row_offset(to) == off;  // 16-byte units of the output line up with the input's
#pragma unroll
  for (int u = 0; u < UNITS; u++) {
    const int p0 = (u * THREADS + tid) * VEC;
    const uint32_t allowed = t.allowed[p0 >> 5] >> (p0 & 31);
    Vec<T, VEC> v;
#pragma unroll
    for (int i = 0; i < VEC; i++) v.v[i] = from_f32<T>((allowed >> i) & 1 ? x[u][i] : -INFINITY);
    const int64_t e = low + p0;
    if (same && e >= 0 && e + VEC <= a.vocab) {
      *reinterpret_cast<Vec<T, VEC>*>(to + e) = v;
    } else {
#pragma unroll
      for (int i = 0; i < VEC; i++)
        if (e + i >= 0 && e + i < a.vocab) to[e + i] = v.v[i];
    }
  }
  if (r.length == 0 && r.biases == 0) return;
  __syncthreads();  // ids with a rule are written after the stream has passed them
  // one thread takes each id that is allowed, by clearing its bit: in place, where the stream has put the same
  // logit back, nobody else may read or write it
  for_ruled<THREADS>(r, a.vocab, low, mine, [&](int p) {
    const uint32_t bit = 1u << (p & 31);
    if (atomicAnd(&t.allowed[p >> 5], ~bit) & bit)
      to[low + p] = from_f32<T>(ruled<THREADS>(to_f32(in[low + p]), p, r, t, count, bias));
  });
}

// One cluster per row; its CTAs take the row's chunks in turn.
template <class T>
__global__ void __launch_bounds__(kSelectThreads, 3) k_logits_select(const __grid_constant__ needle_logits_rules a,
                                                                  int32_t* __restrict__ ids,
                                                                  float* __restrict__ log_probabilities) {
  constexpr int THREADS = kSelectThreads, VEC = 16 / sizeof(T), UNITS = kPerThread / VEC;
  using S = Tables<THREADS>;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  S& t = *reinterpret_cast<S*>(smem_raw);
  uint32_t* count = reinterpret_cast<uint32_t*>(smem_raw + tables_bytes<THREADS>());
  uint32_t* bias = count + (a.history ? S::kChunk : 0);
  cg::cluster_group cluster = cg::this_cluster();
  const int64_t row = blockIdx.y;
  const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, off = row_offset(in);
  const RowRules r = row_rules(a, row);
  // the thread's running best, largest raw logit and sum of exponentials
  uint32_t id = 0xffffffffu;
  float best = -INFINITY, top = -INFINITY, sum = 0.0f;
  uint32_t lowest = 0xffffffffu;  // the lowest allowed id: the choice where every allowed logit is -inf
  for (int64_t c = blockIdx.x; c * S::kChunk - off < a.vocab; c += gridDim.x) {
    const int64_t low = c * S::kChunk - off;
    float x[UNITS][VEC];
#pragma unroll
    for (int u = 0; u < UNITS; u++) load_unit<T, VEC>(in, low + (int64_t)(u * THREADS + tid) * VEC, a.vocab, x[u]);
    if (c != blockIdx.x) __syncthreads();  // the tables of the chunk before are read
    ListPlaces mine;
    lowest = min(lowest, build_tables<THREADS>(r, a.vocab, low, t, count, bias, mine));
    float m = top;
#pragma unroll
    for (int u = 0; u < UNITS; u++)
#pragma unroll
      for (int i = 0; i < VEC; i++) m = fmaxf(m, x[u][i]);
    const float base = m == -INFINITY ? 0.0f : m;
    sum = top == -INFINITY ? 0.0f : sum * exp_below(top - base);
    top = m;
    int at = -1;
#pragma unroll
    for (int u = 0; u < UNITS; u++) {
      const int p0 = (u * THREADS + tid) * VEC, w = p0 >> 5;
      const uint32_t free = (t.allowed[w] & ~(t.seen[w] | t.biased[w])) >> (p0 & 31);  // allowed, without a rule
#pragma unroll
      for (int i = 0; i < VEC; i++) {
        sum += exp_below(x[u][i] - base);
        if (((free >> i) & 1) && x[u][i] > best) {  // ids rise: an equal logit keeps the lower id
          best = x[u][i];
          at = u * VEC + i;
        }
      }
    }
    if (at >= 0) id = (uint32_t)(low + (at / VEC * THREADS + tid) * VEC + at % VEC);
    for_ruled<THREADS>(r, a.vocab, low, mine, [&](int p) {
      if (!bit_of(t.allowed, p)) return;
      const float v = ruled<THREADS>(to_f32(in[low + p]), p, r, t, count, bias);
      const uint32_t i = (uint32_t)(low + p);
      if (v > best || (v == best && i < id && v > -INFINITY)) {
        best = v;
        id = i;
      }
    });
  }
  // warp, CTA, cluster; sums in a fixed order
  auto warp_merge = [&](float& m, float& s) {
    const float m0 = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    s = m0 == -INFINITY ? s : s * exp_below(m0 - m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  };
  auto warp_best = [&](uint32_t& k, uint32_t& i) {
    const uint32_t best = __reduce_max_sync(0xffffffffu, k);
    i = __reduce_min_sync(0xffffffffu, k == best ? i : 0xffffffffu);
    k = best;
  };
  uint32_t k = id == 0xffffffffu ? 0 : order_key(best);
  warp_best(k, id);
  warp_merge(top, sum);
  lowest = __reduce_min_sync(0xffffffffu, lowest);
  if (lane == 0) {
    t.top[warp] = top;
    t.sum[warp] = sum;
    t.key[warp] = k;
    t.id[warp] = id;
    t.lowest[warp] = lowest;
  }
  __syncthreads();
  if (warp == 0) {
    const bool in_use = lane < S::kWarps;
    k = in_use ? t.key[lane] : 0;
    id = in_use ? t.id[lane] : 0xffffffffu;
    lowest = __reduce_min_sync(0xffffffffu, in_use ? t.lowest[lane] : 0xffffffffu);
    top = in_use ? t.top[lane] : -INFINITY;
    sum = in_use ? t.sum[lane] : 0.0f;
    warp_best(k, id);
    warp_merge(top, sum);
    if (lane == 0 && gridDim.x > 1) {
      t.cta_top = top;
      t.cta_sum = sum;
      t.cta_key = k;
      t.cta_id = id;
      t.cta_lowest = lowest;
    }
  }
  if (gridDim.x > 1) cluster.sync();
  if (blockIdx.x == 0 && warp == 0) {
    if (gridDim.x > 1) {
      const bool in_use = lane < (int)gridDim.x;
      const S& o = *cluster.map_shared_rank(&t, in_use ? lane : 0);
      k = in_use ? o.cta_key : 0;
      id = in_use ? o.cta_id : 0xffffffffu;
      lowest = __reduce_min_sync(0xffffffffu, in_use ? o.cta_lowest : 0xffffffffu);
      top = in_use ? o.cta_top : -INFINITY;
      sum = in_use ? o.cta_sum : 0.0f;
      warp_best(k, id);
      warp_merge(top, sum);
    }
    if (lane == 0) {
      if (k == 0) id = lowest;
      ids[row] = (int32_t)id;  // 0xffffffff is -1
      log_probabilities[row] = id != 0xffffffffu ? (to_f32(in[id]) - top) - logf(sum) : -INFINITY;
    }
  }
  if (gridDim.x > 1) cluster.sync();  // shared memory lives until its readers are done
}

// Chunks of a row: one more id range is needed only where rows do not all start on 16 bytes.
int chunks_of(const needle_logits_rules& a, int chunk) {
  const int64_t element = int64_t(type_bytes(a.type));
  const bool lined_up = aligned_to(a.logits, 16) && (a.rows == 1 || a.logits_stride * element % 16 == 0);
  return int((int64_t(a.vocab) + (lined_up ? 0 : 16 / element - 1) + chunk - 1) / chunk);
}

// CTAs that keep the GPU busy: four of kSelectThreads an SM.
constexpr int64_t kSelectCtas = 148 * 4;

int check_rules(const needle_logits_rules* a, int* device, const char* op) {
  if (!a) return refuse("null argument");
  if (a->type < NEEDLE_TYPE_F32 || a->type > NEEDLE_TYPE_BF16) return refuse("unknown element type");
  if (a->rows < 0 || a->vocab < 0) return refuse("bad row or vocabulary count");
  if (a->rows == 0 || a->vocab == 0) return NEEDLE_OK;
  if (a->rows > 65535) return refuse("at most 65535 rows in a call");
  if (!a->logits) return refuse("null argument");
  if (a->rows > 1 && a->logits_stride < a->vocab) return refuse("a row stride is shorter than its row");
  if (!aligned_to(a->logits, type_bytes(a->type))) return refuse("a buffer is not aligned to its element type");
  if (a->history && (!a->history_lengths || a->history_stride < 0)) return refuse("history without lengths");
  if (a->bias_ids && (!a->bias_values || !a->bias_counts || a->bias_stride < 0 || a->bias_stride >= 0x7fffffff))
    return refuse("bias ids without values or counts");
  if (a->masks && (!a->mask_slots || a->mask_count < 0)) return refuse("masks without slots");
  const cudaError_t e = cudaGetDevice(device);
  if (e != cudaSuccess) return refuse_cuda(op, e);
  return check_buffer(a->logits, "logits", *device);
}

template <class K>
cudaError_t set_smem(K kernel, size_t bytes) {
  return bytes <= 48 * 1024 ? cudaSuccess
                            : cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

}  // namespace
}  // namespace needle

using namespace needle;

extern "C" int needle_cuda_logits_rules_dev(const needle_logits_rules* a, void* out, int64_t out_stride, void* stream) {
  return entry([&] {
    int device = 0;
    if (int rc = check_rules(a, &device, "logits_rules")) return rc;
    if (a->rows == 0 || a->vocab == 0) return int(NEEDLE_OK);
    if (!out) return refuse("null argument");
    if (a->rows > 1 && out_stride < a->vocab) return refuse("a row stride is shorter than its row");
    if (!aligned_to(out, type_bytes(a->type))) return refuse("a buffer is not aligned to its element type");
    if (int rc = check_buffer(out, "out", device)) return rc;
    const cudaError_t e = with_type(a->type, [&](auto zero) {
      using T = decltype(zero);
      const size_t smem = smem_bytes<kRulesThreads>(*a);
      cudaError_t err = set_smem(k_logits_rules<T>, smem);
      if (err != cudaSuccess) return err;
      k_logits_rules<T><<<dim3(chunks_of(*a, kRulesThreads * kPerThread), a->rows), kRulesThreads, smem,
                          static_cast<cudaStream_t>(stream)>>>(*a, static_cast<T*>(out), out_stride);
      return cudaGetLastError();
    });
    return e == cudaSuccess ? int(NEEDLE_OK) : refuse_cuda("logits_rules", e);
  });
}

extern "C" int needle_cuda_logits_select_dev(const needle_logits_rules* a, int32_t* ids, float* log_probabilities,
                                             void* stream) {
  return entry([&] {
    int device = 0;
    if (int rc = check_rules(a, &device, "logits_select")) return rc;
    if (a->rows == 0) return int(NEEDLE_OK);
    if (a->vocab == 0) return refuse("an empty vocabulary has no id to select");
    if (!ids || !log_probabilities) return refuse("null argument");
    if (int rc = check_buffer(ids, "ids", device)) return rc;
    if (int rc = check_buffer(log_probabilities, "log_probabilities", device)) return rc;
    const cudaError_t e = with_type(a->type, [&](auto zero) {
      using T = decltype(zero);
      const size_t smem = smem_bytes<kSelectThreads>(*a);
      cudaError_t err = set_smem(k_logits_select<T>, smem);
      if (err != cudaSuccess) return err;
      const int chunks = chunks_of(*a, kSelectThreads * kPerThread);
      int cluster = 1;
      while (cluster < 8 && cluster < chunks && a->rows * int64_t(cluster) < kSelectCtas) cluster *= 2;
      cudaLaunchConfig_t config{};
      config.gridDim = dim3(cluster, a->rows);
      config.blockDim = dim3(kSelectThreads);
      config.dynamicSmemBytes = smem;
      config.stream = static_cast<cudaStream_t>(stream);
      cudaLaunchAttribute attribute{};
      attribute.id = cudaLaunchAttributeClusterDimension;
      attribute.val.clusterDim.x = cluster;
      attribute.val.clusterDim.y = 1;
      attribute.val.clusterDim.z = 1;
      config.attrs = &attribute;
      config.numAttrs = 1;
      err = cudaLaunchKernelEx(&config, k_logits_select<T>, *a, ids, log_probabilities);
      return err == cudaSuccess ? cudaGetLastError() : err;
    });
    return e == cudaSuccess ? int(NEEDLE_OK) : refuse_cuda("logits_select", e);
  });
}
