// logits.cu -- the rules between the vocabulary projection and the choice of a token, and the choice:
// penalties for repeated ids, biases, grammar masks, then (logits_select) the argmax and log
// probability of selectToken (packages/needle.js/src/model/runtime.ts:880-899).
//
//   x = raw logit l;  seen ids:  x = l > 0 ? l / repetition : l * repetition
//   x = x - frequency * c;  c > 0: x = x - presence       (c: times the id was answered)
//   x = x + bias;  ids the mask leaves out: x = -inf       (every step rounded to binary32)
//   id = argmax x, the lowest on ties;  log p = l[id] - max l - log sum exp(l - max l)
//
// A CTA takes a stretch of kChunk ids of one row, its logits held in registers from first to last, so
// a row is read once.  What the rules touch is sparse: per chunk, bitmaps in shared memory say which ids
// are seen, biased and allowed, and only for those a table of counts and bias positions is read; its
// entries are cleared one by one for the ids that occur, not as a whole.
#include <cooperative_groups.h>

#include "serving.cuh"

namespace needle {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreadsL = 512;
constexpr int kPerThread = 16;
constexpr int kChunk = kThreadsL * kPerThread;
constexpr int kWords = kChunk / 32;
constexpr int kWarpsL = kThreadsL / 32;

struct Tables {
  uint32_t count[kChunk];    // times answered
  uint32_t bias[kChunk];     // 1 + position of the id's last bias
  uint32_t seen[kWords], biased[kWords], allowed[kWords];
  // one entry per warp, then the CTA's
  float top[kWarpsL], sum[kWarpsL], raw;
  uint32_t key[kWarpsL], id[kWarpsL];
  float cta_top, cta_sum, cta_raw;
  uint32_t cta_key, cta_id;
};

// Order-preserving key of a binary32 value (-0 as +0, NaN as -inf); 0 is below every key.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v != v ? -INFINITY : v + 0.0f);
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

// Fills the chunk's bitmaps and tables: ids [low, low + kChunk) of the row.
__device__ void build_tables(const needle_logits_rules& a, int64_t row, int64_t low, Tables& t) {
  const int tid = threadIdx.x;
  const int32_t* mask_slots = a.masks ? a.mask_slots : nullptr;
  const int slot = mask_slots ? mask_slots[row] : -1;
  const int words = (a.vocab + 31) >> 5;
  const uint32_t* mask = slot >= 0 && slot < a.mask_count ? a.masks + (int64_t)slot * words : nullptr;
  for (int w = tid; w < kWords; w += kThreadsL) {
    t.seen[w] = 0;
    t.biased[w] = 0;
    // ids low + 32 w .. + 31: two words of the mask, and none outside the vocabulary
    const int64_t first = low + 32 * w;
    uint32_t bits = 0xffffffffu;
    if (mask) {
      const int64_t at = first >> 5;  // floor
      const uint32_t a0 = at >= 0 && at < words ? __ldg(mask + at) : 0;
      const uint32_t a1 = at + 1 >= 0 && at + 1 < words ? __ldg(mask + at + 1) : 0;
      bits = __funnelshift_r(a0, a1, (uint32_t)(first & 31));
    } else if (slot >= a.mask_count && mask_slots) {
      bits = 0;  // a slot that does not exist allows nothing
    }
    if (first < 0) bits &= first <= -32 ? 0u : 0xffffffffu << (int)(-first);
    const int64_t left = (int64_t)a.vocab - first;
    if (left < 32) bits &= left <= 0 ? 0u : 0xffffffffu >> (32 - (int)left);
    t.allowed[w] = bits;
  }
  const int64_t length = a.history ? min((int64_t)max(a.history_lengths[row], 0), a.history_stride) : 0;
  const int64_t prompt = a.prompt_lengths && a.history ? a.prompt_lengths[row] : 0;
  const int64_t biases = a.bias_ids ? min((int64_t)max(a.bias_counts[row], 0), a.bias_stride) : 0;
  const int32_t* history = a.history + row * a.history_stride;
  const int32_t* bias_ids = a.bias_ids + row * a.bias_stride;
  __syncthreads();
  if (length == 0 && biases == 0) return;
  auto place = [&](int32_t id) -> int {  // place in the chunk, or -1
    const int64_t p = (int64_t)id - low;
    return id >= 0 && id < a.vocab && p >= 0 && p < kChunk ? (int)p : -1;
  };
  for (int64_t i = tid; i < length; i += kThreadsL) {
    const int p = place(__ldg(history + i));
    if (p >= 0) {
      t.count[p] = 0;
      atomicOr(&t.seen[p >> 5], 1u << (p & 31));
    }
  }
  for (int64_t i = tid; i < biases; i += kThreadsL) {
    const int p = place(__ldg(bias_ids + i));
    if (p >= 0) {
      t.bias[p] = 0;
      atomicOr(&t.biased[p >> 5], 1u << (p & 31));
    }
  }
  __syncthreads();
  for (int64_t i = max(prompt, (int64_t)0) + tid; i < length; i += kThreadsL) {
    const int p = place(__ldg(history + i));
    if (p >= 0) atomicAdd(&t.count[p], 1u);
  }
  for (int64_t i = tid; i < biases; i += kThreadsL) {
    const int p = place(__ldg(bias_ids + i));
    if (p >= 0) atomicMax(&t.bias[p], (uint32_t)i + 1u);
  }
  __syncthreads();
}

struct RowRules {
  float repetition, frequency, presence;
};

__device__ __forceinline__ RowRules row_rules(const needle_logits_rules& a, int64_t row) {
  return {a.repetition ? a.repetition[row] : 1.0f, a.frequency ? a.frequency[row] : 0.0f,
          a.presence ? a.presence[row] : 0.0f};
}

// x of place p of the chunk (not the mask).
__device__ __forceinline__ float ruled(float l, int p, bool seen, bool biased, const RowRules& r, const Tables& t,
                                       const float* bias_values) {
  float x = l;
  if (seen) {
    x = x > 0.0f ? __fdiv_rn(x, r.repetition) : __fmul_rn(x, r.repetition);
    const uint32_t c = t.count[p];
    if (c) {
      x = __fsub_rn(x, __fmul_rn(r.frequency, (float)c));
      x = __fsub_rn(x, r.presence);
    }
  }
  if (biased) x = __fadd_rn(x, __ldg(bias_values + t.bias[p] - 1));
  return x;
}

template <class T>
__global__ void __launch_bounds__(kThreadsL) k_logits_rules(const needle_logits_rules a, T* __restrict__ out,
                                                            int64_t out_stride) {
  constexpr int VEC = 16 / sizeof(T), UNITS = kPerThread / VEC;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Tables& t = *reinterpret_cast<Tables*>(smem_raw);
  const int64_t row = blockIdx.y;
  const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride;
  T* to = out + row * out_stride;
  const int tid = threadIdx.x, off = row_offset(in);
  const int64_t low = (int64_t)blockIdx.x * kChunk - off;
  if (low >= a.vocab) return;
  float x[UNITS][VEC];
#pragma unroll
  for (int u = 0; u < UNITS; u++) load_unit<T, VEC>(in, low + (int64_t)(u * kThreadsL + tid) * VEC, a.vocab, x[u]);
  build_tables(a, row, low, t);
  const RowRules r = row_rules(a, row);
  const float* bias_values = a.bias_values + row * a.bias_stride;
  const bool same = row_offset(to) == off;  // 16-byte units of the output line up with the input's
#pragma unroll
  for (int u = 0; u < UNITS; u++) {
    const int p0 = (u * kThreadsL + tid) * VEC;
    const uint32_t sh = p0 & 31, all = (1u << VEC) - 1u;
    const uint32_t seen = (t.seen[p0 >> 5] >> sh) & all, biased = (t.biased[p0 >> 5] >> sh) & all,
                   allowed = (t.allowed[p0 >> 5] >> sh) & all;
    if (seen | biased) {
#pragma unroll
      for (int i = 0; i < VEC; i++)
        x[u][i] = ruled(x[u][i], p0 + i, (seen >> i) & 1, (biased >> i) & 1, r, t, bias_values);
    }
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
}

// One cluster per row; its CTAs take the row's chunks in turn.
template <class T>
__global__ void __launch_bounds__(kThreadsL) k_logits_select(const needle_logits_rules a, int32_t* __restrict__ ids,
                                                             float* __restrict__ log_probabilities) {
  constexpr int VEC = 16 / sizeof(T), UNITS = kPerThread / VEC;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Tables& t = *reinterpret_cast<Tables*>(smem_raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int64_t row = blockIdx.y;
  const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, off = row_offset(in);
  const RowRules r = row_rules(a, row);
  const float* bias_values = a.bias_values + row * a.bias_stride;
  // the thread's running best (key, id, raw logit), largest raw logit and sum of exponentials
  uint32_t key = 0, id = 0xffffffffu;
  float raw = 0.0f, top = -INFINITY, sum = 0.0f;
  for (int64_t c = blockIdx.x; c * kChunk - off < a.vocab; c += gridDim.x) {
    const int64_t low = c * kChunk - off;
    float x[UNITS][VEC];
#pragma unroll
    for (int u = 0; u < UNITS; u++) load_unit<T, VEC>(in, low + (int64_t)(u * kThreadsL + tid) * VEC, a.vocab, x[u]);
    if (c != blockIdx.x) __syncthreads();  // the tables of the chunk before are read
    build_tables(a, row, low, t);
    float m = top;
#pragma unroll
    for (int u = 0; u < UNITS; u++)
#pragma unroll
      for (int i = 0; i < VEC; i++) m = fmaxf(m, x[u][i]);
    const float base = m == -INFINITY ? 0.0f : m;
    sum = top == -INFINITY ? 0.0f : sum * expf(top - base);
    top = m;
#pragma unroll
    for (int u = 0; u < UNITS; u++) {
      const int p0 = (u * kThreadsL + tid) * VEC;
      const uint32_t sh = p0 & 31, all = (1u << VEC) - 1u;
      const uint32_t seen = (t.seen[p0 >> 5] >> sh) & all, biased = (t.biased[p0 >> 5] >> sh) & all,
                     allowed = (t.allowed[p0 >> 5] >> sh) & all;
#pragma unroll
      for (int i = 0; i < VEC; i++) {
        const float l = x[u][i];
        sum += expf(l - base);
        if ((allowed >> i) & 1) {
          const float v =
              (seen | biased) ? ruled(l, p0 + i, (seen >> i) & 1, (biased >> i) & 1, r, t, bias_values) : l;
          const uint32_t k = order_key(v);
          if (k > key) {  // ids rise: an equal key keeps the lower id
            key = k;
            id = (uint32_t)(low + p0 + i);
            raw = l;
          }
        }
      }
    }
  }
  // warp, CTA, cluster; sums in a fixed order
  auto warp_merge = [&](float& m, float& s) {
    const float m0 = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    s = m0 == -INFINITY ? s : s * expf(m0 - m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  };
  auto warp_best = [&](uint32_t& k, uint32_t& i) {
    const uint32_t best = __reduce_max_sync(0xffffffffu, k);
    i = __reduce_min_sync(0xffffffffu, k == best ? i : 0xffffffffu);
    k = best;
  };
  uint32_t wk = key, wi = id;
  warp_best(wk, wi);
  warp_merge(top, sum);
  if (lane == 0) {
    t.top[warp] = top;
    t.sum[warp] = sum;
    t.key[warp] = wk;
    t.id[warp] = wi;
  }
  __syncthreads();
  uint32_t k = lane < kWarpsL ? t.key[lane] : 0, i = lane < kWarpsL ? t.id[lane] : 0xffffffffu;
  warp_best(k, i);  // every warp, so that the thread that holds the best knows
  if (k != 0 && i == id && key == k) t.cta_raw = raw;
  if (warp == 0) {
    float m = lane < kWarpsL ? t.top[lane] : -INFINITY, s = lane < kWarpsL ? t.sum[lane] : 0.0f;
    warp_merge(m, s);
    if (lane == 0) {
      t.cta_top = m;
      t.cta_sum = s;
      t.cta_key = k;
      t.cta_id = i;
    }
  }
  if (gridDim.x > 1) cluster.sync();
  else __syncthreads();
  if (blockIdx.x == 0 && warp == 0) {
    const int n = gridDim.x;
    float m = -INFINITY, s = 0.0f, l = 0.0f;
    uint32_t bk = 0, bi = 0xffffffffu;
    if (lane < n) {
      const Tables& o = n > 1 ? *cluster.map_shared_rank(&t, lane) : t;
      m = o.cta_top;
      s = o.cta_sum;
      bk = o.cta_key;
      bi = o.cta_id;
      l = o.cta_raw;
    }
    const uint32_t mine = bk, mine_id = bi;
    warp_best(bk, bi);
    warp_merge(m, s);
    const uint32_t who = __ballot_sync(0xffffffffu, mine == bk && mine_id == bi);
    l = __shfl_sync(0xffffffffu, l, __ffs(who) - 1);
    if (lane == 0) {
      ids[row] = bk ? (int32_t)bi : -1;
      log_probabilities[row] = bk ? (l - m) - logf(s) : -INFINITY;
    }
  }
  if (gridDim.x > 1) cluster.sync();  // shared memory lives until its readers are done
}

int chunks_of(int32_t vocab, size_t element) {
  return int((int64_t(vocab) + int64_t(16 / element) - 1 + kChunk - 1) / kChunk);
}

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
cudaError_t set_smem(K kernel) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Tables));
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
      cudaError_t err = set_smem(k_logits_rules<T>);
      if (err != cudaSuccess) return err;
      k_logits_rules<T><<<dim3(chunks_of(a->vocab, sizeof(T)), a->rows), kThreadsL, sizeof(Tables),
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
      cudaError_t err = set_smem(k_logits_select<T>);
      if (err != cudaSuccess) return err;
      const int chunks = chunks_of(a->vocab, sizeof(T));
      int cluster = 1;
      while (cluster < 8 && cluster < chunks) cluster *= 2;
      cudaLaunchConfig_t config{};
      config.gridDim = dim3(cluster, a->rows);
      config.blockDim = dim3(kThreadsL);
      config.dynamicSmemBytes = sizeof(Tables);
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
