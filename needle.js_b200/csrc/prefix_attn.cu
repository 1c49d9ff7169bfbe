// prefix_attn.cu -- decode attention of a batch whose sequences share a prompt prefix: every row
// attends over the prefix's int8 keys and values, held once, and over its own int8 cache
// (#attention, packages/needle.js/src/model/runtime.ts:719-786, with the prefix taken out of the
// per-sequence caches; any head layout, binary32 arithmetic).
//
//   s_j = scale * (q . code_j) * ks_j,  o = sum_j e^(s_j - m) vs_j code_j / sum_j e^(s_j - m),
//   j over the prefix and the row's own positions;  lse = m + log sum_j e^(s_j - m)
//
// One CTA per (row, KV head, up to 8 of its query heads), each warp taking every fourth position with
// a running maximum and sum; the warps are merged at the end.
#include <cmath>

#include "serving.cuh"

namespace needle {

namespace {

constexpr int kAttendThreads = 128;
constexpr int kAttendWarps = kAttendThreads / 32;
constexpr int kGroupHeads = 8;  // query heads of one KV head taken together

template <class T, int EPL>
__global__ void __launch_bounds__(kAttendThreads) k_prefix_attention(const needle_prefix_attention a, float scale) {
  constexpr int D = EPL * 32;
  __shared__ float sm[kAttendWarps][kGroupHeads], sl[kAttendWarps][kGroupHeads], so[kAttendWarps][kGroupHeads][D];
  const int64_t row = blockIdx.x;
  const int h = blockIdx.y, group = a.heads / a.kv_heads, g0 = blockIdx.z * kGroupHeads;
  const int n = min(kGroupHeads, group - g0);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slot = a.slots ? a.slots[row] : (int)row;
  if (slot < 0 || slot >= a.slot_count) return;
  const int count = min(max(a.counts[row], 0), a.capacity);
  const T* q = static_cast<const T*>(a.q) + row * a.q_stride + (int64_t)(h * group + g0) * D;
  float qr[kGroupHeads][EPL], o[kGroupHeads][EPL], m[kGroupHeads], l[kGroupHeads];
#pragma unroll
  for (int g = 0; g < kGroupHeads; g++) {
    m[g] = -INFINITY;
    l[g] = 0.0f;
#pragma unroll
    for (int i = 0; i < EPL; i++) {
      qr[g][i] = g < n ? to_f32(q[g * D + lane * EPL + i]) * scale : 0.0f;
      o[g][i] = 0.0f;
    }
  }
  for (int64_t j = warp; j < (int64_t)a.prefix_length + count; j += kAttendWarps) {
    const bool shared = j < a.prefix_length;
    const int64_t r = shared ? h * (int64_t)a.prefix_capacity + j
                             : ((int64_t)slot * a.kv_heads + h) * a.capacity + (j - a.prefix_length);
    const Vec<int8_t, EPL> kc = *reinterpret_cast<const Vec<int8_t, EPL>*>(
        (shared ? a.prefix_key_codes : a.key_codes) + r * D + lane * EPL);
    const Vec<int8_t, EPL> vc = *reinterpret_cast<const Vec<int8_t, EPL>*>(
        (shared ? a.prefix_value_codes : a.value_codes) + r * D + lane * EPL);
    const float ks = (shared ? a.prefix_key_scales : a.key_scales)[r];
    const float vs = (shared ? a.prefix_value_scales : a.value_scales)[r];
#pragma unroll
    for (int g = 0; g < kGroupHeads; g++) {
      if (g >= n) break;
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < EPL; i++) s = fmaf(qr[g][i], (float)kc.v[i], s);
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
      s *= ks;
      const float mn = fmaxf(m[g], s), f = expf(m[g] - mn), p = expf(s - mn);
      l[g] = fmaf(l[g], f, p);
#pragma unroll
      for (int i = 0; i < EPL; i++) o[g][i] = fmaf(p * vs, (float)vc.v[i], o[g][i] * f);
      m[g] = mn;
    }
  }
#pragma unroll
  for (int g = 0; g < kGroupHeads; g++) {
    if (lane == 0) {
      sm[warp][g] = m[g];
      sl[warp][g] = l[g];
    }
#pragma unroll
    for (int i = 0; i < EPL; i++) so[warp][g][lane * EPL + i] = o[g][i];
  }
  __syncthreads();
  T* out = static_cast<T*>(a.out) + row * a.out_stride + (int64_t)(h * group + g0) * D;
  for (int e = tid; e < n * D; e += kAttendThreads) {
    const int g = e / D, d = e % D;
    float M = -INFINITY, L = 0.0f, O = 0.0f;
    for (int w = 0; w < kAttendWarps; w++) M = fmaxf(M, sm[w][g]);
    for (int w = 0; w < kAttendWarps; w++) {
      const float f = sm[w][g] == -INFINITY ? 0.0f : expf(sm[w][g] - M);
      L = fmaf(sl[w][g], f, L);
      O = fmaf(so[w][g][d], f, O);
    }
    out[g * D + d] = from_f32<T>(L > 0.0f ? O / L : 0.0f);
    if (d == 0 && a.lse) a.lse[row * a.heads + h * group + g0 + g] = L > 0.0f ? M + logf(L) : -INFINITY;
  }
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
    *bytes = 0;
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
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return refuse_cuda("prefix_attention", e);
    if (int rc = check_buffer(a->out, "out", device)) return rc;
    if (int rc = check_buffer(a->q, "q", device)) return rc;
    const float scale = a->scale > 0.0f ? a->scale : 1.0f / std::sqrt(float(a->head_dim));
    const int group = a->heads / a->kv_heads;
    e = with_type(a->type, [&](auto zero) {
      using T = decltype(zero);
      auto go = [&](auto kernel) {
        kernel<<<dim3(a->rows, a->kv_heads, (group + kGroupHeads - 1) / kGroupHeads), kAttendThreads, 0,
                 static_cast<cudaStream_t>(stream)>>>(*a, scale);
        return cudaGetLastError();
      };
      return a->head_dim == 64 ? go(k_prefix_attention<T, 2>) : go(k_prefix_attention<T, 4>);
    });
    return e == cudaSuccess ? int(NEEDLE_OK) : refuse_cuda("prefix_attention", e);
  });
}
