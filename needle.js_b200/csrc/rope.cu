// rope.cu -- rotary positions with the head norms before them and the int8 cache append after them
// (the Q / K path of NeedleRuntime.step, packages/needle.js/src/model/runtime.ts:471-501, 679-717,
// for any head layout, element type and frequency table).
//
//   y = (1 + s) x / sqrt(mean x^2 + 1e-6)                 (heads with a norm; stored in binary32)
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t) m,   t = position * w_i, pair i of `rotary`
//   scale = max(1e-12, max |y|) / 127,  code = round-half-even(y / scale)
//
// Keys are computed in binary64 and rounded to binary32 exactly where the engine stores them, so the
// codes are the engine's: a key one ulp off would round to the other code next to a border.  The scale is
// the binary64 product with 1 / 127, at most one binary64 ulp from the quotient and several times cheaper;
// only a value within 2^-52 of a border between codes could tell the two apart.
// Queries in binary32 are computed the same way; 16-bit queries in binary32, whose error (2^-23) is far
// below the rounding to 16 bits (2^-11, 2^-8).
//
// One CTA per token: its threads first compute the token's cosines and sines (binary64, shared by all
// heads), then each warp takes whole head rows, lanes holding consecutive elements.
#include <cmath>
#include <type_traits>

#include "serving.cuh"

namespace needle {

namespace {

constexpr int kRopeThreads = 256;
constexpr int kMaxPairs = 64;  // rotated pairs of a head of 128

struct RopeArgs {
  needle_rope_append a;
  double inverse[kMaxPairs];
};

// code of x at binary64 scale s = top / 127: the quotient is first taken in binary32 (error below
// 2^-15 of a code step at |code| <= 127), and only quotients that near a border are divided in binary64.
__device__ __forceinline__ int quantise(float x, float inverse, double scale) {
  const float t = x * inverse;
  float r = rintf(t);
  if (!(fabsf(t - r) < 0.4999f)) r = (float)rint((double)x / scale);
  return r != r ? 0 : (int)fminf(fmaxf(r, -127.0f), 127.0f);
}

template <class T, int EPL>
__device__ __forceinline__ void load_row(const T* p, int lane, bool vec, float* x) {
  if (vec) {
    const Vec<T, EPL> v = *reinterpret_cast<const Vec<T, EPL>*>(p + lane * EPL);
#pragma unroll
    for (int i = 0; i < EPL; i++) x[i] = to_f32(v.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < EPL; i++) x[i] = to_f32(p[lane * EPL + i]);
  }
}

template <class T, int EPL>
__device__ __forceinline__ void store_row(T* p, int lane, bool vec, const float* x) {
  if (vec) {
    Vec<T, EPL> v;
#pragma unroll
    for (int i = 0; i < EPL; i++) v.v[i] = from_f32<T>(x[i]);
    *reinterpret_cast<Vec<T, EPL>*>(p + lane * EPL) = v;
  } else {
#pragma unroll
    for (int i = 0; i < EPL; i++) p[lane * EPL + i] = from_f32<T>(x[i]);
  }
}

// Norm and rotation of one head row (EPL consecutive elements per lane) in arithmetic A.
template <class A, int EPL>
__device__ __forceinline__ void turn_row(float* x, const float* norm, const double2* cs, int lane, int rotary,
                                         bool interleaved) {
  if (norm) {
    A sum = 0;
#pragma unroll
    for (int i = 0; i < EPL; i++) sum = fma((A)x[i], (A)x[i], sum);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const A inverse = (A)1 / sqrt(sum / (A)(EPL * 32) + (A)1e-6);
#pragma unroll
    for (int i = 0; i < EPL; i++) x[i] = (float)(((A)1 + (A)__ldg(norm + lane * EPL + i)) * (A)x[i] * inverse);
  }
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < EPL; i += 2) {
      const int e = lane * EPL + i;
      if (e < rotary) {
        const A c = (A)cs[e >> 1].x, s = (A)cs[e >> 1].y, a = (A)x[i], b = (A)x[i + 1];
        x[i] = (float)(a * c - b * s);
        x[i + 1] = (float)(b * c + a * s);
      }
    }
    return;
  }
  // pairs (e, e + half): the partner of a lane's element i is register (i +- half) % EPL of another lane
  const int half = rotary >> 1, shift = half % EPL;
  float y[EPL];
#pragma unroll
  for (int i = 0; i < EPL; i++) {
    const int e = lane * EPL + i;
    const int up = ((e + half) / EPL) & 31, down = ((e - half + 32 * EPL) / EPL) & 31;
    if (shift == 0) {
      y[i] = __shfl_sync(0xffffffffu, x[i], e < half ? up : down);
    } else {
      float from_up = 0.0f, from_down = 0.0f;
#pragma unroll
      for (int j = 0; j < EPL; j++) {
        if ((i + shift) % EPL == j) from_up = x[j];
        if ((i + EPL - shift) % EPL == j) from_down = x[j];
      }
      from_up = __shfl_sync(0xffffffffu, from_up, up);
      from_down = __shfl_sync(0xffffffffu, from_down, down);
      y[i] = e < half ? from_up : from_down;
    }
  }
#pragma unroll
  for (int i = 0; i < EPL; i++) {
    const int e = lane * EPL + i;
    if (e < rotary) {
      const bool first = e < half;
      const double2 t = cs[first ? e : e - half];
      const A c = (A)t.x, s = (A)t.y;
      x[i] = (float)(first ? (A)x[i] * c - (A)y[i] * s : (A)x[i] * c + (A)y[i] * s);
    }
  }
}

template <class T, int EPL>
__global__ void __launch_bounds__(kRopeThreads) k_rope_append(const __grid_constant__ RopeArgs args, bool q_vec,
                                                               bool k_vec, bool v_vec, bool qo_vec, bool ko_vec,
                                                               bool vo_vec) {
  constexpr int kDimension = EPL * 32;
  __shared__ double2 cs[kMaxPairs];
  const needle_rope_append& a = args.a;
  const int64_t t = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31;
  const int pairs = a.rotary_dim >> 1;
  if (tid < pairs) {
    double s, c;
    sincos((double)a.positions[t] * args.inverse[tid], &s, &c);
    cs[tid] = make_double2(c * a.magnitude, s * a.magnitude);
  }
  const int slot = a.slots[t], entry = a.entries[t];
  const bool stored = slot >= 0 && slot < a.slot_count && entry >= 0 && entry < a.capacity;
  __syncthreads();
  using Query = typename std::conditional<sizeof(T) == 4, double, float>::type;
  for (int r = tid >> 5; r < a.heads + 2 * a.kv_heads; r += kRopeThreads / 32) {
    float x[EPL];
    if (r < a.heads) {
      load_row<T, EPL>(static_cast<const T*>(a.q) + t * a.q_stride + (int64_t)r * kDimension, lane, q_vec, x);
      turn_row<Query, EPL>(x, a.q_norm, cs, lane, a.rotary_dim, a.interleaved != 0);
      store_row<T, EPL>(static_cast<T*>(a.q_out) + t * a.q_out_stride + (int64_t)r * kDimension, lane, qo_vec, x);
      continue;
    }
    const bool key = r < a.heads + a.kv_heads;
    const int h = r - a.heads - (key ? 0 : a.kv_heads);
    if (key) {
      load_row<T, EPL>(static_cast<const T*>(a.k) + t * a.k_stride + (int64_t)h * kDimension, lane, k_vec, x);
      turn_row<double, EPL>(x, a.k_norm, cs, lane, a.rotary_dim, a.interleaved != 0);
    } else {
      load_row<T, EPL>(static_cast<const T*>(a.v) + t * a.v_stride + (int64_t)h * kDimension, lane, v_vec, x);
    }
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < EPL; i++) top = fmaxf(top, fabsf(x[i]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const double scale = fmax(1e-12, (double)top) * (1.0 / 127.0);
    const float scale32 = (float)scale, inverse = (float)(1.0 / scale);
    Vec<int8_t, EPL> code;
    float value[EPL];
#pragma unroll
    for (int i = 0; i < EPL; i++) {
      const int c = quantise(x[i], inverse, scale);
      code.v[i] = (int8_t)c;
      value[i] = (float)c * scale32;
    }
    if (stored) {
      const int64_t row = ((int64_t)slot * a.kv_heads + h) * a.capacity + entry;
      *reinterpret_cast<Vec<int8_t, EPL>*>((key ? a.key_codes : a.value_codes) + row * kDimension + lane * EPL) = code;
      if (lane == 0) (key ? a.key_scales : a.value_scales)[row] = scale32;
    }
    void* out = key ? a.k_out : a.v_out;
    if (out)
      store_row<T, EPL>(static_cast<T*>(out) + t * (key ? a.k_out_stride : a.v_out_stride) + (int64_t)h * kDimension,
                        lane, key ? ko_vec : vo_vec, value);
  }
}

// Whether every head row of a [tokens][*][dim] view can be accessed in a lane's whole share at once.
bool rows_aligned(const void* p, int64_t stride, int32_t dim, size_t element) {
  const size_t share = size_t(dim) / 32 * element;
  return aligned_to(p, share) && (stride * int64_t(element)) % int64_t(share) == 0;
}

cudaError_t launch_rope(const RopeArgs& args, cudaStream_t s) {
  const needle_rope_append& a = args.a;
  return with_type(a.type, [&](auto zero) {
    using T = decltype(zero);
    const size_t e = sizeof(T);
    auto go = [&](auto kernel) {
      kernel<<<(unsigned)a.tokens, kRopeThreads, 0, s>>>(
          args, rows_aligned(a.q, a.q_stride, a.head_dim, e), rows_aligned(a.k, a.k_stride, a.head_dim, e),
          rows_aligned(a.v, a.v_stride, a.head_dim, e), rows_aligned(a.q_out, a.q_out_stride, a.head_dim, e),
          rows_aligned(a.k_out, a.k_out_stride, a.head_dim, e), rows_aligned(a.v_out, a.v_out_stride, a.head_dim, e));
      return cudaGetLastError();
    };
    return a.head_dim == 64 ? go(k_rope_append<T, 2>) : go(k_rope_append<T, 4>);
  });
}

}  // namespace
}  // namespace needle

using namespace needle;

extern "C" int needle_cuda_rope_append_dev(const needle_rope_append* a, const double* inverse_frequencies,
                                           void* stream) {
  return entry([&] {
    if (!a) return refuse("null argument");
    if (a->type < NEEDLE_TYPE_F32 || a->type > NEEDLE_TYPE_BF16) return refuse("unknown element type");
    if (a->head_dim != 64 && a->head_dim != 128) return refuse("head dimensions of 64 and 128 only");
    if (a->tokens < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads > 65536 || a->kv_heads > 65536 ||
        a->slot_count < 0 || a->capacity < 0)
      return refuse("bad token, head, slot or entry count");
    if (a->rotary_dim < 0 || a->rotary_dim > a->head_dim || (a->rotary_dim & 1))
      return refuse("rotary_dim must be even and at most head_dim");
    if (a->rotary_dim > 0 && !inverse_frequencies) return refuse("null argument");
    if (a->tokens == 0) return int(NEEDLE_OK);
    if (!a->q || !a->k || !a->v || !a->q_out || !a->positions || !a->slots || !a->entries || !a->key_codes ||
        !a->key_scales || !a->value_codes || !a->value_scales)
      return refuse("null argument");
    const int64_t d = a->head_dim;
    if (a->tokens > 1 && (a->q_stride < a->heads * d || a->q_out_stride < a->heads * d || a->k_stride < a->kv_heads * d ||
                          a->v_stride < a->kv_heads * d || (a->k_out && a->k_out_stride < a->kv_heads * d) ||
                          (a->v_out && a->v_out_stride < a->kv_heads * d)))
      return refuse("a row stride is shorter than its row");
    const size_t e = type_bytes(a->type);
    for (const void* p : {a->q, a->k, a->v, (const void*)a->q_out, (const void*)a->k_out, (const void*)a->v_out})
      if (!aligned_to(p, e)) return refuse("a buffer is not aligned to its element type");
    if (!aligned_to(a->key_codes, 16) || !aligned_to(a->value_codes, 16))
      return refuse("key/value codes must be 16-byte aligned");
    RopeArgs args{};
    args.a = *a;
    for (int i = 0; i < a->rotary_dim / 2; i++) {
      if (!std::isfinite(inverse_frequencies[i])) return refuse("an inverse frequency is not finite");
      args.inverse[i] = inverse_frequencies[i];
    }
    if (!std::isfinite(a->magnitude)) return refuse("the magnitude is not finite");
    int device = 0;
    cudaError_t err = cudaGetDevice(&device);
    if (err != cudaSuccess) return refuse_cuda("rope_append", err);
    if (int rc = check_buffer(a->q_out, "q_out", device)) return rc;
    if (int rc = check_buffer(a->key_codes, "key_codes", device)) return rc;
    err = launch_rope(args, static_cast<cudaStream_t>(stream));
    return err == cudaSuccess ? int(NEEDLE_OK) : refuse_cuda("rope_append", err);
  });
}

extern "C" int needle_cuda_rope_frequencies(const needle_rope_scaling* s, int32_t rotary_dim,
                                            double* inverse_frequencies, double* magnitude) {
  return entry([&] {
    if (!s || !inverse_frequencies || !magnitude) return refuse("null argument");
    if (rotary_dim < 2 || rotary_dim > 2 * kMaxPairs || (rotary_dim & 1))
      return refuse("rotary_dim must be even and at most 128");
    if (!(s->theta > 0.0) || !std::isfinite(s->theta)) return refuse("theta must be positive");
    if (s->kind < NEEDLE_ROPE_PLAIN || s->kind > NEEDLE_ROPE_PARTS) return refuse("unknown rotary scaling");
    if (s->kind != NEEDLE_ROPE_PLAIN && (!(s->factor > 0.0) || !std::isfinite(s->factor)))
      return refuse("the scaling factor must be positive");
    if (s->kind == NEEDLE_ROPE_NTK && rotary_dim < 4) return refuse("NTK scaling needs two pairs or more");
    if (s->kind == NEEDLE_ROPE_PARTS && (!(s->trained_length > 0.0) || !(s->fast_turns > s->slow_turns) ||
                                         !std::isfinite(s->trained_length) || !std::isfinite(s->fast_turns) ||
                                         !std::isfinite(s->slow_turns)))
      return refuse("scaling by parts needs a trained length and fast_turns above slow_turns");
    const double pi = 3.14159265358979323846;
    const int n = rotary_dim / 2;
    double theta = s->theta;
    if (s->kind == NEEDLE_ROPE_NTK) theta *= std::pow(s->factor, rotary_dim / (rotary_dim - 2.0));
    *magnitude = 1.0;
    if (s->kind == NEEDLE_ROPE_PARTS && s->factor > 1.0) *magnitude = 0.1 * std::log(s->factor) + 1.0;
    for (int i = 0; i < n; i++) {
      double w = std::pow(theta, -2.0 * i / rotary_dim);
      if (s->kind == NEEDLE_ROPE_LINEAR) w /= s->factor;
      if (s->kind == NEEDLE_ROPE_PARTS) {
        const double turns = s->trained_length * w / (2.0 * pi);
        const double keep =
            std::fmin(1.0, std::fmax(0.0, (turns - s->slow_turns) / (s->fast_turns - s->slow_turns)));
        w = w * keep + w / s->factor * (1.0 - keep);
      }
      inverse_frequencies[i] = w;
    }
    return int(NEEDLE_OK);
  });
}
