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
// the binary64 product with 1 / 127, several times cheaper than the quotient; rounded to binary32, as it is
// stored, it is the same for every binary32 maximum (all of them were compared).  The two differ by one
// binary64 ulp in one row of ten, which only a value exactly on a border between codes can tell: half of a
// row's largest value, in most rows.  There binary32 rows, the engine's type, are divided by the quotient and
// get the engine's codes; 16-bit rows, where such values are common (one in 2.4% of bf16 rows of 128 normal
// values gets another code), keep the product: 63 or 64 for 63.5 steps, equally near.
// Queries in binary32 are computed the same way; 16-bit queries in binary32, whose error (2^-23) is far
// below the rounding to 16 bits (2^-11, 2^-8).
//
// A warp reads kRows head rows at once, 16 bytes a lane, and works on one token (or a part of one, where there are
// few): it computes the token's angles in binary64, leaves them in shared memory, and walks over the keys, the
// values and the queries, whose pieces come to a place of each lane in shared memory kAhead turns before they are
// used (cp.async: a register a load in flight would cost resident warps).  Bytes bound the operator (every row is read
// and written once), then instructions: about 90 for 256 query elements, 250 for 256 key elements, of which the
// binary64 rotation and its conversions (quarter rate) are the larger part.
// Measured, 8191 tokens of 32 / 8 heads of 128 in bf16 (217 MB): 131 us with a CTA a token and 8-byte accesses; 100 us
// with a warp a token; 64 us with the exact division only for quotients next to a border, in a loop over them (inlined
// for every element it held registers), and accesses whose width is known at compile time; 48 us = 4.5 TB/s, 69% of a
// copy's rate, with the loads in shared memory (in registers: 61 us; 8 ahead instead of 4: 49 us).  4 resident CTAs of
// 64 registers: 3 take 51 us, 5 take 60 us (spills).  4096 tokens of 8 / 4 heads of 64 in binary32 (36 MB): 13.9 us,
// bound by conversions; 4 tokens: 3.7 us.
// At 64 registers the 16-bit kernels spill 16 bytes (pairs), 36 (halves) and 160 (any), those of binary32 none.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "serving.cuh"

namespace needle {

namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeWarps = kRopeThreads / 32;
constexpr int kMaxPairs = 64;        // rotated pairs of a head of 128
constexpr int kRopeFill = 148 * 3;   // CTAs that keep the GPU busy (148 * 6: as fast; 148 * 12: 4096 tokens 14 -> 19 us)
constexpr int kRopeResident = 4;     // CTAs of an SM
constexpr int kAhead = 4;            // 16-byte loads of a lane in flight

// What a kernel is built for, E being the elements of a lane: pairs (2i, 2i + 1) and 16-byte accesses; pairs
// (i, i + half), half a multiple of E (a lane's partners are then one lane), and 16-byte accesses; or any pairs and
// any alignment, an element an access and nothing loaded ahead: halves that are no multiple of E (a rotary size of 24,
// 40 or 50 in 16 bits), and rows that do not begin on 16 bytes.
enum Form { kInterleaved, kHalves, kAny };

struct RopeArgs {
  needle_rope_append a;
  int32_t parts;  // warps that share a token: 1, 2, 4 or 8
  double inverse[kMaxPairs];
};

// a c - b s; binary64 rounds every step as the engine's JavaScript does.
__device__ __forceinline__ float turned(double a, double c, double b, double s) { return (float)(a * c - b * s); }
__device__ __forceinline__ float turned(float a, float c, float b, float s) { return fmaf(a, c, -b * s); }

// Where pair i's (cosine, sine) lies: lanes whose pairs are 4 or 8 apart meet different banks.
__device__ __forceinline__ int angle_at(int pair) { return pair ^ (pair >> 3 & 7); }

// The norm and rotation of rows of D elements, E of them in each of D / E lanes, in arithmetic A.  Angles and norm
// factors (1 + s) in binary64 are read from shared memory for every row: in registers they would cost half the
// resident warps.  Binary32 angles are kept.
template <class A, int D, int E, int FORM, bool BF16 = false>
struct Turn {
  using Angle = typename std::conditional<std::is_same<A, double>::value, double2, float2>::type;
  static constexpr int kLanes = D / E, kAngles = FORM == kInterleaved ? E / 2 : E;
  static constexpr bool kKept = std::is_same<A, float>::value && FORM != kAny;
  const A* factors;     // of this lane
  const Angle* angles;  // of the token
  Angle kept[kKept ? kAngles : 1];
  int sub, half, other, pair0;
  bool normed, interleaved, first, turns, whole;  // whole: all of the lane's elements turn

  __device__ __forceinline__ Turn(bool normed, const A* factors, const Angle* angles, int sub, int rotary, bool interleaved)
      : factors(factors + sub * E), angles(angles), sub(sub), half(rotary >> 1), normed(normed), interleaved(interleaved) {
    const int e0 = sub * E;
    turns = e0 < rotary;
    whole = e0 + E <= rotary;
    first = e0 < half;
    other = first ? sub + half / E : sub - half / E;
    pair0 = FORM == kInterleaved ? e0 / 2 : first ? e0 : e0 - half;
    if constexpr (kKept) {
#pragma unroll
      for (int i = 0; i < kAngles; i++) kept[i] = turns ? angles[angle_at(pair0 + i)] : Angle{1.0f, 0.0f};
    }
  }
  __device__ __forceinline__ Angle angle(int i) const {
    if constexpr (kKept)
      return kept[i];
    else
      return angles[angle_at(pair0 + i)];
  }
  static __device__ __forceinline__ void turn_pair(float& x, float& y, const Angle& t) {
    const A a = (A)x, b = (A)y;
    x = turned(a, t.x, b, t.y);
    y = turned(b, t.x, -a, t.y);
  }

  __device__ __forceinline__ void operator()(float (&x)[E]) const {
    if (normed) {
      auto squares = [&] {
        A sum = 0;
#pragma unroll
        for (int i = 0; i < E; i++) sum = fma((A)x[i], (A)x[i], sum);
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        return sum;
      };
      A sum = squares(), least = (A)1e-6;
      // Squares of bf16 values beyond 2^60 can pass binary32's range: such a row is brought nearer first, where 1e-6 is
      // nothing beside its mean (8191 tokens of 32 / 8 heads with norms: 59.5 us, 58.3 us without)
      if constexpr (BF16 && std::is_same<A, float>::value) {
        const bool far = sum == INFINITY;
        if (__any_sync(0xffffffffu, far)) {
#pragma unroll
          for (int i = 0; i < E; i++) x[i] *= far ? 0x1p-68f : 1.0f;
          sum = squares();
          least = far ? 0.0f : least;
        }
      }
      const A inverse = rsqrt(sum * (A)(1.0 / D) + least);
      constexpr int kPiece = 16 / sizeof(A);
#pragma unroll
      for (int i = 0; i < E; i += kPiece) {
        const Vec<A, kPiece> f = *reinterpret_cast<const Vec<A, kPiece>*>(factors + i);
#pragma unroll
        for (int j = 0; j < kPiece; j++) x[i + j] = (float)(f.v[j] * (A)x[i + j] * inverse);
      }
    }
    if (FORM == kInterleaved) {
      if (whole) {
#pragma unroll
        for (int i = 0; i < E; i += 2) turn_pair(x[i], x[i + 1], angle(i / 2));
      } else if (turns) {
#pragma unroll
        for (int i = 0; i < E; i += 2)
          if (sub * E + i < 2 * half) turn_pair(x[i], x[i + 1], angle(i / 2));
      }
    } else if (FORM == kHalves) {
      float y[E];
#pragma unroll
      for (int i = 0; i < E; i++) y[i] = __shfl_sync(0xffffffffu, x[i], other, kLanes);
      if (turns) {
#pragma unroll
        for (int i = 0; i < E; i++) {
          const Angle t = angle(i);
          x[i] = turned((A)x[i], t.x, first ? (A)y[i] : -(A)y[i], t.y);
        }
      }
    } else if (interleaved) {
#pragma unroll
      for (int i = 0; i < E; i += 2)
        if (sub * E + i < 2 * half) turn_pair(x[i], x[i + 1], angles[angle_at((sub * E + i) / 2)]);
    } else {  // the partner of element i is element (i +- half) % E of a lane that depends on i
      const int shift = half % E;
      float y[E];
#pragma unroll
      for (int i = 0; i < E; i++) {
        float from_up = 0.0f, from_down = 0.0f;
#pragma unroll
        for (int j = 0; j < E; j++) {
          if ((i + shift) % E == j) from_up = x[j];
          if ((i + E - shift) % E == j) from_down = x[j];
        }
        from_up = __shfl_sync(0xffffffffu, from_up, sub + (i + half) / E, kLanes);
        from_down = __shfl_sync(0xffffffffu, from_down, sub - (half - i + E - 1) / E, kLanes);
        y[i] = sub * E + i < half ? from_up : from_down;
      }
#pragma unroll
      for (int i = 0; i < E; i++) {
        const int e = sub * E + i;
        if (e < 2 * half) {
          const Angle t = angles[angle_at(e < half ? e : e - half)];
          x[i] = turned((A)x[i], t.x, e < half ? (A)y[i] : -(A)y[i], t.y);
        }
      }
    }
  }
};

template <class T, int E, int FORM>
__device__ __forceinline__ void store_piece(T* p, const float (&x)[E]) {
  Vec<T, E> v;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < E; i++) v.v[i] = x[i];
  } else {
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(x[i], x[i + 1]);
        v.v[i] = h.x, v.v[i + 1] = h.y;
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[i], x[i + 1]);
        v.v[i] = h.x, v.v[i + 1] = h.y;
      }
    }
  }
  if constexpr (FORM != kAny) {
    *reinterpret_cast<Vec<T, E>*>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < E; i++) p[i] = v.v[i];
  }
}

template <class T, int D, int FORM>
__global__ void __launch_bounds__(kRopeThreads, kRopeResident) k_rope_append(const __grid_constant__ RopeArgs args) {
  constexpr int E = 16 / sizeof(T), kLanes = D / E, kRows = 32 / kLanes;
  constexpr bool kNarrow = sizeof(T) == 2;
  using Query = typename std::conditional<kNarrow, float, double>::type;
  using Piece = Vec<T, E>;
  __shared__ double2 angles[kRopeWarps][kMaxPairs];
  __shared__ float2 angles32[kNarrow ? kRopeWarps : 1][kMaxPairs];
  __shared__ alignas(16) double k_factors[D];
  __shared__ alignas(16) Query q_factors[D];
  __shared__ Piece pieces[FORM == kAny ? 1 : kAhead][kRopeThreads];  // each lane's own
  const needle_rope_append& a = args.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = lane / kLanes, sub = lane % kLanes;
  const int parts = args.parts, mine = warp / parts, part = warp % parts;
  const int64_t token = (int64_t)blockIdx.x * (kRopeWarps / parts) + mine;
  const bool live = token < a.tokens;
  const int step = parts * kRows;  // heads a turn
  // the first head of this warp, of each kind: few heads are spread over the warps
  const int q0 = part * kRows, k0 = (parts - 1 - part) * kRows, v0 = (part + parts / 2) % parts * kRows;
  // The warp's turns: its key rows, its value rows, its query rows.
  auto turns_of = [&](int head, int heads) { return (max(heads - head, 0) + step - 1) / step; };
  const int k_turns = turns_of(k0, a.kv_heads), kv_turns = k_turns + turns_of(v0, a.kv_heads);
  const int turns = kv_turns + turns_of(q0, a.heads);
  // The lane's elements of a turn, NULL where the group has no row.
  auto piece_of = [&](int turn) -> const T* {
    const bool key = turn < k_turns, query = turn >= kv_turns;
    const int head = group + (key ? k0 + turn * step : query ? q0 + (turn - kv_turns) * step : v0 + (turn - k_turns) * step);
    if (head >= (query ? a.heads : a.kv_heads)) return nullptr;
    const void* base = key ? a.k : query ? a.q : a.v;
    return static_cast<const T*>(base) + token * (key ? a.k_stride : query ? a.q_stride : a.v_stride) + (int64_t)head * D + sub * E;
  };
  auto ask = [&](int turn) {
    if constexpr (FORM != kAny) {
      const T* p = turn < turns ? piece_of(turn) : nullptr;
      if (p)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared_address(&pieces[turn % kAhead][threadIdx.x])),
                     "l"(p)
                     : "memory");
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  };
  auto take = [&](int turn, float (&x)[E]) {
    Piece v{};
    if constexpr (FORM != kAny) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
      v = pieces[turn % kAhead][threadIdx.x];  // (of no use where the group has no row)
      ask(turn + kAhead);
    } else if (const T* p = piece_of(turn)) {
#pragma unroll
      for (int i = 0; i < E; i++) v.v[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < E; i++) x[i] = to_f32(v.v[i]);
  };
  int64_t at = -1;
  if (live) {
    for (int turn = 0; turn < kAhead; turn++) ask(turn);  // on their way while the angles are computed
    const int slot = a.slots[token], entry = a.entries[token];
    if (slot >= 0 && slot < a.slot_count && entry >= 0 && entry < a.capacity)
      at = (int64_t)slot * a.kv_heads * a.capacity + entry;
    const double position = a.positions[token];
    for (int i = part * 32 + lane; i < a.rotary_dim >> 1; i += parts * 32) {
      double s, c;
      sincos(position * args.inverse[i], &s, &c);
      c *= a.magnitude, s *= a.magnitude;
      angles[mine][angle_at(i)] = make_double2(c, s);
      if constexpr (kNarrow) angles32[mine][angle_at(i)] = make_float2((float)c, (float)s);
    }
  }
  if (a.k_norm)
    for (int i = threadIdx.x; i < D; i += kRopeThreads) k_factors[i] = 1.0 + (double)a.k_norm[i];
  if (a.q_norm)
    for (int i = threadIdx.x; i < D; i += kRopeThreads) q_factors[i] = (Query)1 + (Query)a.q_norm[i];
  if (parts > 1 || a.k_norm || a.q_norm)
    __syncthreads();
  else
    __syncwarp();
  if (!live) return;

  int turn = 0;
  auto keep = [&](float (&x)[E], int head, int8_t* codes, float* scales, void* out, int64_t stride) {
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < E; i++) top = fmaxf(top, fabsf(x[i]));
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const double scale = fmax(1e-12, (double)top) * (1.0 / 127.0);
    const float scale32 = (float)scale, inverse = 1.0f / scale32;
    // The quotient in binary32 is within 2^-15 of the exact one; adding 1.5 * 2^23 rounds it to an integer,
    // which the sum's lowest byte holds.  One that near a border between codes, or a NaN, is divided in binary64
    // (by the quotient in binary32 rows, whose division only these few pay for).
    constexpr float kRound = 12582912.0f;
    uint32_t border = 0;
    float r[E];
#pragma unroll
    for (int i = 0; i < E; i++) {
      const float t = x[i] * inverse;
      r[i] = t + kRound;
      border |= !(fabsf(t - (r[i] - kRound)) < 0.4999f) ? 1u << i : 0u;
    }
    while (border) {
      const int at = __ffs(border) - 1;
      border &= border - 1;
      float value = x[0];
#pragma unroll
      for (int i = 1; i < E; i++) value = i == at ? x[i] : value;
      float code = (float)rint((double)value / (kNarrow ? scale : fmax(1e-12, (double)top) / 127.0));
      code = code != code ? 0.0f : fminf(fmaxf(code, -127.0f), 127.0f);
#pragma unroll
      for (int i = 0; i < E; i++) r[i] = i == at ? code + kRound : r[i];
    }
    Vec<int8_t, E> code;
#pragma unroll
    for (int i = 0; i < E; i++) {
      code.v[i] = (int8_t)__float_as_int(r[i]);
      x[i] = (r[i] - kRound) * scale32;
    }
    if (head + group >= a.kv_heads) return;
    if (at >= 0) {
      const int64_t row = at + (int64_t)(head + group) * a.capacity;
      *reinterpret_cast<Vec<int8_t, E>*>(codes + row * D + sub * E) = code;
      if (sub == 0) scales[row] = scale32;
    }
    if (out) store_piece<T, E, FORM>(static_cast<T*>(out) + token * stride + (int64_t)(head + group) * D + sub * E, x);
  };
  const Turn<double, D, E, FORM> turn_key(a.k_norm != nullptr, k_factors, angles[mine], sub, a.rotary_dim,
                                          a.interleaved);
  for (int head = k0; head < a.kv_heads; head += step, turn++) {
    float x[E];
    take(turn, x);
    turn_key(x);
    keep(x, head, a.key_codes, a.key_scales, a.k_out, a.k_out_stride);
  }
  for (int head = v0; head < a.kv_heads; head += step, turn++) {
    float x[E];
    take(turn, x);
    keep(x, head, a.value_codes, a.value_scales, a.v_out, a.v_out_stride);
  }
  const auto* query_angles = [&] {
    if constexpr (kNarrow)
      return angles32[mine];
    else
      return angles[mine];
  }();
  const Turn<Query, D, E, FORM, std::is_same<T, __nv_bfloat16>::value> turn_query(a.q_norm != nullptr, q_factors, query_angles,
                                                                                  sub, a.rotary_dim, a.interleaved);
  for (int head = q0; head < a.heads; head += step, turn++) {
    float x[E];
    take(turn, x);
    turn_query(x);
    if (head + group < a.heads)
      store_piece<T, E, FORM>(static_cast<T*>(a.q_out) + token * a.q_out_stride + (int64_t)(head + group) * D + sub * E, x);
  }
}

cudaError_t launch_rope(RopeArgs& args, cudaStream_t s) {
  const needle_rope_append& a = args.a;
  const int e = int(type_bytes(a.type)), half = a.rotary_dim / 2;
  // A warp a token computes its angles once and waits for no other; with few tokens, several share one.
  args.parts = 1;
  while (args.parts < kRopeWarps && int64_t(a.tokens) * args.parts < int64_t(kRopeFill) * kRopeWarps) args.parts *= 2;
  auto wide = [&](const void* p, int64_t stride) { return aligned_to(p, 16) && (a.tokens == 1 || stride * e % 16 == 0); };
  const bool all_wide = wide(a.q, a.q_stride) && wide(a.k, a.k_stride) && wide(a.v, a.v_stride) &&
                        wide(a.q_out, a.q_out_stride) && wide(a.k_out, a.k_out_stride) && wide(a.v_out, a.v_out_stride);
  const unsigned grid = unsigned((int64_t(a.tokens) * args.parts + kRopeWarps - 1) / kRopeWarps);
  return with_type(a.type, [&](auto zero) {
    using T = decltype(zero);
    auto go = [&](auto* interleaved, auto* halves, auto* any) {
      // (one pair is the same pair either way)
      auto* kernel = !all_wide ? any : a.interleaved || half == 1 ? interleaved : half % (16 / e) == 0 ? halves : any;
      kernel<<<grid, kRopeThreads, 0, s>>>(args);
      return cudaGetLastError();
    };
    return a.head_dim == 64
               ? go(k_rope_append<T, 64, kInterleaved>, k_rope_append<T, 64, kHalves>, k_rope_append<T, 64, kAny>)
               : go(k_rope_append<T, 128, kInterleaved>, k_rope_append<T, 128, kHalves>, k_rope_append<T, 128, kAny>);
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
    // (with another stride a token's output would be another token's input)
    if (a->tokens > 1 && ((a->q_out == a->q && a->q_out_stride != a->q_stride) ||
                          (a->k_out == a->k && a->k_out_stride != a->k_stride) ||
                          (a->v_out == a->v && a->v_out_stride != a->v_stride)))
      return refuse("q_out may be q, k_out k and v_out v only with the same row stride");
    const size_t e = type_bytes(a->type);
    const Buffers buffers = {{a->q, "q", e}, {a->k, "k", e}, {a->v, "v", e}, {a->q_out, "q_out", e}, {a->k_out, "k_out", e},
                             {a->v_out, "v_out", e}, {a->q_norm, "q_norm", 4}, {a->k_norm, "k_norm", 4},
                             {a->positions, "positions", 4}, {a->slots, "slots", 4}, {a->entries, "entries", 4},
                             {a->key_codes, "key_codes", 1}, {a->key_scales, "key_scales", 4},
                             {a->value_codes, "value_codes", 1}, {a->value_scales, "value_scales", 4}};
    if (int rc = check_alignment(buffers)) return rc;
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
    if (int rc = check_buffers(buffers, device)) return rc;
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
