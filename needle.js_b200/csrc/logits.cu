// logits.cu -- the rules between the vocabulary projection and the choice of a token, and the choice:
// penalties for repeated ids, biases, grammar masks, then (logits_select) the argmax and log
// probability of selectToken (packages/needle.js/src/model/runtime.ts:880-899).
//
//   x = raw logit l;  seen ids:  x = l > 0 ? l / repetition : l * repetition
//   x = x - frequency * c;  c > 0: x = x - presence       (c: times the id was answered)
//   x = x + bias;  ids the mask leaves out: x = -inf       (every step rounded to binary32)
//   id = argmax x, the lowest on ties;  log p = l[id] - max l - log sum exp(l - max l)
//
// A row is read once.  What the rules touch is sparse, so the stream over a row knows only one bit an id (allowed by
// the mask; in selection, without a rule too).  The ids with a rule (history, biases) go into a hash table in shared
// memory, which counts them and keeps their last bias; its entries are ruled one by one from a second, gathered read
// of their logits.  CTAs take parts of rows (at most kPartIds ids; several CTAs or one a row as the batch needs), one
// after another, and build the table for each.  Each of the four warps that stream has its slice of a part come through
// a ring of its own in shared memory, filled by bulk copies that run on over the ends of parts and rows: the copies
// never pause, and no barrier is needed for them.
//
// Bytes bound the stream, the lists' chains of dependent accesses the rest.  512 rows of 50001 bf16 ids (102 MB) with
// histories of up to 1000 ids, 50 biases and masks take 32 us, 23 us without rules.  Select: 4096 rows of 8192
// binary32 ids with histories of 256: 60 us (2.2 TB/s), 41 us without rules; 200 rows of 128000 fp16 ids with
// histories of 2000: 46 us (1.1 TB/s; each of a row's two CTAs builds a table), 25 us without.  Binary32 rules: 60 us for
// 4096 rows of 8192 ids (4.5 TB/s), 46 us for 512 rows of 50001.
// Measured beside it (the three sizes; 42, 61, 46 us then, before the rules had list warps): chunks of a row in
// registers, direct tables of counts instead of the hash, one CTA a chunk: 47, 72, 63 us; the hash 5/4 of its lists
// instead of twice: 50, 66, 55 us (probes), four times: 71, 66, 129 us (fewer CTAs resident); one warp a row: 110 us
// for the 4096 rows (too few warps hide the lists' latency); parts of 32 KB in shared memory with the lists ruled
// there, 8 warps: 51, 81, 85 us (every warp repeats a part's fixed work); twice the parts: 48, 66, 87 us (each
// rescans the lists).
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "serving.cuh"

namespace needle {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kRingBytes = kWarps * 32 * 16 * 8;  // of a CTA: eight 16-byte units a thread, in two steps or four
constexpr int kPartIds = 65536;                  // most ids of a part: 8 KB of bits
constexpr int kListIds = 2;                      // list ids of a thread loaded at once (4: 4096 x 8192 61 -> 66 us)
constexpr int kMostEntries = 4096;               // hash entries of a part; a part of as many ids never has more

// Ids of a step of the stream with `units` 16-byte units a thread.
__host__ __device__ constexpr int step_ids(size_t element, int units) { return kThreads * units * 16 / int(element); }
constexpr int kRulesUnits = 2, kSelectUnits = 4;
// CTAs of an SM by the registers of k_logits_select: a thread holds 16 binary32 logits of a step, or 32 of 16 bits.
__host__ __device__ constexpr int resident(size_t element) { return element == 4 ? 6 : 4; }
constexpr int kRulesResident = 4;  // of k_logits_rules, with its list warps

// The hash table of a part's ids with a rule.  word: bit 31 the mask allows the id, bit 0 it is in the prompt,
// bits 1..30 how often it was answered.
struct Table {
  uint32_t *key, *word, *bias;  // key: id + 1, 0 for a free slot; bias: 1 + position of the id's last bias
  uint32_t* free;               // bit per id of the part
  int slots;                    // a multiple of 4, more than the part can have entries
};

// How a call is cut (plan_for).
struct LogitsPlan {
  int part;   // ids of a part (a multiple of a step's)
  int parts;  // parts of a row
  int slots;  // of the hash table; 0: no lists
};

// Order-preserving key of a binary32 value that is not NaN (-0 as +0); 0 is below every key.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ float exp_below(float v) { return power2f(v * kLog2e); }  // e^v, v <= 0

// First id (possibly below 0) of 16-byte unit 0 of the row: rows that do not start on a 16-byte
// boundary are taken from the boundary before them, with the ids outside the row left out.
template <class T>
__device__ __forceinline__ int row_offset(const T* row) {
  return (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
}

// Ids of a unit whose bit is not set become -inf.
template <int VEC>
__device__ __forceinline__ void keep_free(Vec<float, VEC>& v, uint32_t free) {
#pragma unroll
  for (int i = 0; i < VEC; i++)
    if (!(free & (1u << i))) v.v[i] = -INFINITY;
}
template <class T, int VEC>
__device__ __forceinline__ void keep_free(Vec<T, VEC>& v, uint32_t free) {
  static_assert(sizeof(T) == 2, "two ids a word");
  const uint32_t low = sizeof(T) == 2 && std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;  // -inf twice
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
  free &= (1u << VEC) - 1u;
#pragma unroll
  for (int i = 0; i < VEC / 2; i++) {
    const uint32_t b = free >> (2 * i), keep = ((b | (b << 15)) & 0x00010001u) * 0xffffu;  // bits 0, 1 as two halves
    w[i] = (w[i] & keep) | (low & ~keep);
  }
}

// What the rules of a row need from memory, loaded ahead.
struct RowRules {
  float repetition, frequency, presence;
  int length, prompt, biases;
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
  r.length = a.history ? (int)min((int64_t)max(__ldg(a.history_lengths + row), 0), a.history_stride) : 0;
  r.prompt = a.history && a.prompt_lengths ? __ldg(a.prompt_lengths + row) : 0;
  r.biases = a.bias_ids ? (int)min((int64_t)max(__ldg(a.bias_counts + row), 0), a.bias_stride) : 0;
  r.history = a.history + row * a.history_stride;
  r.bias_ids = a.bias_ids + row * a.bias_stride;
  r.bias_values = a.bias_values + row * a.bias_stride;
  const int slot = a.masks ? __ldg(a.mask_slots + row) : -1;
  r.none = a.masks && slot >= a.mask_count;  // a slot that does not exist
  r.mask = slot >= 0 && !r.none ? a.masks + (int64_t)slot * ((a.vocab + 31) >> 5) : nullptr;
  return r;
}

// Slot of an id of the part (claimed for it when it has none yet).  CLAIM: the id leaves the stream.
template <bool CLAIM>
__device__ __forceinline__ int slot_of(const Table& t, int id, int low) {
  const uint32_t key = (uint32_t)id + 1u;
  uint32_t s = __umulhi((uint32_t)id * 2654435761u, (uint32_t)t.slots);  // multiplicative hashing
  for (;;) {
    const uint32_t k = atomicCAS(&t.key[s], 0u, key);
    if (k == 0u) {
      if (CLAIM) {
        const int p = id - low;
        const uint32_t bit = 1u << (p & 31);
        if (atomicAnd(&t.free[p >> 5], ~bit) & bit) atomicOr(&t.word[s], 0x80000000u);
      }
      return (int)s;
    }
    if (k == key) return (int)s;
    if (++s == (uint32_t)t.slots) s = 0;  // there are more slots than ids, so this ends
  }
}

// The share of thread `tid` of kThreads in a list, kListIds loads at a time, the first of them issued by begin().
struct List {
  const int32_t* list;
  int length, tid;
  int32_t ids[kListIds];

  __device__ __forceinline__ void load(int i0) {
#pragma unroll
    for (int k = 0; k < kListIds; k++)
      if (i0 + k * kThreads < length) ids[k] = __ldg(list + i0 + k * kThreads);
  }
  __device__ __forceinline__ void begin(const int32_t* l, int n, int thread) {
    list = l;
    length = n;
    tid = thread;
    load(tid);
  }
  // Calls f(id, position).
  template <class F>
  __device__ __forceinline__ void each(F f) {
    for (int i0 = tid; i0 < length; i0 += kListIds * kThreads) {
      if (i0 != tid) load(i0);
#pragma unroll
      for (int k = 0; k < kListIds; k++)
        if (i0 + k * kThreads < length) f(ids[k], i0 + k * kThreads);
    }
  }
};

// The bits of ids [low, low + len) of a row (low may be below 0 by less than a unit): allowed by the mask.  Gives the
// lowest id the thread found allowed, 0xffffffff for none.
__device__ __forceinline__ uint32_t allowed_bits(const RowRules& r, const Table& t, int vocab, int low, int len, int tid) {
  uint32_t lowest = 0xffffffffu;
  const int words = (vocab + 31) >> 5;
#pragma unroll 4
  for (int w = tid; w < len / 32; w += kThreads) {
    // ids first .. first + 31: two words of the mask, and none outside the vocabulary
    const int first = low + 32 * w;
    uint32_t bits = r.none ? 0u : 0xffffffffu;
    if (r.mask) {
      const int word = first >> 5;  // floor
      const uint32_t a0 = (uint32_t)word < (uint32_t)words ? __ldg(r.mask + word) : 0;
      const uint32_t a1 = (uint32_t)(word + 1) < (uint32_t)words ? __ldg(r.mask + word + 1) : 0;
      bits = __funnelshift_r(a0, a1, (uint32_t)(first & 31));
    }
    if (first < 0) bits &= 0xffffffffu << -first;
    const int left = vocab - first;
    if (left < 32) bits &= left <= 0 ? 0u : 0xffffffffu >> (32 - left);
    t.free[w] = bits;
    if (bits) lowest = min(lowest, (uint32_t)(first + __ffs(bits) - 1));
  }
  return lowest;
}

__device__ __forceinline__ void clear_table(const Table& t, int tid) {
  // key, word and, where there are biases, bias lie behind one another
  for (int s = tid * 4; s < t.slots * (t.bias ? 3 : 2); s += kThreads * 4)
    *reinterpret_cast<uint4*>(t.key + s) = make_uint4(0, 0, 0, 0);
}

// The lists' ids among [low, low + len) into a cleared table (CLAIM: behind the part's bits).
template <bool CLAIM>
__device__ __forceinline__ void fill_table(const RowRules& r, const Table& t, int vocab, int low, int len, List& history,
                                           List& biases) {
  const int from = max(low, 0), to = min(vocab - low, len) + low;
  history.each([&](int id, int i) {
    if (id < from || id >= to) return;
    const int s = slot_of<CLAIM>(t, id, low);
    if (i >= r.prompt) atomicAdd(&t.word[s], 2u);
    else atomicOr(&t.word[s], 1u);
  });
  biases.each([&](int id, int i) {
    if (id >= from && id < to) atomicMax(&t.bias[slot_of<CLAIM>(t, id, low)], (uint32_t)i + 1u);
  });
}

// Calls f(slot, id, raw logit, ruled logit) for the share of thread `tid` of kThreads in the table's ids (CLAIM: those
// allowed).  Four gathers at a time are in flight.
template <bool CLAIM, class T, class F>
__device__ __forceinline__ void for_ruled(const RowRules& r, const Table& t, const T* row, int tid, F f) {
  for (int s0 = tid; s0 < t.slots; s0 += 4 * kThreads) {
    uint32_t key[4], word[4];
    float raw[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int s = s0 + k * kThreads;
      key[k] = s < t.slots ? t.key[s] : 0;
      word[k] = key[k] ? t.word[s] : 0;
      if (CLAIM && !(word[k] & 0x80000000u)) key[k] = 0;
      raw[k] = key[k] ? to_f32(row[key[k] - 1u]) : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
      if (key[k] == 0) continue;
      const int s = s0 + k * kThreads;
      float x = raw[k];
      const uint32_t seen = word[k] & 0x7fffffffu, c = seen >> 1;
      if (seen) x = x > 0.0f ? __fdiv_rn(x, r.repetition) : __fmul_rn(x, r.repetition);
      if (c) {
        x = __fsub_rn(x, __fmul_rn(r.frequency, (float)c));
        x = __fsub_rn(x, r.presence);
      }
      if (t.bias) {
        const uint32_t b = t.bias[s];
        if (b) x = __fadd_rn(x, __ldg(r.bias_values + b - 1));
      }
      f(s, (int)(key[k] - 1u), raw[k], x);
    }
  }
}

// A barrier of kThreads threads, all stream or all list warps.
__device__ __forceinline__ void group_sync(int id) { asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(kThreads) : "memory"); }

// The table lies behind the warps' rings.
template <class T>
__device__ __forceinline__ Table table_in(unsigned char* smem, const needle_logits_rules& a, const LogitsPlan& plan) {
  Table t;
  t.slots = plan.slots;
  t.key = reinterpret_cast<uint32_t*>(smem + kRingBytes);
  t.word = t.key + plan.slots;
  t.bias = a.bias_ids ? t.word + plan.slots : nullptr;
  t.free = t.key + plan.slots * (a.bias_ids ? 3 : 2);
  return t;
}

// The steps a CTA streams: the rows blockIdx.y, + gridDim.y, ..., of each the parts blockIdx.x, + gridDim.x, ...
template <class T, int UNITS>
struct Steps {
  const T* in;   // the row
  int64_t row;
  int off, part, at, end;  // the step's first id, and where its part ends

  __device__ __forceinline__ void begin_part(const needle_logits_rules& a, const LogitsPlan& plan) {
    at = part * plan.part - off;
    end = min(at + plan.part, a.vocab);
  }
  // The next row, from this one on, that has ids in the CTA's first part (a row's units may begin before it, so
  // the last part of a row can be empty where another's is not).
  __device__ __forceinline__ void begin_row(const needle_logits_rules& a, const LogitsPlan& plan) {
    part = blockIdx.x;
    for (; row < a.rows; row += gridDim.y) {
      in = static_cast<const T*>(a.logits) + row * a.logits_stride;
      off = row_offset(in);
      begin_part(a, plan);
      if (at < a.vocab) return;
    }
  }
  __device__ __forceinline__ void next(const needle_logits_rules& a, const LogitsPlan& plan) {
    at += step_ids(sizeof(T), UNITS);
    if (at < end) return;
    part += gridDim.x;
    begin_part(a, plan);
    if (part < plan.parts && at < a.vocab) return;
    row += gridDim.y;
    begin_row(a, plan);
  }
};

// A warp's stream: its slice of every step, kStages of them in shared memory or on their way.
template <class T, int UNITS>
struct Stream {
  // ids of a 16-byte unit, units of a lane, ids of a step
  static constexpr int VEC = 16 / sizeof(T), N = UNITS, kSlice = 32 * VEC * N;
  static constexpr int kStages = 8 / UNITS;  // steps of the ring
  T* ring;
  uint64_t* bars;  // kStages of them
  Steps<T, UNITS> steps;  // what is copied next
  int stage;       // of the next step to be read
  uint32_t parity;
  bool ok;

  // Whole units of a slice that begins with id e inside the row: from unit `begin` to unit `end`.
  static __device__ __forceinline__ void whole_units(int e, int vocab, int& begin, int& end) {
    begin = e < 0 ? (-e + VEC - 1) / VEC : 0;
    end = max(begin, min(32 * N, (vocab - e) / VEC));
    if (e >= vocab) end = begin;
  }
  __device__ __forceinline__ void copy(const needle_logits_rules& a, const LogitsPlan& plan, int s) {
    if (steps.row >= a.rows) return;
    if ((threadIdx.x & 31) == 0) {
      const int e = steps.at + (int)(threadIdx.x >> 5) * kSlice;
      int begin, end;
      whole_units(e, a.vocab, begin, end);
      const uint32_t bytes = (uint32_t)(end - begin) * 16;
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(shared_address(&bars[s])), "r"(bytes) : "memory");
      if (bytes) copy_bulk(ring + s * kSlice + begin * VEC, steps.in + e + begin * VEC, bytes, &bars[s]);
    }
    steps.next(a, plan);
  }
  __device__ __forceinline__ void begin(const needle_logits_rules& a, const LogitsPlan& plan, unsigned char* smem, uint64_t* all) {
    const int warp = threadIdx.x >> 5;
    ring = reinterpret_cast<T*>(smem) + warp * kStages * kSlice;
    bars = all + warp * kStages;
    if ((threadIdx.x & 31) == 0) {
      for (int s = 0; s < kStages; s++) barrier_init(&bars[s], 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    steps.row = blockIdx.y;
    steps.begin_row(a, plan);
    for (int s = 0; s < kStages; s++) copy(a, plan, s);
    stage = 0;
    parity = 0;
    ok = true;
  }
  // The lane's units of the next step, which begins at id `at` of row `in`; ids outside [0, vocab) are -inf.
  // After a wait that ran out everything is NaN.
  __device__ __forceinline__ void read(const T* in, int at, int vocab, Vec<T, VEC> (&v)[N]) {
    const int lane = threadIdx.x & 31, e = at + (int)(threadIdx.x >> 5) * kSlice;
    ok = ok && barrier_wait_warp(&bars[stage], parity);
    const Vec<T, VEC>* p = reinterpret_cast<const Vec<T, VEC>*>(ring + stage * kSlice) + lane;
    if (ok && e >= 0 && e <= vocab - kSlice) {
#pragma unroll
      for (int u = 0; u < N; u++) v[u] = p[u * 32];
      return;
    }
    int begin, end;
    whole_units(e, vocab, begin, end);
#pragma unroll
    for (int u = 0; u < N; u++) {
      const int k = u * 32 + lane, first = e + k * VEC;
      if (k >= begin && k < end) {
        v[u] = p[u * 32];
      } else {
#pragma unroll
        for (int i = 0; i < VEC; i++) v[u].v[i] = first + i >= 0 && first + i < vocab ? in[first + i] : from_f32<T>(-INFINITY);
      }
      if (!ok) {
#pragma unroll
        for (int i = 0; i < VEC; i++) v[u].v[i] = from_f32<T>(NAN);
      }
    }
  }
  // The step's units have been taken: its place is filled again.
  __device__ __forceinline__ void advance(const needle_logits_rules& a, const LogitsPlan& plan) {
    __syncwarp();
    if (ok) copy(a, plan, stage);
    if (++stage == kStages) {
      stage = 0;
      parity ^= 1;
    }
  }
  // Before the warp ends: a wait that ran out is reported, and copies on their way get their time.
  __device__ __forceinline__ void finish(uint32_t* wait_words) {
    if (ok) return;
    if ((threadIdx.x & 31) == 0) {
      report_wait_timeout(wait_words, kWaitLogits);
      for (int s = 0; s < kStages; s++) barrier_wait(&bars[s], parity);
    }
    __syncwarp();
  }
};

// Four warps stream; where there are lists, four more build the part's table and rule its ids meanwhile: the stream
// writes the ids that the mask allows as they are, ruled or not, so it waits for no list, and the ruled logits are
// written behind it.  (out may be logits: an allowed logit that is gathered is the same before and after it was
// written.)  512 x 50001 bf16 with lists: 32 us (3.2 TB/s of logits in and out), 41.7 us with four warps that do one
// after the other.  Steps of two units a thread: 64 registers hold them, with four units 39.5 us, with one 38.9 us.
template <class T>
__global__ void __launch_bounds__(2 * kThreads, kRulesResident) k_logits_rules(const __grid_constant__ needle_logits_rules a,
                                                                               const LogitsPlan plan, T* out,
                                                                               int64_t out_stride, uint32_t* wait_words) {
  using S = Stream<T, kRulesUnits>;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) uint64_t bars[kWarps * S::kStages];
  const Table t = table_in<T>(smem, a, plan);
  const bool lists = threadIdx.x >= kThreads;  // a list warp
  const int tid = threadIdx.x & (kThreads - 1), lane = tid & 31, slice = (tid >> 5) * S::kSlice;
  S stream;
  if (!lists) stream.begin(a, plan, smem, bars);
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride;
    T* to = out + row * out_stride;
    const int off = row_offset(in);
    const RowRules r = row_rules(a, row);
    const bool listed = r.length > 0 || r.biases > 0;
    // whole units can be written where the output's 16-byte units line up with the input's
    const bool same = row_offset(to) == off;
    for (int part = blockIdx.x; part < plan.parts; part += gridDim.x) {
      const int low = part * plan.part - off, end = min(low + plan.part, a.vocab);
      if (low >= a.vocab) break;
      if (lists) {
        if (listed) {
          List history, biases;
          history.begin(r.history, r.length, tid);
          biases.begin(r.bias_ids, r.biases, tid);
          clear_table(t, tid);
          group_sync(1);
          fill_table<false>(r, t, a.vocab, low, plan.part, history, biases);
          group_sync(1);
          for_ruled<false>(r, t, in, tid, [&](int s, int, float, float x) { t.word[s] = __float_as_uint(x); });
        }
      } else {
        allowed_bits(r, t, a.vocab, low, plan.part, tid);
        group_sync(2);
        for (int at = low; at < end; at += step_ids(sizeof(T), kRulesUnits)) {
          Vec<T, S::VEC> x[S::N];
          stream.read(in, at, a.vocab, x);
          stream.advance(a, plan);
          const int e0 = at + slice + lane * S::VEC;
          const bool whole = same && at + slice >= 0 && at + slice <= a.vocab - S::kSlice;
#pragma unroll
          for (int u = 0; u < S::N; u++) {
            const int e = e0 + u * 32 * S::VEC, p = e - low;
            const uint32_t free = t.free[p >> 5] >> (p & 31);
            keep_free(x[u], free);
            if (whole || (same && e >= 0 && e <= a.vocab - S::VEC)) {
              *reinterpret_cast<Vec<T, S::VEC>*>(to + e) = x[u];
            } else {
#pragma unroll
              for (int i = 0; i < S::VEC; i++)
                if (e + i >= 0 && e + i < a.vocab) to[e + i] = x[u].v[i];
            }
          }
        }
      }
      __syncthreads();
      if (listed) {
        for (int s = threadIdx.x; s < t.slots; s += 2 * kThreads) {
          const uint32_t key = t.key[s];
          const int id = (int)(key - 1u), p = id - low;
          if (key && (t.free[p >> 5] >> (p & 31) & 1u)) to[id] = from_f32<T>(__uint_as_float(t.word[s]));
        }
        __syncthreads();
      }
    }
  }
  if (!lists) stream.finish(wait_words);
}

// One cluster per row (and the rows gridDim.y on); its CTAs take the row's parts in turn.  The stream has to know which
// ids have a rule before it chooses.  List warps beside it, as in k_logits_rules, that mark the ids first and build the
// table meanwhile: 80 instead of 60 us (4096 x 8192), 50 instead of 46 us (200 x 128000): they take the registers of
// stream warps, and steps of two units cost more instructions an id than steps of four (69, 51 us by themselves).
template <class T>
__global__ void __launch_bounds__(kThreads, resident(sizeof(T))) k_logits_select(const __grid_constant__ needle_logits_rules a,
                                                             const LogitsPlan plan, int32_t* __restrict__ ids,
                                                             float* __restrict__ log_probabilities, uint32_t* wait_words) {
  using S = Stream<T, kSelectUnits>;
  struct Best {  // of a warp, of a CTA
    float top, sum, raw;
    uint32_t key, id, lowest;
  };
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) uint64_t bars[kWarps * S::kStages];
  __shared__ Best of_warp[kWarps], of_cta;
  const Table t = table_in<T>(smem, a, plan);
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, slice = warp * S::kSlice;
  S stream;
  stream.begin(a, plan, smem, bars);
  // sums in a fixed order
  auto merge = [&](Best& b) {
    const float m = b.top;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) b.top = fmaxf(b.top, __shfl_xor_sync(0xffffffffu, b.top, o));
    b.sum = m == -INFINITY ? b.sum : b.sum * exp_below(m - b.top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) b.sum += __shfl_xor_sync(0xffffffffu, b.sum, o);
    const uint32_t key = __reduce_max_sync(0xffffffffu, b.key);
    const uint32_t id = __reduce_min_sync(0xffffffffu, b.key == key ? b.id : 0xffffffffu);
    const uint32_t who = __ballot_sync(0xffffffffu, b.key == key && b.id == id);
    b.raw = __shfl_sync(0xffffffffu, b.raw, __ffs(who) - 1);
    b.key = key;
    b.id = id;
    b.lowest = __reduce_min_sync(0xffffffffu, b.lowest);
  };
  const Best nothing = {-INFINITY, 0.0f, 0.0f, 0u, 0xffffffffu, 0xffffffffu};
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride;
    const int off = row_offset(in);
    const RowRules r = row_rules(a, row);
    const bool listed = r.length > 0 || r.biases > 0;
    // the warp's best of the stream; the thread's best of the ids with a rule and its raw logit; the thread's
    // largest raw logit and sum of exponentials
    float best = -INFINITY, ruled_best = -INFINITY, raw = 0.0f, top = -INFINITY, sum = 0.0f;
    uint32_t id = 0xffffffffu, ruled_id = 0xffffffffu;
    uint32_t lowest = 0xffffffffu;  // the lowest allowed id: the choice where every allowed logit is -inf
    for (int part = blockIdx.x; part < plan.parts; part += gridDim.x) {
      const int low = part * plan.part - off, end = min(low + plan.part, a.vocab);
      if (low >= a.vocab) break;
      if (part != (int)blockIdx.x) __syncthreads();  // the table of the part before has been read
      {
        List history, biases;  // on their way beside the mask
        history.begin(r.history, r.length, tid);
        biases.begin(r.bias_ids, r.biases, tid);
        lowest = min(lowest, allowed_bits(r, t, a.vocab, low, plan.part, tid));
        if (listed) clear_table(t, tid);
        __syncthreads();
        if (listed) {
          fill_table<true>(r, t, a.vocab, low, plan.part, history, biases);
          __syncthreads();
        }
      }
      for (int at = low; at < end; at += step_ids(sizeof(T), kSelectUnits)) {
        float x[S::N][S::VEC];
        {
          Vec<T, S::VEC> v[S::N];
          stream.read(in, at, a.vocab, v);
#pragma unroll
          for (int u = 0; u < S::N; u++)
#pragma unroll
            for (int i = 0; i < S::VEC; i++) x[u][i] = to_f32(v[u].v[i]);
        }
        stream.advance(a, plan);
        float most = -INFINITY;
#pragma unroll
        for (int u = 0; u < S::N; u++)
#pragma unroll
          for (int i = 0; i < S::VEC; i += 2) most = max3(most, x[u][i], x[u][i + 1]);
        const float m = fmaxf(top, most), base = m == -INFINITY ? 0.0f : m;
        sum = top == -INFINITY ? 0.0f : sum * exp_below(top - base);
        top = m;
        if (fabsf(base) < 1e6f) {
          // 2^(x log2 e - p) with p = m log2 e rounded: a term is 2^off times its value, off = m log2 e - p up to
          // 2^-24 |m|, exact in a fused product.  The factor goes out once a step (no slower: 200 x 128000 45.6 us).
          // Further from zero, where binary32 logits are 2^-4 apart and more, m is subtracted first
          const float2 scale = make_float2(kLog2e, kLog2e), minus = make_float2(-base * kLog2e, -base * kLog2e);
          const float off = fmaf(base, kLog2e, minus.x);
          float2 more = make_float2(0.0f, 0.0f);
#pragma unroll
          for (int u = 0; u < S::N; u++)
#pragma unroll
            for (int i = 0; i < S::VEC; i += 2) {
              float2 d = __ffma2_rn(make_float2(x[u][i], x[u][i + 1]), scale, minus);
              d.x = power2f(d.x);
              d.y = power2f(d.y);
              more = __fadd2_rn(more, d);
            }
          sum += (more.x + more.y) * power2f(-off);
        } else {
#pragma unroll
          for (int u = 0; u < S::N; u++)
#pragma unroll
            for (int i = 0; i < S::VEC; i++) sum += exp_below(x[u][i] - base);
        }
        // the free ids matter only where some id of the step beats the best one so far
        if (__any_sync(0xffffffffu, most > best)) {
          uint32_t free[S::N];
          float top_free = -INFINITY;
#pragma unroll
          for (int u = 0; u < S::N; u++) {
            const int p = at - low + slice + (u * 32 + lane) * S::VEC;
            free[u] = t.free[p >> 5] >> (p & 31);
#pragma unroll
            for (int i = 0; i < S::VEC; i++)
              if (free[u] & (1u << i)) top_free = fmaxf(top_free, x[u][i]);
          }
          const uint32_t key = __reduce_max_sync(0xffffffffu, order_key(top_free));
          if (key > order_key(best)) {
            uint32_t mine = 0xffffffffu;
            if (order_key(top_free) == key) {
#pragma unroll
              for (int u = S::N - 1; u >= 0; u--)
#pragma unroll
                for (int i = S::VEC - 1; i >= 0; i--)
                  if ((free[u] & (1u << i)) && x[u][i] == top_free)
                    mine = (uint32_t)(at + slice + (u * 32 + lane) * S::VEC + i);
            }
            id = __reduce_min_sync(0xffffffffu, mine);
            best = __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
          }
        }
      }
      if (listed) for_ruled<true>(r, t, in, tid, [&](int, int id_of, float l, float v) {
        const uint32_t i = (uint32_t)id_of;
        if (v > ruled_best || (v == ruled_best && i < ruled_id && v > -INFINITY)) {
          ruled_best = v;
          raw = l;
          ruled_id = i;
        }
      });
    }
    // warp, CTA, cluster
    if (best > ruled_best || (best == ruled_best && id < ruled_id)) {
      ruled_best = raw = best;
      ruled_id = id;
    }
    Best b = {top, sum, raw, ruled_id == 0xffffffffu ? 0u : order_key(ruled_best), ruled_id, lowest};
    merge(b);
    if (lane == 0) of_warp[warp] = b;
    __syncthreads();
    if (warp == 0) {
      b = lane < kWarps ? of_warp[lane] : nothing;
      merge(b);
      if (lane == 0 && gridDim.x > 1) of_cta = b;
    }
    if (gridDim.x > 1) cluster.sync();
    if (blockIdx.x == 0 && warp == 0) {
      if (gridDim.x > 1) {
        b = nothing;
        if (lane < (int)gridDim.x) b = *cluster.map_shared_rank(&of_cta, lane);
        merge(b);
      }
      if (lane == 0) {
        const bool only = b.key == 0 && b.lowest != 0xffffffffu;  // no allowed logit above -inf
        if (only) {
          b.id = b.lowest;
          b.raw = to_f32(in[b.id]);
        }
        ids[row] = (int32_t)b.id;  // 0xffffffff is -1
        log_probabilities[row] = b.id != 0xffffffffu ? (b.raw - b.top) - logf(b.sum) : -INFINITY;
      }
    }
    if (gridDim.x > 1) cluster.sync();  // the CTAs' results have been read
  }
  stream.finish(wait_words);
}

size_t smem_bytes(const needle_logits_rules& a, const LogitsPlan& p) {
  return size_t(kRingBytes) + size_t(p.slots) * (a.bias_ids ? 12 : 8) + size_t(p.part) / 8;
}

// CTAs that the GPU holds at once: by shared memory, and by registers.
int64_t resident_ctas(int by_registers, size_t smem) {
  return 148 * std::max<int64_t>(1, std::min<int64_t>(by_registers, int64_t(226 * 1024 / (smem + 1536))));
}

// Rows a CTA (or cluster) of `parts` CTAs takes side by side with the others: as few turns as the GPU can hold,
// all of them full.
unsigned rows_at_once(const needle_logits_rules& a, int by_registers, size_t smem, int parts) {
  const int64_t fit = std::max<int64_t>(1, resident_ctas(by_registers, smem) / parts), turns = (a.rows + fit - 1) / fit;
  return unsigned((a.rows + turns - 1) / turns);
}

LogitsPlan plan_for(const needle_logits_rules& a, int units, int most_parts) {
  LogitsPlan p{};
  const int64_t element = int64_t(type_bytes(a.type));
  const bool lined_up = aligned_to(a.logits, 16) && (a.rows == 1 || a.logits_stride * element % 16 == 0);
  const int64_t ids = int64_t(a.vocab) + (lined_up ? 0 : 16 / element - 1);  // with those before a row's first unit
  const int64_t entries = (a.history ? a.history_stride : 0) + (a.bias_ids ? a.bias_stride : 0);
  const int64_t step = step_ids(size_t(element), units), steps = (ids + step - 1) / step;
  // parts: as many as keep the GPU busy, each rescanning the lists (148 * 8: 512 x 50001 32 -> 38 us, 200 x 128000
  // 46 -> 86 us); small enough for their bits and, with long lists, for a table that has room for every id of the part.
  // What counts is the lists' room, not their lengths, which are on the device.  200 x 128000, 100 biases, histories of
  // up to 2000 ids (of 10): room for 2000: 47 us; 3900: 121 us (72): a table twice as large, cleared and walked whole, and
  // half the CTAs; 5000 and 32768: 943 us (662): 32 parts a row.  512 x 50001, up to 1000 (10): 31 us, 761 us (351).
  const int64_t most = (entries > kMostEntries ? kMostEntries : kPartIds) / step;
  int64_t parts = std::max<int64_t>(1, std::min<int64_t>({steps, 148 * 4 / a.rows, most_parts}));
  parts = std::max(parts, (steps + most - 1) / most);
  const int64_t per = (steps + parts - 1) / parts;
  p.part = int(per * step);
  p.parts = int((steps + per - 1) / per);
  if (entries > 0) p.slots = int((std::min(entries, int64_t(p.part)) * 2 + 35) / 4 * 4);
  return p;
}

int check_rules(const needle_logits_rules* a) {
  if (!a) return refuse("null argument");
  if (a->type < NEEDLE_TYPE_F32 || a->type > NEEDLE_TYPE_BF16) return refuse("unknown element type");
  if (a->rows < 0 || a->vocab < 0) return refuse("bad row or vocabulary count");
  if (a->rows == 0 || a->vocab == 0) return NEEDLE_OK;
  if (a->rows > 65535) return refuse("at most 65535 rows in a call");
  if (a->vocab > 1 << 30) return refuse("at most 2^30 ids");
  if (!a->logits) return refuse("null argument");
  if (a->rows > 1 && a->logits_stride < a->vocab) return refuse("a row stride is shorter than its row");
  if (a->history && (!a->history_lengths || a->history_stride < 0)) return refuse("history without lengths");
  if (a->bias_ids && (!a->bias_values || !a->bias_counts || a->bias_stride < 0))
    return refuse("bias ids without values or counts");
  if ((a->history && a->history_stride >= 1 << 30) || (a->bias_ids && a->bias_stride >= 1 << 30))  // counts have 30 bits
    return refuse("fewer than 2^30 history entries and biases a row");
  if (a->masks && (!a->mask_slots || a->mask_count < 0)) return refuse("masks without slots");
  return NEEDLE_OK;
}

// The buffers' alignment and device; gives the current device.
int check_rules_buffers(const needle_logits_rules* a, Buffers outputs, int* device, const char* op) {
  const Buffers buffers = {{a->logits, "logits", type_bytes(a->type)}, {a->history, "history", 4},
                           {a->history_lengths, "history_lengths", 4}, {a->prompt_lengths, "prompt_lengths", 4},
                           {a->repetition, "repetition", 4}, {a->presence, "presence", 4}, {a->frequency, "frequency", 4},
                           {a->bias_ids, "bias_ids", 4}, {a->bias_values, "bias_values", 4}, {a->bias_counts, "bias_counts", 4},
                           {a->masks, "masks", 4}, {a->mask_slots, "mask_slots", 4}};
  if (int rc = check_alignment(buffers)) return rc;
  if (int rc = check_alignment(outputs)) return rc;
  const cudaError_t e = cudaGetDevice(device);
  if (e != cudaSuccess) return refuse_cuda(op, e);
  if (int rc = check_buffers(buffers, *device)) return rc;
  return check_buffers(outputs, *device);
}

// Always the same limit, so that calls at the same time cannot lower each other's: rings, a table of kMostEntries
// with their biases, and a bit an id of the largest part.
constexpr size_t kMostSmem = kRingBytes + (kMostEntries * 2 + 36) * 12 + kPartIds / 8;
template <class K>
cudaError_t set_smem(K kernel) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kMostSmem));
}

}  // namespace
}  // namespace needle

using namespace needle;

extern "C" int needle_cuda_logits_rules_dev(const needle_logits_rules* a, void* out, int64_t out_stride, void* stream) {
  return entry([&] {
    if (int rc = check_rules(a)) return rc;
    if (a->rows == 0 || a->vocab == 0) return int(NEEDLE_OK);
    if (!out) return refuse("null argument");
    if (a->rows > 1 && out_stride < a->vocab) return refuse("a row stride is shorter than its row");
    if (a->rows > 1 && out == a->logits && out_stride != a->logits_stride)
      return refuse("out may be logits only with the same row stride");
    int device = 0;
    if (int rc = check_rules_buffers(a, {{out, "out", type_bytes(a->type)}}, &device, "logits_rules")) return rc;
    if (check_wait_status(device) != NEEDLE_OK) return int(NEEDLE_BACKEND_UNAVAILABLE);
    const LogitsPlan plan = plan_for(*a, kRulesUnits, 1 << 30);
    const size_t smem = smem_bytes(*a, plan);
    const cudaError_t e = with_type(a->type, [&](auto zero) {
      using T = decltype(zero);
      const cudaError_t err = set_smem(k_logits_rules<T>);
      if (err != cudaSuccess) return err;
      const dim3 grid(plan.parts, rows_at_once(*a, kRulesResident, smem, plan.parts));
      k_logits_rules<T><<<grid, plan.slots > 0 ? 2 * kThreads : kThreads, smem, static_cast<cudaStream_t>(stream)>>>(
          *a, plan, static_cast<T*>(out), out_stride, wait_status_words(device));
      return cudaGetLastError();
    });
    return e == cudaSuccess ? int(NEEDLE_OK) : refuse_cuda("logits_rules", e);
  });
}

extern "C" int needle_cuda_logits_select_dev(const needle_logits_rules* a, int32_t* ids, float* log_probabilities,
                                             void* stream) {
  return entry([&] {
    if (int rc = check_rules(a)) return rc;
    if (a->rows == 0) return int(NEEDLE_OK);
    if (a->vocab == 0) return refuse("an empty vocabulary has no id to select");
    if (!ids || !log_probabilities) return refuse("null argument");
    int device = 0;
    if (int rc = check_rules_buffers(a, {{ids, "ids", 4}, {log_probabilities, "log_probabilities", 4}}, &device, "logits_select"))
      return rc;
    if (check_wait_status(device) != NEEDLE_OK) return int(NEEDLE_BACKEND_UNAVAILABLE);
    const LogitsPlan plan = plan_for(*a, kSelectUnits, 8);  // a row's CTAs are one cluster
    const size_t smem = smem_bytes(*a, plan);
    const cudaError_t e = with_type(a->type, [&](auto zero) {
      using T = decltype(zero);
      const cudaError_t err = set_smem(k_logits_select<T>);
      if (err != cudaSuccess) return err;
      const int cluster = std::min(8, plan.parts);
      cudaLaunchAttribute attribute{};
      attribute.id = cudaLaunchAttributeClusterDimension;
      attribute.val.clusterDim.x = cluster;
      attribute.val.clusterDim.y = 1;
      attribute.val.clusterDim.z = 1;
      cudaLaunchConfig_t config{};
      config.gridDim = dim3(cluster, rows_at_once(*a, resident(sizeof(T)), smem, cluster));
      config.blockDim = dim3(kThreads);
      config.dynamicSmemBytes = smem;
      config.stream = static_cast<cudaStream_t>(stream);
      config.attrs = &attribute;
      config.numAttrs = 1;
      return cudaLaunchKernelEx(&config, k_logits_select<T>, *a, plan, ids, log_probabilities, wait_status_words(device));
    });
    return e == cudaSuccess ? int(NEEDLE_OK) : refuse_cuda("logits_select", e);
  });
}
