// Operators on language-model logits z [rows, cols], x = z / temperature:
// log-probabilities of given tokens with the row's entropy and its most likely
// alternatives (credit_token_logprob_*), and the divergence from a teacher's
// top entries (credit_topk_distill_*), each with its gradient.
//
// The forwards read the logits once and write a few numbers a row: one
// streaming pass keeps, per lane, a reference r, s = sum e^(x - r) and, for the
// entropy, t = sum e^(x - r) (x - r) (in base 2: one v_exp_f32 an element).  The
// reference is raised only where a term passes it by 2^8, so that the usual
// batch does no rescaling; floating point keeps the same relative precision
// wherever the reference lies.  The backwards are elementwise given the
// forward's row statistics.  All of them are bound by HBM where the rows fill
// the device and by latency, launch to last store, where they do not.
//
// Rows start at any element address and may be apart by more than cols: a row
// is read in 16-byte vectors from the 128-byte line that its first element lies
// in, and the elements of its first and last vector that are not its own are
// masked.
#include <float.h>

#include <type_traits>

#include "api_internal.hpp"
#include "common.hpp"
#include "logits_rules.hpp"
#include "rows.hpp"

namespace credit {
namespace {

constexpr int kThreads = 256;
constexpr int kNW = kThreads / kWave;
constexpr int kLane = 32;                     // elements of a lane in a batch
constexpr int kBatch = kThreads * kLane;      // elements of a workgroup in a batch
constexpr int kMaxEntries = kThreads;         // tokens, alternatives or teacher entries a row
constexpr uintptr_t kLine = 128;              // bytes
constexpr int64_t kMaxGridRows = int64_t{1} << 23;  // a grid's threads fit 32 bits
constexpr int64_t kMaxCols = int64_t{1} << 29;  // a row's bytes fit 32-bit offsets
constexpr float kNegInf = -__builtin_inff();
constexpr float kNaN = __builtin_nanf("");
constexpr double kLn2 = 0.693147180559945309417232;

template <class T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int kN = 4;  // elements of a 16-byte vector
  __device__ static float get(const float* p) { return *p; }
  __device__ static void put(float* p, float v) { *p = v; }
};
template <>
struct Elem<uint16_t> {
  static constexpr int kN = 8;
  __device__ static float get(const uint16_t* p) { return bf16_to_f32(*p); }
  __device__ static void put(uint16_t* p, float v) { *p = f32_to_bf16(v); }
};
template <class T>
constexpr int kN = Elem<T>::kN;
template <class T>
constexpr int kU = kLane / kN<T>;  // vectors of a lane in a batch

// A row from the start of its first 128-byte line on: element e of the frame is
// column e - head, and the row's own are those in [head, end).  Whole waves then
// read and write whole lines, wherever the row starts.  Vectors wholly before
// the row are not accessed: their offsets wrap around, past the buffer's end.
struct Frame {
  buffer_rsrc_t r;  // from the 16 bytes that hold the row's first element
  uint32_t skip;    // bytes of the frame before those
  int head, end;
};
// Of them, the loads reach those below `upto`.
template <class T>
__device__ __forceinline__ Frame frame_of(const T* row, int cols, int upto = 0x7FFFFFFF) {
  Frame f;
  const uintptr_t a = reinterpret_cast<uintptr_t>(row);
  const uint32_t in_line = static_cast<uint32_t>(a & (kLine - 1));
  f.skip = in_line & ~15u;
  f.head = static_cast<int>(in_line / sizeof(T));
  f.end = f.head + cols;
  // Whole dwords: the last one holds the row's last element.
  f.r = make_rsrc(reinterpret_cast<const void*>(a & ~uintptr_t{15}),
                  (static_cast<uint32_t>(min(f.end, upto)) * static_cast<uint32_t>(sizeof(T)) + 3u &
                   ~3u) - f.skip);
  return f;
}
__device__ __forceinline__ u32x4 load_vec(const Frame& f, int vec) {
  return buffer_load(f.r, static_cast<uint32_t>(vec) * 16u - f.skip);
}
__device__ __forceinline__ u32x4 load_vec_nt(const Frame& f, int vec) {
  return buffer_load_nt(f.r, static_cast<uint32_t>(vec) * 16u - f.skip);
}

template <class T, int N>
__device__ __forceinline__ void unpack(float (&f)[N * kN<T>], const u32x4 (&v)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t w = v[k][e];
      if constexpr (std::is_same_v<T, float>) {
        f[4 * k + e] = __builtin_bit_cast(float, w);
      } else {
        f[8 * k + 2 * e] = bf16_lo(w);
        f[8 * k + 2 * e + 1] = bf16_hi(w);
      }
    }
}
template <class T>
__device__ __forceinline__ void load_batch(u32x4 (&v)[kU<T>], const Frame& f, int b) {
#pragma unroll
  for (int k = 0; k < kU<T>; ++k)
    v[k] = load_vec_nt(f, (b * kU<T> + k) * kThreads + static_cast<int>(threadIdx.x));
}
// The lane's elements of batch b that are not the row's, bit i the i-th.
template <class T>
__device__ __forceinline__ uint32_t outside(const Frame& f, int b) {
  uint32_t drop = 0;
#pragma unroll
  for (int k = 0; k < kU<T>; ++k) {
    const int e = ((b * kU<T> + k) * kThreads + static_cast<int>(threadIdx.x)) * kN<T>;
    const int from = min(max(f.head - e, 0), kN<T>), to = min(max(f.end - e, 0), kN<T>);
    const uint32_t own = (1u << to) - (1u << from);  // from > to: nothing is own
    drop |= (to > from ? ~own & ((1u << kN<T>) - 1) : (1u << kN<T>) - 1) << (k * kN<T>);
  }
  return drop;
}
// -inf in the place of the elements that `drop` names, vector by vector where
// any lane has one.
template <class T>
__device__ __forceinline__ void hide(u32x4 (&v)[kU<T>], uint32_t drop) {
#pragma unroll
  for (int k = 0; k < kU<T>; ++k) {
    const uint32_t d = drop >> (k * kN<T>);
    if (__builtin_amdgcn_ballot_w64((d & ((1u << kN<T>) - 1)) != 0) == 0) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t w = v[k][e];
      if constexpr (std::is_same_v<T, float>) {
        w = (d >> e & 1u) != 0 ? 0xFF800000u : w;
      } else {
        w = (d >> (2 * e) & 1u) != 0 ? (w & 0xFFFF0000u) | 0xFF80u : w;
        w = (d >> (2 * e + 1) & 1u) != 0 ? (w & 0xFFFFu) | 0xFF800000u : w;
      }
      v[k][e] = w;
    }
  }
}

// ---------------------------------------------------------- streaming pass --
// s and t of the values a lane has seen, about a reference r in the exponent's
// base-2 units: s = sum 2^(z c - r), t = sum 2^(z c - r) (z c - r), c = log2(e)/T;
// mx their maximum (NaN-propagating).  One fused multiply-add makes an exponent,
// exact but for its last rounding, as long as |z c| stays below kFar; a row
// whose maximum does not (or one of lowest values alone) is streamed once more
// in the CAREFUL form, whose reference is a logit: 2^((z - r) c).
constexpr float kFar = 1048576.0f;
constexpr float kRaise = 8.0f;  // 2^8 x 2^29 columns is far from overflow
struct Lane {
  float r, s = 0.0f, t = 0.0f, mx = kNegInf;
};
template <bool CAREFUL>
__device__ __forceinline__ Lane new_lane() {
  return Lane{CAREFUL ? -FLT_MAX : -2.0f * kFar};
}

template <bool ENT, bool CAREFUL, bool CLAMP>
__device__ __forceinline__ void add_terms(float& s, float& t, const float (&z)[kLane], float r,
                                          float c) {
  float s2[2] = {0.0f, 0.0f}, t2[2] = {0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < kLane; ++i) {
    const float x = CAREFUL ? (z[i] - r) * c : __builtin_fmaf(z[i], c, -r);
    const float e = __builtin_amdgcn_exp2f(x);
    s2[i & 1] += e;
    // 2^-1000 is 0 as 2^-inf is, and 0 (-1000) is 0.
    if (ENT) t2[i & 1] = __builtin_fmaf(e, CLAMP ? __builtin_fmaxf(x, -1000.0f) : x, t2[i & 1]);
  }
  s = s2[0] + s2[1];
  t = t2[0] + t2[1];
}

// Takes a batch; vm: the maxima of the lane's vectors.  A column of -inf
// makes the plain t NaN: then, and only then, the terms are formed again with
// the exponent clamped (the clamp costs an eighth of the loop's instructions).
template <class T, bool ENT, bool CAREFUL>
__device__ __forceinline__ void absorb(Lane& a, float c, const u32x4 (&v)[kU<T>],
                                       float (&vm)[kU<T>]) {
  float z[kLane];
  unpack<T, kU<T>>(z, v);
#pragma unroll
  for (int k = 0; k < kU<T>; ++k) {
    const float* y = z + k * kN<T>;
    vm[k] = fmax_nan(y[0], y[1]);
#pragma unroll
    for (int i = 2; i < kN<T>; i += 2) vm[k] = fmax_nan(vm[k], fmax_nan(y[i], y[i + 1]));
  }
  float bm = vm[0];
#pragma unroll
  for (int k = 1; k < kU<T>; ++k) bm = fmax_nan(bm, vm[k]);
  a.mx = fmax_nan(a.mx, bm);
  const float over = CAREFUL ? (bm - a.r) * c : __builtin_fmaf(bm, c, -a.r);
  if (__builtin_amdgcn_ballot_w64(over > kRaise) != 0) {
    const float r = over > kRaise ? (CAREFUL ? bm : bm * c) : a.r;
    const float d = CAREFUL ? (a.r - r) * c : a.r - r;
    const float f = __builtin_amdgcn_exp2f(d);
    // f = 0: d may be infinite.
    if (ENT) a.t = f == 0.0f ? 0.0f : f * __builtin_fmaf(d, a.s, a.t);
    a.s *= f;
    a.r = r;
  }
  float s, t;
  add_terms<ENT, CAREFUL, CAREFUL>(s, t, z, a.r, c);
  if (ENT && !CAREFUL && __builtin_amdgcn_ballot_w64(t != t) != 0) {
    // From the packed values: what the first pass computed need not be kept.
    u32x4 w[kU<T>];
#pragma unroll
    for (int k = 0; k < kU<T>; ++k) {
      w[k] = v[k];
      __asm__ volatile("" : "+v"(w[k]));
    }
    unpack<T, kU<T>>(z, w);
    add_terms<ENT, CAREFUL, true>(s, t, z, a.r, c);
  }
  a.s += s;
  if (ENT) a.t += t;
}

// The workgroup's lanes joined, about the maximum m of them all: s = sum
// e^((z - m)/T), t the same terms times their base-2 exponents; every thread has
// the result.
struct Joined {
  float m;
  double s, t;
};
struct JoinSlots {
  float m[kNW];
  double st[2][kNW];
};
template <bool CAREFUL>
__device__ __forceinline__ Joined join_lanes(const Lane& a, float c, JoinSlots& slots) {
  Joined j;
  j.m = rows::block_max<kNW>(a.mx, slots.m);
  j.s = j.t = 0.0;
  if (a.s != 0.0f) {  // not of NaN: then s is NaN
    const float d = CAREFUL ? (a.r - j.m) * c : __builtin_fmaf(j.m, -c, a.r);
    const double f = __builtin_amdgcn_exp2f(d);
    j.s = f * a.s;
    j.t = f * (static_cast<double>(a.t) + static_cast<double>(d) * a.s);
    // A lane that is too far below the maximum to count.
    if (f == 0.0) j.t = 0.0;
  }
  if (j.m != j.m) j.s = kNaN;
  rows::block_sum2<kNW>(j.s, j.t, slots.st);
  // The maximum's own e^0 is in the sum, formed as 2^d 2^-d of two roundings.
  // Parts and segments keep this: the one with the maximum joins with a factor of 1.
  if (j.m != kNegInf && j.s < 1.0) j.s = 1.0;
  return j;
}

// Two results about their own maxima, as one (s alone).
__device__ __forceinline__ Joined merge(const Joined& a, const Joined& b, float temperature) {
  Joined j{fmax_nan(a.m, b.m), 0.0, 0.0};
  if (a.s != 0.0) j.s += a.s * ::exp((static_cast<double>(a.m) - j.m) / temperature);
  if (b.s != 0.0) j.s += b.s * ::exp((static_cast<double>(b.m) - j.m) / temperature);
  return j;
}

// Batches [b0, b1) of a row: dropped(b) names further elements of batch b to
// leave out, seen(b, vm) takes the maxima of the lane's vectors of each batch in
// order.  A batch is 32 elements a lane (16 a lane, 512 or 1024 lanes, or two
// batches ahead measured the same or slower), loaded while the one before is
// absorbed: a wave spends some 30 cycles on 64 bf16 elements (unpack, multiply-
// add, exponential at a quarter rate, add, two-input share of a maximum), two
// thirds of the time that HBM takes for them, half of that for fp32.
template <class T, bool ENT, bool CAREFUL, class Dropped, class Seen>
__device__ __forceinline__ Lane stream(const Frame& f, int b0, int b1, float c, Dropped&& dropped,
                                       Seen&& seen) {
  Lane lane = new_lane<CAREFUL>();
  u32x4 v[kU<T>];
  load_batch<T>(v, f, b0);
#pragma unroll 1
  for (int b = b0; b < b1; ++b) {
    u32x4 next[kU<T>];
    load_batch<T>(next, f, b + 1);  // past the row: zeros, no access
    uint32_t drop = dropped(b);
    if ((b == 0 && f.head != 0) || (b + 1) * kBatch > f.end) drop |= outside<T>(f, b);
    if (__builtin_amdgcn_ballot_w64(drop != 0) != 0) hide<T>(v, drop);
    float vm[kU<T>];
    absorb<T, ENT, CAREFUL>(lane, c, v, vm);
    seen(b, vm);
#pragma unroll
    for (int k = 0; k < kU<T>; ++k) v[k] = next[k];
  }
  return lane;
}
template <class T, bool ENT, class Dropped, class Seen>
__device__ __forceinline__ Joined scan(const Frame& f, int b0, int b1, float c, JoinSlots& slots,
                                       Dropped&& dropped, Seen&& seen) {
  const Joined j = join_lanes<false>(stream<T, ENT, false>(f, b0, b1, c, dropped, seen), c, slots);
  if (__builtin_fabsf(j.m * c) <= kFar || __builtin_isinf(j.m) || j.m != j.m) return j;
  __syncthreads();
  return join_lanes<true>(stream<T, ENT, true>(f, b0, b1, c, dropped, seen), c, slots);
}
// ------------------------------------------------ a row in several parts --
// Few rows leave most CUs idle on a workgroup each, and one workgroup draws a row
// at 35 GB/s (bf16).  A row is then cut into parts of whole batches; each leaves
// its result (and its units) in the workspace, and the part that finds all others
// arrived joins them and goes on as a whole row's workgroup does.  Nothing waits
// for another workgroup; the row's counter is 0 again afterwards.  Published and
// read past the L2s, as the exchange of the SPLIT kernels (common.hpp).
constexpr int kBufferPastL2 = 16;  // cache-policy operand: sc1, as device-scope loads have
constexpr int kMaxParts = kWave;  // a lane each where they are joined
constexpr int kPartValues = 4;    // m, s, t, whether a column was named twice
struct Parts {
  int n = 1, batches = 0;     // parts of a row, batches of a part
  double* values = nullptr;   // [row][part][kPartValues]
  float* units = nullptr;     // [row][batch][lane]
  uint32_t* arrived = nullptr;  // kGroupCounterStride apart
};
// Every thread, with what the workgroup has published; true for the last part.
__device__ __forceinline__ bool last_part(const Parts& p, int64_t row) {
  __shared__ int last;
  publish_wait();
  lds_barrier();
  if (threadIdx.x == 0) {
    uint32_t* arrived = p.arrived + row * kGroupCounterStride;
    last = arrive(arrived) == static_cast<uint32_t>(p.n - 1);
    if (last) counter_reset(arrived);
  }
  __syncthreads();
  return last != 0;
}
__device__ __forceinline__ void publish_part(const Parts& p, int64_t row, const Joined& j,
                                             bool repeated) {
  if (threadIdx.x != 0) return;
  double* v = p.values + (row * p.n + blockIdx.x) * kPartValues;
  publish(v, static_cast<double>(j.m));
  publish(v + 1, j.s);
  publish(v + 2, j.t);
  publish(v + 3, repeated ? 1.0 : 0.0);
}
// The lane's part of the row, read before the parts are joined.
struct PartValues {
  double m, s, t, twice;
};
__device__ __forceinline__ PartValues fetch_part(const Parts& p, int64_t row) {
  const int lane = threadIdx.x & (kWave - 1);
  // Without a branch: loads that follow need not wait for these.
  const double* v = p.values + (row * p.n + min(lane, p.n - 1)) * kPartValues;
  return PartValues{fetch(v), fetch(v + 1), fetch(v + 2), fetch(v + 3)};
}
// All parts' results joined, in every thread.
__device__ __forceinline__ Joined join_parts(const PartValues& p, int parts, float c,
                                             bool* repeated) {
  const bool mine = static_cast<int>(threadIdx.x & (kWave - 1)) < parts;
  const float m = mine ? static_cast<float>(p.m) : kNegInf;
  double s = mine ? p.s : 0.0, t = p.t;
  Joined j;
  j.m = wave_reduce(m, MaxOp{});
  if (s == 0.0) {
    t = 0.0;
  } else {
    const float d = (m - j.m) * c;
    const double f = __builtin_amdgcn_exp2f(d);
    t = f == 0.0 ? 0.0 : f * (t + static_cast<double>(d) * s);
    s *= f;
  }
  j.s = wave_reduce_sum_f64(s);
  j.t = wave_reduce_sum_f64(t);
  if (j.m != j.m) j.s = kNaN;
  *repeated = __builtin_amdgcn_ballot_w64(p.twice != 0.0) != 0;
  return j;
}

__device__ __forceinline__ uint32_t none_dropped(int) { return 0; }
constexpr auto unseen = [](int, auto&&) {};

// ------------------------------------------------------------ the largest --
// Order of the alternatives: by value, NaN above everything and -0 as 0, equal
// ones by column.  key: as unsigned, the order of the values.
__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t u = __builtin_bit_cast(uint32_t, z + 0.0f);
  const uint32_t k = (u >> 31) != 0 ? ~u : u | 0x80000000u;
  return z != z ? 0xFFFFFFFFu : k;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  if (key == 0xFFFFFFFFu) return kNaN;
  return __builtin_bit_cast(float, (key >> 31) != 0 ? key & 0x7FFFFFFFu : ~key);
}

// A unit is the 64 (bf16) or 128 (fp32) contiguous bytes that kU lanes read at
// once; its maximum goes, while the row streams by, to the one of those lanes
// whose number is the vector's: a lane leaves one unit a batch in LDS.
// Afterwards every wave finds a bound that its share of the K reaches among its
// 128 group maxima (a lane's units, even and odd batches); the least of the
// waves' bounds is one that K elements of the row reach, and not many more: of n
// elements in G groups about G ln(1/(1 - K/G)) pass the K-th largest group
// maximum (74 for K = 64 of 512).  Only units that reach the bound are read
// again (units of one lane's 32 elements, which lie in four or eight lines, took
// a third of the row's traffic at 4096 x 65536 and K = 64).  A row with fewer
// than K columns above its mask, or with many equal to the bound, gives those
// above it and then the first that equal it.  What crowds a few units otherwise
// takes write_top_any, which reads the row several times.
constexpr int kBins = 256;
constexpr int kCands = 1024;
// Group maxima that a wave takes out one by one rather than bisecting the bits of
// their bound: 64 x 131072 bf16 13.1 us against 14.4 where it takes 2 (K = 5),
// 13.9 against 14.5 at 5, 14.9 both at 8.
constexpr uint32_t kTakeOut = 6;
constexpr int kUnitList = 256;  // units that a wave lists
constexpr size_t kMaxUnitBytes = 32768;
struct TopSlots {
  uint32_t hist[kBins];
  union {
    uint16_t units[kNW][kUnitList];
    uint64_t order[kMaxEntries];  // the first candidates, once the units are read
  };
  uint32_t n, bin, above, count, crowded[2];
  uint32_t wave[kNW], bound[kNW];
};
// The lane's unit of a batch, from the maxima of its vectors: the lanes of a unit
// halve what they hold step by step, each sending its partner what that keeps.
template <int CTRL, int N>
__device__ __forceinline__ void halve(float* m, bool upper) {
#pragma unroll
  for (int k = 0; k < N / 2; ++k) {
    const float keep = upper ? m[k + N / 2] : m[k], send = upper ? m[k] : m[k + N / 2];
    m[k] = fmax_nan(keep, dpp_f32<CTRL>(send));
  }
}
template <class T>
__device__ __forceinline__ float unit_max(const float (&vm)[kU<T>]) {
  float m[kU<T>];
#pragma unroll
  for (int k = 0; k < kU<T>; ++k) m[k] = vm[k];
  // Partners lane ^ 7, ^ 2, ^ 1: those of a step hold the same vectors.
  if constexpr (kU<T> == 8) halve<kDppHalfMirror, 8>(m, (threadIdx.x & 4) != 0);
  halve<kDppXor2, 4>(m, (threadIdx.x & 2) != 0);
  halve<kDppXor1, 2>(m, (threadIdx.x & 1) != 0);
  return m[0];
}
// A candidate: its key above ~column, so that the larger is nearer the front.
// They lie where the units were.
typedef uint64_t __attribute__((address_space(3))) * CandPtr;
typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
typedef u64x2 __attribute__((address_space(3))) * Cand2Ptr;
// Units are kept in the logits' type, which holds them exactly.
__device__ __forceinline__ void put_unit(float* u, float v) { *u = v; }
__device__ __forceinline__ void put_unit(uint16_t* u, float v) {
  *u = static_cast<uint16_t>(__builtin_bit_cast(uint32_t, v) >> 16);
}

template <class T, class Fn>
__device__ __forceinline__ void each_value(const Frame& f, Fn&& fn) {
  const int vecs = (f.end + kN<T> - 1) / kN<T>;
  for (int v = threadIdx.x; v < vecs; v += kThreads) {
    const u32x4 raw[1] = {load_vec(f, v)};
    float z[kN<T>];
    unpack<T, 1>(z, raw);
#pragma unroll
    for (int i = 0; i < kN<T>; ++i) {
      const int e = v * kN<T> + i;
      if (e >= f.head && e < f.end) fn(e - f.head, key_of(z[i]));
    }
  }
}

// Sum over this lane and those below it.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  int x = static_cast<int>(v);
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast 15 to rows 1, 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast 31 to rows 2, 3
  return static_cast<uint32_t>(x);
}

// The bin that holds the `need`-th largest of the histogram (bin 0 the largest)
// and what lies above it; every thread.
__device__ __forceinline__ void find_bin(TopSlots& s, uint32_t need) {
  if (threadIdx.x < kWave) {
    const int lane = threadIdx.x;
    uint32_t h[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += h[i] = s.hist[4 * lane + i];
    uint32_t above = wave_scan(sum) - sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (above < need && above + h[i] >= need) {
        s.bin = 4 * lane + i;
        s.above = above;
        s.count = h[i];
      }
      above += h[i];
    }
  }
  __syncthreads();
}

// Keys [lo, hi] narrowed around the `need`-th largest of what each() gives
// (each(fn): fn(key) for the thread's keys; at least `need` lie in [lo, hi]):
// afterwards `above` keys lie above hi and `in` in [lo, hi], together at most
// `enough` unless lo = hi.
struct Range {
  uint32_t lo, hi, above, in;
};
template <class Each>
__device__ __forceinline__ Range narrow(TopSlots& s, uint32_t lo, uint32_t hi, uint32_t need,
                                        uint32_t enough, Each&& each) {
  Range r{lo, hi, 0, 0};
  for (;;) {
    const int bits = 32 - __builtin_clz((r.hi - r.lo) | 1u);
    const int shift = bits > 8 ? bits - 8 : 0;
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.hist[i] = 0;
    __syncthreads();
    each([&](uint32_t key) {
      if (key >= r.lo && key <= r.hi) atomicAdd(&s.hist[(r.hi - key) >> shift], 1u);
    });
    __syncthreads();
    find_bin(s, need - r.above);
    r.above += s.above;
    r.in = s.count;
    r.hi -= s.bin << shift;
    const uint32_t span = (1u << shift) - 1u;
    r.lo = r.hi - r.lo > span ? r.hi - span : r.lo;
    __syncthreads();
    if (r.above + r.in <= enough || r.lo == r.hi) return r;
  }
}

// Orders the n candidates by counting, four lanes to a candidate; put(rank, key,
// column) for the first `top`.
template <class Put>
__device__ __forceinline__ void rank_candidates(TopSlots& s, CandPtr cand, int n, int top,
                                                Put&& put) {
  const int padded = (n + 31) & ~31;  // zeros, which are larger than none
  if (static_cast<int>(threadIdx.x) < padded - n) cand[n + threadIdx.x] = 0;
  __syncthreads();
  const int quarter = threadIdx.x & 3;
#pragma unroll 1
  for (int i0 = threadIdx.x / kWave * (kWave / 4); i0 < n; i0 += kThreads / 4) {
    const int i = i0 + static_cast<int>(threadIdx.x & (kWave - 1)) / 4;
    const uint64_t mine = i < n ? cand[i] : ~uint64_t{0};
    int rank = 0;
#pragma unroll 1
    for (int j = 0; j < padded; j += 32)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const u64x2 two = *(Cand2Ptr)(cand + j + 8 * k + 2 * quarter);
        rank += (two[0] > mine) + (two[1] > mine);
      }
    rank += __builtin_amdgcn_update_dpp(0, rank, kDppXor1, 0xf, 0xf, false);
    rank += __builtin_amdgcn_update_dpp(0, rank, kDppXor2, 0xf, 0xf, false);
    if (quarter == 0 && rank < top && i < n) s.order[rank] = mine;
  }
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < min(n, top)) {
    const uint64_t c = s.order[threadIdx.x];
    put(static_cast<int>(threadIdx.x), static_cast<uint32_t>(c >> 32),
        static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(c)));
  }
}
// The first place, in a list that *n counts, for each lane's `wanted` entries:
// one atomic a wave.
__device__ __forceinline__ uint32_t places(uint32_t* n, uint32_t wanted) {
  const uint32_t upto = wave_scan(wanted);
  uint32_t base = 0;
  if ((threadIdx.x & (kWave - 1)) == kWave - 1) base = atomicAdd(n, upto);
  return __builtin_amdgcn_readlane(base, kWave - 1) + upto - wanted;
}
__device__ __forceinline__ void put_candidate(CandPtr cand, uint32_t at, uint32_t key, int col) {
  if (at < kCands)
    cand[at] = static_cast<uint64_t>(key) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(col));
}

// The first columns whose values have this key, from place `found` on up to `top`.
template <class T, class Put>
__device__ __forceinline__ void put_equal(const Frame& f, uint32_t key, int found, int top,
                                          TopSlots& s, Put&& put) {
  const int vecs = (f.end + kN<T> - 1) / kN<T>;
  for (int v0 = 0; v0 < vecs && found < top; v0 += kThreads) {
    const int v = v0 + threadIdx.x;
    const u32x4 raw[1] = {load_vec(f, v)};
    float z[kN<T>];
    unpack<T, 1>(z, raw);
    uint32_t hit = 0;
#pragma unroll
    for (int i = 0; i < kN<T>; ++i) {
      const int e = v * kN<T> + i;
      if (e >= f.head && e < f.end && key_of(z[i]) == key) hit |= 1u << i;
    }
    const uint32_t mine = __builtin_popcount(hit);
    const uint32_t incl = wave_scan(mine);
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    if (lane == kWave - 1) s.wave[wave] = incl;
    __syncthreads();
    int at = found + static_cast<int>(incl - mine), all = 0;
    for (int w = 0; w < kNW; ++w) {
      if (w < wave) at += s.wave[w];
      all += s.wave[w];
    }
    for (; hit != 0 && at < top; hit &= hit - 1, ++at)
      put(at, key, v * kN<T> + __builtin_ctz(hit) - f.head);
    found += all;
    __syncthreads();
  }
}

// The `top` largest of any row: the range that holds the last of them is
// narrowed until what is at or above it fits the candidates, or until it is a
// single value, whose first columns are then taken in order.
template <class T, class Put>
__device__ __forceinline__ void write_top_any(const Frame& f, int top, TopSlots& s, CandPtr cand,
                                              Put&& put) {
  const Range r = narrow(s, 0u, 0xFFFFFFFFu, top, kCands, [&](auto&& fn) {
    each_value<T>(f, [&](int, uint32_t key) { fn(key); });
  });
  const bool ties = r.above + r.in > kCands;
  if (threadIdx.x == 0) s.n = 0;
  __syncthreads();
  each_value<T>(f, [&](int col, uint32_t key) {
    if (ties ? key > r.hi : key >= r.lo) put_candidate(cand, atomicAdd(&s.n, 1u), key, col);
  });
  __syncthreads();
  const int n = static_cast<int>(s.n);
  rank_candidates(s, cand, n, top, put);
  if (ties) put_equal<T>(f, r.hi, n, top, s, put);
}

// The `top` largest of a row whose units (of 2^fold batches each, `groups` of
// them a lane) are known.  A row's end costs instructions, not traffic (five
// workgroups a CU come to it together): hence masks and one scan for many units,
// and vectors dealt out to whole waves.
template <class T, class Put>
__device__ __forceinline__ void write_top(const Frame& f, const T* units, CandPtr cand, int groups,
                                          int fold, int top, TopSlots& s, Put&& put) {
  const int wave = threadIdx.x / kWave;
  float g[2] = {kNegInf, kNegInf};
  // Sixteen of the lane's units at once, -inf past the last.
  const auto sixteen = [&](float (&v)[16], int u0) {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      v[j] = Elem<T>::get(units + min(u0 + j, groups - 1) * kThreads + threadIdx.x);
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = u0 + j < groups ? v[j] : kNegInf;
  };
  float kept[16];  // the first, for the list below
  sixteen(kept, 0);
#pragma unroll
  for (int j = 0; j < 16; ++j) g[j & 1] = fmax_nan(g[j & 1], kept[j]);
#pragma unroll 1
  for (int u0 = 16; u0 < groups; u0 += 16) {
    float v[16];
    sixteen(v, u0);
#pragma unroll
    for (int j = 0; j < 16; ++j) g[j & 1] = fmax_nan(g[j & 1], v[j]);
  }
  const uint32_t k0 = key_of(g[0]), k1 = key_of(g[1]);
  const auto reach = [&](uint32_t t) {
    return static_cast<uint32_t>(__builtin_popcountll(__builtin_amdgcn_ballot_w64(k0 >= t)) +
                                 __builtin_popcountll(__builtin_amdgcn_ballot_w64(k1 >= t)));
  };
  // Groups of the wave that hold anything; its share of the row's `top`.
  const uint32_t full = reach(key_of(kNegInf) + 1);
  if (threadIdx.x % kWave == 0) s.wave[wave] = full;
  if (threadIdx.x == 0) s.n = s.crowded[0] = s.crowded[1] = 0;
  __syncthreads();
  uint32_t all = 0;
  for (int w = 0; w < kNW; ++w) all += s.wave[w];
  uint32_t bound = key_of(kNegInf);  // any column reaches that
  bool above = all < static_cast<uint32_t>(top);
  if (!above) {
    const uint32_t need = full * kNW == all ? (static_cast<uint32_t>(top) + kNW - 1) / kNW
                                            : (top * full + all - 1) / all;
    const uint32_t enough = need + need / 4;
    bound = 0xFFFFFFFFu;
    if (need != 0 && need <= kTakeOut) {
      // The largest taken out until `need` are; NaN reaches what infinity does.
      float x = g[0] == g[0] ? g[0] : __builtin_inff(), y = g[1] == g[1] ? g[1] : __builtin_inff();
      float m;
      uint32_t n = 0;
      do {
        m = wave_reduce(__builtin_fmaxf(x, y), MaxOp{});
        n += static_cast<uint32_t>(__builtin_popcountll(__builtin_amdgcn_ballot_w64(x == m)) +
                                   __builtin_popcountll(__builtin_amdgcn_ballot_w64(y == m)));
        x = x == m ? kNegInf : x;
        y = y == m ? kNegInf : y;
      } while (n < need);
      bound = key_of(m);
    } else if (need != 0) {
      const float most = wave_reduce(fmax_nan(g[0], g[1]), MaxOp{});
      // The least group maximum above -inf, of those that are no NaN.
      const float few = -wave_reduce(fmax_nan(g[0] > kNegInf ? -g[0] : kNegInf,
                                              g[1] > kNegInf ? -g[1] : kNegInf), MaxOp{});
      // Bit by bit below what the largest and the least group have in common.
      const uint32_t hi = __builtin_amdgcn_readfirstlane(key_of(most));
      const uint32_t lo = __builtin_amdgcn_readfirstlane(key_of(few));
      uint32_t bit = most != most || lo > hi ? 0x80000000u
                     : lo == hi              ? 0u
                                             : 0x80000000u >> __builtin_clz(lo ^ hi);
      bound = bit == 0 ? hi : hi & ~(bit | (bit - 1));
#pragma unroll 1
      for (uint32_t n = ~0u; n > enough && bit != 0; bit >>= 1) {
        const uint32_t at = reach(bound | bit);
        n = at >= need ? at : n;
        bound |= at >= need ? bit : 0u;
      }
    }
    if (threadIdx.x % kWave == 0) s.bound[wave] = bound;
    __syncthreads();
    for (int w = 0; w < kNW; ++w) bound = s.bound[w] < bound ? s.bound[w] : bound;
    bound = __builtin_amdgcn_readfirstlane(bound);
  }
  // Values that reach the bound, or that are above it and then the first columns
  // that hold it: where a mask leaves fewer groups than `top`, and where more
  // reach it than the lists take.  key >= k is !(z < value_of(k)), of the values'
  // keys up to that of infinity.
  constexpr uint32_t kInfKey = 0xFF800000u;
  uint16_t* mine = s.units[wave];
  int listed;
  bool crowded;
  float least;
  for (;;) {
    least = value_of(bound + (above ? 1u : 0u));
    listed = 0;
    if (__builtin_amdgcn_ballot_w64(!(fmax_nan(g[0], g[1]) < least)) != 0) {
#pragma unroll 1
      for (int u0 = 0; u0 < groups; u0 += 16) {
        float v[16];
        if (u0 != 0)
          sixteen(v, u0);
        else
          for (int j = 0; j < 16; ++j) v[j] = kept[j];
        uint32_t hits = 0;
#pragma unroll
        for (int j = 0; j < 16; ++j)
          hits |= !(v[j] < least) && u0 + j < groups ? 1u << j : 0u;
        const int count = __builtin_popcount(hits);
        const int upto = static_cast<int>(wave_scan(count));
        for (int at = listed + upto - count; hits != 0; hits &= hits - 1, ++at)
          if (at < kUnitList)
            mine[at] = static_cast<uint16_t>((u0 + __builtin_ctz(hits)) * kThreads + threadIdx.x);
        listed += __builtin_amdgcn_readlane(upto, kWave - 1);
      }
    }
    if (listed > kUnitList && threadIdx.x % kWave == 0) s.crowded[above] = 1;
    // Every wave has read the units: candidates may take their place.
    __syncthreads();
    crowded = s.crowded[above] != 0;
    if (!crowded || above || bound >= kInfKey) break;
    above = true;
  }
  constexpr int kPer = kU<T> == 4 ? 2 : 3;  // vectors of a unit in a batch: 4 or 8
  static_assert(kU<T> == 1 << kPer);
  const int per = kPer + fold, vecs = listed << per;
  // The lane's vector of the listed units' i0-th and following.
  const auto vector_at = [&](int i0) {
    const int i = i0 + static_cast<int>(threadIdx.x & (kWave - 1));
    const int unit = mine[i < vecs ? i >> per : 0];
    // Vector `first % kU` of lanes first / kU kU + [0, kU), in batch b.
    const int b = (unit / kThreads << fold) + (i >> kPer & ((1 << fold) - 1));
    const int first = unit % kThreads;
    return (b * kU<T> + first % kU<T>)*kThreads + first / kU<T> * kU<T> + i % kU<T>;
  };
  int n = kCands + 1;
  while (!crowded) {
    int vec = 0, next_vec = 0;
    u32x4 raw[1] = {}, next = {};
    if (vecs != 0) next = load_vec(f, next_vec = vector_at(0));
#pragma unroll 1
    for (int i0 = 0; i0 < vecs; i0 += kWave) {
      const int i = i0 + static_cast<int>(threadIdx.x & (kWave - 1));
      raw[0] = next;
      vec = next_vec;
      if (i0 + kWave < vecs) next = load_vec(f, next_vec = vector_at(i0 + kWave));
      const int e0 = vec * kN<T>;
      float z[kN<T>];
      unpack<T, 1>(z, raw);
      uint32_t hits = 0;
#pragma unroll
      for (int e = 0; e < kN<T>; ++e) hits |= !(z[e] < least) ? 1u << e : 0u;
      // The row's own elements, of a vector that this lane has.
      const int from = min(max(f.head - e0, 0), kN<T>), to = min(max(f.end - e0, 0), kN<T>);
      hits = i < vecs && to > from ? hits & ((1u << to) - (1u << from)) : 0u;
      uint32_t at = places(&s.n, __builtin_popcount(hits));
      for (; hits != 0; hits &= hits - 1, ++at) {
        const int e = __builtin_ctz(hits);
        float x = z[0];
#pragma unroll
        for (int k = 1; k < kN<T>; ++k) x = e == k ? z[k] : x;
        put_candidate(cand, at, key_of(x), e0 + e - f.head);
      }
    }
    __syncthreads();
    n = static_cast<int>(s.n);
    if (n <= kCands || above || bound >= kInfKey) break;
    above = true;
    least = value_of(bound + 1u);
    __syncthreads();
    if (threadIdx.x == 0) s.n = 0;
    __syncthreads();
  }
  if (n > kCands) return write_top_any<T>(f, top, s, cand, put);
  rank_candidates(s, cand, n, top, put);
  if (n < top) put_equal<T>(f, bound, n, top, s, put);
}

// -------------------------------------------------------- token log-probs --
template <class T>
struct LogprobArgs {
  const T* logits;
  int64_t ld;
  const int64_t* tokens;
  float* logp;
  float* stats;
  float* entropy;
  float* top_logp;
  int64_t* top_ids;
  int64_t first = 0;  // row of the launch's first workgroup
  int cols, n_tokens, n_top;
  int fold;      // a unit has 2^fold batches
  float c;       // log2(e) / temperature
  double inv_t;
  Parts parts;
};

// ln s of s >= 1 to 4e-8: the exponent's part in 64 bits, that of a mantissa in
// [1/sqrt 2, sqrt 2) by logf.
__device__ __forceinline__ double ln_sum(double s) {
  int e;
  double m = ::frexp(s, &e);
  if (m < 0.70710678118654752) m *= 2.0, e -= 1;
  return e * kLn2 + static_cast<double>(::logf(static_cast<float>(m)));
}

// The row's units from all parts, in LDS, four lanes' to a load.  They come from
// past the L2: 16 batches take 4000 cycles, as many as one does.
template <class T>
__device__ __forceinline__ void fetch_units(const Parts& p, int64_t row, int batches, int groups,
                                            int fold, T* units) {
  const int lanes = threadIdx.x % kWave * 4;
  const size_t all = static_cast<size_t>(p.n) * p.batches * kThreads;
  const buffer_rsrc_t r = make_rsrc(p.units + row * all, static_cast<uint32_t>(all * 4));
#pragma unroll 4
  for (int g = threadIdx.x / kWave; g < groups; g += kNW) {
    float unit[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
    for (int b = g << fold; b < min((g + 1) << fold, batches); ++b) {
      const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(r, (b * kThreads + lanes) * 4, 0,
                                                            kBufferPastL2);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = v[i];
        unit[i] = fmax_nan(unit[i], __builtin_bit_cast(float, w));
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) put_unit(units + g * kThreads + lanes + i, unit[i]);
  }
  __syncthreads();
}

// One read of the logits.  512 x 262144 fp32 with the entropy 77.8 us, 6.90 TB/s
// (a kernel that reads alone reaches 7.08); 2048 x 131072 bf16 83 us without
// alternatives (6.5 TB/s) and 93 with 64 (5.80): the workgroups that a CU holds
// reach their rows' ends together, where a row's choice of alternatives, some
// 9000 cycles of latency, has no loads to hide it.  64 x 131072 in four parts
// each, K = 20: 13.4 us, of which the stream 4, the parts' meeting and the units
// from past the L2 2.5, the choice 3.5.
template <class T, bool ENT, bool TOP, bool SPLIT>
__global__ __launch_bounds__(kThreads) void token_logprob_fwd_kernel(LogprobArgs<T> a) {
  extern __shared__ __attribute__((aligned(16))) char dynamic_lds[];
  __shared__ JoinSlots join;
  T* units = reinterpret_cast<T*>(dynamic_lds);
  const int64_t row = SPLIT ? blockIdx.y : a.first + blockIdx.x;
  const T* z = a.logits + row * a.ld;
  // The thread's token, read ahead of the row.
  int64_t token = -1;
  float chosen = kNaN;  // a token >= cols
  if (static_cast<int>(threadIdx.x) < a.n_tokens) {
    token = a.tokens[row * a.n_tokens + threadIdx.x];
    if (token >= 0 && token < a.cols) chosen = Elem<T>::get(z + token);
  }
  const Frame f = frame_of(z, a.cols);
  const int batches = (f.end + kBatch - 1) / kBatch;
  const int groups = (batches + (1 << a.fold) - 1) >> a.fold;
  Joined j;
  if constexpr (SPLIT) {
    const int b0 = blockIdx.x * a.parts.batches, b1 = min(b0 + a.parts.batches, batches);
    const Frame own = frame_of(z, a.cols, b1 * kBatch);  // the next part's batch is not read ahead
    float* out = a.parts.units + (row * a.parts.n * a.parts.batches) * kThreads + threadIdx.x;
    j = scan<T, ENT>(own, b0, b1, a.c, join, none_dropped, [&](int b, const float (&vm)[kU<T>]) {
      if constexpr (TOP) publish(out + b * kThreads, unit_max<T>(vm));
    });
    publish_part(a.parts, row, j, false);
    if (!last_part(a.parts, row)) return;
    const PartValues values = fetch_part(a.parts, row);
    if constexpr (TOP) fetch_units<T>(a.parts, row, batches, groups, a.fold, units);
    bool unused;
    j = join_parts(values, a.parts.n, a.c, &unused);
  } else {
    float unit = kNegInf;
    j = scan<T, ENT>(f, 0, batches, a.c, join, none_dropped, [&](int b, const float (&vm)[kU<T>]) {
      if constexpr (TOP) {
        if ((b & ((1 << a.fold) - 1)) == 0) unit = kNegInf;
        unit = fmax_nan(unit, unit_max<T>(vm));
        put_unit(units + (b >> a.fold) * kThreads + threadIdx.x, unit);
      }
    });
  }
  __shared__ double shared_ln_s;
  if (threadIdx.x < kWave) {
    const bool empty = j.m == kNegInf;
    const double ln_s = empty ? 0.0 : j.s == j.s ? ln_sum(j.s) : j.s;
    if (threadIdx.x == 0) {
      shared_ln_s = ln_s;
      a.stats[2 * row] = j.m;
      a.stats[2 * row + 1] = static_cast<float>(j.s);
      if (ENT) {
        const float h = empty ? 0.0f : static_cast<float>(ln_s - kLn2 * j.t / j.s);
        a.entropy[row] = h < 0.0f ? 0.0f : h;  // NaN stays
      }
    }
  }
  const auto log_p = [&](float v) {
    const double ln_s = shared_ln_s;
    return v == kNegInf && ln_s == ln_s
               ? kNegInf
               : static_cast<float>((static_cast<double>(v) - j.m) * a.inv_t - ln_s);
  };
  if constexpr (TOP) {
    __shared__ TopSlots top;
    write_top<T>(f, units, (CandPtr)(dynamic_lds), groups, a.fold, a.n_top, top,
                 [&](int rank, uint32_t key, int col) {
                   a.top_logp[row * a.n_top + rank] = log_p(value_of(key));
                   a.top_ids[row * a.n_top + rank] = col;
                 });
  } else {
    __syncthreads();
  }
  if (static_cast<int>(threadIdx.x) < a.n_tokens)
    a.logp[row * a.n_tokens + threadIdx.x] = token < 0 ? 0.0f : log_p(chosen);
}

// ------------------------------------------------------------- gradients --
// A workgroup writes kGradVecs vectors a lane of a row's gradient, in place too: a
// lane writes what it has read.  The entries that a row names (its tokens, the
// teacher's columns) get their own value in the registers of the lane that holds
// them (patched in memory afterwards, 2048 x 131072 bf16 with 64 entries took
// 173.6 us instead of 169.8, 8192 x 32768 with 256 260 instead of 176).
constexpr int kGradVecs = 4;
template <class T>
constexpr int kGradBatch = kThreads * kGradVecs * kN<T>;

// Stores the row's own elements of a vector; VEC: in and out lie alike in their
// 16-byte lines.
template <class T, bool VEC>
__device__ __forceinline__ void store_grad(T* row, const Frame& f, int e, const float (&g)[kN<T>]) {
  if (VEC && e >= f.head && e + kN<T> <= f.end) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same_v<T, float>)
        v[i] = __builtin_bit_cast(uint32_t, g[i]);
      else
        v[i] = pack_bf16x2(g[2 * i], g[2 * i + 1]);
    }
    store_nt(reinterpret_cast<u32x4*>(row + (e - f.head)), v);
  } else {
#pragma unroll
    for (int i = 0; i < kN<T>; ++i)
      if (e + i >= f.head && e + i < f.end) Elem<T>::put(row + (e + i - f.head), g[i]);
  }
}

// The workgroup's part of a row, and value(z) over it (0 where `zero`); own(column,
// z) of the lane's elements that `named` has a bit for.
template <class T>
__device__ __forceinline__ void load_part(u32x4 (&v)[kGradVecs], const Frame& f, int part) {
#pragma unroll
  for (int k = 0; k < kGradVecs; ++k)
    v[k] = load_vec_nt(f, (part * kGradVecs + k) * kThreads + static_cast<int>(threadIdx.x));
}
template <class T, bool VEC, class Fn, class Own>
__device__ __forceinline__ void write_part(const u32x4 (&v)[kGradVecs], const Frame& f, T* out,
                                           int part, bool zero, uint32_t named, Fn&& value,
                                           Own&& own) {
#pragma unroll
  for (int k = 0; k < kGradVecs; ++k) {
    const u32x4 raw[1] = {v[k]};
    float z[kN<T>], g[kN<T>];
    unpack<T, 1>(z, raw);
#pragma unroll
    for (int i = 0; i < kN<T>; ++i) g[i] = zero ? 0.0f : value(z[i]);
    const int e = ((part * kGradVecs + k) * kThreads + static_cast<int>(threadIdx.x)) * kN<T>;
    for (uint32_t d = named >> (k * kN<T>) & ((1u << kN<T>) - 1); d != 0; d &= d - 1) {
      const int at = __builtin_ctz(d);
      float x = z[0];
#pragma unroll
      for (int i = 1; i < kN<T>; ++i) x = at == i ? z[i] : x;
      x = own(e + at - f.head, x);
#pragma unroll
      for (int i = 0; i < kN<T>; ++i) g[i] = at == i ? x : g[i];
    }
    store_grad<T, VEC>(out, f, e, g);
  }
}

template <class T>
struct LogprobGradArgs {
  const T* logits;
  int64_t ld;
  const int64_t* tokens;
  const float* stats;
  const float* entropy;
  const float* dlogp;
  const float* dentropy;
  T* dlogits;
  int64_t ldd;
  int64_t rows;
  int cols, n_tokens;
  float inv_t, c;
};

// One read, one write; a workgroup's part is four vectors a lane, all loaded
// before the first is used.
// 2048 x 131072 bf16 with the entropy's gradient 173.2 us, 6.20 TB/s (a kernel
// that reads and writes as much and does nothing else reaches 6.37).
template <class T, bool ENT, bool VEC>
__global__ __launch_bounds__(kThreads) void token_logprob_bwd_kernel(LogprobGradArgs<T> a) {
  const int lane = threadIdx.x & (kWave - 1);
  const int part = blockIdx.x;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const T* z = a.logits + row * a.ld;
    T* out = a.dlogits + row * a.ldd;
    const Frame f = frame_of(z, a.cols);
    const int first = part * kGradBatch<T> - f.head;  // the part's first column
    if (first >= a.cols) continue;
    const int64_t* tokens = a.tokens + row * a.n_tokens;
    const float* dlogp = a.dlogp + row * a.n_tokens;
    // Every wave by itself: the tokens' weight, and the lane's elements that they name.
    double weight = 0.0;
    bool live = false;
    uint32_t named = 0;
    for (int k0 = 0; k0 < a.n_tokens; k0 += kWave) {
      const int k = k0 + lane;
      const int64_t tok = k < a.n_tokens ? tokens[k] : -1;
      const float g = k < a.n_tokens ? dlogp[k] : 0.0f;
      const bool counts = tok >= 0 && g != 0.0f;
      live |= counts;
      if (counts) weight += tok >= a.cols ? kNaN : g;
      const int64_t e = tok - first;
      uint64_t here = __builtin_amdgcn_ballot_w64(counts && tok < a.cols && e >= 0 &&
                                                  e < kGradBatch<T>);
      for (; here != 0; here &= here - 1) {
        const int at = __builtin_amdgcn_readlane(static_cast<int>(e), __builtin_ctzll(here));
        const int vec = at / kN<T>;
        if (vec % kThreads == static_cast<int>(threadIdx.x))
          named |= 1u << (vec / kThreads * kN<T> + at % kN<T>);
      }
    }
    const float gsum = static_cast<float>(wave_reduce_sum_f64(weight));
    live = __builtin_amdgcn_ballot_w64(live) != 0;
    const float m = a.stats[2 * row], s = a.stats[2 * row + 1];
    const float h = ENT ? a.dentropy[row] : 0.0f;
    // dz = e^(x - m/T) (A + B log2 e^(x - m/T)).
    const float k = a.inv_t / s;
    float A = gsum, B = 0.0f;
    if (ENT && h != 0.0f) {
      live = true;
      A += h * (a.entropy[row] - ::logf(s));
      B = -h * static_cast<float>(kLn2) * k;
    }
    A *= -k;
    const bool zero = !live || m == kNegInf;
    const auto value = [&](float v) {
      const float x = (v - m) * a.c;
      const float e = __builtin_amdgcn_exp2f(x);
      return ENT ? e * __builtin_fmaf(B, __builtin_fmaxf(x, -1000.0f), A) : e * A;
    };
    u32x4 v[kGradVecs] = {};
    if (!zero) load_part<T>(v, f, part);
    if (zero) named = 0;
    write_part<T, VEC>(v, f, out, part, zero, named, value, [&](int col, float x) {
      double g = 0.0;
      for (int j = 0; j < a.n_tokens; ++j)
        if (tokens[j] == col) g += dlogp[j];
      return static_cast<float>(g) * a.inv_t + value(x);
    });
  }
}

// ------------------------------------------------------------ distillation --
// Columns of the frame that a row's entries name, a bit each, for the batches
// of one segment: bit i of word (b, lane) is the lane's i-th element of batch b.
constexpr int kSegBatches = 16;
constexpr int kSegWords = kSegBatches * kThreads;

template <class T>
struct DistillArgs {
  const T* logits;
  int64_t ld;
  const int64_t* ids;
  const float* teacher;
  float* loss;
  float* stats;
  int64_t first = 0;  // row of the launch's first workgroup
  int cols, n_top;
  float temperature, c;
  Parts parts;
};
// Row statistics [rows, 8] for the backward, which takes the teacher's softmax
// about its maximum and leaves the log-sum to the caller.
enum DistillStat { kMax, kSum, kTailMax, kTailSum, kMass, kTailGrad, kTeacherLse, kUnused };

// Marks element e of the frame if it lies in batches [b0, b1); whether it was
// marked before.
template <class T>
__device__ __forceinline__ bool mark(uint32_t* bits, int e, int b0, int b1) {
  const int v = e / kN<T>;
  const int b = v / (kThreads * kU<T>);
  if (b < b0 || b >= b1) return false;
  const uint32_t bit = 1u << (v / kThreads % kU<T> * kN<T> + e % kN<T>);
  return (atomicOr(&bits[(b - b0) * kThreads + v % kThreads], bit) & bit) != 0;
}

// The tail is summed directly, over the columns that no entry names (1 - sum p of
// the named ones would lose it where it is small): their bits are marked in LDS
// for 16 batches at a time.  2048 x 131072 bf16, K = 64, tail 87.6 us, 6.15 TB/s;
// without it the same; 8192 x 32768 108 us against 85: 64 named columns in four
// batches leave hardly a wave's batch without one to mask.
// Rows whose entries repeat a column, found by their marks, sum its entries
// before q ln q: with a repeat in every row 90.6 us without the tail, 90.9 with
// it; 16 x 262144 fp32, K = 256 11.5 against 8.3.
template <class T, bool TAIL, bool SPLIT>
__global__ __launch_bounds__(kThreads) void topk_distill_fwd_kernel(DistillArgs<T> a) {
  __shared__ JoinSlots join;
  __shared__ float max_slots[2][kNW];
  __shared__ double sum_slots[4][kNW];
  __shared__ int flags[kNW];
  __shared__ int repeated;
  // Marks of the columns that entries name: with the tail a segment's, without it
  // all of the row's by their number modulo 2^17 (of 64 entries in 2^18 columns
  // two that differ may meet in one row of 130, which is then looked at for
  // nothing).
  __shared__ __attribute__((aligned(16))) uint32_t bits[kSegWords];
  const int64_t row = SPLIT ? blockIdx.y : a.first + blockIdx.x;
  const T* z = a.logits + row * a.ld;
  const int k = threadIdx.x;
  if constexpr (!TAIL)
    for (int i = threadIdx.x; i < kSegWords / 4; i += kThreads)
      reinterpret_cast<u32x4*>(bits)[i] = u32x4{0, 0, 0, 0};
  // The thread's entry.
  int64_t id = -1;
  float t = kNegInf;
  if (k < a.n_top) {
    id = a.ids[row * a.n_top + k];
    t = a.teacher[row * a.n_top + k];
  }
  const bool bad = id >= a.cols;
  const bool live = id >= 0 && !bad;
  const uint64_t any_live = __builtin_amdgcn_ballot_w64(live);
  const uint64_t any_bad = __builtin_amdgcn_ballot_w64(bad);
  if ((threadIdx.x & (kWave - 1)) == 0)
    flags[threadIdx.x / kWave] = (any_live != 0) | (any_bad != 0) << 1;
  if (threadIdx.x == 0) repeated = 0;
  const float tm = rows::block_max<kNW>(id >= 0 ? t : kNegInf, max_slots[0]);
  int flag = 0;
  for (int w = 0; w < kNW; ++w) flag |= flags[w];
  float* stats = a.stats + 8 * row;
  if (flag == 0 || (!TAIL && tm == kNegInf)) {  // no entry to learn from
    if (SPLIT && blockIdx.x != 0) return;
    if (threadIdx.x == 0) a.loss[row] = 0.0f;
    if (threadIdx.x < 8) stats[threadIdx.x] = 0.0f;
    return;
  }
  const float zk = live ? Elem<T>::get(z + id) : kNegInf;

  const Frame f = frame_of(z, a.cols);
  const int batches = (f.end + kBatch - 1) / kBatch;
  const int first_batch = SPLIT ? blockIdx.x * a.parts.batches : 0;
  const int end_batch = SPLIT ? min(first_batch + a.parts.batches, batches) : batches;
  const Frame own = SPLIT ? frame_of(z, a.cols, end_batch * kBatch) : f;
  Joined j{kNegInf, 0.0, 0.0};  // of a part without batches
  if constexpr (TAIL) {
    // The segments' results joined as the lanes' are.
    for (int b0 = first_batch; b0 < end_batch; b0 += kSegBatches) {
      const int b1 = min(b0 + kSegBatches, end_batch);
      if (b0 != first_batch) __syncthreads();
      for (int b = 0; b < b1 - b0; ++b) bits[b * kThreads + threadIdx.x] = 0;
      __syncthreads();
      if (live && mark<T>(bits, static_cast<int>(id) + f.head, b0, b1)) repeated = 1;
      __syncthreads();
      const Joined p = scan<T, false>(
          own, b0, b1, a.c, join, [&](int b) { return bits[(b - b0) * kThreads + threadIdx.x]; },
          unseen);
      j = b0 == first_batch ? p : merge(j, p, a.temperature);
    }
  } else {
    uint32_t met = 0;
    if (live) {
      const uint32_t at = static_cast<uint32_t>(id) % (32u * kSegWords), bit = 1u << (at & 31u);
      met = atomicOr(&bits[at / 32u], bit) & bit;
    }
    // Looked at once the row's first loads are under way.
    j = scan<T, false>(own, first_batch, end_batch, a.c, join, none_dropped, [&](int b, auto&&) {
      if (b == first_batch && met != 0) repeated = 1;
    });
  }
  bool twice = repeated != 0;
  if constexpr (SPLIT) {
    j.t = 0.0;
    publish_part(a.parts, row, j, twice);
    if (!last_part(a.parts, row)) return;
    j = join_parts(fetch_part(a.parts, row), a.parts.n, a.c, &twice);
  }
  // Over the entries, in one go: the mass that the row has outside the tail,
  // and with w = q (tail) or q times its normalisation, W a column's sum of w:
  // w, W ln W once a column, w ln(p S).
  const float m = TAIL ? fmax_nan(j.m, rows::block_max<kNW>(zk, max_slots[1])) : j.m;
  double w = 0.0, ln_w = 0.0;
  if (live) {
    ln_w = TAIL ? static_cast<double>(t) : (static_cast<double>(t) - tm) / a.temperature;
    w = ::exp(ln_w);
  }
  bool first = live;  // of the entries that name one column: the lowest stands for it
  double all = w;     // W
  if (twice) {
    // The marks are done with.
    int* ids = reinterpret_cast<int*>(bits);
    double* ws = reinterpret_cast<double*>(bits + kMaxEntries);
    static_assert(3 * kMaxEntries <= kSegWords && kMaxEntries % 32 == 0);
    ids[k] = live ? static_cast<int>(id) : -1;
    ws[k] = w;
    __syncthreads();
    bool shared = false;
    for (int i0 = 0; i0 < a.n_top; i0 += 32) {
      u32x4 four[8];
#pragma unroll
      for (int v = 0; v < 8; ++v) four[v] = reinterpret_cast<const u32x4*>(ids + i0)[v];
      uint32_t same = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i)
        same |= four[i / 4][i % 4] == static_cast<uint32_t>(id) ? 1u << i : 0u;
      if (k / 32 == i0 / 32) same &= ~(1u << k % 32);
      if (same == 0) continue;
      shared = true;
      first = first && i0 + __builtin_ctz(same) > k;
      for (; same != 0; same &= same - 1) all += ws[i0 + __builtin_ctz(same)];
    }
    if (first && shared) ln_w = ::log(all);
  }
  double sums[4] = {0.0, 0.0, 0.0, 0.0};
  if (live) {
    const double x = zk == kNegInf && m == m && m != __builtin_inff()
                         ? static_cast<double>(kNegInf)
                         : (static_cast<double>(zk) - m) / a.temperature;
    if (TAIL && first && zk != kNegInf) sums[0] = ::exp(x);
    sums[1] = w;
    if (first && all != 0.0) sums[2] = all * ln_w;
    if (w != 0.0) sums[3] = w * x;
  }
  block_reduce_sum_f64_multi<kNW, 4>(sums, sum_slots);
  if (threadIdx.x >= kWave) return;
  double s = j.s;
  if (TAIL) {
    s = sums[0];
    if (j.s != 0.0) s += j.s * ::exp((static_cast<double>(j.m) - m) / a.temperature);
  }
  const double ln_s = m == kNegInf ? 0.0 : ::log(s);
  double q = sums[1], loss, rest = 0.0, tail_grad = 0.0, lse = 0.0;
  if constexpr (TAIL) {
    loss = sums[2] - sums[3] + q * ln_s;
    rest = q < 1.0 ? 1.0 - q : (q == q ? 0.0 : q);
    double share = 0.0;
    // Without mass outside the entries (all of it masked) nothing is held against
    // them: neither the loss nor its gradient has that term.
    if (j.s == 0.0) {
      rest = 0.0;
    } else {
      const double ln_tail = (static_cast<double>(j.m) - m) / a.temperature + ::log(j.s) - ln_s;
      share = ::exp(ln_tail);
      if (rest != 0.0) loss += rest * (::log(rest) - ln_tail);
    }
    tail_grad = (q + rest) * share - rest;
  } else {
    const double ln_w = ::log(q);
    loss = (sums[2] - sums[3]) / q - ln_w + ln_s;
    lse = static_cast<double>(tm) / a.temperature + ln_w;
    q = q == q ? 1.0 : q;
  }
  if ((flag & 2) != 0) loss = q = tail_grad = kNaN;
  if (threadIdx.x == 0) {
    a.loss[row] = static_cast<float>(loss);
    stats[kMax] = m;
    stats[kSum] = static_cast<float>(s);
    stats[kTailMax] = TAIL ? j.m : 0.0f;
    stats[kTailSum] = TAIL ? static_cast<float>(j.s) : 0.0f;
    stats[kMass] = static_cast<float>(q + rest);
    stats[kTailGrad] = static_cast<float>(tail_grad);
    stats[kTeacherLse] = static_cast<float>(lse);
    stats[kUnused] = 0.0f;
  }
}

template <class T>
struct DistillGradArgs {
  const T* logits;
  int64_t ld;
  const int64_t* ids;
  const float* teacher;
  const float* stats;
  const float* dloss;
  T* dlogits;
  int64_t ldd;
  int64_t rows;
  int cols, n_top;
  float temperature, c;
};

// One read, one write, as token_logprob_bwd_kernel: 2048 x 131072 bf16, K = 64
// 171.9 us, 6.25 TB/s; 512 x 262144 fp32, K = 128, tail 172.0.
template <class T, bool TAIL, bool VEC>
__global__ __launch_bounds__(kThreads) void topk_distill_bwd_kernel(DistillGradArgs<T> a) {
  // The entries whose columns lie in this part, in their order; a bit for each of a
  // lane's elements that one names, and which; whether two name the same.
  __shared__ int here_col[kMaxEntries];
  __shared__ float here_q[kMaxEntries];
  __shared__ uint32_t here_bits[kThreads];
  __shared__ uint8_t here_at[kGradBatch<T>];
  __shared__ int here_n[kNW], here_twice;
  __shared__ float teacher_max[kNW], teacher_sum[kNW];
  const int lane = threadIdx.x & (kWave - 1);
  const int part = blockIdx.x;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const T* z = a.logits + row * a.ld;
    T* out = a.dlogits + row * a.ldd;
    const Frame f = frame_of(z, a.cols);
    const int first = part * kGradBatch<T> - f.head;
    if (first >= a.cols) continue;
    const float* st = a.stats + 8 * row;
    const float m = st[kMax], s = st[kSum], mass = st[kMass];
    const float g = a.dloss[row] / a.temperature;
    // S = 0: a row without entries, or of -inf alone.
    const bool zero = s == 0.0f || g == 0.0f || mass == 0.0f;
    u32x4 v[kGradVecs] = {};
    int n = 0;
    uint32_t named = 0;
    if (!zero) {
      // A thread an entry; all of the row's loads are in flight together.
      const int k = threadIdx.x, wave = k / kWave;
      int64_t id = -1;
      float t = 0.0f;
      if (k < a.n_top) {
        id = a.ids[row * a.n_top + k];
        t = a.teacher[row * a.n_top + k];
      }
      load_part<T>(v, f, part);
      const bool here = id >= 0 && id < a.cols && id >= first && id - first < kGradBatch<T>;
      const uint64_t mask = __builtin_amdgcn_ballot_w64(here);
      const bool live = id >= 0 && id < a.cols;
      const float most = TAIL ? 0.0f : wave_reduce(live ? t : kNegInf, MaxOp{});
      if (lane == 0) here_n[wave] = __builtin_popcountll(mask), teacher_max[wave] = most;
      here_bits[k] = 0;
      if (k == 0) here_twice = 0;
      lds_barrier();
      int at = __builtin_popcountll(mask & ((uint64_t{1} << lane) - 1));
      for (int w = 0; w < kNW; ++w) {
        at += w < wave ? here_n[w] : 0;
        n += here_n[w];
      }
      // q about the teacher's maximum, as the forward has it: the log-sum of logits
      // near 20 is off by 10^-6 in fp32, and with it every q formed from that.
      float q = 0.0f;
      if (n != 0 && live) {
        float tm = kNegInf;
        if (!TAIL)
          for (int w = 0; w < kNW; ++w) tm = fmax_nan(tm, teacher_max[w]);
        q = exp_accurate(TAIL ? t : (t - tm) / a.temperature);
      }
      if (!TAIL && n != 0) {
        const float sum = wave_reduce(q, SumOp{});
        if (lane == 0) teacher_sum[wave] = sum;
      }
      if (here) {
        here_col[at] = static_cast<int>(id);
        here_q[at] = q;
        const int e = static_cast<int>(id) - first, vec = e / kN<T>;
        const uint32_t bit = 1u << (vec / kThreads * kN<T> + e % kN<T>);
        here_at[e] = static_cast<uint8_t>(at);
        if ((atomicOr(&here_bits[vec % kThreads], bit) & bit) != 0) here_twice = 1;
      }
      if (n != 0) {
        lds_barrier();
        named = here_bits[k];
      }
    }
    float ref = m, A = g * mass / s;
    if (TAIL) {
      const bool some = st[kTailSum] != 0.0f;  // else every column is named or without mass
      ref = some ? st[kTailMax] : m;
      A = some ? g * st[kTailGrad] / st[kTailSum] : g * st[kTailGrad];
    }
    write_part<T, VEC>(
        v, f, out, part, zero, named,
        [&](float x) { return __builtin_amdgcn_exp2f((x - ref) * a.c) * A; },
        [&](int col, float x) {
          float q = 0.0f;
          if (here_twice == 0)
            q = here_q[here_at[col - first]];
          else
            for (int j = 0; j < n; ++j) q += here_col[j] == col ? here_q[j] : 0.0f;
          if (!TAIL) {
            float sum = 0.0f;
            for (int w = 0; w < kNW; ++w) sum += teacher_sum[w];
            q /= sum;
          }
          return g * (mass * exp_accurate((x - m) / a.temperature) / s - q);
        });
    if (row + gridDim.y < a.rows) lds_barrier();  // before the next row's list
  }
}

// ---------------------------------------------------------------- host ----
using logits::kMaxSplitRows;
using logits::part_values_bytes;
using logits::parts_bytes;
static_assert(kMaxSplitRows <= kMaxGroupsPerLaunch);
static_assert(logits::kMaxParts == kMaxParts && logits::kPartValues == kPartValues &&
              logits::kBatch == kBatch && logits::kThreads == kThreads);
// Batches of the widest frame that a row of this alignment has.
template <class T>
int64_t row_batches(const T* logits, int64_t ld, int64_t rows, int64_t cols, int batch = kBatch) {
  const bool lines = reinterpret_cast<uintptr_t>(logits) % kLine == 0 &&
                     (rows == 1 || ld * static_cast<int64_t>(sizeof(T)) % kLine == 0);
  const int64_t head = lines ? 0 : kLine / sizeof(T) - 1;
  return (cols + head + batch - 1) / batch;
}
int check_logits(const void* p, const char* name, int64_t ld, int64_t rows, int64_t cols,
                 size_t elem) {
  CREDIT_TRY(check_row_ptr(p, name, rows));
  CREDIT_TRY(check_aligned(p, elem, name));
  if (rows > 1 && ld < cols)
    return set_error(CREDIT_ERR_BAD_SHAPE, "%s: rows of %lld columns are %lld elements apart",
                     name, static_cast<long long>(cols), static_cast<long long>(ld));
  if (rows > 1 && ld > (int64_t{1} << 62) / (rows * 4))
    return set_error(CREDIT_ERR_BAD_SHAPE, "%s: %lld rows %lld elements apart", name,
                     static_cast<long long>(rows), static_cast<long long>(ld));
  return CREDIT_OK;
}
// An operand with something for every row, its elements at their own alignment.
int check_operand(const void* p, const char* name, int64_t rows, size_t elem) {
  CREDIT_TRY(check_row_ptr(p, name, rows));
  return check_aligned(p, elem, name);
}
int check_entries(int32_t n, int32_t least, int64_t most, const char* what) {
  if (n < least || n > most)
    return set_error(CREDIT_ERR_BAD_SHAPE, "%d %s a row: need %d to %lld", n, what, least,
                     static_cast<long long>(most));
  return CREDIT_OK;
}
int check_temperature(float t) {
  if (!(t >= 1e-4f && t <= 1e4f))
    return set_error(CREDIT_ERR_BAD_CONFIG, "temperature %g outside [1e-4, 1e4]",
                     static_cast<double>(t));
  return CREDIT_OK;
}
int check_variant(const credit_cfg* cfg, bool forward) {
  CREDIT_TRY(check_cfg(cfg));
  const int v = cfg_variant(cfg);
  if (v == CREDIT_VARIANT_STAGED || (v == CREDIT_VARIANT_SPLIT && !forward))
    return set_error(CREDIT_ERR_UNSUPPORTED, "this logits operator has no variant %d", v);
  return CREDIT_OK;
}

// Parts of a row that the call takes (parts->n 1: one workgroup a row), with
// their workspace.  `units`: also the units'.
int plan_parts(const credit_cfg* cfg, int64_t rows, int64_t batches, bool units, Parts* parts) {
  const int variant = cfg_variant(cfg);
  const int64_t want = variant == CREDIT_VARIANT_READ ? 1
                       : variant == CREDIT_VARIANT_SPLIT && cfg_split(cfg) > 0
                           ? cfg_split(cfg)
                           : logits::auto_parts(rows, batches, units);
  const int64_t each = (batches + want - 1) / want;
  const int64_t n = (batches + each - 1) / each;
  if (n < 2 || rows > kMaxSplitRows) return CREDIT_OK;
  if (cfg == nullptr || cfg->workspace == nullptr) {
    // A graph replays on any stream, beside the eager calls of the one it was
    // captured on: it may not share that one's workspace.
    if (!keeps_scratch(cfg_stream(cfg))) {
      if (variant == CREDIT_VARIANT_SPLIT)
        return set_error(CREDIT_ERR_WORKSPACE,
                         "SPLIT under capture or on the per-thread stream needs cfg->workspace");
      return CREDIT_OK;
    }
  }
  char* base = nullptr;
  CREDIT_TRY(acquire_workspace(cfg, parts_bytes(rows, n, each, units), &base));
  parts->n = static_cast<int>(n);
  parts->batches = static_cast<int>(each);
  parts->values = reinterpret_cast<double*>(ws_scratch(base));
  parts->units = reinterpret_cast<float*>(ws_scratch(base) + part_values_bytes(rows, n));
  parts->arrived = ws_counters(base) + kGroupCounterBase;
  return CREDIT_OK;
}
float log2e_over(float temperature) {
  return static_cast<float>(1.44269504088896340736 / static_cast<double>(temperature));
}
// Whether rows of in and out lie alike in their 16-byte lines.
bool alike(const void* in, int64_t ld, const void* out, int64_t ldd, int64_t rows, size_t elem) {
  const uintptr_t d = reinterpret_cast<uintptr_t>(in) - reinterpret_cast<uintptr_t>(out);
  return d % 16 == 0 && (rows == 1 || (ld - ldd) * static_cast<int64_t>(elem) % 16 == 0);
}
int check_overlap(const void* in, int64_t ld, const void* out, int64_t ldd, int64_t rows,
                  int64_t cols, size_t elem) {
  if (logits::may_share(reinterpret_cast<uintptr_t>(in), ld, reinterpret_cast<uintptr_t>(out), ldd,
                        rows, cols, elem))
    return CREDIT_OK;
  return set_error(CREDIT_ERR_BAD_CONFIG, "dlogits overlaps logits without being it");
}
template <class T>
dim3 grad_grid(const T* logits, int64_t ld, int64_t rows, int64_t cols) {
  const int64_t parts = row_batches(logits, ld, rows, cols, kGradBatch<T>);
  return dim3(static_cast<unsigned>(parts), static_cast<unsigned>(rows < 65535 ? rows : 65535));
}

// A workgroup a row, or a part of one (of at most kMaxSplitRows rows).
dim3 forward_grid(const Parts& parts, int64_t rows) {
  if (parts.n > 1) return dim3(parts.n, static_cast<unsigned>(rows));
  return dim3(static_cast<unsigned>(rows < kMaxGridRows ? rows : kMaxGridRows));
}

// fn(bool_constant...) for the values of `flags`.
template <class Fn, class... Flags>
void choose(Fn&& fn, bool flag, Flags... flags) {
  if constexpr (sizeof...(flags) == 0) {
    flag ? fn(std::true_type{}) : fn(std::false_type{});
  } else {
    const auto with = [&](auto... rest) {
      flag ? fn(std::true_type{}, rest...) : fn(std::false_type{}, rest...);
    };
    choose(with, flags...);
  }
}

template <class T>
int logprob_fwd(const T* logits, int64_t ld, const int64_t* tokens, float* logp, float* stats,
                float* entropy, float* top_logp, int64_t* top_ids, int64_t rows, int64_t cols,
                int32_t n_tokens, int32_t n_top, float temperature, const credit_cfg* cfg) {
  CREDIT_TRY(check_shape(rows, cols, kMaxCols));
  CREDIT_TRY(check_logits(logits, "logits", ld, rows, cols, sizeof(T)));
  CREDIT_TRY(check_entries(n_tokens, 0, kMaxEntries, "tokens"));
  CREDIT_TRY(check_entries(n_top, 0, cols < kMaxEntries ? cols : kMaxEntries, "alternatives"));
  CREDIT_TRY(check_operand(stats, "stats", rows, sizeof(float)));
  if (n_tokens > 0) {
    CREDIT_TRY(check_operand(tokens, "tokens", rows, sizeof(int64_t)));
    CREDIT_TRY(check_operand(logp, "logp", rows, sizeof(float)));
  }
  if (n_top > 0) {
    CREDIT_TRY(check_operand(top_logp, "top_logp", rows, sizeof(float)));
    CREDIT_TRY(check_operand(top_ids, "top_ids", rows, sizeof(int64_t)));
  }
  CREDIT_TRY(check_aligned(entropy, sizeof(float), "entropy"));
  CREDIT_TRY(check_temperature(temperature));
  CREDIT_TRY(check_variant(cfg, true));
  if (rows == 0) return CREDIT_OK;
  LogprobArgs<T> a{logits,   ld,
                   tokens,   logp,
                   stats,    entropy,
                   top_logp, top_ids,
                   0,        static_cast<int>(cols),
                   n_tokens, n_top,
                   0,        log2e_over(temperature),
                   1.0 / static_cast<double>(temperature),
                   Parts{}};
  const int64_t batches = row_batches(logits, ld, rows, cols);
  CREDIT_TRY(plan_parts(cfg, rows, batches, n_top > 0, &a.parts));
  const auto unit_bytes = [&] {
    return static_cast<size_t>((batches + (int64_t{1} << a.fold) - 1) >> a.fold) * kThreads *
           sizeof(T);
  };
  while (unit_bytes() > kMaxUnitBytes) ++a.fold;
  // The candidates take the units' place once those are listed.
  const size_t lds = n_top > 0 ? std::max(unit_bytes(), size_t{kCands} * sizeof(uint64_t)) : 0;
  hipStream_t stream = cfg_stream(cfg);
  const auto launch = [&](auto ent, auto top, auto split) {
    for (; a.first < rows; a.first += kMaxGridRows)
      token_logprob_fwd_kernel<T, decltype(ent)::value, decltype(top)::value,
                               decltype(split)::value>
          <<<forward_grid(a.parts, rows - a.first), kThreads, lds, stream>>>(a);
  };
  choose(launch, entropy != nullptr, n_top > 0, a.parts.n > 1);
  return check_launch("token_logprob_fwd_kernel");
}

template <class T>
int logprob_bwd(const T* logits, int64_t ld, const int64_t* tokens, const float* stats,
                const float* entropy, const float* dlogp, const float* dentropy, T* dlogits,
                int64_t ldd, int64_t rows, int64_t cols, int32_t n_tokens, float temperature,
                const credit_cfg* cfg) {
  CREDIT_TRY(check_shape(rows, cols, kMaxCols));
  CREDIT_TRY(check_logits(logits, "logits", ld, rows, cols, sizeof(T)));
  CREDIT_TRY(check_logits(dlogits, "dlogits", ldd, rows, cols, sizeof(T)));
  CREDIT_TRY(check_entries(n_tokens, 0, kMaxEntries, "tokens"));
  CREDIT_TRY(check_operand(stats, "stats", rows, sizeof(float)));
  if (n_tokens > 0) {
    CREDIT_TRY(check_operand(tokens, "tokens", rows, sizeof(int64_t)));
    CREDIT_TRY(check_operand(dlogp, "dlogp", rows, sizeof(float)));
  }
  if (dentropy != nullptr) {
    CREDIT_TRY(check_operand(entropy, "entropy", rows, sizeof(float)));
    CREDIT_TRY(check_aligned(dentropy, sizeof(float), "dentropy"));
  }
  CREDIT_TRY(check_temperature(temperature));
  CREDIT_TRY(check_variant(cfg, false));
  if (rows == 0) return CREDIT_OK;
  CREDIT_TRY(check_overlap(logits, ld, dlogits, ldd, rows, cols, sizeof(T)));
  const LogprobGradArgs<T> a{logits,
                             ld,
                             tokens,
                             stats,
                             entropy,
                             dlogp,
                             dentropy,
                             dlogits,
                             ldd,
                             rows,
                             static_cast<int>(cols),
                             n_tokens,
                             1.0f / temperature,
                             log2e_over(temperature)};
  hipStream_t stream = cfg_stream(cfg);
  const dim3 grid = grad_grid(logits, ld, rows, cols);
  const auto launch = [&](auto ent, auto vec) {
    token_logprob_bwd_kernel<T, decltype(ent)::value, decltype(vec)::value>
        <<<grid, kThreads, 0, stream>>>(a);
  };
  choose(launch, dentropy != nullptr, alike(logits, ld, dlogits, ldd, rows, sizeof(T)));
  return check_launch("token_logprob_bwd_kernel");
}

template <class T>
int distill_fwd(const T* logits, int64_t ld, const int64_t* ids, const float* teacher, float* loss,
                float* stats, int64_t rows, int64_t cols, int32_t n_top, int32_t tail,
                float temperature, const credit_cfg* cfg) {
  CREDIT_TRY(check_shape(rows, cols, kMaxCols));
  CREDIT_TRY(check_logits(logits, "logits", ld, rows, cols, sizeof(T)));
  CREDIT_TRY(check_entries(n_top, 1, kMaxEntries, "teacher entries"));
  CREDIT_TRY(check_operand(ids, "teacher_ids", rows, sizeof(int64_t)));
  CREDIT_TRY(check_operand(teacher, "teacher", rows, sizeof(float)));
  CREDIT_TRY(check_operand(loss, "loss", rows, sizeof(float)));
  CREDIT_TRY(check_operand(stats, "stats", rows, sizeof(float)));
  CREDIT_TRY(check_temperature(temperature));
  CREDIT_TRY(check_variant(cfg, true));
  if (rows == 0) return CREDIT_OK;
  DistillArgs<T> a{logits, ld,    ids,         teacher,
                   loss,   stats, 0, static_cast<int>(cols),
                   n_top,  temperature, log2e_over(temperature),
                   Parts{}};
  CREDIT_TRY(plan_parts(cfg, rows, row_batches(logits, ld, rows, cols), false, &a.parts));
  hipStream_t stream = cfg_stream(cfg);
  const auto launch = [&](auto has_tail, auto split) {
    for (; a.first < rows; a.first += kMaxGridRows)
      topk_distill_fwd_kernel<T, decltype(has_tail)::value, decltype(split)::value>
          <<<forward_grid(a.parts, rows - a.first), kThreads, 0, stream>>>(a);
  };
  choose(launch, tail != 0, a.parts.n > 1);
  return check_launch("topk_distill_fwd_kernel");
}

template <class T>
int distill_bwd(const T* logits, int64_t ld, const int64_t* ids, const float* teacher,
                const float* stats, const float* dloss, T* dlogits, int64_t ldd, int64_t rows,
                int64_t cols, int32_t n_top, int32_t tail, float temperature,
                const credit_cfg* cfg) {
  CREDIT_TRY(check_shape(rows, cols, kMaxCols));
  CREDIT_TRY(check_logits(logits, "logits", ld, rows, cols, sizeof(T)));
  CREDIT_TRY(check_logits(dlogits, "dlogits", ldd, rows, cols, sizeof(T)));
  CREDIT_TRY(check_entries(n_top, 1, kMaxEntries, "teacher entries"));
  CREDIT_TRY(check_operand(ids, "teacher_ids", rows, sizeof(int64_t)));
  CREDIT_TRY(check_operand(teacher, "teacher", rows, sizeof(float)));
  CREDIT_TRY(check_operand(stats, "stats", rows, sizeof(float)));
  CREDIT_TRY(check_operand(dloss, "dloss", rows, sizeof(float)));
  CREDIT_TRY(check_temperature(temperature));
  CREDIT_TRY(check_variant(cfg, false));
  if (rows == 0) return CREDIT_OK;
  CREDIT_TRY(check_overlap(logits, ld, dlogits, ldd, rows, cols, sizeof(T)));
  const DistillGradArgs<T> a{logits,
                             ld,
                             ids,
                             teacher,
                             stats,
                             dloss,
                             dlogits,
                             ldd,
                             rows,
                             static_cast<int>(cols),
                             n_top,
                             temperature,
                             log2e_over(temperature)};
  hipStream_t stream = cfg_stream(cfg);
  const dim3 grid = grad_grid(logits, ld, rows, cols);
  const auto launch = [&](auto has_tail, auto vec) {
    topk_distill_bwd_kernel<T, decltype(has_tail)::value, decltype(vec)::value>
        <<<grid, kThreads, 0, stream>>>(a);
  };
  choose(launch, tail != 0, alike(logits, ld, dlogits, ldd, rows, sizeof(T)));
  return check_launch("topk_distill_bwd_kernel");
}

}  // namespace
}  // namespace credit

using namespace credit;

extern "C" {

int credit_token_logprob_fwd_f32(const float* logits, int64_t ld, const int64_t* tokens,
                                 float* logp, float* stats, float* entropy, float* top_logp,
                                 int64_t* top_ids, int64_t rows, int64_t cols, int32_t n_tokens,
                                 int32_t n_top, float temperature, const credit_cfg* cfg) {
  return logprob_fwd(logits, ld, tokens, logp, stats, entropy, top_logp, top_ids, rows, cols,
                     n_tokens, n_top, temperature, cfg);
}
int credit_token_logprob_fwd_bf16(const uint16_t* logits, int64_t ld, const int64_t* tokens,
                                  float* logp, float* stats, float* entropy, float* top_logp,
                                  int64_t* top_ids, int64_t rows, int64_t cols, int32_t n_tokens,
                                  int32_t n_top, float temperature, const credit_cfg* cfg) {
  return logprob_fwd(logits, ld, tokens, logp, stats, entropy, top_logp, top_ids, rows, cols,
                     n_tokens, n_top, temperature, cfg);
}
int credit_token_logprob_bwd_f32(const float* logits, int64_t ld, const int64_t* tokens,
                                 const float* stats, const float* entropy, const float* dlogp,
                                 const float* dentropy, float* dlogits, int64_t ldd, int64_t rows,
                                 int64_t cols, int32_t n_tokens, float temperature,
                                 const credit_cfg* cfg) {
  return logprob_bwd(logits, ld, tokens, stats, entropy, dlogp, dentropy, dlogits, ldd, rows, cols,
                     n_tokens, temperature, cfg);
}
int credit_token_logprob_bwd_bf16(const uint16_t* logits, int64_t ld, const int64_t* tokens,
                                  const float* stats, const float* entropy, const float* dlogp,
                                  const float* dentropy, uint16_t* dlogits, int64_t ldd,
                                  int64_t rows, int64_t cols, int32_t n_tokens, float temperature,
                                  const credit_cfg* cfg) {
  return logprob_bwd(logits, ld, tokens, stats, entropy, dlogp, dentropy, dlogits, ldd, rows, cols,
                     n_tokens, temperature, cfg);
}
int credit_topk_distill_fwd_f32(const float* logits, int64_t ld, const int64_t* teacher_ids,
                                const float* teacher, float* loss, float* stats, int64_t rows,
                                int64_t cols, int32_t n_top, int32_t tail, float temperature,
                                const credit_cfg* cfg) {
  return distill_fwd(logits, ld, teacher_ids, teacher, loss, stats, rows, cols, n_top, tail,
                     temperature, cfg);
}
int credit_topk_distill_fwd_bf16(const uint16_t* logits, int64_t ld, const int64_t* teacher_ids,
                                 const float* teacher, float* loss, float* stats, int64_t rows,
                                 int64_t cols, int32_t n_top, int32_t tail, float temperature,
                                 const credit_cfg* cfg) {
  return distill_fwd(logits, ld, teacher_ids, teacher, loss, stats, rows, cols, n_top, tail,
                     temperature, cfg);
}
int credit_topk_distill_bwd_f32(const float* logits, int64_t ld, const int64_t* teacher_ids,
                                const float* teacher, const float* stats, const float* dloss,
                                float* dlogits, int64_t ldd, int64_t rows, int64_t cols,
                                int32_t n_top, int32_t tail, float temperature,
                                const credit_cfg* cfg) {
  return distill_bwd(logits, ld, teacher_ids, teacher, stats, dloss, dlogits, ldd, rows, cols,
                     n_top, tail, temperature, cfg);
}
int credit_topk_distill_bwd_bf16(const uint16_t* logits, int64_t ld, const int64_t* teacher_ids,
                                 const float* teacher, const float* stats, const float* dloss,
                                 uint16_t* dlogits, int64_t ldd, int64_t rows, int64_t cols,
                                 int32_t n_top, int32_t tail, float temperature,
                                 const credit_cfg* cfg) {
  return distill_bwd(logits, ld, teacher_ids, teacher, stats, dloss, dlogits, ldd, rows, cols,
                     n_top, tail, temperature, cfg);
}

}  // extern "C"
