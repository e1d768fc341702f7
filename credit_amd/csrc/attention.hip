// Attention of a batch's new tokens over a paged cache
// (credit_paged_attention_bf16): o = sum_j p_j v_j, p = softmax(scale q k_j) over
// the positions j up to the token's own.
//
// A wave holds 32 query rows, a row one head of one token: the heads that share
// keys are rows of one tile, so that keys and values are read once for them.  In
// one pass over the positions it keeps each row's maximum m, sum l and output o in
// registers (the online softmax): S^T = K Q^T on v_mfma_f32_32x32x16_bf16 leaves a
// row's scores in one lane pair, so maxima and sums need one exchange, and the
// weights, packed to bf16, are already the other product's operand, O^T = V^T P^T,
// whose V^T comes from row-major LDS through transposing reads.  Products are
// exact and summed in fp32; the weights' rounding to bf16 (2^-8 of each, sums are
// taken before it) is what matrix units of this rate take.  m is that of the first
// step, raised only where a score passes it by 2^16: floating point keeps the same
// relative precision wherever it lies, and the usual step rescales nothing.
//
// Large tiles: four waves of 32 rows share every step's keys and values in LDS.
// Small tiles (few rows, decode): four waves share the rows and take steps of the
// positions in turn, each with its own LDS; their results meet at the end.  The
// positions of a tile may be cut into parts whose results meet in the workspace;
// the last to arrive joins them in the parts' order and none waits for another.
#include <math.h>

#include <type_traits>

#include "api_internal.hpp"
#include "attention_rules.hpp"
#include "common.hpp"

namespace credit {
namespace {

using attention::Divisor;
using attention::kFew;
using attention::kMany;
using heads::Place;

constexpr int kThreads = 256;
constexpr int kNW = kThreads / kWave;
constexpr float kNegInf = -__builtin_inff();
constexpr float kRaise = 16.0f;  // log2 of the weights' largest value

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) bf16x4_t lds_bf16x4_t;
typedef __attribute__((address_space(3))) void* lds_ptr_t;

// LDS by its own 32-bit addresses: those of a step's reads differ in bits that an
// exclusive or sets, one instruction each.  The kernels' LDS is one dynamic array,
// which begins at address 0; its steps lie at multiples of 1 KiB.
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(lds_ptr_t)(const_cast<void*>(p));
}
template <class T>
__device__ __forceinline__ T lds_read(uint32_t at) {
  return *(__attribute__((address_space(3))) const T*)(uintptr_t)at;
}
// Four positions of one element (column) for each lane of a group of 16: lane j of
// it addresses row j / 4, columns 4 (j % 4) .. + 3, and gets column j of the rows.
__device__ __forceinline__ bf16x4_t read_transposed(uint32_t at) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4_t*)(uintptr_t)at);
}

// The kernel's arguments, opaque to the compiler: read again where they are used
// instead of kept in scalar registers over a loop that has none to spare.
template <class A>
__device__ __forceinline__ const A& arguments() {
  auto p = __builtin_amdgcn_kernarg_segment_ptr();
  __asm__ volatile("" : "+s"(p));
  return *(const A*)p;
}

struct Cache {
  const uint16_t* data;
  int64_t page, slot, head;  // strides
};
struct Args {
  const uint16_t* q;
  int64_t q_token, q_head;
  Cache k, v;
  const int32_t* pages;  // [batch, columns]
  int64_t pages_ld;
  const int32_t* q_start;
  const int32_t* kv_len;
  uint16_t* out;
  int64_t out_token, out_head;
  float* lse;  // [tokens, heads] or nullptr
  float* partial;      // parts' results, two a workgroup; nullptr: no parts
  uint32_t partial_bytes;
  uint32_t* arrived;
  int64_t tokens;
  int batch, heads, kv_heads, group, dim;
  int page_size, n_pages, positions;  // positions: most that a row of pages holds
  Divisor by_page, by_group;
  int window, units, tiles;  // units: workgroups a key head
  int least_steps;           // of a unit
  float scale, scale_log2;  // scale, scale log2(e)
};

__device__ __forceinline__ int divide(int n, const Divisor& d) {
  return static_cast<int>(
      (__umulhi(static_cast<uint32_t>(n), d.mul) + static_cast<uint32_t>(n)) >> d.shift);
}

// The lane, opaque to the compiler: what is derived from it within a step is not
// kept in registers from step to step.
__device__ __forceinline__ int opaque_lane() { return opaque_lane_index() & (kWave - 1); }

// A tile: rows row0 .. of sequence b, whose token i sees positions up to ahead + i.
struct Tile {
  int b;
  int64_t first;  // token of the sequence's row 0
  int rows, row0;
  int kv, ahead;
};
// The value of any lane of a wave that all hold one.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ const void* uniform(const void* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = static_cast<uint32_t>(uniform(static_cast<int>(v)));
  const uint32_t hi = static_cast<uint32_t>(uniform(static_cast<int>(v >> 32)));
  return reinterpret_cast<const void*>(static_cast<uint64_t>(hi) << 32 | lo);
}

__device__ __forceinline__ int64_t start_of(const Args& a, int b) {
  const int64_t s = a.q_start[b];
  return s < 0 ? 0 : s < a.tokens ? s : a.tokens;
}
__device__ __forceinline__ int rows_of(const Args& a, int b) {
  const int64_t n = start_of(a, b + 1) - start_of(a, b);
  return n > 0 ? static_cast<int>(n * a.group) : 0;
}
__device__ __forceinline__ int positions_of(const Args& a, int b) {
  return min(max(a.kv_len[b], 0), a.positions);
}

// Work on a tile: `take` of its steps from the skip-th on, which is part `part` of
// `parts`; unit: the one with part 0, inside: whether the tile begins within it.
struct Work {
  Tile t;
  int head, skip, take, part, parts, unit, inside;
};
template <int ROWS>
__device__ __forceinline__ void tile_of(Work& w, const Args& a, int b, int tile) {
  Tile& t = w.t;
  t.b = uniform(b);
  t.first = uniform(static_cast<int>(start_of(a, t.b)));
  t.rows = uniform(rows_of(a, t.b));
  t.row0 = uniform(tile) * ROWS;
  t.kv = uniform(positions_of(a, t.b));
  t.ahead = t.kv - divide(t.rows, a.by_group);
}

// A sequence's tiles and the steps of each, at least one.
struct Count {
  int tiles, steps;
};
template <int ROWS, int KEYS>
__device__ __forceinline__ Count count_of(const Args& a, int b) {
  if (b >= a.batch) return {0, 0};
  const int rows = rows_of(a, b), kv = positions_of(a, b);
  Count c{(rows + ROWS - 1) / ROWS, max(1, (kv + KEYS - 1) / KEYS)};
  if (a.window > 0) {  // those in front of the window are not walked
    const int64_t seen = static_cast<int64_t>(a.window) + divide(ROWS - 1, a.by_group) + 1;
    c.steps = static_cast<int>(min(static_cast<int64_t>(kv), seen) + KEYS - 1) / KEYS + 1;
  }
  return c;
}

// What a workgroup does, tile by tile.  Key heads lie next to each other in the
// grid: the dies take workgroups in turn, so that tiles of one head's keys tend to
// share one die's L2.
//
// With parts: the steps of all tiles of a key head, one sequence behind the other,
// are dealt to its units in runs of one length, whatever the sequences' lengths:
// the device is busy evenly to the end, and only a run's first and last tile can be
// shared with other units.  Each wave counts the sequences through.
// Without: a unit is a tile's slot, sequence b's from floor(first row / ROWS) + b
// on, found by a search; later tiles, which see more, first.
template <int ROWS, int KEYS, bool PARTS>
struct Cursor {
  int head, unit, each;
  int64_t at, end;  // steps of the unit's run, -1: without parts
  int upto;         // of this lane's sequence among the first 64: steps up to its end
  Count count;

  __device__ __forceinline__ static int scan(int v) {
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
      const int u = __shfl_up(v, d);
      if (lane >= d) v += u;
    }
    return v;
  }
  __device__ __forceinline__ void start(const Args& a) {
    const int i = static_cast<int>(blockIdx.x);
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    head = i % a.kv_heads;
    unit = i / a.kv_heads;
    at = end = -1;
    if constexpr (!PARTS) return;
    count = count_of<ROWS, KEYS>(a, lane);
    upto = scan(count.tiles * count.steps);
    constexpr double kTile = 1ull << 39;  // tiles and steps summed as one number
    double sum = count.tiles * (kTile + count.steps);
    for (int b = lane + kWave; b - lane < a.batch; b += kWave) {
      const Count more = count_of<ROWS, KEYS>(a, b);
      sum += more.tiles * (kTile + more.steps);
    }
    sum = wave_reduce_sum_f64(sum);
    const double tiles = __builtin_floor(sum / kTile);
    // More tiles than the rows make: q_start does not rise.  Nothing is done.
    const int all = tiles > a.tiles ? 0 : uniform(static_cast<int>(sum - tiles * kTile));
    each = max(a.least_steps, (all + a.units - 1) / a.units);
    at = static_cast<int64_t>(unit) * each;
    end = min(at + each, static_cast<int64_t>(all));
  }
  // The next tile's work; false: none.
  __device__ __forceinline__ bool next(Work& w, const Args& a) {
    w.head = head;
    if constexpr (!PARTS) return search(w, a, a.units - 1 - unit);
    if (at >= end) return false;
    const int now = uniform(static_cast<int>(at));
    int before = 0, to = upto;
    Count c = count;
    for (int b0 = 0;; b0 += kWave) {
      if (b0 > 0) {
        c = count_of<ROWS, KEYS>(a, b0 + static_cast<int>(threadIdx.x & (kWave - 1)));
        to = scan(c.tiles * c.steps);
      }
      const uint64_t past = __builtin_amdgcn_ballot_w64(now < before + to);
      if (past == 0) {  // ends: now is less than the last sequence's
        before += __builtin_amdgcn_readlane(to, kWave - 1);
        continue;
      }
      const int in = __builtin_ctzll(past);
      const int steps = __builtin_amdgcn_readlane(c.steps, in);
      const int first = before + __builtin_amdgcn_readlane(to - c.tiles * c.steps, in);
      const int tile = (now - first) / steps;
      const int from = first + tile * steps;
      tile_of<ROWS>(w, a, b0 + in, tile);
      w.skip = now - from;
      w.take = min(static_cast<int>(end) - now, steps - w.skip);
      w.unit = from / each;
      w.inside = from != w.unit * each;
      w.parts = (from + steps - 1) / each - w.unit + 1;
      w.part = unit - w.unit;
      at += w.take;
      return true;
    }
  }
  __device__ __forceinline__ static bool search(Work& w, const Args& a, int slot) {
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    int lo = 0, n = a.batch;
    while (n > 1) {
      const int step = (n + kWave - 1) / kWave;
      const int b = lo + lane * step;
      const bool at =
          lane * step < n && start_of(a, b) * a.group / ROWS + b <= static_cast<int64_t>(slot);
      const int count = __builtin_popcountll(__builtin_amdgcn_ballot_w64(at));
      if (count == 0) return false;
      const int skip = (count - 1) * step;
      lo += skip;
      n = min(step, n - skip);
    }
    lo = uniform(lo);
    const int64_t first = start_of(a, lo) * a.group / ROWS + lo;
    if (slot < first || (slot - first) * ROWS >= rows_of(a, lo)) return false;
    tile_of<ROWS>(w, a, lo, static_cast<int>(slot - first));
    w.skip = w.part = 0;
    w.take = 1 << 30;
    w.parts = 1;
    return true;
  }
};

// Layout of a step's keys and values in LDS: rows of D elements, or the power of two
// above, 16-byte chunk c of row r at place c ^ swizzle(r), so that the reads below
// meet no bank twice: of the keys 16 rows' same chunk, of the values 4 rows' 64 bytes.
template <int D>
struct Lds {
  static constexpr int kWidth = D <= 64 ? 64 : D <= 128 ? 128 : 256;
  static constexpr int kChunks = kWidth / 8;
  static constexpr int kRowBytes = kWidth * 2;
  __device__ static int key(int row, int chunk) {
    const int s = D == 64 ? (row >> 1) & 7 : row & 15;
    return row * kRowBytes + (chunk ^ s) * 16;
  }
  __device__ static int value(int row, int chunk) {
    const int s = D == 64 ? ((row >> 1) & 1) * 4 : (row & 3) * 4;
    return row * kRowBytes + (chunk ^ s) * 16;
  }
};

// What a wave keeps of its 32 rows: lane l has row l % 32.
template <int D>
struct State {
  f32x16 o[D / 32];  // element (i): column 32 db + 8 (i / 4) + 4 (l / 32) + i % 4
  float m, l;        // maximum of the scores (raw) that o and l refer to
};
template <int D>
__device__ __forceinline__ void clear(State<D>& s) {
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) s.o[db][i] = 0.0f;
  s.m = kNegInf;
  s.l = 0.0f;
}
// The maximum to subtract: of a row that has seen nothing 0, so that its weights
// are 0.
__device__ __forceinline__ float base_of(float m) { return m == kNegInf ? 0.0f : m; }

// Of lane l and lane l ^ 32: both values, in some order.
__device__ __forceinline__ float2_t both_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v),
                                                  __builtin_bit_cast(uint32_t, v), false, false);
  const uint32_t a = r[0], b = r[1];  // a bit_cast of r[1] itself takes r[0]
  return {__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)};
}

// The queries of a wave's rows: lane l holds elements 16 ks + 8 (l / 32) .. + 7 of
// row l % 32.
template <int D>
__device__ __forceinline__ void load_queries(bf16x8_t (&q)[D / 16], const Args& a, const Tile& t,
                                             int lane, int row, int kv_head) {
  const int token = divide(row, a.by_group), head = row - token * a.group;
  const uint16_t* p = a.q + (t.first + token) * a.q_token +
                      static_cast<int64_t>(kv_head * a.group + head) * a.q_head;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) {
    const int e = 16 * ks + 8 * (lane >> 5);
    u32x4 v = {0, 0, 0, 0};
    if (row < t.rows && e < a.dim) v = *reinterpret_cast<const u32x4*>(p + e);
    q[ks] = __builtin_bit_cast(bf16x8_t, v);
  }
}

// A lane's places in a step's keys and values.  Its first chunk of keys (row l % 32,
// chunk l / 32); those of elements 16 ks on are 32 ks away by exclusive or, those of
// row 32 nb + l % 32 32 nb rows on.  Of the values the row and columns that it
// addresses for a fragment of columns 0 .. 31; those of columns 32 db on are 64 db
// away by exclusive or.
struct Places {
  uint32_t key, value;
};
template <int D>
__device__ __forceinline__ Places places_of(int lane) {
  const int row = 4 * (lane >> 5) + ((lane & 15) >> 2);
  const int column = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  return {static_cast<uint32_t>(Lds<D>::key(lane & 31, lane >> 5)),
          static_cast<uint32_t>(Lds<D>::value(row, column >> 3) + (column & 7) * 2)};
}
// A fragment of V^T: column 32 db + l % 32 of the 16 positions from 16 ts on, in
// the weights' order (element e: position 16 ts + 8 (e / 4) + 4 (l / 32) + e % 4).
template <int D>
__device__ __forceinline__ bf16x8_t value_fragment(uint32_t v, int db, int ts) {
  const uint32_t at = (v ^ (64u * db)) + 16 * ts * Lds<D>::kRowBytes;
  const bf16x4_t lo = read_transposed(at);
  const bf16x4_t hi = read_transposed(at + 8 * Lds<D>::kRowBytes);
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// In steps where a mask hides positions from some rows, a value that is not finite
// would make NaN of its weight of 0: whether there are any among `ROWS` rows.
template <int D, int ROWS>
__device__ __forceinline__ bool any_special(uint32_t v) {
  const uint32_t own = v + static_cast<uint32_t>(opaque_lane()) * 16;
  uint32_t bad = 0;
#pragma unroll 4
  for (int i = 0; i < ROWS * Lds<D>::kRowBytes / (16 * kWave); ++i) {
    const u32x4 w = lds_read<u32x4>(own + i * kWave * 16);
#pragma unroll
    for (int e = 0; e < 4; ++e)  // bit 31 or 15: an exponent of all ones
      bad |= ((w[e] & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
  }
  return __builtin_amdgcn_ballot_w64(bad != 0) != 0;
}
// 0 in their place.
__device__ __forceinline__ bf16x8_t without_special(bf16x8_t v) {
  u32x4 w = __builtin_bit_cast(u32x4, v);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    w[e] &= ((w[e] & 0x7F80u) == 0x7F80u ? 0u : 0xFFFFu) |
            ((w[e] & 0x7F800000u) == 0x7F800000u ? 0u : 0xFFFF0000u);
  return __builtin_bit_cast(bf16x8_t, w);
}
// Adds them to the outputs of the rows that see them, whatever their weight.
template <int D, int ROWS>
__device__ __forceinline__ void add_special(State<D>& s, uint32_t v, int j0, int low, int last) {
#pragma unroll 1
  for (int r = 0; r < ROWS; ++r) {
    const int lane = opaque_lane();
    const bool seen = j0 + r >= low && j0 + r <= last;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int column = 32 * db + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
        const uint16_t bits =
            lds_read<uint16_t>(v + Lds<D>::value(r, column >> 3) + (column & 7) * 2);
        s.o[db][i] += seen && (bits & 0x7F80u) == 0x7F80u ? bf16_to_f32(bits) : 0.0f;
      }
  }
}

// A step: NB blocks of 32 positions from j0 on, keys at k, values at v in LDS;
// masked: a row sees those in [low, last] alone.
struct Step {
  uint32_t k, v;
  int j0;
  bool masked;
  int low, last;
};
// What a step came to.  kRaise, kSpecial: nothing yet; the rows' maxima have to be
// raised first, or the values hold what the mask must be kept from.  The loops over
// the steps leave such steps to code behind them: a second way to the outputs inside
// costs a copy of them in every step (64 registers; a prompt of 8192 tokens 602 us
// against 575).
enum class Outcome { kDone, kRaise, kSpecial };

// fn(integral_constant 0 .. N - 1).
template <int N, int I = 0, class Fn>
__device__ __forceinline__ void unrolled(Fn&& fn) {
  if constexpr (I < N) {
    fn(std::integral_constant<int, I>{});
    unrolled<N, I + 1>(fn);
  }
}

// The order of a run of matrix products and the reads from LDS that feed them: PER
// reads a product, those of AHEAD products on their way before the first, where the
// compiler by itself waits for each read (us, without -> with: a prompt of 4096 with 16
// heads of 192 168 -> 149, of 256 404 -> 375, of 8192 with 32 heads of 128 578 -> 570;
// of 4096 with 32 heads of 64 90 -> 92).
template <int D, int PRODUCTS, int PER, int AHEAD>
__device__ __forceinline__ void in_order() {
  constexpr int kProduct = 0x008, kRead = 0x100;
  if constexpr (D > 64) {
    __builtin_amdgcn_sched_group_barrier(kRead, PER * AHEAD, 0);
    unrolled<PRODUCTS - AHEAD>([](auto) {
      __builtin_amdgcn_sched_group_barrier(kProduct, 1, 0);
      __builtin_amdgcn_sched_group_barrier(kRead, PER, 0);
    });
    __builtin_amdgcn_sched_group_barrier(kProduct, AHEAD, 0);
  }
}

template <int D, int NB>
__device__ __forceinline__ void scores(f32x16 (&x)[NB], const bf16x8_t (&q)[D / 16],
                                       const Places& places, const Step& at) {
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int i = 0; i < 16; ++i) x[nb][i] = 0.0f;
  const uint32_t key = places.key + at.k;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
      x[nb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
          lds_read<bf16x8_t>((key ^ (32u * ks)) + 32 * nb * Lds<D>::kRowBytes), q[ks], x[nb], 0, 0,
          0);
  }
  in_order<D, NB * D / 16, 1, 4>();
}
template <int NB>
__device__ __forceinline__ void hide(f32x16 (&x)[NB], const Step& at) {
  const int j0 = at.j0 + 4 * (opaque_lane() >> 5);
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int j = j0 + 32 * nb + 8 * (i >> 2) + (i & 3);
      x[nb][i] = j >= at.low && j <= at.last ? x[nb][i] : kNegInf;
    }
}
// The scores' maximum of each row; NaN makes its row NaN.
template <int NB>
__device__ __forceinline__ float most(const f32x16 (&x)[NB]) {
  float m = fmax_nan(x[0][0], x[0][1]);
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int i = nb == 0 ? 2 : 0; i < 16; ++i) m = fmax_nan(m, x[nb][i]);
  const float2_t ms = both_halves(m);
  return fmax_nan(ms.x, ms.y);
}
// The weights, as the other product's operand, and their sum.
template <int NB>
__device__ __forceinline__ float weights(bf16x8_t (&p)[2 * NB], const f32x16 (&x)[NB], float m,
                                         float scale_log2) {
  const float base = base_of(m) * scale_log2;
  float sum = 0.0f;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = __builtin_amdgcn_exp2f(
            __builtin_fmaf(x[nb][8 * h + 2 * e], scale_log2, -base));
        const float b = __builtin_amdgcn_exp2f(
            __builtin_fmaf(x[nb][8 * h + 2 * e + 1], scale_log2, -base));
        sum += a + b;
        w[e] = pack_bf16x2(a, b);
      }
      p[2 * nb + h] = __builtin_bit_cast(bf16x8_t, w);
    }
  return sum;
}
// Whether a row's maximum has to be raised for a step's m; the first is taken as it
// is, while o and l are 0 (or NaN).
template <int D>
__device__ __forceinline__ bool to_raise(State<D>& s, float m, float scale_log2) {
  s.m = s.m == kNegInf ? m : s.m;
  return __builtin_amdgcn_ballot_w64((m - s.m) * scale_log2 > kRaise) != 0;
}
// scored() runs once the keys have been read, ready() before the values are.
template <int D, int NB, class Scored, class Ready>
__device__ __forceinline__ Outcome step(State<D>& s, const bf16x8_t (&q)[D / 16],
                                        const Places& places, const Step& at, float scale_log2,
                                        Scored&& scored, Ready&& ready) {
  if (at.masked) {
    ready();
    if (any_special<D, 32 * NB>(at.v)) return Outcome::kSpecial;
  }
  f32x16 x[NB];
  scores<D, NB>(x, q, places, at);
  if (at.masked) hide<NB>(x, at);
  const float m = most<NB>(x);
  if (to_raise(s, m, scale_log2)) return Outcome::kRaise;
  scored();
  bf16x8_t p[2 * NB];
  s.l += weights<NB>(p, x, s.m, scale_log2);
  ready();
  const uint32_t value = places.value + at.v;
#pragma unroll
  for (int db = 0; db < D / 32; ++db) {
#pragma unroll
    for (int ts = 0; ts < 2 * NB; ++ts)
      s.o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(value_fragment<D>(value, db, ts), p[ts],
                                                        s.o[db], 0, 0, 0);
  }
  in_order<D, 2 * NB * D / 32, 2, 4>();
  return Outcome::kDone;
}
// Raises the maxima of the rows to those of the step.
template <int D, int NB>
__device__ __forceinline__ void raise(State<D>& s, const bf16x8_t (&q)[D / 16],
                                      const Places& places, const Step& at, float scale_log2) {
  f32x16 x[NB];
  scores<D, NB>(x, q, places, at);
  if (at.masked) hide<NB>(x, at);
  const float raised = fmax_nan(s.m, most<NB>(x));
  const float factor =
      s.m == kNegInf ? 1.0f : __builtin_amdgcn_exp2f((s.m - raised) * scale_log2);
  s.m = raised;
  s.l *= factor;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) s.o[db][i] *= factor;
}
// A masked step over values that are not finite; the same bits as step()'s where
// they are hidden.
template <int D, int NB>
__device__ __forceinline__ void special_step(State<D>& s, const bf16x8_t (&q)[D / 16],
                                             const Places& places, const Step& at,
                                             float scale_log2) {
  f32x16 x[NB];
  scores<D, NB>(x, q, places, at);
  hide<NB>(x, at);
  if (to_raise(s, most<NB>(x), scale_log2)) raise<D, NB>(s, q, places, at, scale_log2);
  bf16x8_t p[2 * NB];
  s.l += weights<NB>(p, x, s.m, scale_log2);
  const uint32_t value = places.value + at.v;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int ts = 0; ts < 2 * NB; ++ts)
      s.o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
          without_special(value_fragment<D>(value, db, ts)), p[ts], s.o[db], 0, 0, 0);
  add_special<D, 32 * NB>(s, at.v, at.j0, at.low, at.last);
}
// The steps first, first + by, .. below last: at(i) gives one, begin(i) runs before
// each, scored(i) and ready(i) as in step(), end(i) behind each.
template <int D, int NB, class At, class Begin, class Scored, class Ready, class End>
__device__ __forceinline__ void walk(State<D>& s, const bf16x8_t (&q)[D / 16],
                                     const Places& places, float scale_log2, int first, int last,
                                     int by, At&& at, Begin&& begin, Scored&& scored,
                                     Ready&& ready, End&& end) {
  int i = first;
  if (i >= last) return;
  begin(i);
  while (true) {
    Outcome out;
    while (true) {
      out = step<D, NB>(s, q, places, at(i), scale_log2, [&] { scored(i); }, [&] { ready(i); });
      if (out != Outcome::kDone) break;
      end(i);
      i += by;
      if (i >= last) return;
      begin(i);
    }
    if (out == Outcome::kRaise) {
      raise<D, NB>(s, q, places, at(i), scale_log2);
      continue;
    }
    special_step<D, NB>(s, q, places, at(i), scale_log2);
    scored(i);
    end(i);
    i += by;
    if (i >= last) return;
    begin(i);
  }
}

__device__ __forceinline__ float inverse_of(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }
// l = 0: nothing was seen.
__device__ __forceinline__ float lse_of(const Args& a, float m, float l) {
  return l == 0.0f ? kNegInf : base_of(m) * a.scale + logf(l);
}
// What scales a wave's or part's results to the maximum m of all (nothing seen: its
// sums are 0, or NaN).
__device__ __forceinline__ float weight_of(const Args& a, float own, float m) {
  return own == kNegInf ? 1.0f : __builtin_amdgcn_exp2f((own - base_of(m)) * a.scale_log2);
}
// Head and token of a row; its place in an array of rows.
struct Row {
  int64_t token;
  int head;
};
__device__ __forceinline__ Row row_of(const Args& a, const Work& w, int row) {
  const int token = divide(row, a.by_group);
  return {w.t.first + token, w.head * a.group + row - token * a.group};
}

// A wave's rows, finished.
template <int D>
__device__ __forceinline__ void finish(const State<D>& s, const Args& a, const Work& w, int row) {
  const int lane = opaque_lane();
  if (row >= w.t.rows) return;
  const Row r = row_of(a, w, row);
  const float inv = inverse_of(s.l);
  uint16_t* p = a.out + r.token * a.out_token + r.head * a.out_head;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = 32 * db + 8 * i + 4 * (lane >> 5);
      const uint32_t lo = pack_bf16x2(s.o[db][4 * i] * inv, s.o[db][4 * i + 1] * inv);
      const uint32_t hi = pack_bf16x2(s.o[db][4 * i + 2] * inv, s.o[db][4 * i + 3] * inv);
      if (d < a.dim)
        *reinterpret_cast<uint64_t*>(p + d) = lo | static_cast<uint64_t>(hi) << 32;
    }
  if (a.lse != nullptr && lane < 32) a.lse[r.token * a.heads + r.head] = lse_of(a, s.m, s.l);
}

// A part's results in the workspace: ROWS rows of D outputs, then the rows' maxima
// and sums; its first float.  A unit's first place is for the tile that it begins
// in, its second for the one that begins within it.
template <int D, int ROWS>
__device__ __forceinline__ uint32_t part_at(const Args& a, const Work& w, int part) {
  const uint32_t place = 2u * (w.unit + part) + (part == 0 ? w.inside : 0);
  return (place * a.kv_heads + w.head) * (ROWS * (D + 2));
}
// Stores and loads of them at device scope (sc1: past the die's own L2).
constexpr int kDeviceScope = 16;
__device__ __forceinline__ buffer_rsrc_t parts_rsrc(const Args& a) {
  return make_rsrc(a.partial, a.partial_bytes);
}
__device__ __forceinline__ void publish_quad(buffer_rsrc_t parts, uint32_t at, f32x4 v) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), parts, at * 4, 0,
                                         kDeviceScope);
}
__device__ __forceinline__ f32x4 fetch_quad(buffer_rsrc_t parts, uint32_t at) {
  return __builtin_bit_cast(
      f32x4, __builtin_amdgcn_raw_buffer_load_b128(parts, at * 4, 0, kDeviceScope));
}

// All parts of a tile joined by its workgroup, in their order: first the rows'
// maxima and sums over all parts, then, kMost parts at a time, each part's weight of
// each row into LDS and four columns of a row a thread and turn, the reads of kTurns
// turns and kParts parts in flight together.  Of few rows the parts are dealt to
// several threads, which meet in LDS.
template <int D, int ROWS>
__device__ __forceinline__ void join(const Args& a, const Work& w, char* smem) {
  const buffer_rsrc_t all = parts_rsrc(a);
  constexpr int kQuads = D / 4;
  constexpr int kTurns = ROWS == kFew ? 1 : 4, kParts = ROWS == kFew ? 8 : 4;
  constexpr int kMost = ROWS == kFew ? kWave : 16;
  const int rows = min(ROWS, w.t.rows - w.t.row0), items = rows * kQuads;
  const int thread = static_cast<int>(threadIdx.x);
  const int lane = thread & (kWave - 1), wave = thread / kWave;
  float* weight = reinterpret_cast<float*>(smem);           // [kMost][ROWS]
  float2_t* total = reinterpret_cast<float2_t*>(weight + kMost * ROWS);  // maximum, 1 / sum
  f32x4* meet = reinterpret_cast<f32x4*>(total + ROWS);     // [kThreads]
  const auto most_of = [&](int part, int row) {
    return fetch(a.partial + part_at<D, ROWS>(a, w, part) + ROWS * D + row);
  };
  const auto sum_of = [&](int part, int row) {
    return fetch(a.partial + part_at<D, ROWS>(a, w, part) + ROWS * (D + 1) + row);
  };
  const auto finished = [&](int row, float m, float l) {
    total[row] = float2_t{m, inverse_of(l)};
    const Row r = row_of(a, w, w.t.row0 + row);
    if (a.lse != nullptr) a.lse[r.token * a.heads + r.head] = lse_of(a, m, l);
  };
  if constexpr (ROWS == kFew) {  // a lane a part
#pragma unroll 1
    for (int row = wave; row < rows; row += kNW) {
      float m = kNegInf, l = 0.0f;
#pragma unroll 1
      for (int p = lane; p < w.parts; p += kWave) {
        const float own = most_of(p, row), sum = sum_of(p, row);
        const float raised = fmax_nan(m, own);
        l = l * weight_of(a, m, raised) + sum * weight_of(a, own, raised);
        m = raised;
      }
      const float raised = wave_reduce(m, MaxOp());
      l = wave_reduce(l * weight_of(a, m, raised), SumOp());
      if (lane == 0) finished(row, raised, l);
    }
  } else if (thread < rows) {  // a thread a row
    float m = kNegInf, l = 0.0f;
#pragma unroll 4
    for (int p = 0; p < w.parts; ++p) {
      const float own = most_of(p, thread), sum = sum_of(p, thread);
      const float raised = fmax_nan(m, own);
      l = l * weight_of(a, m, raised) + sum * weight_of(a, own, raised);
      m = raised;
    }
    finished(thread, m, l);
  }
  __syncthreads();
  // Threads of a (row, quad).
  const int several = items * 2 > kThreads ? 1 : kThreads / items;
  const int which = several > 1 ? thread / items : 0;
  const int own = several > 1 ? thread - which * items : thread;
#pragma unroll 1
  for (int turn = 0; turn * kThreads < items; turn += kTurns) {
    f32x4 o[kTurns];
    int item[kTurns];
#pragma unroll
    for (int n = 0; n < kTurns; ++n) {
      o[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      item[n] = min(own + (several > 1 ? 0 : (turn + n) * kThreads), items - 1);
    }
#pragma unroll 1
    for (int p0 = 0; p0 < w.parts; p0 += kMost) {
      const int parts = min(kMost, w.parts - p0);
      if (turn == 0 || w.parts > kMost) {
        __syncthreads();
#pragma unroll 2
        for (int i = thread; i < parts * rows; i += kThreads) {
          const int p = i / rows, row = i - p * rows;
          const float2_t of = total[row];
          weight[p * ROWS + row] = weight_of(a, most_of(p0 + p, row), of.x) * of.y;
        }
        __syncthreads();
      }
#pragma unroll 1
      for (int p1 = which; p1 < parts; p1 += several * kParts) {
        f32x4 v[kParts][kTurns];
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
          const uint32_t at = part_at<D, ROWS>(a, w, p0 + min(p1 + p * several, parts - 1));
#pragma unroll
          for (int n = 0; n < kTurns; ++n) v[p][n] = fetch_quad(all, at + 4 * item[n]);
        }
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
          const int part = p1 + p * several;
#pragma unroll
          for (int n = 0; n < kTurns; ++n) {
            const float f = weight[min(part, parts - 1) * ROWS + item[n] / kQuads];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              o[n][e] = part < parts ? __builtin_fmaf(v[p][n][e], f, o[n][e]) : o[n][e];
          }
        }
      }
    }
    if (several > 1) {
      meet[thread] = o[0];
      __syncthreads();
      for (int n = 1; n < several && which == 0; ++n) o[0] += meet[n * items + own];
    }
#pragma unroll
    for (int n = 0; n < kTurns; ++n) {
      const int i = own + (several > 1 ? 0 : (turn + n) * kThreads);
      if (i >= items || (several > 1 && (n > 0 || which > 0))) continue;
      const int row = i / kQuads, d = i % kQuads * 4;
      if (d >= a.dim) continue;
      const Row r = row_of(a, w, w.t.row0 + row);
      *reinterpret_cast<uint64_t*>(a.out + r.token * a.out_token + r.head * a.out_head + d) =
          pack_bf16x2(o[n][0], o[n][1]) |
          static_cast<uint64_t>(pack_bf16x2(o[n][2], o[n][3])) << 32;
    }
  }
}

// A step's positions through registers into LDS, for pages of any size: W waves
// copy ROWS positions from j0 on.  Those from `end` on are not read: their values are
// 0, as those of pages outside the cache, whose keys are NaN.
template <int D, int ROWS, int W>
__device__ __forceinline__ void copy_step(const Args& a, const int32_t* pages, int head, int j0,
                                          int end, int thread, char* key, char* value) {
#pragma unroll 2
  for (int i = 0; i < ROWS * Lds<D>::kChunks / (kWave * W); ++i) {
    const int at = thread + i * kWave * W;
    const int row = at / Lds<D>::kChunks, chunk = at % Lds<D>::kChunks;
    const int j = j0 + row;
    u32x4 k = {0, 0, 0, 0}, v = k;
    if (j < end && chunk * 8 < a.dim) {
      const int column = divide(j, a.by_page);
      const int page = pages[column];
      if (page >= 0 && page < a.n_pages) {
        const int64_t slot = j - column * a.page_size;
        k = *reinterpret_cast<const u32x4*>(a.k.data + page * a.k.page + slot * a.k.slot +
                                            head * a.k.head + chunk * 8);
        v = *reinterpret_cast<const u32x4*>(a.v.data + page * a.v.page + slot * a.v.slot +
                                            head * a.v.head + chunk * 8);
      } else {
        k = u32x4{0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u};
      }
    }
    *reinterpret_cast<u32x4*>(key + Lds<D>::key(row, chunk)) = k;
    *reinterpret_cast<u32x4*>(value + Lds<D>::value(row, chunk)) = v;
  }
}

// One LDS-direct load: 16 bytes a lane from offset `off` of the resource to LDS at
// `lds` + AT + 16 lane.  In inline assembly, as the compiler would wait for every
// such load before any read of LDS; the waits are those written below.  s_nop covers
// the write of M0, which nothing else here reads.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// NT: with the nontemporal hint.
template <uint32_t AT, bool NT>
__device__ __forceinline__ void load_to_lds(buffer_rsrc_t rsrc, uint32_t off, uint32_t lds) {
  if constexpr (NT)
    asm volatile(
        "s_add_u32 m0, %2, %3\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %0, %1, 0 offen nt lds"
        :
        : "v"(off), "s"(rsrc), "s"(lds), "i"(AT)
        : "memory", "m0", "scc");
  else
    asm volatile(
        "s_add_u32 m0, %2, %3\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %0, %1, 0 offen lds"
        :
        : "v"(off), "s"(rsrc), "s"(lds), "i"(AT)
        : "memory", "m0", "scc");
}
#pragma clang diagnostic pop
// s_waitcnt vmcnt(N), the other counters at their maxima.
template <int N>
__device__ __forceinline__ void wait_loads() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(((N >> 4) << 14) | (0xF << 8) | (0x7 << 4) | (N & 15));
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}
// Every read of LDS has returned.
__device__ __forceinline__ void wait_reads() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0xC07F);
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// Keys of pages that are not there: NaN.
__device__ const u32x4 kNoKeys = {0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u};

typedef const __attribute__((address_space(4))) int32_t* scalar_i32_t;

// The same step without registers, where whole pieces of PIECE rows lie in one page
// (page_size a multiple of PIECE): a piece's address is uniform, and rows behind
// `end`, or of a page that is not there, are out of its resource's bounds, which
// makes them 0.  A wave loads ROWS / W consecutive rows.
template <int D, int ROWS, int W, int PIECE>
struct Direct {
  static constexpr int kRows = kWave / Lds<D>::kChunks;  // of a load
  static constexpr int kMine = ROWS / W;                 // of a wave
  static constexpr int kPieces = kMine / PIECE;
  static constexpr int kLoads = PIECE / kRows;  // of a piece, of keys or values
  static constexpr int kPer = kMine / kRows;    // of a step, of keys or values
  // Loads apart whose rows swizzle alike.
  static constexpr int kTurn = kPer < 16 / kRows ? kPer : 16 / kRows;
  int page[kPieces];
  uint32_t k_off[kTurn], v_off[kTurn];

  // Byte offsets of the lanes' loads within a piece: row and the chunk that lands
  // at the lane's place.
  __device__ __forceinline__ void init(const Args& a, int lane, int wave) {
    const int in_row = lane / Lds<D>::kChunks, place = lane % Lds<D>::kChunks;
    const uint32_t bytes = static_cast<uint32_t>(a.dim) * 2u;
#pragma unroll
    for (int i = 0; i < kTurn; ++i) {
      const int r = wave * kMine + i * kRows + in_row;
      const uint32_t ck = Lds<D>::key(r, place) - r * Lds<D>::kRowBytes;
      const uint32_t cv = Lds<D>::value(r, place) - r * Lds<D>::kRowBytes;
      const uint32_t row = static_cast<uint32_t>(i % kLoads * kRows + in_row) * 2u;
      k_off[i] = ck < bytes ? row * static_cast<uint32_t>(a.k.slot) + ck : 0xFFFFFFF0u;
      v_off[i] = cv < bytes ? row * static_cast<uint32_t>(a.v.slot) + cv : 0xFFFFFFF0u;
    }
  }
  // The pages of the step at j0, ahead of its loads.
  __device__ __forceinline__ void look_up(const Args& a, const int32_t* pages, int j0, int end,
                                          int wave) {
    const scalar_i32_t table = (scalar_i32_t)(reinterpret_cast<uintptr_t>(pages));
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
      page[i] = table[divide(min(j0 + wave * kMine + i * PIECE, end - 1), a.by_page)];
  }
  // KEYS: the keys, else the values.  lds: of the wave's first row of them.
  template <bool KEYS, bool NT>
  __device__ __forceinline__ void load(const Args& a, int head, int j0, int end, int wave,
                                       uint32_t lds) const {
    unrolled<kPieces>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      const int j = j0 + wave * kMine + i * PIECE;
      const int n = min(max(end - j, 0), PIECE);  // rows that are read
      const bool there = page[i] >= 0 && page[i] < a.n_pages;
      const int64_t at = there ? page[i] : 0;
      const int in_page = j - divide(j, a.by_page) * a.page_size;
      const Cache& c = KEYS ? a.k : a.v;
      const uint32_t extent = n > 0 ? static_cast<uint32_t>(n - 1) *
                                              static_cast<uint32_t>(c.slot) * 2u +
                                          static_cast<uint32_t>(a.dim) * 2u
                                    : 0u;
      const void* first =
          c.data + at * c.page + static_cast<int64_t>(in_page) * c.slot + head * c.head;
      const bool keys_gone = KEYS && !there;
      const buffer_rsrc_t rsrc =
          make_rsrc(uniform(keys_gone ? static_cast<const void*>(&kNoKeys) : first),
                    static_cast<uint32_t>(uniform(
                        static_cast<int>(keys_gone ? 16u : there ? extent : 0u))));
      unrolled<kLoads>([&](auto lc) {
        constexpr int l = i * kLoads + decltype(lc)::value;
        const uint32_t off = KEYS ? (there ? k_off[l % kTurn] : 0u) : v_off[l % kTurn];
        load_to_lds<l * 1024, NT>(rsrc, off, static_cast<uint32_t>(uniform(static_cast<int>(lds))));
      });
    });
  }
};

// The steps [first, last) of a tile's work.
struct Range {
  int first, last;
  int end;  // positions that any row sees end here
};
__device__ __forceinline__ Range range_of(const Args& a, const Work& w, int rows, int keys) {
  const Tile& t = w.t;
  const int last = t.ahead + divide(min(t.row0 + rows, t.rows) - 1, a.by_group);
  int low = 0;
  if (a.window > 0) low = max(0, t.ahead + divide(t.row0, a.by_group) - a.window + 1);
  const int from = low / keys, to = last < 0 ? 0 : last / keys + 1;
  return {from + w.skip, min(to, from + w.skip + w.take), last + 1};
}

__device__ __forceinline__ uint32_t* counter_of(const Args& a, const Work& w) {
  return a.arrived + (static_cast<int64_t>(w.unit) * a.kv_heads + w.head) * kGroupCounterStride;
}
// Whether this workgroup is the last of the tile's parts; its own results are
// published.
__device__ __forceinline__ bool last_of(uint32_t* counter, int parts, char* smem) {
  publish_wait();
  __syncthreads();  // smem is free, too
  uint32_t* before = reinterpret_cast<uint32_t*>(smem);
  if (threadIdx.x == 0) {
    *before = arrive(counter);
    if (*before + 1 == static_cast<uint32_t>(parts)) counter_reset(counter);
  }
  __syncthreads();
  const bool last = *before + 1 == static_cast<uint32_t>(parts);
  __syncthreads();
  return last;
}

constexpr int kKeys = attention::kKeys;

// A tile of 128 rows: 32 a wave, keys and values of 64 positions in one of two stages
// of LDS, the next step's on their way into the other (64 KiB for heads up to 128: two
// workgroups a CU, so that one's products run under the other's exponentials).  Bound
// by the matrix units and what stands between their products: a wave's step of heads
// of 128 is 32 products of 32 x 32 x 16 and the exponentials of 2048 scores.
// Measured, 32 heads over 8 key heads of 128: a prompt of 8192 550-570 us (960-1000
// TFLOP/s; a large product alone 1268), of 2048 59-62; 4 chunks of 1024 tokens over 8192
// positions 505-520 (990-1020), 512 tokens over 8192 in parts 88-93; heads of 64, a prompt
// of 4096 88 us (780), of 192 (16 heads) 146-150 (690-705); chunks of 6 sequences of up
// to 500 tokens over 6000 positions, 14 heads of 80 over 2 key heads, pages of 24, a window
// of 4096 80-88.
template <int D, int PIECE, bool PARTS>
__device__ __forceinline__ void work_on_many(const Args& a, const Work& w, char* smem) {
  constexpr int kStage = 2 * kKeys * Lds<D>::kRowBytes;
  const Tile& t = w.t;
  const Range r = range_of(a, w, kMany, kKeys);
  const int lane = opaque_lane();
  const int wave = uniform(opaque_lane_index() / kWave);
  const int row = t.row0 + 32 * wave + (lane & 31);
  const int last = row < t.rows ? t.ahead + divide(row, a.by_group) : -1;
  const int low = a.window > 0 ? last - a.window + 1 : 0;
  // What all of the wave's rows see.
  const int wave_row = t.row0 + 32 * wave;
  // Rows that are not there need no mask: nothing of theirs is written.
  const int all_last = wave_row < t.rows ? t.ahead + divide(wave_row, a.by_group) : -1;
  const int any_last =
      wave_row < t.rows ? t.ahead + divide(min(wave_row + 31, t.rows - 1), a.by_group) : -1;
  const int all_low = a.window > 0 ? any_last - a.window + 1 : 0;
  bf16x8_t q[D / 16];
  load_queries<D>(q, a, t, lane, row, w.head);
  State<D> s;
  clear(s);
  const int32_t* pages = a.pages + t.b * a.pages_ld;
  const Places places = places_of<D>(lane);
  const uint32_t lds = static_cast<uint32_t>(uniform(static_cast<int>(lds_address(smem))));
  const auto step_at = [&](int i) {
    const uint32_t k = lds + ((i - r.first) & 1) * kStage;
    const int j0 = i * kKeys;
    return Step{k, k + kStage / 2, j0, j0 + kKeys - 1 > all_last || j0 < all_low, low, last};
  };
  const auto none = [](int) {};
  if constexpr (PIECE > 0) {
    const uint32_t own = lds + wave * (kKeys / kNW) * Lds<D>::kRowBytes;
    Direct<D, kKeys, kNW, PIECE> loads;
    loads.init(a, lane, wave);
    const auto load = [&](int i) {
      const uint32_t to = own + ((i - r.first) & 1) * kStage;
      loads.template load<true, false>(a, w.head, i * kKeys, r.end, wave, to);
      loads.template load<false, false>(a, w.head, i * kKeys, r.end, wave, to + kStage / 2);
      loads.look_up(a, pages, min(i + 1, r.last - 1) * kKeys, r.end, wave);
    };
    if (r.first < r.last) {
      loads.look_up(a, pages, r.first * kKeys, r.end, wave);
      load(r.first);
    }
    walk<D, kKeys / 32>(
        s, q, places, a.scale_log2, r.first, r.last, 1, step_at,
        [&](int i) {
          // This step's loads have landed; every wave has read the step before.
          wait_loads<0>();
          lds_barrier();
          if (i + 1 < r.last) load(i + 1);
        },
        none, none, none);
  } else {
    walk<D, kKeys / 32>(
        s, q, places, a.scale_log2, r.first, r.last, 1, step_at,
        [&](int i) {
          char* to = smem + ((i - r.first) & 1) * kStage;
          copy_step<D, kKeys, kNW>(a, pages, w.head, i * kKeys, r.end,
                                   static_cast<int>(threadIdx.x), to, to + kStage / 2);
          __syncthreads();
        },
        none, none, none);
  }
  const float2_t halves = both_halves(s.l);
  s.l = halves.x + halves.y;
  if (!PARTS || w.parts == 1) {
    finish(s, a, w, row);
    return;
  }
  const uint32_t at = part_at<D, kMany>(a, w, w.part);
  const buffer_rsrc_t all = parts_rsrc(a);
  const int in_tile = 32 * wave + (lane & 31);
  if (row < t.rows) {
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        publish_quad(all, at + in_tile * D + 32 * db + 8 * i + 4 * (lane >> 5),
                     f32x4{s.o[db][4 * i], s.o[db][4 * i + 1], s.o[db][4 * i + 2],
                           s.o[db][4 * i + 3]});
  }
  if (lane < 32) {
    publish(a.partial + at + kMany * D + in_tile, s.m);
    publish(a.partial + at + kMany * (D + 1) + in_tile, s.l);
  }
  if (last_of(counter_of(a, w), w.parts, smem)) join<D, kMany>(a, w, smem);
}

template <int D, int PIECE, bool PARTS>
__global__ __launch_bounds__(kThreads, D <= 128 ? 2 : 1) void paged_attention_many_kernel(
    const Args a) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  Cursor<kMany, kKeys, PARTS> cursor;
  Work w;
  cursor.start(a);
  if constexpr (PARTS) {
    while (cursor.next(w, arguments<Args>())) {
      work_on_many<D, PIECE, true>(arguments<Args>(), w, smem);
      __syncthreads();
    }
  } else if (cursor.next(w, a)) {
    work_on_many<D, PIECE, false>(a, w, smem);
  }
}

// A wave's LDS operations run in order; this keeps the compiler to it where lanes
// read what other lanes have written.
__device__ __forceinline__ void wave_fence() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_wave_barrier();
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

using attention::kFewKeys;  // positions of a wave's step

// A tile of up to 32 rows: each wave takes every fourth step of 32 positions, with a
// stage of LDS of its own and no barrier; its keys are replaced by the next step's as
// soon as they are read, the values likewise, so that loads never stop.  Bound by HBM
// where there are steps enough, else by a chain of latencies: find the work, the first
// keys, the meeting of the waves and of the parts.  Nothing is read twice: nontemporal.
// Measured, 32 heads over 8 key heads of 128: one token over 32 positions 5.3-6.1 us, 8192
// 13.3-14.7, 131072 94-98 (5.5-5.7 TB/s); 64 sequences of 8192 327-357 us (6.0-6.6 TB/s of
// the 7.1 that reads alone reach), of up to 16384 355-363 (6.2-6.4); one key head, 512
// sequences of 8192 344 (6.2); 128 with heads of 64 402 (5.3).  Prompts with heads of 256, 4096
// tokens and 16 heads, 346 us (397 TFLOP/s): 20 to 46 of a wave's registers spill, as the
// code behind its loop has copies of the outputs and 64 hold queries; and 32 rows share a
// read of keys and values.

// LDS of a workgroup's steps, where its waves' results meet behind them.
template <int D>
constexpr size_t kFewBytes = std::max<size_t>(size_t{kNW} * 2 * kFewKeys * Lds<D>::kRowBytes,
                                              size_t{kNW} * kFew * (D + 4) * sizeof(float));

template <int D, int PIECE, bool PARTS>
__device__ __forceinline__ void work_on_few(const Args& a, const Work& w, char* smem) {
  using Rows = float[kNW][kFew];
  Rows& ms = *reinterpret_cast<Rows*>(smem + kFewBytes<D>);  // the waves' maxima, sums
  Rows& ls = *reinterpret_cast<Rows*>(smem + kFewBytes<D> + sizeof(Rows));
  constexpr int kStage = 2 * kFewKeys * Lds<D>::kRowBytes;
  const Tile& t = w.t;
  const Range r = range_of(a, w, kFew, kFewKeys);
  const int lane = opaque_lane();
  const int wave = uniform(opaque_lane_index() / kWave);
  const int row = t.row0 + (lane & 31);
  const int last = row < t.rows ? t.ahead + divide(row, a.by_group) : -1;
  const int low = a.window > 0 ? last - a.window + 1 : 0;
  // Rows that are not there need no mask: nothing of theirs is written.
  const int last_row = min(t.row0 + 31, t.rows - 1);
  const int all_last = t.ahead + divide(t.row0, a.by_group);
  const int all_low =
      a.window > 0 ? t.ahead + divide(last_row, a.by_group) - a.window + 1 : 0;
  bf16x8_t q[D / 16];
  load_queries<D>(q, a, t, lane, row, w.head);
  State<D> s;
  clear(s);
  const int32_t* pages = a.pages + t.b * a.pages_ld;
  char* own = smem + wave * kStage;
  const Places places = places_of<D>(lane);
  const uint32_t lds = static_cast<uint32_t>(uniform(static_cast<int>(lds_address(own))));
  const auto step_at = [&](int i) {
    const int j0 = i * kFewKeys;
    return Step{lds, lds + kStage / 2, j0, j0 + kFewKeys - 1 > all_last || j0 < all_low, low,
                last};
  };
  const auto none = [](int) {};
  if constexpr (PIECE > 0) {
    Direct<D, kFewKeys, 1, PIECE> loads;
    constexpr int kPer = Direct<D, kFewKeys, 1, PIECE>::kPer;
    loads.init(a, lane, 0);
    const auto load_keys = [&](int i) {
      loads.template load<true, true>(a, w.head, i * kFewKeys, r.end, 0, lds);
    };
    const auto load_values = [&](int i) {
      loads.template load<false, true>(a, w.head, i * kFewKeys, r.end, 0, lds + kStage / 2);
      // Of the step after this one.
      loads.look_up(a, pages, min(i + kNW, r.last - 1) * kFewKeys, r.end, 0);
    };
    const int first = r.first + wave;
    if (first < r.last) {
      loads.look_up(a, pages, first * kFewKeys, r.end, 0);
      load_keys(first);
      load_values(first);
    }
    // In flight as a step begins: its keys, then its values.  The next step's keys
    // are loaded once its own have been read, the values likewise.
    walk<D, kFewKeys / 32>(
        s, q, places, a.scale_log2, first, r.last, kNW, step_at,
        [&](int) { wait_loads<kPer>(); },
        [&](int i) {
          wait_reads();
          if (i + kNW < r.last) load_keys(i + kNW);
        },
        [&](int i) {
          // A masked step waits for its values before the next keys are loaded.
          if (i + kNW < r.last && !step_at(i).masked)
            wait_loads<kPer>();
          else
            wait_loads<0>();
        },
        [&](int i) {
          wait_reads();
          if (i + kNW < r.last) load_values(i + kNW);
        });
  } else {
    walk<D, kFewKeys / 32>(
        s, q, places, a.scale_log2, r.first + wave, r.last, kNW, step_at,
        [&](int i) {
          wave_fence();
          copy_step<D, kFewKeys, 1>(a, pages, w.head, i * kFewKeys, r.end, lane, own,
                                    own + kStage / 2);
          wave_fence();
        },
        none, none, none);
  }
  const float2_t halves = both_halves(s.l);
  s.l = halves.x + halves.y;
  // The waves' results, added in their order: rows of D and four more floats, which
  // spreads a column of rows over the banks.
  constexpr int kPitch = D + 4;
  float* sums = reinterpret_cast<float*>(smem);  // [waves][kFew][kPitch]
  if (lane < 32) {
    ms[wave][lane] = s.m;
    ls[wave][lane] = s.l;
  }
  __syncthreads();
  float m = kNegInf;
#pragma unroll
  for (int v = 0; v < kNW; ++v) m = fmaxf(m, ms[v][lane & 31]);
  const float factor = weight_of(a, s.m, m);
  if (row < t.rows) {
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4*>(sums + (wave * kFew + (lane & 31)) * kPitch + 32 * db + 8 * i +
                                  4 * (lane >> 5)) =
            f32x4{s.o[db][4 * i], s.o[db][4 * i + 1], s.o[db][4 * i + 2], s.o[db][4 * i + 3]} *
            factor;
  }
  __syncthreads();
  const int rows = min(kFew, t.rows - t.row0);
  const bool parted = PARTS && w.parts > 1;
  const uint32_t at = parted ? part_at<D, kFew>(a, w, w.part) : 0;
  const auto sum_of = [&](int in_tile, float& most) {
    most = kNegInf;
#pragma unroll
    for (int v = 0; v < kNW; ++v) most = fmaxf(most, ms[v][in_tile]);
    float l = 0.0f;
#pragma unroll
    for (int v = 0; v < kNW; ++v) l += ls[v][in_tile] * weight_of(a, ms[v][in_tile], most);
    return l;
  };
  for (int i = static_cast<int>(threadIdx.x); i < rows * (D / 4); i += kThreads) {
    const int in_tile = i / (D / 4), d = i % (D / 4) * 4;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < kNW; ++n)
      v += *reinterpret_cast<const f32x4*>(sums + (n * kFew + in_tile) * kPitch + d);
    if (parted) {
      publish_quad(parts_rsrc(a), at + in_tile * D + d, v);
    } else if (d < a.dim) {
      float most;
      v *= inverse_of(sum_of(in_tile, most));
      const Row r0 = row_of(a, w, t.row0 + in_tile);
      *reinterpret_cast<uint64_t*>(a.out + r0.token * a.out_token + r0.head * a.out_head + d) =
          pack_bf16x2(v[0], v[1]) | static_cast<uint64_t>(pack_bf16x2(v[2], v[3])) << 32;
    }
  }
  if (static_cast<int>(threadIdx.x) < kFew) {
    const int in_tile = static_cast<int>(threadIdx.x);
    float most;
    const float l = sum_of(in_tile, most);
    if (parted) {
      publish(a.partial + at + kFew * D + in_tile, most);
      publish(a.partial + at + kFew * (D + 1) + in_tile, l);
    } else if (in_tile < rows && a.lse != nullptr) {
      const Row r0 = row_of(a, w, t.row0 + in_tile);
      a.lse[r0.token * a.heads + r0.head] = lse_of(a, most, l);
    }
  }
  if constexpr (PARTS)
    if (parted && last_of(counter_of(a, w), w.parts, smem)) join<D, kFew>(a, w, smem);
}

template <int D, int PIECE, bool PARTS>
__global__ __launch_bounds__(kThreads, D <= 128 ? 2 : 1) void paged_attention_few_kernel(
    const Args a) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  Cursor<kFew, kFewKeys, PARTS> cursor;
  Work w;
  cursor.start(a);
  if constexpr (PARTS) {
    while (cursor.next(w, arguments<Args>())) {
      work_on_few<D, PIECE, true>(arguments<Args>(), w, smem);
      __syncthreads();
    }
  } else if (cursor.next(w, a)) {
    work_on_few<D, PIECE, false>(a, w, smem);
  }
}

// ------------------------------------------------------------------- host --

// A kernel with more dynamic LDS than the default limit: allowed once per process
// and kernel (the attribute belongs to the kernel, not to a device).
template <auto KERNEL>
int launch_with(const Args& a, size_t lds, hipStream_t stream, const char* name) {
  static const hipError_t err =
      hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL),
                          hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
  CREDIT_HIP(err);
  const dim3 grid(static_cast<unsigned>(a.units) * static_cast<unsigned>(a.kv_heads));
  KERNEL<<<grid, kThreads, lds, stream>>>(a);
  return check_launch(name);
}
template <int D>
int launch(const Args& a, int rows, hipStream_t stream) {
  // Pieces of 16 rows or 8, or through registers where pages hold no whole number of
  // them or a piece's offsets pass 31 bits.  us with pages of 16 / 8 / 12 positions: 64
  // sequences of 8192, one token each 343 / 346 / 602, 4 chunks of 1024 over 8192
  // 514 / 539 / 871.
  constexpr int64_t kMost = int64_t{1} << 25;
  const bool near = a.k.slot < kMost && a.v.slot < kMost;
  const auto choose = [&](auto&& with) {
    const auto parts = [&](auto piece) {
      return a.partial != nullptr ? with(piece, std::true_type{}) : with(piece, std::false_type{});
    };
    if (near && a.page_size % 16 == 0) return parts(std::integral_constant<int, 16>{});
    if (near && a.page_size % 8 == 0) return parts(std::integral_constant<int, 8>{});
    return parts(std::integral_constant<int, 0>{});
  };
  const auto few = [&](auto piece, auto parts) {
    constexpr size_t kBytes = kFewBytes<D> + 2 * sizeof(float[kNW][kFew]);
    return launch_with<
        paged_attention_few_kernel<D, decltype(piece)::value, decltype(parts)::value>>(
        a, kBytes, stream, "paged_attention_few_kernel");
  };
  if constexpr (D <= attention::kManyDim) {
    if (rows == kMany)
      return choose([&](auto piece, auto parts) {
        constexpr size_t kBytes = size_t{4} * kKeys * Lds<D>::kRowBytes;
        return launch_with<
            paged_attention_many_kernel<D, decltype(piece)::value, decltype(parts)::value>>(
            a, kBytes, stream, "paged_attention_many_kernel");
      });
  }
  return choose(few);
}

// Largest calls: rows are tokens times query heads, positions those of a row of pages.
constexpr int64_t kMaxRows = int64_t{1} << 30, kMaxPositions = int64_t{1} << 30;
constexpr int64_t kMaxSequences = int64_t{1} << 20;

int check_vectors(const Place& p, const char* name) {
  if (p.at % 16 == 0 && (p.run | p.step | p.lead) % 16 == 0) return CREDIT_OK;
  return set_error(CREDIT_ERR_ALIGNMENT, "%s: address and strides are not all multiples of 16 bytes",
                   name);
}

int attend(const credit_heads* q, const credit_pages* k_cache, const credit_pages* v_cache,
           const int32_t* pages, int64_t pages_ld, int64_t pages_cols, const int32_t* q_start,
           const int32_t* kv_len, const credit_heads* out, float* lse, int64_t tokens,
           int64_t batch, int32_t dim, float scale, int32_t window, const credit_cfg* cfg) {
  constexpr size_t kElem = sizeof(uint16_t);
  CREDIT_TRY(check_tokens(tokens, dim, attention::kMaxDim));
  if (dim % 8 != 0)
    return set_error(CREDIT_ERR_BAD_SHAPE, "dim %d is not a multiple of 8", dim);
  if (batch < 0 || batch > kMaxSequences)
    return set_error(CREDIT_ERR_BAD_SHAPE, "batch %lld outside [0, 2^20]",
                     static_cast<long long>(batch));
  Place pq, po, kc, vc;
  CREDIT_TRY(check_heads(q, "q", tokens, dim, kElem, &pq));
  CREDIT_TRY(check_output(out, "out", q, tokens, dim, kElem, &po));
  CREDIT_TRY(check_cache(k_cache, "k_cache", dim, kElem, &kc));
  CREDIT_TRY(check_cache(v_cache, "v_cache", dim, kElem, &vc));
  if (k_cache->pages != v_cache->pages || k_cache->page_size != v_cache->page_size ||
      k_cache->heads != v_cache->heads)
    return set_error(CREDIT_ERR_BAD_SHAPE, "k_cache and v_cache have different pages");
  if (q->heads % k_cache->heads != 0)
    return set_error(CREDIT_ERR_BAD_SHAPE, "%d query heads are not a multiple of %d key heads",
                     q->heads, k_cache->heads);
  if (pages_cols < 0 || pages_ld < pages_cols || pages_ld > (int64_t{1} << 40) ||
      static_cast<double>(pages_cols) * k_cache->page_size > static_cast<double>(kMaxPositions))
    return set_error(CREDIT_ERR_BAD_SHAPE,
                     "pages: rows of %lld entries, %lld apart, of %d positions each",
                     static_cast<long long>(pages_cols), static_cast<long long>(pages_ld),
                     k_cache->page_size);
  if (static_cast<double>(tokens) * q->heads > static_cast<double>(kMaxRows))
    return set_error(CREDIT_ERR_BAD_SHAPE, "%lld tokens of %d heads are more than 2^30 rows",
                     static_cast<long long>(tokens), q->heads);
  const int64_t sequences = tokens == 0 ? 0 : batch;
  if (pages_cols > 0) CREDIT_TRY(check_row_ptr(pages, "pages", sequences));
  CREDIT_TRY(check_row_ptr(q_start, "q_start", sequences));
  CREDIT_TRY(check_row_ptr(kv_len, "kv_len", sequences));
  CREDIT_TRY(check_aligned(pages, 4, "pages"));
  CREDIT_TRY(check_aligned(q_start, 4, "q_start"));
  CREDIT_TRY(check_aligned(kv_len, 4, "kv_len"));
  CREDIT_TRY(check_aligned(lse, 4, "lse"));
  if (!(scale > 0.0f) || !__builtin_isfinite(scale) || !__builtin_isfinite(scale * 1.5f))
    return set_error(CREDIT_ERR_BAD_CONFIG, "scale %g is not a finite number above 0", scale);
  if (window < 0) return set_error(CREDIT_ERR_BAD_CONFIG, "window %d is negative", window);
  CREDIT_TRY(check_only_auto(cfg));
  if (sequences == 0) return CREDIT_OK;
  CREDIT_TRY(check_vectors(pq, "q"));
  CREDIT_TRY(check_vectors(po, "out"));
  CREDIT_TRY(check_vectors(kc, "k_cache"));
  CREDIT_TRY(check_vectors(vc, "v_cache"));
  CREDIT_TRY(check_places_apart(po, "out", pq, "q"));
  CREDIT_TRY(check_places_apart(po, "out", kc, "k_cache"));
  CREDIT_TRY(check_places_apart(po, "out", vc, "v_cache"));
  const NamedPlace table{Place{reinterpret_cast<uintptr_t>(pages), pages_ld * 4, 0, batch, 1,
                               pages_cols * 4},
                         "pages"};
  const NamedPlace starts{flat_place(q_start, batch + 1, 4), "q_start"};
  const NamedPlace lengths{flat_place(kv_len, batch, 4), "kv_len"};
  CREDIT_TRY(check_outputs_apart({{po, "out"}}, {table, starts, lengths}));
  CREDIT_TRY(check_outputs_apart(
      {{flat_place(lse, tokens * q->heads, sizeof(float)), "lse"}},
      {{pq, "q"}, {po, "out"}, {kc, "k_cache"}, {vc, "v_cache"}, table, starts, lengths}));
  Args a{};
  a.q = static_cast<const uint16_t*>(q->data);
  a.q_token = q->token_stride;
  a.q_head = q->head_stride;
  const auto cache = [](const credit_pages* c) {
    return Cache{static_cast<const uint16_t*>(c->data), c->page_stride, c->slot_stride,
                 c->head_stride};
  };
  a.k = cache(k_cache);
  a.v = cache(v_cache);
  a.pages = pages;
  a.pages_ld = pages_ld;
  a.q_start = q_start;
  a.kv_len = kv_len;
  a.out = static_cast<uint16_t*>(out->data);
  a.out_token = out->token_stride;
  a.out_head = out->head_stride;
  a.lse = lse;
  a.tokens = tokens;
  a.batch = static_cast<int>(batch);
  a.heads = q->heads;
  a.kv_heads = k_cache->heads;
  a.group = a.heads / a.kv_heads;
  a.dim = dim;
  a.page_size = k_cache->page_size;
  a.n_pages = static_cast<int>(k_cache->pages);
  a.positions = static_cast<int>(pages_cols * k_cache->page_size);
  a.by_page = attention::divisor(a.page_size);
  a.by_group = attention::divisor(a.group);
  // A window of at least the positions that there may be hides none of them.  Those
  // left are below 2^30, as are rows: a border of theirs lies within 32 bits, also
  // where a sequence has fewer positions than new tokens.
  a.window = window = window < a.positions ? window : 0;
  a.scale = scale;
  a.scale_log2 = static_cast<float>(1.44269504088896340736 * static_cast<double>(scale));
  const int rows =
      attention::tile_rows(tokens, batch, a.heads, a.kv_heads, dim, a.positions);
  a.tiles = static_cast<int>(attention::tiles(tokens, batch, a.group, rows));
  attention::Parts parts = attention::parts(tokens, batch, a.heads, a.kv_heads, dim,
                                             a.positions, window);
  hipStream_t stream = cfg_stream(cfg);
  if (static_cast<int64_t>(parts.units) * a.kv_heads > kMaxGroupsPerLaunch ||
      ((cfg == nullptr || cfg->workspace == nullptr) && !keeps_scratch(stream)))
    parts.units = 0;
  a.units = parts.units > 0 ? parts.units : a.tiles;
  if (static_cast<int64_t>(a.units) * a.kv_heads > (int64_t{1} << 23))
    return set_error(CREDIT_ERR_BAD_SHAPE, "%d tiles of %d key heads are too many for a launch",
                     a.units, a.kv_heads);
  if (parts.units > 0) {
    a.least_steps = parts.least_steps;
    char* base = nullptr;
    const size_t bytes =
        attention::workspace(tokens, batch, a.heads, a.kv_heads, dim, a.positions, window);
    CREDIT_TRY(acquire_workspace(cfg, bytes, &base));
    a.partial_bytes = static_cast<uint32_t>(bytes);
    a.partial = reinterpret_cast<float*>(ws_scratch(base));
    a.arrived = ws_counters(base) + kGroupCounterBase;
  }
  switch (attention::padded_dim(dim)) {
    case 64:
      return launch<64>(a, rows, stream);
    case 96:
      return launch<96>(a, rows, stream);
    case 128:
      return launch<128>(a, rows, stream);
    case 192:
      return launch<192>(a, rows, stream);
    default:
      return launch<256>(a, rows, stream);
  }
}

}  // namespace
}  // namespace credit

using namespace credit;

extern "C" {

int credit_paged_attention_bf16(const credit_heads* q, const credit_pages* k_cache,
                                const credit_pages* v_cache, const int32_t* pages,
                                int64_t pages_ld, int64_t pages_cols, const int32_t* q_start,
                                const int32_t* kv_len, const credit_heads* out, float* lse,
                                int64_t tokens, int64_t batch, int32_t dim, float scale,
                                int32_t window, const credit_cfg* cfg) {
  return attend(q, k_cache, v_cache, pages, pages_ld, pages_cols, q_start, kv_len, out, lse,
                tokens, batch, dim, scale, window, cfg);
}

size_t credit_paged_attention_workspace_bytes(int64_t tokens, int64_t batch, int32_t q_heads,
                                              int32_t kv_heads, int32_t dim, int64_t positions) {
  // What the call refuses takes none, and sizes of its range keep the rules in theirs.
  if (tokens <= 0 || tokens > kMaxRows || batch <= 0 || batch > kMaxSequences || q_heads <= 0 ||
      kv_heads <= 0 || q_heads % kv_heads != 0 || tokens * q_heads > kMaxRows || dim <= 0 ||
      dim > attention::kMaxDim || dim % 8 != 0 || positions <= 0 || positions > kMaxPositions)
    return 0;
  const size_t body =
      attention::workspace(tokens, batch, q_heads, kv_heads, dim, positions, 0);
  return body == 0 ? 0 : kScratchOffset + body;
}

}  // extern "C"
