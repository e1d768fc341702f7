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
// taken before it) is what matrix units of this rate take.  m is raised only where
// a score passes it by 2^8, so that the usual step rescales nothing.
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
constexpr float kRaise = 8.0f;  // log2 of the weights' largest value

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) bf16x4_t lds_bf16x4_t;
typedef __attribute__((address_space(3))) void* lds_ptr_t;

// Four positions of one element (column) for each lane of a group of 16: lane j of
// it addresses row j / 4, columns 4 (j % 4) .. + 3, and gets column j of the rows.
__device__ __forceinline__ bf16x4_t read_transposed(const char* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
      reinterpret_cast<lds_bf16x4_t*>((lds_ptr_t)(const_cast<char*>(p))));
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
  float* partial;
  uint32_t* arrived;
  int64_t tokens;
  int batch, heads, kv_heads, group, dim;
  int page_size, n_pages, positions;  // positions: most that a row of pages holds
  Divisor by_page, by_group;
  int window, parts, tiles;
  float scale, scale_log2;  // scale, scale log2(e)
};

__device__ __forceinline__ int divide(int n, const Divisor& d) {
  return static_cast<int>(
      (__umulhi(static_cast<uint32_t>(n), d.mul) + static_cast<uint32_t>(n)) >> d.shift);
}

// A tile: rows row0 .. of sequence b, whose token i sees positions up to ahead + i.
struct Tile {
  int b;
  int64_t first;  // token of the sequence's row 0
  int rows, row0;
  int kv, ahead;
};
__device__ __forceinline__ int64_t start_of(const Args& a, int b) {
  const int64_t s = a.q_start[b];
  return s < 0 ? 0 : s < a.tokens ? s : a.tokens;
}
// False: no rows here.
template <int ROWS>
__device__ __forceinline__ bool find_tile(Tile& t, const Args& a, int index) {
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  int lo = 0, n = a.batch;
  while (n > 1) {
    const int step = (n + kWave - 1) / kWave;
    const int b = lo + lane * step;
    const bool at = lane * step < n &&
                    start_of(a, b) * a.group / ROWS + b <= static_cast<int64_t>(index);
    const int count = __builtin_popcountll(__builtin_amdgcn_ballot_w64(at));
    if (count == 0) return false;
    const int skip = (count - 1) * step;
    lo += skip;
    n = min(step, n - skip);
  }
  t.b = __builtin_amdgcn_readfirstlane(lo);
  t.first = start_of(a, t.b);
  const int64_t slot = t.first * a.group / ROWS + t.b;
  const int64_t rows = (start_of(a, t.b + 1) - t.first) * a.group;
  const int64_t row0 = (index - slot) * ROWS;
  if (row0 < 0 || row0 >= rows) return false;
  t.rows = static_cast<int>(rows);
  t.row0 = static_cast<int>(row0);
  const int kv = a.kv_len[t.b];
  t.kv = kv < 0 ? 0 : kv < a.positions ? kv : a.positions;
  t.ahead = t.kv - t.rows / a.group;
  return true;
}

// Layout of a step's keys and values in LDS: rows of D elements, 16-byte chunk c
// of row r at place c ^ swizzle(r), so that the reads below meet no bank twice:
// of the keys 16 rows' same chunk, of the values 4 rows' 64 bytes.
template <int D>
struct Lds {
  static constexpr int kChunks = D / 8;
  static constexpr int kRowBytes = D * 2;
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

// The lane, opaque to the compiler: what is derived from it within a step is not
// kept in registers from step to step.
__device__ __forceinline__ int opaque_lane() { return opaque_lane_index() & (kWave - 1); }

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32); }

// The queries of a wave's rows: lane l holds elements 16 ks + 8 (l / 32) .. + 7 of
// row l % 32.
template <int D>
__device__ __forceinline__ void load_queries(bf16x8_t (&q)[D / 16], const Args& a, const Tile& t,
                                             int row, int kv_head) {
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
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

// A fragment of V^T: column 32 db + l % 32 of the 16 positions from 16 ts on, in
// the weights' order (element e: position 16 ts + 8 (e / 4) + 4 (l / 32) + e % 4).
template <int D>
__device__ __forceinline__ bf16x8_t value_fragment(const char* v, int lane, int db, int ts) {
  const int row = 16 * ts + 4 * (lane >> 5) + ((lane & 15) >> 2);
  const int column = 32 * db + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  const int at = Lds<D>::value(row, column >> 3) + (column & 7) * 2;
  const bf16x4_t lo = read_transposed(v + at);
  // 8 rows on: the swizzle is the same.
  const bf16x4_t hi = read_transposed(v + at + 8 * Lds<D>::kRowBytes);
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// In steps where a mask hides positions from some rows, a value that is not finite
// would make NaN of its weight of 0: whether there are any among `ROWS` rows.
template <int D, int ROWS>
__device__ __forceinline__ bool any_special(const char* v) {
  const int lane = opaque_lane();
  uint32_t bad = 0;
#pragma unroll 4
  for (int i = 0; i < ROWS * Lds<D>::kRowBytes / (16 * kWave); ++i) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(v + (i * kWave + lane) * 16);
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
__device__ __forceinline__ void add_special(State<D>& s, const char* v, int j0, int low,
                                            int last) {
#pragma unroll 1
  for (int r = 0; r < ROWS; ++r) {
    const int lane = opaque_lane();
    const bool seen = j0 + r >= low && j0 + r <= last;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int column = 32 * db + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
        const uint16_t bits = *reinterpret_cast<const uint16_t*>(
            v + Lds<D>::value(r, column >> 3) + (column & 7) * 2);
        s.o[db][i] += seen && (bits & 0x7F80u) == 0x7F80u ? bf16_to_f32(bits) : 0.0f;
      }
  }
}

// One step: NB blocks of 32 positions from j0 on, keys at k, values at v in LDS.
// MASKED: a row sees those in [low, last] alone.
template <int D, int NB, bool MASKED>
__device__ __forceinline__ void step(State<D>& s, const bf16x8_t (&q)[D / 16], const char* k,
                                     const char* v, int j0, int low, int last, float scale_log2) {
  const int lane = opaque_lane();
  f32x16 x[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[nb][i] = 0.0f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const int row = 32 * nb + (lane & 31);
      const bf16x8_t f = *reinterpret_cast<const bf16x8_t*>(
          k + Lds<D>::key(row, 2 * ks + (lane >> 5)));
      x[nb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f, q[ks], x[nb], 0, 0, 0);
    }
  }
  float m = kNegInf;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if constexpr (MASKED) {
        const int j = j0 + 32 * nb + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
        x[nb][i] = j >= low && j <= last ? x[nb][i] : kNegInf;
      }
      m = fmaxf(m, x[nb][i]);
    }
  m = fmaxf(m, other_half(m));
  if (__builtin_amdgcn_ballot_w64((m - s.m) * scale_log2 > kRaise ||
                                  (s.m == kNegInf && m != kNegInf)) != 0) {
    const float raised = fmaxf(s.m, m);
    const float by = __builtin_amdgcn_exp2f((s.m - base_of(raised)) * scale_log2);
    const float factor = s.m == kNegInf ? 0.0f : by;
    s.m = raised;
    s.l *= factor;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) s.o[db][i] *= factor;
  }
  const float base = base_of(s.m) * scale_log2;
  bf16x8_t p[2 * NB];
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
  s.l += sum;
  const bool special = MASKED && any_special<D, 32 * NB>(v);
  if (!special) {
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int ts = 0; ts < 2 * NB; ++ts)
        s.o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(value_fragment<D>(v, lane, db, ts), p[ts],
                                                          s.o[db], 0, 0, 0);
  } else {
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int ts = 0; ts < 2 * NB; ++ts)
        s.o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            without_special(value_fragment<D>(v, lane, db, ts)), p[ts], s.o[db], 0, 0, 0);
    add_special<D, 32 * NB>(s, v, j0, low, last);
  }
}

// The rows' outputs from o, l (of all lanes' halves) and m.
template <int D>
__device__ __forceinline__ void finish(const State<D>& s, const Args& a, const Tile& t, int row,
                                       int kv_head, int from, int to) {
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  if (row >= t.rows) return;
  const int token = divide(row, a.by_group);
  const int head = kv_head * a.group + row - token * a.group;
  const float inv = s.l == 0.0f ? 0.0f : 1.0f / s.l;
  uint16_t* p = a.out + (t.first + token) * a.out_token + head * a.out_head;
#pragma unroll
  for (int db = 0; db < D / 32; ++db) {
    if (db < from || db >= to) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = 32 * db + 8 * i + 4 * (lane >> 5);
      // l = 0: nothing was seen and o is 0.
      const uint32_t lo = pack_bf16x2(s.o[db][4 * i] * inv, s.o[db][4 * i + 1] * inv);
      const uint32_t hi = pack_bf16x2(s.o[db][4 * i + 2] * inv, s.o[db][4 * i + 3] * inv);
      if (d < a.dim)
        *reinterpret_cast<uint64_t*>(p + d) = lo | static_cast<uint64_t>(hi) << 32;
    }
  }
  if (a.lse != nullptr && lane < 32 && from == 0)
    a.lse[(t.first + token) * a.heads + head] =
        s.l == 0.0f ? kNegInf : base_of(s.m) * a.scale + logf(s.l);
}

// A part's results in the workspace: per 32 rows, o in the order of its lanes, then
// m and l.
template <int D>
__device__ __forceinline__ float* part_at(const Args& a, int tile, int part, int block, int rows) {
  return a.partial + ((static_cast<int64_t>(tile) * a.parts + part) * rows + block * 32) *
                         (D + 2);
}
template <int D>
__device__ __forceinline__ void leave(float* at, const State<D>& s, int db) {
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2_t v = {s.o[db][2 * i], s.o[db][2 * i + 1]};
    publish(reinterpret_cast<double*>(at) + (db * 8 + i) * kWave + lane,
            __builtin_bit_cast(double, v));
  }
}
// All of the tile's parts joined: those of the 32 rows at block, column blocks
// from .. to.
template <int D>
__device__ __forceinline__ void join(State<D>& s, const Args& a, int tile, int parts, int block,
                                     int rows, int from, int to) {
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  clear(s);
  for (int part = 0; part < parts; ++part) {
    const float* at = part_at<D>(a, tile, part, block, rows);
    const float m = fetch(at + 32 * D + (lane & 31));
    s.m = fmaxf(s.m, m);
  }
  const float base = base_of(s.m);
  for (int part = 0; part < parts; ++part) {
    const float* at = part_at<D>(a, tile, part, block, rows);
    const float m = fetch(at + 32 * D + (lane & 31));
    const float l = fetch(at + 32 * D + 32 + (lane & 31));
    // A part that saw nothing has m = -inf and l = 0.
    const float w = m == kNegInf ? 0.0f
                                 : __builtin_amdgcn_exp2f((m - base) * a.scale_log2);
    s.l += m == kNegInf ? l : l * w;
#pragma unroll
    for (int db = 0; db < D / 32; ++db) {
      if (db < from || db >= to) continue;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2_t v = __builtin_bit_cast(
            float2_t,
            fetch(reinterpret_cast<const double*>(at) + (db * 8 + i) * kWave + lane));
        s.o[db][2 * i] += m == kNegInf ? v.x : v.x * w;
        s.o[db][2 * i + 1] += m == kNegInf ? v.y : v.y * w;
      }
    }
  }
}

// Steps of a wave or workgroup: positions through registers into LDS.  W waves
// load one step of ROWS positions together.
template <int D, int ROWS, int W>
struct Loader {
  static constexpr int kPer = ROWS * Lds<D>::kChunks / (kWave * W);  // 16-byte loads a lane
  u32x4 k[kPer], v[kPer];

  // Positions j0 + r, r < ROWS; those from `end` on are not read: their values
  // are 0, as those of pages outside the cache, whose keys are NaN.
  __device__ __forceinline__ void load(const Args& a, const int32_t* pages, int head, int j0,
                                       int end, int thread) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int at = thread + i * kWave * W;
      const int row = at / Lds<D>::kChunks, chunk = at % Lds<D>::kChunks;
      const int j = j0 + row;
      u32x4 kv = {0, 0, 0, 0}, vv = kv;
      if (j < end && chunk * 8 < a.dim) {
        const int column = divide(j, a.by_page);
        const int page = pages[column];
        if (page >= 0 && page < a.n_pages) {
          const int64_t slot = j - column * a.page_size;
          kv = *reinterpret_cast<const u32x4*>(a.k.data + page * a.k.page + slot * a.k.slot +
                                               head * a.k.head + chunk * 8);
          vv = *reinterpret_cast<const u32x4*>(a.v.data + page * a.v.page + slot * a.v.slot +
                                               head * a.v.head + chunk * 8);
        } else {
          kv = u32x4{0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u};
        }
      }
      k[i] = kv;
      v[i] = vv;
    }
  }
  __device__ __forceinline__ void put(char* key, char* value, int thread) const {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int at = thread + i * kWave * W;
      const int row = at / Lds<D>::kChunks, chunk = at % Lds<D>::kChunks;
      *reinterpret_cast<u32x4*>(key + Lds<D>::key(row, chunk)) = k[i];
      *reinterpret_cast<u32x4*>(value + Lds<D>::value(row, chunk)) = v[i];
    }
  }
};

// One LDS-direct load: 16 bytes a lane from offset `off` of the resource to LDS at
// `lds` + 16 lane.  In inline assembly, as the compiler would wait for every such
// load before any read of LDS; the waits are those written below.  s_nop covers
// the write of M0, which nothing else here reads.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(buffer_rsrc_t rsrc, uint32_t off, uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %0, %1, 0 offen lds"
      :
      : "v"(off), "s"(rsrc), "s"(lds)
      : "memory", "m0");
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

// The same step without registers, where the kRows rows of a wave's load lie in one
// page (page_size a multiple of kRows): its address is uniform, and rows behind
// `end`, or of a page that is not there, are out of the resource's bounds, which
// makes them 0.
template <int D, int ROWS, int W>
struct Direct {
  static constexpr int kRows = kWave / Lds<D>::kChunks;  // of a load
  static constexpr int kPer = ROWS / kRows / W;          // loads a wave, of keys or values
  int page[kPer];

  // The pages of the step at j0, ahead of its loads.
  __device__ __forceinline__ void look_up(const Args& a, const int32_t* pages, int j0, int end,
                                          int wave) {
    const scalar_i32_t table = (scalar_i32_t)(reinterpret_cast<uintptr_t>(pages));
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      page[i] = table[divide(min(j0 + (i * W + wave) * kRows, end - 1), a.by_page)];
  }
  __device__ __forceinline__ void load(const Args& a, int head, int j0, int end, int wave,
                                       uint32_t lds) const {
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    const int in_row = lane / Lds<D>::kChunks, place = lane % Lds<D>::kChunks;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int r0 = (i * W + wave) * kRows;
      const int j = min(j0 + r0, end - 1);
      const int n = min(max(end - (j0 + r0), 0), kRows);  // rows that are read
      const bool there = page[i] >= 0 && page[i] < a.n_pages;
      const int64_t at = there ? page[i] : 0;
      const int64_t slot = j - divide(j, a.by_page) * a.page_size;
      const int r = r0 + in_row;
      const int ck = Lds<D>::key(r, place) - r * Lds<D>::kRowBytes;  // bytes of a row
      const int cv = Lds<D>::value(r, place) - r * Lds<D>::kRowBytes;
      const uint32_t bytes = static_cast<uint32_t>(a.dim) * 2u;
      const auto offset = [&](int c, const Cache& cache) {
        return static_cast<uint32_t>(c) < bytes
                   ? static_cast<uint32_t>(in_row * static_cast<int>(cache.slot) * 2 + c)
                   : 0xFFFFFFF0u;
      };
      const auto extent = [&](const Cache& cache) {
        return n > 0 ? static_cast<uint32_t>((n - 1) * static_cast<int>(cache.slot)) * 2u + bytes
                     : 0u;
      };
      const uint16_t* k = a.k.data + at * a.k.page + slot * a.k.slot + head * a.k.head;
      const uint16_t* v = a.v.data + at * a.v.page + slot * a.v.slot + head * a.v.head;
      const uint32_t to = lds + static_cast<uint32_t>((i * W + wave) * 1024);
      load_to_lds(there ? make_rsrc(k, extent(a.k)) : make_rsrc(&kNoKeys, 16u),
                  there ? offset(ck, a.k) : 0u, to);
      load_to_lds(make_rsrc(v, there ? extent(a.v) : 0u), offset(cv, a.v),
                  to + ROWS * Lds<D>::kRowBytes);
    }
  }
};

// The steps of a part: [first, last) of those of `keys` positions, and how many
// parts have any.
struct Range {
  int first, last, parts;
  int end;  // positions that any row sees end here
};
__device__ __forceinline__ Range range_of(const Args& a, const Tile& t, int rows, int part,
                                          int keys) {
  const int last_row = min(t.row0 + rows, t.rows) - 1;
  const int last = t.ahead + divide(last_row, a.by_group);
  int low = 0;
  if (a.window > 0) low = max(0, t.ahead + divide(t.row0, a.by_group) - a.window + 1);
  Range r;
  r.end = last + 1;
  const int from = low / keys, to = last < 0 ? 0 : last / keys + 1;
  const int n = max(0, to - from);
  const int each = max(1, (n + a.parts - 1) / a.parts);
  r.parts = max(1, (n + each - 1) / each);
  r.first = from + part * each;
  r.last = min(to, r.first + each);
  return r;
}

// Whether this workgroup is the last of the tile's parts; its own results are
// published.
__device__ __forceinline__ bool last_of(uint32_t* counter, int parts, uint32_t* shared) {
  publish_wait();
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t before = arrive(counter);
    *shared = before;
    if (before + 1 == static_cast<uint32_t>(parts)) counter_reset(counter);
  }
  __syncthreads();
  return *shared + 1 == static_cast<uint32_t>(parts);
}

struct Work {
  int tile, part, head;
};
// Key heads next to each other: the dies take workgroups in turn, so that tiles of
// one head's keys tend to share one die's L2.  Later tiles, which see more, first.
__device__ __forceinline__ Work work_of(const Args& a) {
  const int i = static_cast<int>(blockIdx.x);
  Work w;
  w.head = i % a.kv_heads;
  const int j = i / a.kv_heads;
  w.part = j % a.parts;
  w.tile = a.tiles - 1 - j / a.parts;
  return w;
}

constexpr int kKeys = attention::kKeys;

template <int D, bool DIRECT>
__global__ __launch_bounds__(kThreads, D <= 128 ? 2 : 1) void paged_attention_many_kernel(
    const Args a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ uint32_t shared;
  constexpr int kStage = 2 * kKeys * Lds<D>::kRowBytes;
  const Work w = work_of(a);
  Tile t;
  if (!find_tile<kMany>(t, a, w.tile)) return;
  const Range r = range_of(a, t, kMany, w.part, kKeys);
  if (w.part >= r.parts) return;
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const int row = t.row0 + 32 * wave + (lane & 31);
  const int last = row < t.rows ? t.ahead + divide(row, a.by_group) : -1;
  const int low = a.window > 0 ? last - a.window + 1 : 0;
  // Of the wave's rows: what all of them see and what any does.
  const int wave_row = t.row0 + 32 * wave;
  // Rows that are not there need no mask: nothing of theirs is written.
  const int all_last = wave_row < t.rows ? t.ahead + divide(wave_row, a.by_group) : -1;
  const int any_last =
      wave_row < t.rows ? t.ahead + divide(min(wave_row + 31, t.rows - 1), a.by_group) : -1;
  const int all_low = a.window > 0 ? any_last - a.window + 1 : 0;
  const int any_low =
      a.window > 0 ? t.ahead + divide(min(wave_row, t.rows - 1), a.by_group) - a.window + 1 : 0;
  bf16x8_t q[D / 16];
  load_queries<D>(q, a, t, row, w.head);
  State<D> s;
  clear(s);
  const int32_t* pages = a.pages + t.b * a.pages_ld;
  const auto compute = [&](int i, const char* k) {
    const int j0 = i * kKeys;
    if (j0 > any_last || j0 + kKeys <= any_low) return;
    if (j0 + kKeys - 1 <= all_last && j0 >= all_low)
      step<D, kKeys / 32, false>(s, q, k, k + kStage / 2, j0, low, last, a.scale_log2);
    else
      step<D, kKeys / 32, true>(s, q, k, k + kStage / 2, j0, low, last, a.scale_log2);
  };
  if constexpr (DIRECT) {
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_ptr_t)smem;
    Direct<D, kKeys, kNW> loads;
    if (r.first < r.last) {
      loads.look_up(a, pages, r.first * kKeys, r.end, wave);
      loads.load(a, w.head, r.first * kKeys, r.end, wave, lds);
      loads.look_up(a, pages, min(r.first + 1, r.last - 1) * kKeys, r.end, wave);
    }
    for (int i = r.first; i < r.last; ++i) {
      const int stage = (i - r.first) & 1;
      // This step's loads have landed; every wave has read the step before.
      wait_loads<0>();
      lds_barrier();
      if (i + 1 < r.last) {
        loads.load(a, w.head, (i + 1) * kKeys, r.end, wave, lds + (stage ^ 1) * kStage);
        loads.look_up(a, pages, min(i + 2, r.last - 1) * kKeys, r.end, wave);
      }
      compute(i, smem + stage * kStage);
    }
  } else {
    Loader<D, kKeys, kNW> loader;
    const int thread = static_cast<int>(threadIdx.x);
    if (r.first < r.last) {
      loader.load(a, pages, w.head, r.first * kKeys, r.end, thread);
      loader.put(smem, smem + kStage / 2, thread);
    }
    for (int i = r.first; i < r.last; ++i) {
      __syncthreads();
      char* next = smem + ((i - r.first + 1) & 1) * kStage;
      const bool more = i + 1 < r.last;
      if (more) loader.load(a, pages, w.head, (i + 1) * kKeys, r.end, thread);
      compute(i, smem + ((i - r.first) & 1) * kStage);
      if (more) loader.put(next, next + kStage / 2, thread);
    }
  }
  s.l += other_half(s.l);
  const int tile = w.tile * a.kv_heads + w.head;
  if (r.parts > 1) {
    float* at = part_at<D>(a, tile, w.part, wave, kMany);
#pragma unroll
    for (int db = 0; db < D / 32; ++db) leave(at, s, db);
    if (lane < 32) {
      publish(at + 32 * D + lane, s.m);
      publish(at + 32 * D + 32 + lane, s.l);
    }
    if (!last_of(a.arrived + static_cast<int64_t>(tile) * kGroupCounterStride, r.parts, &shared))
      return;
    join(s, a, tile, r.parts, wave, kMany, 0, D / 32);
  }
  finish(s, a, t, row, w.head, 0, D / 32);
}

// A wave's LDS operations run in order; this keeps the compiler to it where lanes
// read what other lanes have written.
__device__ __forceinline__ void wave_fence() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_wave_barrier();
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// Positions of a wave's step, and its stages in LDS: two where four waves' fit.
constexpr int kFewKeys = 32;
template <int D>
constexpr int kFewStages = D <= 128 ? 2 : 1;

template <int D, bool DIRECT>
__global__ __launch_bounds__(kThreads) void paged_attention_few_kernel(const Args a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ uint32_t shared;
  __shared__ float ms[kNW][32], ls[kNW][32];
  constexpr int kStage = 2 * kFewKeys * Lds<D>::kRowBytes;
  const Work w = work_of(a);
  Tile t;
  if (!find_tile<kFew>(t, a, w.tile)) return;
  const Range r = range_of(a, t, kFew, w.part, kFewKeys);
  if (w.part >= r.parts) return;
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const int row = t.row0 + (lane & 31);
  const int last = row < t.rows ? t.ahead + divide(row, a.by_group) : -1;
  const int low = a.window > 0 ? last - a.window + 1 : 0;
  // Rows that are not there need no mask: nothing of theirs is written.
  const int last_row = min(t.row0 + 31, t.rows - 1);
  const int all_last = t.ahead + divide(t.row0, a.by_group);
  const int all_low =
      a.window > 0 ? t.ahead + divide(last_row, a.by_group) - a.window + 1 : 0;
  bf16x8_t q[D / 16];
  load_queries<D>(q, a, t, row, w.head);
  State<D> s;
  clear(s);
  const int32_t* pages = a.pages + t.b * a.pages_ld;
  char* own = smem + wave * kFewStages<D> * kStage;
  const auto compute = [&](int i, const char* k) {
    const int j0 = i * kFewKeys;
    if (j0 + kFewKeys - 1 <= all_last && j0 >= all_low)
      step<D, kFewKeys / 32, false>(s, q, k, k + kStage / 2, j0, low, last, a.scale_log2);
    else
      step<D, kFewKeys / 32, true>(s, q, k, k + kStage / 2, j0, low, last, a.scale_log2);
  };
  if constexpr (DIRECT) {
    const uint32_t lds = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(
        static_cast<int>((uint32_t)(uintptr_t)(lds_ptr_t)own)));
    Direct<D, kFewKeys, 1> loads;
    int i = r.first + wave;
    if (i < r.last) {
      loads.look_up(a, pages, i * kFewKeys, r.end, 0);
      loads.load(a, w.head, i * kFewKeys, r.end, 0, lds);
      loads.look_up(a, pages, min(i + kNW, r.last - 1) * kFewKeys, r.end, 0);
    }
    for (int stage = 0; i < r.last; i += kNW) {
      const bool more = i + kNW < r.last;
      if (kFewStages<D> == 2 && more) {
        // The other stage's step was read before this one's wait.
        wait_reads();
        loads.load(a, w.head, (i + kNW) * kFewKeys, r.end, 0, lds + (stage ^ 1) * kStage);
        loads.look_up(a, pages, min(i + 2 * kNW, r.last - 1) * kFewKeys, r.end, 0);
        wait_loads<2 * Direct<D, kFewKeys, 1>::kPer>();
      } else {
        wait_loads<0>();
      }
      compute(i, own + stage * kStage);
      if (kFewStages<D> == 2) {
        stage ^= 1;
      } else if (more) {
        wait_reads();
        loads.load(a, w.head, (i + kNW) * kFewKeys, r.end, 0, lds);
        loads.look_up(a, pages, min(i + 2 * kNW, r.last - 1) * kFewKeys, r.end, 0);
      }
    }
  } else {
    Loader<D, kFewKeys, 1> loader;
    int i = r.first + wave;
    if (i < r.last) loader.load(a, pages, w.head, i * kFewKeys, r.end, lane);
    for (; i < r.last; i += kNW) {
      loader.put(own, own + kStage / 2, lane);
      wave_fence();
      if (i + kNW < r.last)
        loader.load(a, pages, w.head, (i + kNW) * kFewKeys, r.end, lane);
      compute(i, own);
      wave_fence();
    }
  }
  s.l += other_half(s.l);
  // The waves' results, in their order.
  if (lane < 32) {
    ms[wave][lane] = s.m;
    ls[wave][lane] = s.l;
  }
  __syncthreads();
  float m = kNegInf, l = 0.0f;
#pragma unroll
  for (int v = 0; v < kNW; ++v) m = fmaxf(m, ms[v][lane & 31]);
  const float base = base_of(m);
#pragma unroll
  for (int v = 0; v < kNW; ++v) {
    const float mv = ms[v][lane & 31];
    l += mv == kNegInf ? ls[v][lane & 31]
                       : ls[v][lane & 31] * __builtin_amdgcn_exp2f((mv - base) * a.scale_log2);
  }
  const float factor = s.m == kNegInf ? 1.0f
                                      : __builtin_amdgcn_exp2f((s.m - base) * a.scale_log2);
  float* sums = reinterpret_cast<float*>(smem);  // [waves][16][64] of one column block
  s.m = m;
  s.l = l;
#pragma unroll
  for (int db = 0; db < D / 32; ++db) {
#pragma unroll
    for (int e = 0; e < 16; ++e) sums[(wave * 16 + e) * kWave + lane] = s.o[db][e] * factor;
    __syncthreads();
    if (db % kNW == wave) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float v = 0.0f;
#pragma unroll
        for (int n = 0; n < kNW; ++n) v += sums[(n * 16 + e) * kWave + lane];
        s.o[db][e] = v;
      }
    }
    __syncthreads();
  }
  const int tile = w.tile * a.kv_heads + w.head;
  const bool parted = r.parts > 1;
  if (parted) {
    float* at = part_at<D>(a, tile, w.part, 0, kFew);
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
      if (db % kNW == wave) leave(at, s, db);
    if (wave == 0 && lane < 32) {
      publish(at + 32 * D + lane, s.m);
      publish(at + 32 * D + 32 + lane, s.l);
    }
    if (!last_of(a.arrived + static_cast<int64_t>(tile) * kGroupCounterStride, r.parts, &shared))
      return;
  }
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
    if (db % kNW == wave) {
      if (parted) join(s, a, tile, r.parts, 0, kFew, db, db + 1);
      finish(s, a, t, row, w.head, db, db + 1);
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
  const dim3 grid(static_cast<unsigned>(a.tiles) * static_cast<unsigned>(a.parts) *
                  static_cast<unsigned>(a.kv_heads));
  KERNEL<<<grid, kThreads, lds, stream>>>(a);
  return check_launch(name);
}
template <int D>
int launch(const Args& a, int rows, hipStream_t stream) {
  // Rows of a load in one page, and their offsets within 31 bits.
  constexpr int kRows = Direct<D, kKeys, kNW>::kRows;
  const int64_t most = int64_t{1} << 28;
  const bool direct = a.page_size % kRows == 0 && a.k.slot < most / kRows * 2 &&
                      a.v.slot < most / kRows * 2;
  if (rows == kFew) {
    constexpr const char* kName = "paged_attention_few_kernel";
    constexpr size_t kBytes = std::max<size_t>(
        size_t{kNW} * kFewStages<D> * 2 * kFewKeys * Lds<D>::kRowBytes, kNW * 16 * kWave * 4);
    return direct ? launch_with<paged_attention_few_kernel<D, true>>(a, kBytes, stream, kName)
                  : launch_with<paged_attention_few_kernel<D, false>>(a, kBytes, stream, kName);
  }
  constexpr const char* kName = "paged_attention_many_kernel";
  constexpr size_t kBytes = size_t{4} * kKeys * Lds<D>::kRowBytes;
  return direct ? launch_with<paged_attention_many_kernel<D, true>>(a, kBytes, stream, kName)
                : launch_with<paged_attention_many_kernel<D, false>>(a, kBytes, stream, kName);
}

int check_vectors(const Place& p, const char* name) {
  if (p.at % 16 == 0 && p.run % 16 == 0 && p.step % 16 == 0) return CREDIT_OK;
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
  if (batch < 0 || batch > (1 << 20))
    return set_error(CREDIT_ERR_BAD_SHAPE, "batch %lld outside [0, 2^20]",
                     static_cast<long long>(batch));
  Place pq, po, kc, vc, kslots, vslots;
  CREDIT_TRY(check_heads(q, "q", tokens, dim, kElem, &pq));
  CREDIT_TRY(check_output(out, "out", q, tokens, dim, kElem, &po));
  CREDIT_TRY(check_cache(k_cache, "k_cache", dim, kElem, &kc, &kslots));
  CREDIT_TRY(check_cache(v_cache, "v_cache", dim, kElem, &vc, &vslots));
  if (k_cache->pages != v_cache->pages || k_cache->page_size != v_cache->page_size ||
      k_cache->heads != v_cache->heads)
    return set_error(CREDIT_ERR_BAD_SHAPE, "k_cache and v_cache have different pages");
  if (q->heads % k_cache->heads != 0)
    return set_error(CREDIT_ERR_BAD_SHAPE, "%d query heads are not a multiple of %d key heads",
                     q->heads, k_cache->heads);
  if (pages_cols < 0 || pages_ld < pages_cols || pages_ld > (int64_t{1} << 40) ||
      static_cast<double>(pages_cols) * k_cache->page_size > static_cast<double>(1 << 30))
    return set_error(CREDIT_ERR_BAD_SHAPE,
                     "pages: rows of %lld entries, %lld apart, of %d positions each",
                     static_cast<long long>(pages_cols), static_cast<long long>(pages_ld),
                     k_cache->page_size);
  if (static_cast<double>(tokens) * q->heads > static_cast<double>(1 << 30))
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
  CREDIT_TRY(check_vectors(kslots, "k_cache"));
  CREDIT_TRY(check_vectors(vc, "v_cache"));
  CREDIT_TRY(check_vectors(vslots, "v_cache"));
  CREDIT_TRY(check_places_apart(po, "out", pq, "q"));
  CREDIT_TRY(check_places_apart(po, "out", kc, "k_cache"));
  CREDIT_TRY(check_places_apart(po, "out", vc, "v_cache"));
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
  a.window = window;
  a.scale = scale;
  a.scale_log2 = static_cast<float>(1.44269504088896340736 * static_cast<double>(scale));
  const int rows = attention::tile_rows(tokens, batch, a.group);
  const int64_t tiles = attention::tiles(tokens, batch, a.group, rows);
  int64_t parts =
      attention::parts(tokens, batch, a.heads, a.kv_heads, a.positions);
  hipStream_t stream = cfg_stream(cfg);
  if (tiles * a.kv_heads > kMaxGroupsPerLaunch) parts = 1;
  if (parts > 1 && (cfg == nullptr || cfg->workspace == nullptr) && !keeps_scratch(stream))
    parts = 1;
  if (tiles * parts * a.kv_heads > (int64_t{1} << 23))
    return set_error(CREDIT_ERR_BAD_SHAPE, "%lld tiles of %d key heads are too many for a launch",
                     static_cast<long long>(tiles), a.kv_heads);
  a.parts = static_cast<int>(parts);
  a.tiles = static_cast<int>(tiles);
  if (parts > 1) {
    char* base = nullptr;
    CREDIT_TRY(acquire_workspace(
        cfg, attention::workspace(tokens, batch, a.heads, a.kv_heads, dim, a.positions), &base));
    a.partial = reinterpret_cast<float*>(ws_scratch(base));
    a.arrived = ws_counters(base) + kGroupCounterBase;
  }
  switch (attention::padded_dim(dim)) {
    case 64:
      return launch<64>(a, rows, stream);
    case 128:
      return launch<128>(a, rows, stream);
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
  if (tokens <= 0 || batch <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 ||
      dim <= 0 || dim > attention::kMaxDim || positions <= 0)
    return 0;
  const size_t body =
      attention::workspace(tokens, batch, q_heads, kv_heads, dim, positions);
  return body == 0 ? 0 : kScratchOffset + body;
}

}  // extern "C"
