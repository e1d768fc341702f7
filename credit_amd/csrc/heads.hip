// Operators on the heads of queries, keys and values: rotary positions
// (credit_rope_*), RMS norm of each head with the rotation in the same pass and
// its gradients (credit_qk_norm_rope_*), and the same on the way into a paged
// cache (credit_paged_append_*).
//
// A head is held by a group of lanes (4 to 64 of them), each with two units of N
// consecutive elements: units p and p + rot/2N of the rotated part where pairs
// are half of it apart, so that a pair never leaves its lane, else neighbours.
// The only exchange is the head's sum of squares.  A group's lanes take the sines
// and cosines of their N pairs of a token once and use them for every head that
// the group turns (groups_of).  All are bound by HBM where the rows fill the
// device, by latency, launch to last store, where they do not.
#include <math.h>

#include <mutex>
#include <type_traits>

#include "api_internal.hpp"
#include "common.hpp"
#include "heads_rules.hpp"
#include "workspace_cache.hpp"

namespace credit {
namespace {

using heads::kMaxDim;
using heads::Place;

constexpr int kThreads = 256;

template <class T, int N>
using Raw = T __attribute__((ext_vector_type(N)));
template <class T, int N>
struct Unit {
  Raw<T, N> v;
};
template <class T>
struct Unit<T, 1> {
  T v;
};
template <class T>
__device__ __forceinline__ float widen(T v) {
  if constexpr (std::is_same_v<T, float>)
    return v;
  else
    return bf16_to_f32(v);
}
template <class T, int N, bool NT = false>
__device__ __forceinline__ Unit<T, N> load_unit(const T* p) {
  Unit<T, N> u;
  if constexpr (N == 1)
    u.v = *p;
  else if constexpr (NT)
    u.v = __builtin_nontemporal_load(reinterpret_cast<const Raw<T, N>*>(p));
  else
    u.v = *reinterpret_cast<const Raw<T, N>*>(p);
  return u;
}
template <class T, int N>
__device__ __forceinline__ void widen_unit(float (&f)[N], const Unit<T, N>& u) {
  if constexpr (N == 1) {
    f[0] = widen(u.v);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = widen<T>(u.v[j]);
  }
}
template <class T, int N>
__device__ __forceinline__ Unit<T, N> narrow_unit(const float (&f)[N]) {
  Unit<T, N> u;
  if constexpr (std::is_same_v<T, float>) {
    if constexpr (N == 1) {
      u.v = f[0];
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) u.v[j] = f[j];
    }
  } else if constexpr (N == 1) {
    u.v = f32_to_bf16(f[0]);
  } else {
    uint32_t w[N / 2];
#pragma unroll
    for (int j = 0; j < N / 2; ++j) w[j] = pack_bf16x2(f[2 * j], f[2 * j + 1]);
    __builtin_memcpy(&u.v, w, sizeof(w));
  }
  return u;
}
template <class T, int N, bool NT = false>
__device__ __forceinline__ void store_unit(T* p, const Unit<T, N>& u) {
  if constexpr (N == 1)
    *p = u.v;
  else if constexpr (NT)
    __builtin_nontemporal_store(u.v, reinterpret_cast<Raw<T, N>*>(p));
  else
    *reinterpret_cast<Raw<T, N>*>(p) = u.v;
}

// The sum over the G lanes of a group, in each of them.
template <int G>
__device__ __forceinline__ float group_sum(float v) {
  if constexpr (G >= 2) v += dpp_f32<kDppXor1>(v);
  if constexpr (G >= 4) v += dpp_f32<kDppXor2>(v);
  if constexpr (G >= 8) v += dpp_f32<kDppHalfMirror>(v);
  if constexpr (G >= 16) v += dpp_f32<kDppMirror>(v);
  if constexpr (G >= 32) v += __shfl_xor(v, 16);
  if constexpr (G >= 64) v += __shfl_xor(v, 32);
  return v;
}

// sin and cos of an angle of `turns`, its nearest quarter taken off in 64 bits: of
// positions up to 2^31 more than 20 bits behind the point stay.  What is left lies in
// +-pi/4, where the Taylor polynomials of degree 9 and 10 are within 2e-9 and 1e-10 of
// the functions.
__device__ __forceinline__ void sincos_of(double turns, float& s, float& c) {
  constexpr float k2Pi = 6.28318530717958647692528f;
  const double part = turns - __builtin_rint(turns);  // [-1/2, 1/2]
  const double quarter = __builtin_rint(4.0 * part);
  const float x = static_cast<float>(__builtin_fma(quarter, -0.25, part)) * k2Pi;
  const int q = static_cast<int>(quarter);
  const float x2 = x * x;
  float ps = 1.0f / 362880.0f;
  ps = __builtin_fmaf(ps, x2, -1.0f / 5040.0f);
  ps = __builtin_fmaf(ps, x2, 1.0f / 120.0f);
  ps = __builtin_fmaf(ps, x2, -1.0f / 6.0f);
  ps = __builtin_fmaf(ps * x2, x, x);
  float pc = -1.0f / 3628800.0f;
  pc = __builtin_fmaf(pc, x2, 1.0f / 40320.0f);
  pc = __builtin_fmaf(pc, x2, -1.0f / 720.0f);
  pc = __builtin_fmaf(pc, x2, 1.0f / 24.0f);
  pc = __builtin_fmaf(pc, x2, -0.5f);
  pc = __builtin_fmaf(pc, x2, 1.0f);
  const float ss = (q & 1) != 0 ? pc : ps, cc = (q & 1) != 0 ? ps : pc;
  s = (q & 2) != 0 ? -ss : ss;
  c = ((q + 1) & 2) != 0 ? -cc : cc;
}

struct Rotation {
  const int64_t* positions;
  const float* inv_freq;
  int rot;
  int interleaved;
  float magnitude;
  float sign;  // of the angle: -1 for the transposed
  int whole;   // every element is turned
};

// The two units of lane `p` of a head and what turns them.
template <int N>
struct Seat {
  int ea, eb;     // first elements
  bool has_a, has_b, turn_a, turn_b;
};
template <int N>
__device__ __forceinline__ Seat<N> seat_of(int p, int dim, const Rotation& r) {
  Seat<N> s;
  const int half = r.rot / 2;
  int ua = 2 * p, ub = 2 * p + 1;
  // N == 1: an interleaved pair is two units of one element.
  if (r.interleaved == 0 && p * N < half) {
    ua = p;
    ub = p + half / N;
  }
  s.ea = ua * N;
  s.eb = ub * N;
  s.has_a = s.ea < dim;
  s.has_b = s.eb < dim;
  s.turn_a = s.ea < r.rot;
  s.turn_b = s.eb < r.rot;
  return s;
}
// Turns a position of lane p's pairs.
template <int N>
__device__ __forceinline__ void turns_of(double (&f)[N], int p, const Rotation& r) {
  constexpr double kInv2Pi = 0.15915494309189533576888;
#pragma unroll
  for (int j = 0; j < N; ++j)
    f[j] = p * N + j < r.rot / 2 ? static_cast<double>(r.inv_freq[p * N + j]) * kInv2Pi : 0.0;
}
template <int N>
__device__ __forceinline__ void angles_of(float (&c)[N], float (&s)[N], const double (&f)[N],
                                          int64_t token, const Rotation& r) {
  const double position = static_cast<double>(r.positions[token]);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    sincos_of(position * f[j], s[j], c[j]);
    c[j] *= r.magnitude;
    s[j] *= r.magnitude * r.sign;
  }
}
// v^(-1/2): the instruction's, within a step, and one step of Newton's method.  The
// instruction takes subnormal numbers for 0, so small ones are raised by 2^64.
__device__ __forceinline__ float inverse_root(float v) {
  const bool small = v < 0x1p-64f;
  const float u = small ? v * 0x1p64f : v;
  float r = __builtin_amdgcn_rsqf(u);
  if (u > 0.0f && u < __builtin_inff())
    r = __builtin_fmaf(0.5f * r, __builtin_fmaf(-u * r, r, 1.0f), r);
  return small ? r * 0x1p32f : r;
}
// Units without a rotated pair keep their elements, whatever the other holds.
template <int N>
__device__ __forceinline__ void turn(float (&a)[N], float (&b)[N], const float (&c)[N],
                                     const float (&s)[N], const Seat<N>& seat, const Rotation& r) {
  if (r.whole != 0 && (N == 1 || r.interleaved == 0)) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float x = a[j], y = b[j];
      a[j] = __builtin_fmaf(x, c[j], -(y * s[j]));
      b[j] = __builtin_fmaf(y, c[j], x * s[j]);
    }
  } else if (N == 1 || r.interleaved == 0) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float x = a[j], y = b[j];
      a[j] = seat.turn_a ? __builtin_fmaf(x, c[j], -(y * s[j])) : x;
      b[j] = seat.turn_a ? __builtin_fmaf(y, c[j], x * s[j]) : y;
    }
  } else if constexpr (N > 1) {
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
      const float x = a[2 * j], y = a[2 * j + 1];
      a[2 * j] = seat.turn_a ? __builtin_fmaf(x, c[j], -(y * s[j])) : x;
      a[2 * j + 1] = seat.turn_a ? __builtin_fmaf(y, c[j], x * s[j]) : y;
      const float z = b[2 * j], w = b[2 * j + 1];
      const float cb = c[N / 2 + j], sb = s[N / 2 + j];
      b[2 * j] = seat.turn_b ? __builtin_fmaf(z, cb, -(w * sb)) : z;
      b[2 * j + 1] = seat.turn_b ? __builtin_fmaf(w, cb, z * sb) : w;
    }
  }
}

// One tensor's way through the forward.
template <class T>
struct Side {
  const T* x;
  T* y;
  const T* w;     // nullptr: no norm
  float* rstd;    // nullptr: not wanted; a token's own `heads` values
  int64_t x_token, x_head, y_token, y_head, rstd_token;
  int64_t y_slot;          // with slots: y_token is the page's stride
  const int64_t* slots;    // nullptr: y by tokens
  int64_t n_slots;
  int page_size;
  int heads;
  int groups_log;          // groups of a token
  int plain;               // copied as it is
  int64_t first_block, units;
};
constexpr int kMaxSides = 3;
template <class T>
struct ForwardArgs {
  Side<T> side[kMaxSides];
  Rotation r;
  int sides, dim;
  float eps;
};

// WHOLE: lanes, units and heads go evenly: dim = 2 N G, and every unit has RUN
// heads.  NT: loads and stores with the nontemporal hint.  us without either -> with
// both, 16384 tokens of 32 + 8 heads of 128 in bf16: turned 68 -> 62, norm and rotation
// 70 -> 65, the gradients of both 122 -> 104.  Workgroups loop over units; a unit's loads are
// all on their way before the sines and cosines of its token are taken.
//
// Measured in bf16, heads of 128 (a copy reaches 5.16 TB/s): norm, rotation and rstd
// of 16384 tokens of 32 + 8 heads 65 us (5.2 TB/s), rotation alone 62 (5.4), 8192
// tokens of 32 queries, 8 keys and values into a cache 41 (4.9); in fp32 8192 tokens
// normed and turned 61 (5.5).  64 tokens 4.8 us, one 4.3, a cache's 64 5.0: launch,
// loads, sines and stores one behind the other.
template <class T, int N, int G, int U, int RUN, bool WHOLE, bool NT>
__global__ __launch_bounds__(kThreads) void heads_fwd_kernel(const ForwardArgs<T> a) {
  int which = 0;
  if (a.sides > 1 && blockIdx.x >= a.side[1].first_block) which = 1;
  if (a.sides > 2 && blockIdx.x >= a.side[2].first_block) which = 2;
  const Side<T>& side = a.side[which];
  const int64_t blocks =
      (which + 1 < a.sides ? a.side[which + 1].first_block : static_cast<int64_t>(gridDim.x)) -
      side.first_block;
  const int lane = static_cast<int>(threadIdx.x) % G;
  const int groups = 1 << side.groups_log;
  const bool turned = a.r.rot > 0 && side.plain == 0;
  Seat<N> seat[U];
  double freq[U][N];
  float wa[U][N], wb[U][N];
  const bool norm = side.w != nullptr;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    seat[u] = seat_of<N>(lane + G * u, a.dim, a.r);
    if constexpr (WHOLE) seat[u].has_a = seat[u].has_b = true;
#pragma unroll
    for (int j = 0; j < N; ++j) wa[u][j] = wb[u][j] = 0.0f;
    if (norm) {
      if (seat[u].has_a) widen_unit<T, N>(wa[u], load_unit<T, N>(side.w + seat[u].ea));
      if (seat[u].has_b) widen_unit<T, N>(wb[u], load_unit<T, N>(side.w + seat[u].eb));
    }
    if (turned) turns_of<N>(freq[u], lane + G * u, a.r);
  }
  const float inv_dim = 1.0f / static_cast<float>(a.dim);
  for (int64_t unit = (blockIdx.x - side.first_block) * (kThreads / G) +
                      static_cast<int>(threadIdx.x) / G;
       unit < side.units; unit += blocks * (kThreads / G)) {
    const int64_t token = unit >> side.groups_log;
    const int first = static_cast<int>(unit & (groups - 1));
    if (!WHOLE && first >= side.heads) continue;
    const T* x = side.x + token * side.x_token + first * side.x_head;
    const int64_t x_step = groups * side.x_head, y_step = groups * side.y_head;
    // On their way while the angles are taken.
    Unit<T, N> ra[RUN][U], rb[RUN][U];
#pragma unroll
    for (int k = 0; k < RUN; ++k) {
      const T* p = x + (WHOLE || first + k * groups < side.heads ? k : 0) * x_step;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        ra[k][u].v = 0;
        rb[k][u].v = 0;
        if (seat[u].has_a) ra[k][u] = load_unit<T, N, NT>(p + seat[u].ea);
        if (seat[u].has_b) rb[k][u] = load_unit<T, N, NT>(p + seat[u].eb);
      }
    }
    T* y = side.y + first * side.y_head;
    bool keep = true;
    if (side.slots != nullptr) {
      const int64_t slot = side.slots[token];
      keep = slot >= 0 && slot < side.n_slots;
      const int64_t page = keep ? slot / side.page_size : 0;
      y += page * side.y_token + (keep ? slot - page * side.page_size : 0) * side.y_slot;
    } else {
      y += token * side.y_token;
    }
    if (side.plain != 0) {
#pragma unroll
      for (int k = 0; k < RUN; ++k) {
        if (!keep || (!WHOLE && first + k * groups >= side.heads)) break;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (seat[u].has_a) store_unit<T, N, NT>(y + k * y_step + seat[u].ea, ra[k][u]);
          if (seat[u].has_b) store_unit<T, N, NT>(y + k * y_step + seat[u].eb, rb[k][u]);
        }
      }
      continue;
    }
    float c[U][N], s[U][N];
    if (turned) {
#pragma unroll
      for (int u = 0; u < U; ++u) angles_of<N>(c[u], s[u], freq[u], token, a.r);
    }
#pragma unroll
    for (int k = 0; k < RUN; ++k) {
      const int h = first + k * groups;
      if (!WHOLE && h >= side.heads) break;
      float fa[U][N], fb[U][N];
      float sum = 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        widen_unit<T, N>(fa[u], ra[k][u]);
        widen_unit<T, N>(fb[u], rb[k][u]);
      }
      if (norm) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < N; ++j)
            sum = __builtin_fmaf(fa[u][j], fa[u][j], __builtin_fmaf(fb[u][j], fb[u][j], sum));
        const float r = inverse_root(__builtin_fmaf(group_sum<G>(sum), inv_dim, a.eps));
        if (side.rstd != nullptr && lane == 0) side.rstd[token * side.rstd_token + h] = r;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < N; ++j) {
            fa[u][j] = fa[u][j] * r * wa[u][j];
            fb[u][j] = fb[u][j] * r * wb[u][j];
          }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (turned) turn<N>(fa[u], fb[u], c[u], s[u], seat[u], a.r);
        T* q = y + k * y_step;
        if (keep && seat[u].has_a)
          store_unit<T, N, NT>(q + seat[u].ea, narrow_unit<T, N>(fa[u]));
        if (keep && seat[u].has_b)
          store_unit<T, N, NT>(q + seat[u].eb, narrow_unit<T, N>(fb[u]));
      }
    }
  }
}

// One tensor's way through the gradients.
template <class T>
struct GradSide {
  const T* x;
  const T* dy;
  T* dx;
  const T* w;
  const float* rstd;
  float* dw;
  float* partial;  // [blocks, dim]
  int64_t x_token, x_head, dy_token, dy_head, dx_token, dx_head;
  int heads, groups_log;
  int64_t first_block, blocks, units;
};
template <class T>
struct GradArgs {
  GradSide<T> side[2];
  Rotation r;
  int64_t rstd_token;
  int dim;
};

// Workgroups loop over tokens with the weight's gradient in registers and leave
// one partial row each, which heads_dw_kernel adds up in their order: no atomics, the
// same bits from call to call.  Measured with it: 16384 tokens of 32 + 8 heads of 128
// in bf16 98 us (5.1 TB/s of reads and writes 2 : 1), 8192 in fp32 92 (5.5), 1000
// tokens of 14 + 2 heads of 80 in fp32 10.7, 64 tokens of 32 + 8 heads 7.7: two launches
// and their latencies.
template <class T, int N, int G, int U, int RUN, bool WHOLE, bool NT>
__global__ __launch_bounds__(kThreads) void heads_bwd_kernel(const GradArgs<T> a) {
  __shared__ float rows[kThreads / G][2 * N * U * G];
  const GradSide<T>& side = a.side[blockIdx.x >= a.side[1].first_block ? 1 : 0];
  const int64_t block = blockIdx.x - side.first_block;
  const int lane = static_cast<int>(threadIdx.x) % G;
  const int groups = 1 << side.groups_log;
  const float inv_dim = 1.0f / static_cast<float>(a.dim);
  const bool turned = a.r.rot > 0;
  Seat<N> seat[U];
  double freq[U][N];
  float wa[U][N], wb[U][N], da[U][N], db[U][N];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    seat[u] = seat_of<N>(lane + G * u, a.dim, a.r);
    if constexpr (WHOLE) seat[u].has_a = seat[u].has_b = true;
#pragma unroll
    for (int j = 0; j < N; ++j) wa[u][j] = wb[u][j] = da[u][j] = db[u][j] = 0.0f;
    if (seat[u].has_a) widen_unit<T, N>(wa[u], load_unit<T, N>(side.w + seat[u].ea));
    if (seat[u].has_b) widen_unit<T, N>(wb[u], load_unit<T, N>(side.w + seat[u].eb));
    if (turned) turns_of<N>(freq[u], lane + G * u, a.r);
  }
  for (int64_t unit = block * (kThreads / G) + static_cast<int>(threadIdx.x) / G;
       unit < side.units; unit += side.blocks * (kThreads / G)) {
    const int64_t token = unit >> side.groups_log;
    const int first = static_cast<int>(unit & (groups - 1));
    if (!WHOLE && first >= side.heads) continue;
    const T* x = side.x + token * side.x_token + first * side.x_head;
    const T* dy = side.dy + token * side.dy_token + first * side.dy_head;
    T* dx = side.dx + token * side.dx_token + first * side.dx_head;
    // On their way while the angles are taken.
    Unit<T, N> xa[RUN][U], xb[RUN][U], ga[RUN][U], gb[RUN][U];
    float rstd[RUN];
#pragma unroll
    for (int k = 0; k < RUN; ++k) {
      const int step = (WHOLE || first + k * groups < side.heads ? k : 0) * groups;
      const T* px = x + step * side.x_head;
      const T* pg = dy + step * side.dy_head;
      rstd[k] = side.rstd[token * a.rstd_token + first + step];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        xa[k][u].v = 0;
        xb[k][u].v = 0;
        ga[k][u].v = 0;
        gb[k][u].v = 0;
        if (seat[u].has_a) xa[k][u] = load_unit<T, N, NT>(px + seat[u].ea);
        if (seat[u].has_b) xb[k][u] = load_unit<T, N, NT>(px + seat[u].eb);
        if (seat[u].has_a) ga[k][u] = load_unit<T, N, NT>(pg + seat[u].ea);
        if (seat[u].has_b) gb[k][u] = load_unit<T, N, NT>(pg + seat[u].eb);
      }
    }
    float c[U][N], s[U][N];
    if (turned) {
#pragma unroll
      for (int u = 0; u < U; ++u) angles_of<N>(c[u], s[u], freq[u], token, a.r);
    }
#pragma unroll
    for (int k = 0; k < RUN; ++k) {
      if (!WHOLE && first + k * groups >= side.heads) break;
      float na[U][N], nb[U][N], fa[U][N], fb[U][N];
      float dot = 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        widen_unit<T, N>(na[u], xa[k][u]);
        widen_unit<T, N>(nb[u], xb[k][u]);
        widen_unit<T, N>(fa[u], ga[k][u]);
        widen_unit<T, N>(fb[u], gb[k][u]);
        if (turned) turn<N>(fa[u], fb[u], c[u], s[u], seat[u], a.r);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          na[u][j] *= rstd[k];
          nb[u][j] *= rstd[k];
          da[u][j] = __builtin_fmaf(fa[u][j], na[u][j], da[u][j]);
          db[u][j] = __builtin_fmaf(fb[u][j], nb[u][j], db[u][j]);
          fa[u][j] *= wa[u][j];
          fb[u][j] *= wb[u][j];
          dot = __builtin_fmaf(fa[u][j], na[u][j], __builtin_fmaf(fb[u][j], nb[u][j], dot));
        }
      }
      const float mean = group_sum<G>(dot) * inv_dim;
      T* q = dx + k * groups * side.dx_head;
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          fa[u][j] = rstd[k] * __builtin_fmaf(-mean, na[u][j], fa[u][j]);
          fb[u][j] = rstd[k] * __builtin_fmaf(-mean, nb[u][j], fb[u][j]);
        }
        if (seat[u].has_a) store_unit<T, N, NT>(q + seat[u].ea, narrow_unit<T, N>(fa[u]));
        if (seat[u].has_b) store_unit<T, N, NT>(q + seat[u].eb, narrow_unit<T, N>(fb[u]));
      }
    }
  }
  const int group = static_cast<int>(threadIdx.x) / G;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (seat[u].has_a) rows[group][seat[u].ea + j] = da[u][j];
      if (seat[u].has_b) rows[group][seat[u].eb + j] = db[u][j];
    }
  __syncthreads();
  for (int d = static_cast<int>(threadIdx.x); d < a.dim; d += kThreads) {
    float sum = 0.0f;
#pragma unroll
    for (int g = 0; g < kThreads / G; ++g) sum += rows[g][d];
    side.partial[block * a.dim + d] = sum;
  }
}

// dw = the sum of the partial rows: 32 columns a workgroup, 32 runs of rows, kAhead
// loads of a thread on their way together (1022 rows one by one 9 us, with
// the latency of each: the gradients above 104 -> 98, of 1000 tokens 15.6 -> 10.7).
constexpr int kSumCols = 32;
constexpr int kSumRuns = 32;
constexpr int kAhead = 16;
struct SumArgs {
  const float* partial[2];
  float* dw[2];
  int rows[2];
  int dim;
};
__global__ __launch_bounds__(kSumCols* kSumRuns) void heads_dw_kernel(const SumArgs a) {
  __shared__ float part[kSumRuns][kSumCols];
  const int side = blockIdx.y;
  const int col = static_cast<int>(threadIdx.x) % kSumCols;
  const int run = static_cast<int>(threadIdx.x) / kSumCols;
  const int d = static_cast<int>(blockIdx.x) * kSumCols + col;
  float sum = 0.0f;
  if (d < a.dim) {
    const float* p = a.partial[side] + d;
    for (int r = run; r < a.rows[side]; r += kSumRuns * kAhead) {
      float v[kAhead];
#pragma unroll
      for (int n = 0; n < kAhead; ++n) {
        const int row = r + n * kSumRuns;
        v[n] = p[(row < a.rows[side] ? row : r) * a.dim];
      }
#pragma unroll
      for (int n = 0; n < kAhead; ++n) sum += r + n * kSumRuns < a.rows[side] ? v[n] : 0.0f;
    }
  }
  part[run][col] = sum;
  __syncthreads();
  if (run == 0 && d < a.dim) {
    sum = 0.0f;
#pragma unroll
    for (int r = 0; r < kSumRuns; ++r) sum += part[r][col];
    a.dw[side][d] = sum;
  }
}

// ------------------------------------------------------------------- host --

int check_own(const Place& out, const char* name, const Place& in, const char* in_name) {
  return heads::same(out, in) ? CREDIT_OK : check_places_apart(out, name, in, in_name);
}
int check_rotation(const credit_rotation* r, int64_t tokens, int dim, bool transposed,
                   Rotation* out) {
  *out = Rotation{nullptr, nullptr, 0, 0, 1.0f, 1.0f, 0};
  if (r == nullptr) return CREDIT_OK;
  if (r->rot < 0 || r->rot > dim || r->rot % 2 != 0)
    return set_error(CREDIT_ERR_BAD_SHAPE, "rot %d is not an even number in [0, %d]", r->rot, dim);
  if (r->rot == 0) return CREDIT_OK;
  CREDIT_TRY(check_row_ptr(r->positions, "positions", tokens));
  CREDIT_TRY(check_aligned(r->positions, sizeof(int64_t), "positions"));
  CREDIT_TRY(check_ptr(r->inv_freq, "inv_freq"));
  CREDIT_TRY(check_aligned(r->inv_freq, sizeof(float), "inv_freq"));
  if (!__builtin_isfinite(r->magnitude))
    return set_error(CREDIT_ERR_BAD_CONFIG, "magnitude %g is not finite", r->magnitude);
  *out = Rotation{r->positions, r->inv_freq, r->rot, r->interleaved != 0, r->magnitude,
                  transposed ? -1.0f : 1.0f, r->rot == dim};
  return CREDIT_OK;
}
int check_eps(float eps) {
  if (!(eps >= 0.0f) || !__builtin_isfinite(eps))
    return set_error(CREDIT_ERR_BAD_CONFIG, "eps %g is not a finite number >= 0", eps);
  return CREDIT_OK;
}
// Whether units of n elements of `elem` bytes serve: every address and the
// borders of the rotation lie on them.
struct Shape {
  int dim;
  const Rotation* r;
  uintptr_t addresses = 0;  // or of all of them
  int64_t strides = 0;      // and of the strides, in bytes

  void add(const Place& p) {
    addresses |= p.at;
    strides |= p.run | p.step | p.lead;
  }
  bool serves(int n, size_t elem) const {
    const int border = r->interleaved != 0 ? r->rot : r->rot / 2;
    return dim % n == 0 && border % n == 0 && addresses % (n * elem) == 0 &&
           strides % static_cast<int64_t>(n * elem) == 0;
  }
};

// fn(N, G, U): elements of a unit, lanes of a group, pairs of units a lane.  The
// widest units that every address takes: 16 bytes (128 elements of bf16: 8 lanes a
// head), else 8, else single elements.  us of 16384 tokens of 32 + 8 heads of 128 in
// bf16, turned: 61 / 80 / 234.
template <class T, class Fn>
void with_units(const Shape& shape, Fn&& fn) {
  const auto lanes = [&](auto n) {
    constexpr int N = decltype(n)::value;
    const int pairs = (shape.dim / N + 1) / 2;
    using std::integral_constant;
    if constexpr (kMaxDim / N / 2 > 32)
      if (pairs > 32) return fn(n, integral_constant<int, 64>{}, integral_constant<int, 1>{});
    if (pairs > 16) return fn(n, integral_constant<int, 32>{}, integral_constant<int, 1>{});
    if (pairs > 8) return fn(n, integral_constant<int, 16>{}, integral_constant<int, 1>{});
    if (pairs > 4) return fn(n, integral_constant<int, 8>{}, integral_constant<int, 1>{});
    return fn(n, integral_constant<int, 4>{}, integral_constant<int, 1>{});
  };
  if constexpr (std::is_same_v<T, uint16_t>)
    if (shape.serves(8, sizeof(T))) return lanes(std::integral_constant<int, 8>{});
  if (shape.serves(4, sizeof(T))) return lanes(std::integral_constant<int, 4>{});
  fn(std::integral_constant<int, 1>{}, std::integral_constant<int, 64>{},
     std::integral_constant<int, kMaxDim / 128>{});
}

int log2_of(int v) { return 31 - __builtin_clz(static_cast<unsigned>(v)); }

// Units of a side, its groups and workgroups: as many as its share, by heads, of
// kBlocks, which loop over them.
struct Deal {
  int groups;
  int64_t units, blocks;
};
inline Deal deal(int64_t tokens, int side_heads, int64_t all_heads, int lanes, int run,
                 int64_t blocks) {
  Deal d;
  d.groups = heads::groups_of(side_heads, run);
  d.units = tokens * d.groups;
  const int64_t share = std::max<int64_t>(1, blocks * side_heads / all_heads);
  const int64_t per = kThreads / lanes;
  d.blocks = std::min(share, (d.units + per - 1) / per);
  return d;
}

// fn(RUN, WHOLE, NT) of heads a group takes at once.  Nontemporal where a call's
// tensors take more than a third of the last-level cache (256 MiB): among the others
// of a step they are not found there again.  us, without -> with, norm and rotation in
// bf16, calls on 1 / 3 / 8 sets of tensors in turn: 81 MiB 21 / 21 / 27 -> 20 / 21 / 21,
// 161 MiB 33 / 42 / 43 -> 36 / 36 / 37, 320 MiB 79 -> 65; rotation in fp32 of strided
// tensors, 80 MiB 17 / 17 / 21 -> 19 / 20 / 20; 192 MiB into a cache 37 / 48 / 48 -> 40 /
// 41 / 42; gradients, 121 MiB 29 / 37 / 37 -> 33 / 34 / 35.
template <int U, int MOST, class Fn>
void with_run(int run, bool even, int64_t bytes, Fn&& fn) {
  using std::integral_constant;
  if constexpr (U > 1) {
    fn(integral_constant<int, 1>{}, std::false_type{}, std::false_type{});
  } else {
    const auto go = [&](auto n) {
      if (!even) return fn(n, std::false_type{}, std::false_type{});
      if constexpr (decltype(n)::value == MOST)
        if (bytes > (int64_t{256} << 20) / 3) return fn(n, std::true_type{}, std::true_type{});
      fn(n, std::true_type{}, std::false_type{});
    };
    if (run == 1) return go(integral_constant<int, 1>{});
    if constexpr (MOST > 2)
      if (run == 2) return go(integral_constant<int, 2>{});
    go(integral_constant<int, MOST>{});
  }
}

// Workgroups of the forward's launch: more than the device holds at once, so that one
// ends while another begins, each with a few units over which its lanes keep weights
// and frequencies.  us at 1024 / 2048 / 4096 / one a unit: norm and rotation of 16384
// tokens of 32 + 8 heads of 128 in bf16 71 / 66 / 65 / 67, of 131072 tokens of 2 + 1
// heads 43 / 42 / 44 / 49, 8192 tokens into a cache 44 / 38 / 38 / 38.
constexpr int64_t kForwardBlocks = 4096;

template <class T>
int launch_forward(ForwardArgs<T>& a, int64_t tokens, const Shape& shape, hipStream_t stream) {
  with_units<T>(shape, [&](auto n, auto g, auto u) {
    constexpr int N = decltype(n)::value, G = decltype(g)::value, U = decltype(u)::value;
    constexpr int kMost = U == 1 ? 4 : 1;
    int64_t blocks = 0, all = 0, bytes = 0;
    int widest = 0;
    for (int i = 0; i < a.sides; ++i) {
      all += a.side[i].heads;
      widest = std::max(widest, a.side[i].heads);
    }
    const int run = heads::run_of(tokens, all, widest, G, kMost);
    bool even = a.dim == 2 * N * G;
    for (int i = 0; i < a.sides; ++i) {
      Side<T>& s = a.side[i];
      const Deal d = deal(tokens, s.heads, all, G, run, kForwardBlocks);
      s.groups_log = log2_of(d.groups);
      s.units = d.units;
      s.first_block = blocks;
      blocks += d.blocks;
      bytes += 2 * tokens * s.heads * a.dim * static_cast<int64_t>(sizeof(T));
    }
    for (int i = 0; i < a.sides; ++i) even = even && a.side[i].heads == run << a.side[i].groups_log;
    const dim3 grid(static_cast<unsigned>(blocks));
    with_run<U, kMost>(run, even, bytes, [&](auto r, auto whole, auto nt) {
      heads_fwd_kernel<T, N, G, U, decltype(r)::value, decltype(whole)::value,
                       decltype(nt)::value><<<grid, kThreads, 0, stream>>>(a);
    });
  });
  return check_launch("heads_fwd_kernel");
}

template <class T>
Side<T> side_of(const credit_heads* in, const credit_heads* out, const T* w) {
  Side<T> s{};
  s.x = static_cast<const T*>(in->data);
  s.y = static_cast<T*>(out->data);
  s.w = w;
  s.x_token = in->token_stride;
  s.x_head = in->head_stride;
  s.y_token = out->token_stride;
  s.y_head = out->head_stride;
  s.heads = in->heads;
  return s;
}
// The small inputs of a call's rotation (none: empty).
NamedPlace positions_of(const Rotation& r, int64_t tokens) {
  return {flat_place(r.positions, tokens, sizeof(int64_t)), "positions"};
}
NamedPlace frequencies_of(const Rotation& r) {
  return {flat_place(r.inv_freq, r.rot / 2, sizeof(float)), "inv_freq"};
}

// Both forwards without a cache; no weights: the rotation alone.
template <class T>
int rotate(const credit_heads* q, const credit_heads* k, const T* q_weight, const T* k_weight,
           const credit_rotation* rotation, const credit_heads* q_out, const credit_heads* k_out,
           float* rstd, int64_t tokens, int32_t dim, float eps, bool norm, bool transposed,
           const credit_cfg* cfg) {
  constexpr size_t kElem = sizeof(T);
  CREDIT_TRY(check_tokens(tokens, dim, kMaxDim));
  ForwardArgs<T> a{};
  CREDIT_TRY(check_rotation(rotation, tokens, dim, transposed, &a.r));
  Shape shape{dim, &a.r};
  Place in[2], out[2];
  const bool keys = norm || k != nullptr || k_out != nullptr;
  CREDIT_TRY(check_heads(q, "q", tokens, dim, kElem, &in[0]));
  CREDIT_TRY(check_output(q_out, "q_out", q, tokens, dim, kElem, &out[0]));
  if (keys) {
    CREDIT_TRY(check_heads(k, "k", tokens, dim, kElem, &in[1]));
    CREDIT_TRY(check_output(k_out, "k_out", k, tokens, dim, kElem, &out[1]));
  }
  if (norm) {
    CREDIT_TRY(check_ptr(q_weight, "q_weight"));
    CREDIT_TRY(check_ptr(k_weight, "k_weight"));
    CREDIT_TRY(check_aligned(q_weight, kElem, "q_weight"));
    CREDIT_TRY(check_aligned(k_weight, kElem, "k_weight"));
    CREDIT_TRY(check_aligned(rstd, sizeof(float), "rstd"));
    CREDIT_TRY(check_eps(eps));
    shape.addresses |= reinterpret_cast<uintptr_t>(q_weight) | reinterpret_cast<uintptr_t>(k_weight);
  }
  CREDIT_TRY(check_only_auto(cfg));
  if (tokens == 0) return CREDIT_OK;
  CREDIT_TRY(check_own(out[0], "q_out", in[0], "q"));
  if (keys) {
    CREDIT_TRY(check_own(out[1], "k_out", in[1], "k"));
    CREDIT_TRY(check_places_apart(out[0], "q_out", in[1], "k"));
    CREDIT_TRY(check_places_apart(out[1], "k_out", in[0], "q"));
    CREDIT_TRY(check_places_apart(out[0], "q_out", out[1], "k_out"));
  }
  const NamedPlace wq{flat_place(q_weight, dim, kElem), "q_weight"};
  const NamedPlace wk{flat_place(k_weight, dim, kElem), "k_weight"};
  const NamedPlace pos = positions_of(a.r, tokens), freq = frequencies_of(a.r);
  CREDIT_TRY(check_outputs_apart({{out[0], "q_out"}}, {wq, wk, pos, freq}));
  CREDIT_TRY(check_outputs_apart({{out[1], "k_out"}}, {wq, wk, pos, freq}));
  if (rstd != nullptr)
    CREDIT_TRY(check_outputs_apart(
        {{flat_place(rstd, tokens * (static_cast<int64_t>(q->heads) + k->heads), sizeof(float)),
          "rstd"}},
        {{in[0], "q"}, {in[1], "k"}, {out[0], "q_out"}, {out[1], "k_out"}, wq, wk, pos, freq}));
  a.sides = keys ? 2 : 1;
  a.dim = dim;
  a.eps = eps;
  for (int i = 0; i < a.sides; ++i) {
    a.side[i] = side_of<T>(i == 0 ? q : k, i == 0 ? q_out : k_out, i == 0 ? q_weight : k_weight);
    shape.add(in[i]);
    shape.add(out[i]);
  }
  if (norm && rstd != nullptr) {
    a.side[0].rstd = rstd;
    a.side[1].rstd = rstd + q->heads;
    a.side[0].rstd_token = a.side[1].rstd_token = q->heads + k->heads;
  }
  return launch_forward<T>(a, tokens, shape, cfg_stream(cfg));
}

// Workgroups of the gradients' launch at most: four a CU of the largest device.
constexpr int64_t kMaxGradBlocks = 1024;

// Where they leave their partial rows: the caller's workspace, else a buffer that only
// they use, one for each (device, stream).  In the library's workspace another thread's
// call of another operator on the stream, between the two launches, would write over them.
int partial_rows(const credit_cfg* cfg, int dim, float** rows) {
  const size_t bytes = qk_norm_rope_bwd_workspace(dim);
  char* base = nullptr;
  if (cfg != nullptr && cfg->workspace != nullptr) {
    CREDIT_TRY(acquire_workspace(cfg, bytes, &base));
    base = ws_scratch(base);
  } else {
    static auto* buffers = new WorkspaceCache<ScratchAlloc>();
    int device = 0;
    CREDIT_HIP(hipGetDevice(&device));
    if (buffers->get(device, cfg_stream(cfg), bytes, &base) != CREDIT_OK)
      return set_error(CREDIT_ERR_HIP, "no memory for %zu bytes of partial rows", bytes);
  }
  *rows = reinterpret_cast<float*>(base);
  return CREDIT_OK;
}

template <class T>
int norm_rope_bwd(const credit_heads* q, const credit_heads* k, const T* q_weight,
                  const T* k_weight, const credit_rotation* rotation, const float* rstd,
                  const credit_heads* dq_out, const credit_heads* dk_out, const credit_heads* dq,
                  const credit_heads* dk, float* dq_weight, float* dk_weight, int64_t tokens,
                  int32_t dim, const credit_cfg* cfg) {
  constexpr size_t kElem = sizeof(T);
  CREDIT_TRY(check_tokens(tokens, dim, kMaxDim));
  GradArgs<T> a{};
  CREDIT_TRY(check_rotation(rotation, tokens, dim, true, &a.r));
  Shape shape{dim, &a.r};
  const credit_heads* x[2] = {q, k};
  const credit_heads* dy[2] = {dq_out, dk_out};
  const credit_heads* dx[2] = {dq, dk};
  const T* w[2] = {q_weight, k_weight};
  float* dw[2] = {dq_weight, dk_weight};
  static const char* const kNames[5][2] = {{"q", "k"},
                                           {"dq_out", "dk_out"},
                                           {"dq", "dk"},
                                           {"q_weight", "k_weight"},
                                           {"dq_weight", "dk_weight"}};
  Place px[2], py[2], pd[2];
  for (int i = 0; i < 2; ++i) {
    CREDIT_TRY(check_heads(x[i], kNames[0][i], tokens, dim, kElem, &px[i]));
    CREDIT_TRY(check_heads(dy[i], kNames[1][i], tokens, dim, kElem, &py[i]));
    if (dy[i]->heads != x[i]->heads)
      return set_error(CREDIT_ERR_BAD_SHAPE, "%s: %d heads, %s has %d", kNames[1][i],
                       dy[i]->heads, kNames[0][i], x[i]->heads);
    CREDIT_TRY(check_output(dx[i], kNames[2][i], x[i], tokens, dim, kElem, &pd[i]));
    CREDIT_TRY(check_ptr(w[i], kNames[3][i]));
    CREDIT_TRY(check_aligned(w[i], kElem, kNames[3][i]));
    CREDIT_TRY(check_ptr(dw[i], kNames[4][i]));
    CREDIT_TRY(check_aligned(dw[i], sizeof(float), kNames[4][i]));
    shape.addresses |= reinterpret_cast<uintptr_t>(w[i]);
    shape.add(px[i]);
    shape.add(py[i]);
    shape.add(pd[i]);
  }
  CREDIT_TRY(check_row_ptr(rstd, "rstd", tokens));
  CREDIT_TRY(check_aligned(rstd, sizeof(float), "rstd"));
  CREDIT_TRY(check_only_auto(cfg));
  for (int i = 0; i < 2 && tokens > 0; ++i) {
    CREDIT_TRY(check_own(pd[i], kNames[2][i], px[i], kNames[0][i]));
    CREDIT_TRY(check_own(pd[i], kNames[2][i], py[i], kNames[1][i]));
    CREDIT_TRY(check_places_apart(pd[i], kNames[2][i], px[1 - i], kNames[0][1 - i]));
    CREDIT_TRY(check_places_apart(pd[i], kNames[2][i], py[1 - i], kNames[1][1 - i]));
  }
  if (tokens > 0) CREDIT_TRY(check_places_apart(pd[0], "dq", pd[1], "dk"));
  const NamedPlace wq{flat_place(q_weight, dim, kElem), "q_weight"};
  const NamedPlace wk{flat_place(k_weight, dim, kElem), "k_weight"};
  const NamedPlace pos = positions_of(a.r, tokens), freq = frequencies_of(a.r);
  const NamedPlace norms{
      flat_place(rstd, tokens * (static_cast<int64_t>(q->heads) + k->heads), sizeof(float)),
      "rstd"};
  CREDIT_TRY(check_outputs_apart({{pd[0], "dq"}, {pd[1], "dk"}}, {wq, wk, pos, freq, norms}));
  CREDIT_TRY(check_outputs_apart({{flat_place(dq_weight, dim, sizeof(float)), "dq_weight"},
                                  {flat_place(dk_weight, dim, sizeof(float)), "dk_weight"}},
                                 {{px[0], "q"}, {px[1], "k"}, {py[0], "dq_out"},
                                  {py[1], "dk_out"}, {pd[0], "dq"}, {pd[1], "dk"}, wq, wk, pos,
                                  freq, norms}));
  hipStream_t stream = cfg_stream(cfg);
  if ((cfg == nullptr || cfg->workspace == nullptr) && !keeps_scratch(stream))
    return set_error(CREDIT_ERR_WORKSPACE,
                     "under capture or on the per-thread stream this needs cfg->workspace");
  // The two launches of a call stay together when threads share a stream.
  static std::mutex* mu = new std::mutex();
  std::lock_guard<std::mutex> lock(*mu);
  float* partial = nullptr;
  CREDIT_TRY(partial_rows(cfg, dim, &partial));
  a.dim = dim;
  a.rstd_token = static_cast<int64_t>(q->heads) + k->heads;
  SumArgs sum{};
  sum.dim = dim;
  with_units<T>(shape, [&](auto n, auto g, auto u) {
    constexpr int N = decltype(n)::value, G = decltype(g)::value, U = decltype(u)::value;
    constexpr int kMost = U == 1 ? 2 : 1;
    int64_t blocks = 0;
    const int64_t all = static_cast<int64_t>(q->heads) + k->heads;
    const int run = heads::run_of(tokens, all, std::max(q->heads, k->heads), G, kMost);
    for (int i = 0; i < 2; ++i) {
      GradSide<T>& s = a.side[i];
      s.x = static_cast<const T*>(x[i]->data);
      s.dy = static_cast<const T*>(dy[i]->data);
      s.dx = static_cast<T*>(dx[i]->data);
      s.w = w[i];
      s.rstd = rstd + (i == 0 ? 0 : q->heads);
      s.dw = dw[i];
      s.x_token = x[i]->token_stride;
      s.x_head = x[i]->head_stride;
      s.dy_token = dy[i]->token_stride;
      s.dy_head = dy[i]->head_stride;
      s.dx_token = dx[i]->token_stride;
      s.dx_head = dx[i]->head_stride;
      s.heads = x[i]->heads;
      const Deal d = deal(tokens, s.heads, all, G, run, kMaxGradBlocks - 1);
      s.groups_log = log2_of(d.groups);
      s.units = d.units;
      s.first_block = blocks;
      s.blocks = d.blocks;
      s.partial = partial + blocks * dim;
      blocks += s.blocks;
      sum.partial[i] = s.partial;
      sum.dw[i] = s.dw;
      sum.rows[i] = static_cast<int>(s.blocks);
    }
    if (blocks == 0) return;
    bool even = dim == 2 * N * G;
    for (const GradSide<T>& s : a.side) even = even && s.heads == run << s.groups_log;
    const dim3 grid(static_cast<unsigned>(blocks));
    with_run<U, kMost>(run, even, 3 * tokens * all * dim * static_cast<int64_t>(sizeof(T)),
                       [&](auto r, auto whole, auto nt) {
                         heads_bwd_kernel<T, N, G, U, decltype(r)::value,
                                          decltype(whole)::value, decltype(nt)::value>
                             <<<grid, kThreads, 0, stream>>>(a);
                       });
  });
  CREDIT_TRY(check_launch("heads_bwd_kernel"));
  heads_dw_kernel<<<dim3(static_cast<unsigned>((dim + kSumCols - 1) / kSumCols), 2),
                    kSumCols * kSumRuns, 0, stream>>>(sum);
  return check_launch("heads_dw_kernel");
}

int check_pages(const credit_pages* c, const char* name, const credit_heads* in, int dim,
                size_t elem, Place* place) {
  CREDIT_TRY(check_ptr(c, name));
  if (c->heads != in->heads)
    return set_error(CREDIT_ERR_BAD_SHAPE, "%s: %d heads, its input has %d", name, c->heads,
                     in->heads);
  return check_cache(c, name, dim, elem, place);
}

int append(const credit_heads* k, const credit_heads* v, const credit_heads* q,
           const uint16_t* k_weight, const uint16_t* q_weight, const credit_rotation* rotation,
           const int64_t* slots, const credit_pages* k_cache, const credit_pages* v_cache,
           const credit_heads* q_out, int64_t tokens, int32_t dim, float eps,
           const credit_cfg* cfg) {
  using T = uint16_t;
  constexpr size_t kElem = sizeof(T);
  CREDIT_TRY(check_tokens(tokens, dim, kMaxDim));
  ForwardArgs<T> a{};
  CREDIT_TRY(check_rotation(rotation, tokens, dim, false, &a.r));
  Shape shape{dim, &a.r};
  const bool queries = q != nullptr || q_out != nullptr;
  Place pk, pv, pq, po, kc, vc;
  CREDIT_TRY(check_heads(k, "k", tokens, dim, kElem, &pk));
  CREDIT_TRY(check_heads(v, "v", tokens, dim, kElem, &pv));
  CREDIT_TRY(check_pages(k_cache, "k_cache", k, dim, kElem, &kc));
  CREDIT_TRY(check_pages(v_cache, "v_cache", v, dim, kElem, &vc));
  if (queries) {
    CREDIT_TRY(check_heads(q, "q", tokens, dim, kElem, &pq));
    CREDIT_TRY(check_output(q_out, "q_out", q, tokens, dim, kElem, &po));
  } else if (q_weight != nullptr) {
    return set_error(CREDIT_ERR_BAD_CONFIG, "q_weight without q");
  }
  if (k_cache->pages != v_cache->pages || k_cache->page_size != v_cache->page_size)
    return set_error(CREDIT_ERR_BAD_SHAPE, "k_cache and v_cache have different pages");
  CREDIT_TRY(check_row_ptr(slots, "slots", tokens));
  CREDIT_TRY(check_aligned(slots, sizeof(int64_t), "slots"));
  CREDIT_TRY(check_aligned(k_weight, kElem, "k_weight"));
  CREDIT_TRY(check_aligned(q_weight, kElem, "q_weight"));
  CREDIT_TRY(check_eps(eps));
  CREDIT_TRY(check_only_auto(cfg));
  if (tokens == 0) return CREDIT_OK;
  CREDIT_TRY(check_places_apart(kc, "k_cache", vc, "v_cache"));
  struct Named {
    const Place* place;
    const char* name;
  };
  const Named inputs[] = {{&pk, "k"}, {&pv, "v"}, {&pq, "q"}, {&po, "q_out"}};
  for (int i = 0; i < (queries ? 4 : 2); ++i) {
    CREDIT_TRY(check_places_apart(kc, "k_cache", *inputs[i].place, inputs[i].name));
    CREDIT_TRY(check_places_apart(vc, "v_cache", *inputs[i].place, inputs[i].name));
  }
  if (queries) {
    CREDIT_TRY(check_own(po, "q_out", pq, "q"));
    CREDIT_TRY(check_places_apart(po, "q_out", pk, "k"));
    CREDIT_TRY(check_places_apart(po, "q_out", pv, "v"));
  }
  CREDIT_TRY(check_outputs_apart({{kc, "k_cache"}, {vc, "v_cache"}, {po, "q_out"}},
                                 {{flat_place(k_weight, dim, kElem), "k_weight"},
                                  {flat_place(q_weight, dim, kElem), "q_weight"},
                                  positions_of(a.r, tokens), frequencies_of(a.r),
                                  {flat_place(slots, tokens, sizeof(int64_t)), "slots"}}));
  a.dim = dim;
  a.eps = eps;
  const auto into = [&](const credit_heads* in, const credit_pages* c, const T* w, bool plain) {
    const credit_heads to{c->data, c->page_stride, c->head_stride, c->heads};
    Side<T> s = side_of<T>(in, &to, w);
    s.y_slot = c->slot_stride;
    s.slots = slots;
    s.n_slots = c->pages * c->page_size;
    s.page_size = c->page_size;
    s.plain = plain;
    a.side[a.sides++] = s;
  };
  if (queries) a.side[a.sides++] = side_of<T>(q, q_out, q_weight);
  into(k, k_cache, k_weight, false);
  into(v, v_cache, nullptr, true);
  for (const Place* p : {&pk, &pv, &pq, &po, &kc, &vc}) shape.add(*p);
  shape.addresses |= reinterpret_cast<uintptr_t>(k_weight) | reinterpret_cast<uintptr_t>(q_weight);
  return launch_forward<T>(a, tokens, shape, cfg_stream(cfg));
}

}  // namespace

namespace {
constexpr int64_t kMaxBytes = int64_t{1} << 60;
}  // namespace

// A tensor by tokens and heads, its place, checked.
int check_heads(const credit_heads* h, const char* name, int64_t tokens, int dim, size_t elem,
                Place* place) {
  CREDIT_TRY(check_ptr(h, name));
  if (h->heads < 1 || h->heads > (1 << 20))
    return set_error(CREDIT_ERR_BAD_SHAPE, "%s: %d heads outside [1, 2^20]", name, h->heads);
  CREDIT_TRY(check_row_ptr(h->data, name, tokens));
  CREDIT_TRY(check_aligned(h->data, elem, name));
  const double bytes = (static_cast<double>(tokens) * h->token_stride +
                        static_cast<double>(h->heads) * h->head_stride + dim) *
                       static_cast<double>(elem);
  if (h->token_stride < 0 || h->head_stride < 0 || bytes > static_cast<double>(kMaxBytes))
    return set_error(CREDIT_ERR_BAD_SHAPE, "%s: strides (%lld, %lld) negative or too large", name,
                     static_cast<long long>(h->token_stride),
                     static_cast<long long>(h->head_stride));
  const int64_t e = static_cast<int64_t>(elem);
  *place = Place{reinterpret_cast<uintptr_t>(h->data), h->token_stride * e, h->head_stride * e,
                 tokens, h->heads, dim * e};
  return CREDIT_OK;
}
int check_output(const credit_heads* h, const char* name, const credit_heads* in, int64_t tokens,
                 int dim, size_t elem, Place* place) {
  CREDIT_TRY(check_heads(h, name, tokens, dim, elem, place));
  if (h->heads != in->heads)
    return set_error(CREDIT_ERR_BAD_SHAPE, "%s: %d heads, its input has %d", name, h->heads,
                     in->heads);
  if (!heads::apart_within(*place))
    return set_error(CREDIT_ERR_BAD_SHAPE, "%s: its heads overlap each other", name);
  return CREDIT_OK;
}
int check_places_apart(const Place& out, const char* name, const Place& other, const char* other_name) {
  if (heads::apart(out, other)) return CREDIT_OK;
  return set_error(CREDIT_ERR_BAD_CONFIG, "%s overlaps %s", name, other_name);
}
int check_outputs_apart(std::initializer_list<NamedPlace> outs,
                        std::initializer_list<NamedPlace> others) {
  for (const NamedPlace* out = outs.begin(); out != outs.end(); ++out) {
    for (const NamedPlace* next = out + 1; next != outs.end(); ++next)
      CREDIT_TRY(check_places_apart(out->place, out->name, next->place, next->name));
    for (const NamedPlace& other : others)
      CREDIT_TRY(check_places_apart(out->place, out->name, other.place, other.name));
  }
  return CREDIT_OK;
}
int check_tokens(int64_t tokens, int32_t dim, int32_t max_dim) {
  if (tokens < 0 || tokens > (int64_t{1} << 31) - 1)
    return set_error(CREDIT_ERR_BAD_SHAPE, "%lld tokens outside [0, 2^31)",
                     static_cast<long long>(tokens));
  if (dim < 1 || dim > max_dim)
    return set_error(CREDIT_ERR_BAD_SHAPE, "dim %d outside [1, %d]", dim, max_dim);
  return CREDIT_OK;
}
int check_only_auto(const credit_cfg* cfg) {
  CREDIT_TRY(check_cfg(cfg));
  if (cfg_variant(cfg) != CREDIT_VARIANT_AUTO || cfg_split(cfg) != 0)
    return set_error(CREDIT_ERR_UNSUPPORTED, "only AUTO without a split is supported");
  return CREDIT_OK;
}

int check_cache(const credit_pages* c, const char* name, int dim, size_t elem, Place* place) {
  CREDIT_TRY(check_ptr(c, name));
  if (c->pages < 0 || c->pages > (int64_t{1} << 31) - 1 || c->page_size < 1 ||
      c->page_size > (1 << 20) || c->heads < 1 || c->heads > (1 << 20))
    return set_error(CREDIT_ERR_BAD_SHAPE, "%s: %lld pages of %d slots of %d heads", name,
                     static_cast<long long>(c->pages), c->page_size, c->heads);
  CREDIT_TRY(check_row_ptr(c->data, name, c->pages));
  CREDIT_TRY(check_aligned(c->data, elem, name));
  const double bytes = (static_cast<double>(c->pages) * c->page_stride +
                        static_cast<double>(c->page_size) * c->slot_stride +
                        static_cast<double>(c->heads) * c->head_stride + dim) *
                       static_cast<double>(elem);
  const int64_t e = static_cast<int64_t>(elem);
  if (c->page_stride < 0 || c->slot_stride < 0 || c->head_stride < 0 ||
      bytes > static_cast<double>(kMaxBytes))
    return set_error(CREDIT_ERR_BAD_SHAPE, "%s: strides negative or too large", name);
  *place = Place{reinterpret_cast<uintptr_t>(c->data), c->slot_stride * e, c->head_stride * e,
                 c->page_size, c->heads, dim * e, c->page_stride * e, c->pages};
  if (!heads::apart_within(*place))
    return set_error(CREDIT_ERR_BAD_SHAPE, "%s: its slots overlap each other", name);
  return CREDIT_OK;
}
size_t qk_norm_rope_bwd_workspace(int64_t dim) {
  return static_cast<size_t>(kMaxGradBlocks) * static_cast<size_t>(dim) * sizeof(float);
}

}  // namespace credit

using namespace credit;

extern "C" {

int credit_rope_f32(const credit_heads* q, const credit_heads* k, const credit_rotation* rotation,
                    const credit_heads* q_out, const credit_heads* k_out, int64_t tokens,
                    int32_t dim, int32_t transposed, const credit_cfg* cfg) {
  return rotate<float>(q, k, nullptr, nullptr, rotation, q_out, k_out, nullptr, tokens, dim, 0.0f,
                       false, transposed != 0, cfg);
}
int credit_rope_bf16(const credit_heads* q, const credit_heads* k,
                     const credit_rotation* rotation, const credit_heads* q_out,
                     const credit_heads* k_out, int64_t tokens, int32_t dim, int32_t transposed,
                     const credit_cfg* cfg) {
  return rotate<uint16_t>(q, k, nullptr, nullptr, rotation, q_out, k_out, nullptr, tokens, dim,
                          0.0f, false, transposed != 0, cfg);
}
int credit_qk_norm_rope_fwd_f32(const credit_heads* q, const credit_heads* k,
                                const float* q_weight, const float* k_weight,
                                const credit_rotation* rotation, const credit_heads* q_out,
                                const credit_heads* k_out, float* rstd, int64_t tokens,
                                int32_t dim, float eps, const credit_cfg* cfg) {
  return rotate<float>(q, k, q_weight, k_weight, rotation, q_out, k_out, rstd, tokens, dim, eps,
                       true, false, cfg);
}
int credit_qk_norm_rope_fwd_bf16(const credit_heads* q, const credit_heads* k,
                                 const uint16_t* q_weight, const uint16_t* k_weight,
                                 const credit_rotation* rotation, const credit_heads* q_out,
                                 const credit_heads* k_out, float* rstd, int64_t tokens,
                                 int32_t dim, float eps, const credit_cfg* cfg) {
  return rotate<uint16_t>(q, k, q_weight, k_weight, rotation, q_out, k_out, rstd, tokens, dim, eps,
                          true, false, cfg);
}
int credit_qk_norm_rope_bwd_f32(const credit_heads* q, const credit_heads* k,
                                const float* q_weight, const float* k_weight,
                                const credit_rotation* rotation, const float* rstd,
                                const credit_heads* dq_out, const credit_heads* dk_out,
                                const credit_heads* dq, const credit_heads* dk, float* dq_weight,
                                float* dk_weight, int64_t tokens, int32_t dim,
                                const credit_cfg* cfg) {
  return norm_rope_bwd<float>(q, k, q_weight, k_weight, rotation, rstd, dq_out, dk_out, dq, dk,
                              dq_weight, dk_weight, tokens, dim, cfg);
}
int credit_qk_norm_rope_bwd_bf16(const credit_heads* q, const credit_heads* k,
                                 const uint16_t* q_weight, const uint16_t* k_weight,
                                 const credit_rotation* rotation, const float* rstd,
                                 const credit_heads* dq_out, const credit_heads* dk_out,
                                 const credit_heads* dq, const credit_heads* dk,
                                 float* dq_weight, float* dk_weight, int64_t tokens, int32_t dim,
                                 const credit_cfg* cfg) {
  return norm_rope_bwd<uint16_t>(q, k, q_weight, k_weight, rotation, rstd, dq_out, dk_out, dq, dk,
                                 dq_weight, dk_weight, tokens, dim, cfg);
}
int credit_paged_append_bf16(const credit_heads* k, const credit_heads* v,
                             const credit_heads* q, const uint16_t* k_weight,
                             const uint16_t* q_weight, const credit_rotation* rotation,
                             const int64_t* slots, const credit_pages* k_cache,
                             const credit_pages* v_cache, const credit_heads* q_out,
                             int64_t tokens, int32_t dim, float eps, const credit_cfg* cfg) {
  return append(k, v, q, k_weight, q_weight, rotation, slots, k_cache, v_cache, q_out, tokens, dim,
                eps, cfg);
}

}  // extern "C"
