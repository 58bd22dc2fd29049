// rope_cache.cu -- what stands between a layer's Q/K/V projection and its
// paged attention: the per-head RMS norms of Q and K, the position rotation,
// and the append of K and V to the paged cache, in one pass over the
// projection's output.  CacheFlow has no counterpart: its forward pass is an
// abstract ForwardFn (src/cacheflow/decode/batch_decode.h:34-42) that hands
// reshape_and_cache (src/cacheflow/cuda/kv_cache_kernels.cu:17-44) finished
// rows.
//
// Mathematics, per (token, head) row x of D elements, in f32:
//   norm    y = x * rsqrt(mean(x^2) + eps) * w        (only with a weight w)
//   rotate  columns below R in pairs (a, b) = (i, i + R/2), or (2i, 2i + 1):
//             a' = a cos_i - b sin_i,  b' = b cos_i + a sin_i
//           with cos / sin of the token's position read from an f32 table
//           (the angles of far positions need more than f32; a table made in
//           f64 holds them to half an f32 ulp).  Columns R.. pass.
//   store   one rounding at the end: to the rows' type, or to e4m3.
//
// Bound: HBM.  A row is read once and written once; the table row of a token
// (R floats) is shared by all its heads.  Measured, of 6.54 TB/s that a copy
// reaches: 8192 tokens of 64 / 8 heads of 128 in bf16 60 us, 5.1 TB/s; 16384
// tokens of 32 / 8 heads with the append 86 us, 4.75 TB/s; 4095 f32 tokens of
// 32 / 32 heads of 64 27 us, 5.05 TB/s.  A decode step of 64 rows is launch
// latency, 4.3 us.  The block-scaled append is bound by its CTAs' chain of
// dependent steps instead: 16384 tokens of 32 / 8 heads in ragged prompts 117
// us, 3.23 TB/s; 1024 decode rows of 64 / 8 heads 18 us.
#include <atomic>
#include <initializer_list>
#include <mutex>
#include <type_traits>

#include "cf_device.cuh"
#include "cf_internal.h"

namespace cfb {

__device__ uint32_t g_rope_errors;

__device__ __forceinline__ void rope_error(uint32_t bits) { atomicOr(&g_rope_errors, bits); }

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// Where a K row goes (V rows exist only with a cache).
enum KDest : int32_t { kDense = 0, kCacheSame = 1, kCacheFp8 = 2 };

struct RopeArgs {
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  void* k_out;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, qo_ts, qo_hs, ko_ts, ko_hs;  // strides in elements
  const int32_t* positions;  // null: no rotation, every token is live
  const float* cos_sin;      // [max_positions, R]: cos, then sin
  const void* q_w;           // [D] or null
  const void* k_w;
  int32_t w_f32;             // weights are f32 (else the rows' type)
  float eps;
  float inv_dim;             // 1 / head_dim
  int32_t num_tokens, num_heads, num_kv_heads, head_dim, rotary, max_positions;
  int32_t dest;              // KDest
  void* kc;                  // [num_blocks, Hkv, block_size, D]
  void* vc;
  const int32_t* slots;
  int32_t block_size;
  int64_t num_slots;
  float k_scale, v_scale;    // kCacheFp8: cache = e4m3(x / scale)
  // Row layout over lanes (row_layout()).
  int32_t rot_units;  // units that rotate
  int32_t units;      // units of a row
  int32_t lanes_log2; // lanes per row
};

// ---------------------------------------------------------------------------
// A row over lanes.  A unit is two vectors of V elements that a lane can
// rotate on its own: columns [uV, uV+V) and [R/2 + uV, ...) of a half-split
// rotation, or 2V neighbouring columns of an interleaved one; both use the
// angles [uV, uV+V).  Past the rotation a unit is 2V neighbouring columns
// (the last one may hold V).  A row takes 2^lanes_log2 >= units / K lanes, K
// units each, so no element crosses lanes: only the norm's sum does.
// ---------------------------------------------------------------------------
template <int kBytes>
struct RawVec;
template <>
struct RawVec<16> { using type = uint4; };
template <>
struct RawVec<8> { using type = uint2; };
template <>
struct RawVec<4> { using type = uint32_t; };
template <>
struct RawVec<2> { using type = uint16_t; };

template <typename T, int V>
using Raw = typename RawVec<V * (int)sizeof(T)>::type;

template <typename T, int V>
__device__ __forceinline__ void unpack(const Raw<T, V>& r, float* f) {
  if constexpr (V * sizeof(T) == 2) {
    f[0] = (float)*reinterpret_cast<const T*>(&r);
  } else {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < V * (int)sizeof(T) / 4; ++i) unpack_word<T>(w[i], f + i * PerWord<T>::kN);
  }
}

template <typename T, int V>
__device__ __forceinline__ Raw<T, V> pack(const float* f) {
  Raw<T, V> r;
  if constexpr (V * sizeof(T) == 2) {
    const T x = from_float<T>(f[0]);
    r = *reinterpret_cast<const uint16_t*>(&x);
  } else if constexpr (sizeof(T) == 4) {
    float* w = reinterpret_cast<float*>(&r);
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] = f[i];
  } else {
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) w[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
  }
  return r;
}

// V floats -> V e4m3 bytes at p (aligned to V).
template <int V>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float* f) {
  if constexpr (V == 1) {
    *p = (uint8_t)f2_to_e4m3x2(f[0], 0.f);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const uint32_t w = (uint32_t)f2_to_e4m3x2(f[i], f[i + 1]) | ((uint32_t)f2_to_e4m3x2(f[i + 2], f[i + 3]) << 16);
      reinterpret_cast<uint32_t*>(p)[i / 4] = w;
    }
  }
}

template <int V>
__device__ __forceinline__ void load_f32(const float* p, float* f) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      const float4 v = reinterpret_cast<const float4*>(p)[i];
      f[4 * i] = v.x;
      f[4 * i + 1] = v.y;
      f[4 * i + 2] = v.z;
      f[4 * i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = p[i];
  }
}

template <typename T, int V>
__device__ __forceinline__ void load_weight(const RopeArgs& a, const void* w, int off, float* f) {
  if (a.w_f32) {
    load_f32<V>(static_cast<const float*>(w) + off, f);
  } else {
    unpack<T, V>(*reinterpret_cast<const Raw<T, V>*>(static_cast<const T*>(w) + off), f);
  }
}

// One lane's unit of a row: its two column offsets and which of them exist.
struct Unit {
  int o1, o2;
  bool rot, has1, has2;
};

// kFull: every lane of a row has a unit that rotates (R = D, a power of two
// of units), known at compile time.
template <int V, bool IL, bool kFull>
__device__ __forceinline__ Unit unit_of(const RopeArgs& a, int u) {
  Unit x;
  x.rot = kFull || u < a.rot_units;
  x.has1 = kFull || u < a.units;
  if (x.rot) {
    x.o1 = IL ? 2 * u * V : u * V;
    x.o2 = IL ? x.o1 + V : a.rotary / 2 + x.o1;
    x.has2 = true;
  } else {
    x.o1 = a.rotary + (u - a.rot_units) * 2 * V;
    x.o2 = x.o1 + V;
    x.has2 = x.has1 && x.o2 < a.head_dim;
  }
  return x;
}

// Two f32 in one register pair; the packed instructions do both at once and
// round each as the scalar ones do.
struct Pair {
  uint64_t v;
};
__device__ __forceinline__ Pair pair(float lo, float hi) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(lo), "f"(hi));
  return p;
}
__device__ __forceinline__ void split(Pair p, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p.v));
}
__device__ __forceinline__ Pair mul2(Pair x, Pair y) {
  Pair p;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(p.v) : "l"(x.v), "l"(y.v));
  return p;
}
__device__ __forceinline__ Pair fma2(Pair x, Pair y, Pair z) {
  Pair p;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(p.v) : "l"(x.v), "l"(y.v), "l"(z.v));
  return p;
}

// What a lane multiplies its pairs (a, b) with, weights and angles in one:
//   a' = a ca + b sb,  b' = b cb + a sa   (ca = ga cos, cb = gb cos, sa = ga
//   sin, sb = -gb sin; columns that do not rotate: a ca, b cb)
// Of V rotating pairs, as packed as the lane's vectors are: p1 holds what
// multiplies the vectors themselves (ca then cb, or ca, cb, ca, ... when
// interleaved), p2 what multiplies their partners.
template <int V>
struct Turn {
  float p1[2 * V], p2[2 * V];
};

template <typename T, int V, int K, bool IL>
__device__ __forceinline__ void load_turn(const RopeArgs& a, const void* w, int pos, int lane, const Unit (&un)[K],
                                          Turn<V> (&tn)[K]) {
  const float* row = a.positions != nullptr ? a.cos_sin + (size_t)pos * a.rotary : nullptr;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float c[V], s[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      c[i] = 1.f;
      s[i] = 0.f;
    }
    if (un[k].rot && row != nullptr) {
      const int i = (lane + (k << a.lanes_log2)) * V;
      load_f32<V>(row + i, c);
      load_f32<V>(row + a.rotary / 2 + i, s);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int ia = IL ? 2 * i : i, ib = IL ? 2 * i + 1 : V + i;
      tn[k].p1[ia] = tn[k].p1[ib] = c[i];
      tn[k].p2[ia] = -s[i];
      tn[k].p2[ib] = s[i];
    }
    if (w != nullptr) {  // p1 has its own column's weight, p2 the partner's
      float g[2 * V];
#pragma unroll
      for (int i = 0; i < 2 * V; ++i) g[i] = 1.f;
      if (un[k].has1) load_weight<T, V>(a, w, un[k].o1, g);
      if (un[k].has2) load_weight<T, V>(a, w, un[k].o2, g + V);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int ia = IL ? 2 * i : i, ib = IL ? 2 * i + 1 : V + i;
        tn[k].p1[ia] *= g[ia];
        tn[k].p1[ib] *= g[ib];
        tn[k].p2[ia] *= g[ib];
        tn[k].p2[ib] *= g[ia];
      }
    }
  }
}

// Sum over the 2^log2 lanes of a row (aligned groups of a warp).
__device__ __forceinline__ float row_sum(float v, int log2) {
  for (int m = (1 << log2) >> 1; m > 0; m >>= 1) v += shfl_xor(v, m);
  return v;
}

// The lane's K units of one Q or K row, normed (if the row kind has a weight:
// the same for the whole warp) and turned, in f32.
template <int V, int K, bool IL>
__device__ __forceinline__ void norm_turn(const RopeArgs& a, float (&f)[K][2 * V], bool norm, const Unit (&un)[K],
                                          const Turn<V> (&tn)[K]) {
  float rs = 1.f;
  if (norm) {
    float ss = 0.f;
    if constexpr (V % 2 == 0) {
      Pair s0 = pair(0.f, 0.f), s1 = s0;  // four chains
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; i += 2) {
          const Pair x = pair(f[k][i], f[k][i + 1]), y = pair(f[k][V + i], f[k][V + i + 1]);
          s0 = fma2(x, x, s0);
          s1 = fma2(y, y, s1);
        }
      float a0, a1, b0, b1;
      split(s0, a0, a1);
      split(s1, b0, b1);
      ss = (a0 + a1) + (b0 + b1);
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) ss = fmaf(f[k][i], f[k][i], ss);
    }
    // 1 / sqrtf, correctly rounded twice, costs 3 us of 60 at 8192 tokens of
    // 32 + 8 heads and moves no output's error against 64 bits
    rs = rsqrtf(fmaf(row_sum(ss, a.lanes_log2), a.inv_dim, a.eps));
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const Turn<V>& t = tn[k];
    if (!un[k].rot) {
#pragma unroll
      for (int i = 0; i < 2 * V; ++i) f[k][i] = f[k][i] * t.p1[i] * rs;
    } else if constexpr (V % 2 == 0) {
      const Pair r = pair(rs, rs);
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        // two neighbouring columns each, and their partners'
        const int j = IL ? 2 * i : i, j2 = IL ? 2 * i + 2 : V + i;
        const Pair x = pair(f[k][j], f[k][j + 1]), y = pair(f[k][j2], f[k][j2 + 1]);
        const Pair xp = IL ? pair(f[k][j + 1], f[k][j]) : y, yp = IL ? pair(f[k][j2 + 1], f[k][j2]) : x;
        Pair u = fma2(x, pair(t.p1[j], t.p1[j + 1]), mul2(xp, pair(t.p2[j], t.p2[j + 1])));
        Pair v = fma2(y, pair(t.p1[j2], t.p1[j2 + 1]), mul2(yp, pair(t.p2[j2], t.p2[j2 + 1])));
        if (norm) {
          u = mul2(u, r);
          v = mul2(v, r);
        }
        split(u, f[k][j], f[k][j + 1]);
        split(v, f[k][j2], f[k][j2 + 1]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int ia = IL ? 2 * i : i, ib = IL ? 2 * i + 1 : V + i;
        const float x = f[k][ia], y = f[k][ib];
        f[k][ia] = fmaf(x, t.p1[ia], y * t.p2[ia]) * rs;
        f[k][ib] = fmaf(y, t.p1[ib], x * t.p2[ib]) * rs;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Row items.  A warp takes 32 / lanes heads of one token and one kind (Q, K
// or V) at a time, U times over: the token's angles and the kind's weights are
// loaded and multiplied once for all of them, and every branch on the kind is
// the whole warp's.  A lane copies its vectors of the next item into its own
// slots of shared memory (cp.async, which only the lane itself waits for)
// while it works on this one, and has the position and slot after that on
// their way.
// ---------------------------------------------------------------------------
constexpr int kItemStages = 2;
template <typename T, int V, int K, int U>
constexpr int kItemBytes = K == 1 ? U * 2 * 32 * V * (int)sizeof(T) : 0;  // of a warp and stage

// One vector into shared memory; zeros where there is none.
template <int kBytes>
__device__ __forceinline__ void copy_or_zero(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(kBytes),
               "r"(there ? kBytes : 0)
               : "memory");
}

template <typename T, int V, int K, int U, bool IL, bool kFull, bool kKv>
__device__ __forceinline__ void row_items(const RopeArgs& a, int64_t warp, int64_t num_warps, uint8_t* buffer) {
  constexpr bool kPipe = K == 1;  // (a lane of one-element vectors loads where it uses them)
  constexpr int VB = V * (int)sizeof(T);
  const int lane = threadIdx.x & 31;
  const int sub = lane & ((1 << a.lanes_log2) - 1);
  const int per_warp = 32 >> a.lanes_log2;
  const int grp = lane >> a.lanes_log2;
  const int nq = (a.num_heads + per_warp * U - 1) / (per_warp * U);
  const int nk = kKv ? (a.num_kv_heads + per_warp * U - 1) / (per_warp * U) : 0;
  const int per_token = nq + nk + (a.dest == kDense ? 0 : nk);
  Unit un[K];
#pragma unroll
  for (int k = 0; k < K; ++k) un[k] = unit_of<V, IL, kFull>(a, sub + (k << a.lanes_log2));

  // item = t * per_token + c, advanced without a division
  struct Item {
    int64_t t;
    int c, pos, slot;
  };
  const int64_t dt = num_warps / per_token;
  const int dc = (int)(num_warps - dt * per_token);
  auto look = [&](Item& x) {
    x.pos = a.positions != nullptr && x.t < a.num_tokens ? a.positions[x.t] : 0;
    x.slot = a.slots != nullptr && x.t < a.num_tokens ? a.slots[x.t] : -1;
  };
  auto advance = [&](Item x) {
    x.t += dt;
    x.c += dc;
    if (x.c >= per_token) {
      x.c -= per_token;
      ++x.t;
    }
    look(x);
    return x;
  };
  auto kind_of = [&](int c) { return !kKv || c < nq ? 0 : (c < nq + nk ? 1 : 2); };
  auto heads_of = [&](int kind) { return kind == 0 ? a.num_heads : a.num_kv_heads; };
  auto head_of = [&](int c, int kind) { return (kind == 0 ? c : kind == 1 ? c - nq : c - nq - nk) * per_warp * U + grp; };
  auto stride_of = [&](int kind) { return kind == 0 ? a.q_hs : kind == 1 ? a.k_hs : a.v_hs; };
  auto row_of = [&](const Item& x, int kind, int head) {
    const T* base = static_cast<const T*>(kind == 0 ? a.q : kind == 1 ? a.k : a.v);
    return base + x.t * (kind == 0 ? a.q_ts : kind == 1 ? a.k_ts : a.v_ts) + head * stride_of(kind);
  };
  uint8_t* mine = buffer + lane * VB;  // [stage][u][2][lane]
  auto copy = [&](const Item& x, int stage) {
    if (x.t < a.num_tokens) {
      const int kind = kind_of(x.c), heads = heads_of(kind), head0 = head_of(x.c, kind);
      const int64_t hs = stride_of(kind);
      const T* p = row_of(x, kind, head0);
      const uint32_t dst = smem_addr(mine) + stage * kItemBytes<T, V, K, U>;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        // where a row or a vector does not exist, nothing is read: the address is the base's
        const bool there = head0 + u * per_warp < heads;
        const T* r = there ? p + (int64_t)(u * per_warp) * hs : static_cast<const T*>(a.k);
        copy_or_zero<VB>(dst + (2 * u) * 32 * VB, r + (there && un[0].has1 ? un[0].o1 : 0), there && un[0].has1);
        copy_or_zero<VB>(dst + (2 * u + 1) * 32 * VB, r + (there && un[0].has2 ? un[0].o2 : 0), there && un[0].has2);
      }
    }
    cp_async_commit();
  };

  Item now;
  now.t = warp / per_token;
  now.c = (int)(warp - now.t * per_token);
  look(now);
  Item next = advance(now);
  if constexpr (kPipe) copy(now, 0);
  for (int stage = 0; now.t < a.num_tokens; stage ^= 1) {
    if constexpr (kPipe) copy(next, stage ^ 1);
    const Item x = now;
    now = next;
    next = advance(next);
    if constexpr (kPipe) asm volatile("cp.async.wait_group 1;" ::: "memory");
    const int kind = kind_of(x.c), heads = heads_of(kind), head0 = head_of(x.c, kind);
    if (a.positions != nullptr) {
      if (x.pos >= a.max_positions && lane == 0) rope_error(CF_DEVERR_POSITION);
      if (x.pos < 0 || x.pos >= a.max_positions) continue;  // a padding token, or one without angles: left out whole
    }
    const bool cached = kind > 0 && a.dest != kDense;
    if (cached) {
      if (x.slot >= a.num_slots && lane == 0) rope_error(CF_DEVERR_SLOT);
      if (x.slot < 0 || x.slot >= a.num_slots) continue;  // a padding row: nothing is appended
    }
    const void* w = kind == 0 ? a.q_w : kind == 1 ? a.k_w : nullptr;
    // the rows' destination, element strides as the source's
    const uint32_t blk = cached ? (uint32_t)x.slot / (uint32_t)a.block_size : 0u;
    const uint32_t off = cached ? (uint32_t)x.slot - blk * (uint32_t)a.block_size : 0u;
    const int64_t dhs = cached ? (int64_t)a.block_size * a.head_dim : kind == 0 ? a.qo_hs : a.ko_hs;
    const int64_t row0 = (cached ? ((int64_t)blk * a.num_kv_heads * a.block_size + off) * a.head_dim
                                 : kind == 0 ? x.t * a.qo_ts : x.t * a.ko_ts) + head0 * dhs;
    void* dbase = cached ? (kind == 1 ? a.kc : a.vc) : kind == 0 ? a.q_out : a.k_out;
    const float sc = kind == 1 ? a.k_scale : a.v_scale;
    const int64_t hs = stride_of(kind);
    const T* src = row_of(x, kind, head0);
    // kTurn: normed and rotated; kQuant: stored as e4m3; neither: moved as
    // they are, bit for bit.  kWhole: every row of the item exists.
    auto finish = [&](auto turn, auto quant, auto whole) {
      constexpr bool kTurn = decltype(turn)::value, kQuant = decltype(quant)::value, kWhole = decltype(whole)::value;
      Turn<V> tn[K];
      if (kTurn) load_turn<T, V, K, IL>(a, w, x.pos, sub, un, tn);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!kWhole && u > 0 && head0 - grp + u * per_warp >= heads) break;  // for the whole warp
        const bool there = kWhole || head0 + u * per_warp < heads;
        Raw<T, V> raw[K][2];
        if constexpr (kPipe) {
          const uint8_t* p = mine + stage * kItemBytes<T, V, K, U> + 2 * u * 32 * VB;
          raw[0][0] = *reinterpret_cast<const Raw<T, V>*>(p);
          raw[0][1] = *reinterpret_cast<const Raw<T, V>*>(p + 32 * VB);
        } else {
          const T* p = src + (int64_t)(u * per_warp) * hs;
#pragma unroll
          for (int k = 0; k < K; ++k) {
            raw[k][0] = raw[k][1] = Raw<T, V>{};
            if (there && un[k].has1) raw[k][0] = *reinterpret_cast<const Raw<T, V>*>(p + un[k].o1);
            if (there && un[k].has2) raw[k][1] = *reinterpret_cast<const Raw<T, V>*>(p + un[k].o2);
          }
        }
        float f[K][2 * V];
        if (kTurn || kQuant) {
#pragma unroll
          for (int k = 0; k < K; ++k) {
            unpack<T, V>(raw[k][0], f[k]);
            unpack<T, V>(raw[k][1], f[k] + V);
          }
        }
        if (kTurn) norm_turn<V, K, IL>(a, f, w != nullptr, un, tn);
        if (!there) continue;
        const int64_t row = row0 + (int64_t)(u * per_warp) * dhs;
        if (kQuant) {
          uint8_t* dst = static_cast<uint8_t*>(dbase) + row;
#pragma unroll
          for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) f[k][i] = __fdiv_rn(f[k][i], sc);
            if (un[k].has1) store_e4m3<V>(dst + un[k].o1, f[k]);
            if (un[k].has2) store_e4m3<V>(dst + un[k].o2, f[k] + V);
          }
        } else {
          T* dst = static_cast<T*>(dbase) + row;
#pragma unroll
          for (int k = 0; k < K; ++k) {
            if (un[k].has1) *reinterpret_cast<Raw<T, V>*>(dst + un[k].o1) = kTurn ? pack<T, V>(f[k]) : raw[k][0];
            if (un[k].has2) *reinterpret_cast<Raw<T, V>*>(dst + un[k].o2) = kTurn ? pack<T, V>(f[k] + V) : raw[k][1];
          }
        }
      }
    };
    using Y = std::true_type;
    using N = std::false_type;
    const bool fp8 = cached && a.dest == kCacheFp8;
    if (!kKv || (kind < 2 && !fp8))
      head0 - grp + U * per_warp <= heads ? finish(Y{}, N{}, Y{}) : finish(Y{}, N{}, N{});
    else if (kind < 2)
      finish(Y{}, Y{}, N{});
    else if (fp8)
      finish(N{}, Y{}, N{});
    else
      finish(N{}, N{}, N{});
  }
  if constexpr (kPipe) cp_async_wait_all();
}

constexpr int kRowThreads = 128;
constexpr int kRowWarps = kRowThreads / 32;

template <typename T, int V, int K, int U, bool IL, bool kFull>
__global__ void __launch_bounds__(kRowThreads) rope_rows_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int kArea = kItemStages * kItemBytes<T, V, K, U>;
  __shared__ __align__(16) uint8_t buffer[kRowWarps * kArea + 16];
  const int warp = threadIdx.x >> 5;
  row_items<T, V, K, U, IL, kFull, true>(a, (int64_t)blockIdx.x * kRowWarps + warp, (int64_t)gridDim.x * kRowWarps,
                                         buffer + warp * kArea);
}

// ---------------------------------------------------------------------------
// Append into e4m3 caches with a scale for each block and KV head.
//
// For the rows N that a call appends to block b, head h (K and V apart):
//   need  the smallest power of two s with max |x| <= 448 s over the finite
//         x in N; 0 if they are all 0
//   fresh N holds the block's offset 0: a new sequence of rows starts there,
//         so s = need, and what the block held before says nothing
//   else  s = max(s_old, need), and where that grew, the block's other rows
//         are stored anew as e4m3(byte * s_old / s)
//   bytes e4m3(x / s), to nearest even, saturating at +-448
// A power of two costs e4m3 nothing: it is a float, so its relative precision
// does not depend on where in the range the values lie, x / s is exact, and
// storing a row anew only moves exponents (it rounds values that fall under
// e4m3's smallest normal 2^-6 s, and no others).
//
// One CTA takes a window of 16 tokens of the call and the blocks whose FIRST
// token lies in it, with all their rows wherever in the call they are: it
// looks through the call's slots for them (a 1024-bit filter first).  So a
// block has one writer for any order of the tokens, and of two tokens with
// one slot the later one is stored.  That search reads num_tokens slots per
// window, 4 / 16 num_tokens^2 bytes from L2 in all; calls beyond kPiece
// tokens run as consecutive pieces.
// ---------------------------------------------------------------------------
constexpr int kBlk = 16;  // tokens of a KV block
constexpr int kPiece = 16384;
constexpr int kHeads = 16;  // heads a CTA works on between two block barriers

struct BlockArgs {
  RopeArgs r;
  float* k_scales;  // [num_blocks, Hkv]
  float* v_scales;
  int32_t head_split;  // CTAs per window, each with every head_split-th head
  int32_t kv_ctas;     // windows * head_split
  int32_t q_ctas;      // for the Q rows, dealt evenly among the others
};

struct BlockSmem {
  int32_t key[kBlk];            // block id of each window token, -1: none
  int32_t lead[kBlk];           // the block this token is the first of in the window, else -1
  int32_t dead[kBlk];           // its first token lies before the window
  int32_t win[kBlk][kBlk];      // token that gives row `off` of block lead[l], -1: none
  uint32_t filter[32];
  uint32_t few[2];              // first slots of the first two blocks led
  int32_t row_tok[kBlk * kBlk]; // the rows to append: token, and l * 16 + off
  int32_t row_lo[kBlk * kBlk];
  int32_t count[kWarps];
  int32_t state[kBlk];          // of a block: its rows in the call, as bits; 0 where it is not this CTA's
  uint32_t top[2][kHeads][kBlk]; // (K, V), heads at a time: max |x| of a block's rows, as f32 bits
  float old[2][kHeads][kBlk];    // its scale before the call
  float now[2][kHeads][kBlk];    // and after it
};

// The smallest power of two s >= 2^-126 with x <= 448 s; 0 for 0.
// 448 = 1.75 * 2^8: for 2^e <= x < 2^(e+1) that is 2^(e-8) up to 1.75 * 2^e
// and 2^(e-7) beyond, read off the exponent and mantissa.
__device__ __forceinline__ float block_scale(uint32_t bits) {
  if (bits == 0) return 0.f;
  int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = e < 1 ? 1 : e;
  return __uint_as_float((uint32_t)e << 23);
}

constexpr int kTasks = 64;  // (K or V, group of rows, head) copied at once: 64 KB
constexpr int kStageOffset = (int)((sizeof(BlockSmem) + 127) / 128 * 128);
// Shared memory of a CTA of either kind.
template <typename T, int V, int K>
constexpr int kBlockBytes = K == 1 ? kStageOffset + kTasks * 2 * 32 * V * (int)sizeof(T) : kStageOffset;

template <typename T, int V, int K, bool IL, bool kFull>
__global__ void __launch_bounds__(kThreads, 2) rope_block_append_kernel(const __grid_constant__ BlockArgs b) {
  const RopeArgs& a = b.r;
  constexpr int U = K == 1 ? 4 : 1, kArea = kItemStages * kItemBytes<T, V, K, U>;
  extern __shared__ __align__(16) uint8_t smem[];
  // Appends wait on memory, Q rows stream it: CTA i is one of the first or of
  // the second kind so that any stretch of them holds both in proportion.
  const int64_t ctas = (int64_t)b.kv_ctas + b.q_ctas;
  const int q_before = (int)((int64_t)blockIdx.x * b.q_ctas / ctas);
  if ((int64_t)(blockIdx.x + 1) * b.q_ctas / ctas > q_before) {
    const int warp = threadIdx.x >> 5;
    row_items<T, V, K, U, IL, kFull, false>(a, (int64_t)q_before * kWarps + warp, (int64_t)b.q_ctas * kWarps,
                                            smem + warp * kArea);
    return;
  }
  const int cta = blockIdx.x - q_before;
  BlockSmem& sm = *reinterpret_cast<BlockSmem*>(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int window = cta / b.head_split;
  const int w0 = window * kBlk;
  const int T_ = a.num_tokens;

  // 1. the window's blocks
  (&sm.win[0][0])[tid] = -1;
  if (tid < 32) sm.filter[tid] = 0u;
  if (tid < 2 * kBlk) {
    sm.top[0][tid / kBlk][tid % kBlk] = 0u;
  }
  // A token without a position in the table counts as little as one without a
  // slot: an earlier one with its slot is stored.
  auto position = [&](int i) { return a.positions != nullptr ? a.positions[i] : 0; };
  auto live = [&](int pos) { return pos >= 0 && pos < a.max_positions; };
  int key = -1;
  if (tid < kBlk) {
    if (w0 + tid < T_) {
      const int64_t slot = a.slots[w0 + tid];
      const int pos = position(w0 + tid);
      if (!live(pos)) {
        if (pos >= 0) rope_error(CF_DEVERR_POSITION);
      } else if (slot >= a.num_slots) {
        rope_error(CF_DEVERR_SLOT);
      } else if (slot >= 0) {
        key = (int)(slot / kBlk);
      }
    }
    sm.key[tid] = key;
    sm.dead[tid] = 0;
  }
  __syncthreads();
  bool leads = false;
  if (tid < kBlk) {
    int first = tid;  // of the window's tokens in this block
    for (int j = kBlk - 1; j >= 0; --j)
      if (j < first && sm.key[j] == key) first = j;
    leads = key >= 0 && first == tid;
    sm.lead[tid] = leads ? key : -1;
    if (leads) atomicOr(&sm.filter[(key >> 5) & 31], 1u << (key & 31));
    const uint32_t leaders = __ballot_sync(0xffffu, leads);
    const int before = __popc(leaders & ((1u << tid) - 1u));
    if (leads && before < 2) sm.few[before] = (uint32_t)key * kBlk;
    if (leads && leaders == 1u << tid) sm.few[1] = (uint32_t)key * kBlk;
    if (key >= 0) atomicMax(&sm.win[first][a.slots[w0 + tid] % kBlk], w0 + tid);
  }
  const int led = __syncthreads_count(leads ? 1 : 0);
  if (led == 0) return;  // padding only

  // 2. their tokens outside the window, wherever they are in the call (seldom
  // more than a run that goes on behind it): four slots a load where they are
  // 16-byte aligned, eight loads in flight.  One or two blocks, as a window of
  // a prompt has, are compared with directly, more of them looked up in the
  // filter (16384 tokens of prompts, 32 / 8 heads: 117 us, 127 with the filter
  // for all; looking up four slots for one bit took 1024 decode rows from 18
  // to 22 us, by the false hits).
  auto hit = [&](int slot) -> uint32_t {
    const int k = slot / kBlk;
    return slot >= 0 ? (sm.filter[(k >> 5) & 31] >> (k & 31)) & 1u : 0u;
  };
  auto match = [&](int i) {
    const int slot = a.slots[i], k = slot / kBlk;
    if (slot < 0 || !live(position(i))) return;
#pragma unroll 1
    for (int l = 0; l < kBlk; ++l) {
      if (sm.lead[l] != k) continue;
      if (i < w0)
        sm.dead[l] = 1;
      else
        atomicMax(&sm.win[l][slot % kBlk], i);
    }
  };
  constexpr int kLook = 8;
  const int quads = (reinterpret_cast<uintptr_t>(a.slots) & 15) == 0 ? T_ / 4 : 0;
#pragma unroll 1
  for (int q0 = tid; q0 < quads; q0 += kThreads * kLook) {
    int4 slot[kLook];
#pragma unroll
    for (int u = 0; u < kLook; ++u) {
      const int q = q0 + u * kThreads;
      const bool look = q < quads && (uint32_t)(q - w0 / 4) >= (uint32_t)(kBlk / 4);
      slot[u] = look ? reinterpret_cast<const int4*>(a.slots)[q] : make_int4(-1, -1, -1, -1);
    }
    uint32_t hits = 0u;
    if (led <= 2) {
      const uint32_t lo0 = sm.few[0], lo1 = sm.few[1];
      auto in = [&](int x) { return (uint32_t)x - lo0 < (uint32_t)kBlk || (uint32_t)x - lo1 < (uint32_t)kBlk; };
#pragma unroll
      for (int u = 0; u < kLook; ++u)
        if (in(slot[u].x) || in(slot[u].y) || in(slot[u].z) || in(slot[u].w)) hits |= 15u << (4 * u);
    } else {
#pragma unroll
      for (int u = 0; u < kLook; ++u)
        hits |= (hit(slot[u].x) | hit(slot[u].y) << 1 | hit(slot[u].z) << 2 | hit(slot[u].w) << 3) << (4 * u);
    }
#pragma unroll 1
    for (; hits != 0u; hits &= hits - 1u) {
      const int j = __ffs(hits) - 1;
      match((q0 + j / 4 * kThreads) * 4 + j % 4);
    }
  }
#pragma unroll 1
  for (int i = 4 * quads + tid; i < T_; i += kThreads)
    if ((uint32_t)(i - w0) >= (uint32_t)kBlk && hit(a.slots[i])) match(i);
  __syncthreads();

  // 3. the rows to append, in (block, offset) order
  int n;
  {
    const int l = tid / kBlk, off = tid % kBlk;
    const int tok = sm.dead[l] ? -1 : sm.win[l][off];
    const uint32_t there = __ballot_sync(0xffffffffu, tok >= 0);
    if (lane == 0) sm.count[warp] = __popc(there);
    __syncthreads();
    sm.win[l][off] = tok;
    int at = __popc(there & ((1u << lane) - 1u));
    n = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) at += sm.count[w];
      n += sm.count[w];
    }
    if (tok >= 0) {
      sm.row_tok[at] = tok;
      sm.row_lo[at] = tid;
    }
    if ((lane & 15) == 0) sm.state[l] = (int32_t)((there >> lane) & 0xffffu);
  }
  __syncthreads();
  if (n == 0) return;  // no row of these blocks is this CTA's

  // 4. the rows, some heads at a time: maxima, scales, bytes.  A warp takes
  // 32 / lanes rows of K or V and walks the heads, so the rows' angles and the
  // weights are loaded once; where that leaves warps over, they share the
  // heads.  All the vectors of these heads are copied into shared memory at
  // once (a lane's own slots, 1 KB a warp, row group and head); both walks,
  // for the maxima and for the bytes, read them there.
  const int sub = lane & ((1 << a.lanes_log2) - 1);
  const int per_warp = 32 >> a.lanes_log2;
  const int groups = (n + per_warp - 1) / per_warp;
  const int sharing = max(1, kWarps / (2 * groups));  // warps per (K or V, group of rows)
  constexpr int VB = V * (int)sizeof(T);
  constexpr int kTaskBytes = 2 * 32 * VB;
  const bool staged = K == 1 && 2 * groups <= kTasks;  // else (rows from all over the call) loaded where used
  const int at_once = staged ? min(kHeads, kTasks / (2 * groups)) : kHeads;
  Unit un[K];
#pragma unroll
  for (int k = 0; k < K; ++k) un[k] = unit_of<V, IL, kFull>(a, sub + (k << a.lanes_log2));
  uint8_t* stage = smem + kStageOffset + lane * VB;

  Turn<V> tn[K];
  float f[K][2 * V];
  auto row = [&](int kv, int e, int head) {  // row e of the list
    return static_cast<const T*>(kv ? a.v : a.k) + (int64_t)sm.row_tok[e] * (kv ? a.v_ts : a.k_ts) +
           (int64_t)head * (kv ? a.v_hs : a.k_hs);
  };
  auto slot_at = [&](int kv, int group, int hi) { return ((kv * groups + group) * at_once + hi) * kTaskBytes; };
  auto turns = [&](int kv) { return kv == 0 && (a.k_w != nullptr || a.positions != nullptr); };
  auto angles = [&](int kv, int e) {
    if (turns(kv) && e < n)
      load_turn<T, V, K, IL>(a, a.k_w, a.positions != nullptr ? a.positions[sm.row_tok[e]] : 0, sub, un, tn);
  };
  auto values = [&](int kv, int group, int e, int hi, int head) {  // normed and turned, in f
    Raw<T, V> raw[K][2];
#pragma unroll
    for (int k = 0; k < K; ++k) raw[k][0] = raw[k][1] = Raw<T, V>{};
    if (K == 1 && staged) {
      const uint8_t* p = stage + slot_at(kv, group, hi);
      raw[0][0] = *reinterpret_cast<const Raw<T, V>*>(p);
      raw[0][1] = *reinterpret_cast<const Raw<T, V>*>(p + 32 * VB);
    } else if (e < n) {
      const T* p = row(kv, e, head);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (un[k].has1) raw[k][0] = *reinterpret_cast<const Raw<T, V>*>(p + un[k].o1);
        if (un[k].has2) raw[k][1] = *reinterpret_cast<const Raw<T, V>*>(p + un[k].o2);
      }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      unpack<T, V>(raw[k][0], f[k]);
      unpack<T, V>(raw[k][1], f[k] + V);
    }
    if (turns(kv)) norm_turn<V, K, IL>(a, f, a.k_w != nullptr, un, tn);
  };
  const int mine = cta % b.head_split;  // heads mine, mine + head_split, ...
  const int heads = (a.num_kv_heads - mine + b.head_split - 1) / b.head_split;
#pragma unroll 1
  for (int h0 = 0; h0 < heads; h0 += at_once) {
    const int nh = min(at_once, heads - h0);
    auto head_of = [&](int i) { return mine + (h0 + i) * b.head_split; };
    // (K or V, group of rows, share of the heads) of this warp
    auto walk = [&](auto&& work) {
#pragma unroll 1
      for (int c = warp; c < 2 * groups * sharing; c += kWarps) {
        const int kv = c % 2, group = c / 2 % groups;
        work(kv, group, group * per_warp + (lane >> a.lanes_log2), c / (2 * groups));
      }
    };
    if (h0 > 0) __syncthreads();
    if constexpr (K == 1) {
      if (staged)
        walk([&](int kv, int group, int e, int share) {
          const bool there = e < n;
          const uint32_t dst = smem_addr(stage) + slot_at(kv, group, 0);
          const T* p = there ? row(kv, e, head_of(share)) : static_cast<const T*>(a.k);
          const int64_t step = there ? (int64_t)(kv ? a.v_hs : a.k_hs) * sharing * b.head_split : 0;
          for (int hi = share; hi < nh; hi += sharing, p += step) {
            copy_or_zero<VB>(dst + hi * kTaskBytes, p + (there && un[0].has1 ? un[0].o1 : 0), there && un[0].has1);
            copy_or_zero<VB>(dst + hi * kTaskBytes + 32 * VB, p + (there && un[0].has2 ? un[0].o2 : 0),
                             there && un[0].has2);
          }
        });
      cp_async_commit();
    }
    for (int i = tid; i < 2 * kHeads * kBlk; i += kThreads) {
      const int kv = i / (kHeads * kBlk), hi = i / kBlk % kHeads, l = i % kBlk;
      float s = 0.f;
      if (hi < nh && sm.state[l] != 0)
        s = (kv ? b.v_scales : b.k_scales)[(int64_t)sm.lead[l] * a.num_kv_heads + head_of(hi)];
      sm.old[kv][hi][l] = s > 0.f && s < INFINITY ? s : 0.f;
      sm.top[kv][hi][l] = 0u;
    }
    __syncthreads();
    const bool once = 2 * groups * sharing <= kWarps;  // a warp has one kind and group: its angles stay
    walk([&](int kv, int group, int e, int share) {
      angles(kv, e);
      if (K == 1) cp_async_wait_all();
#pragma unroll 1
      for (int hi = share; hi < nh; hi += sharing) {
        values(kv, group, e, hi, head_of(hi));
        float top = 0.f;  // over the finite values: fmaxf leaves NaN out, infinities are looked for after
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) top = fmaxf(top, fabsf(f[k][i]));
        if (top == INFINITY) {
          top = 0.f;
#pragma unroll
          for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) top = fmaxf(top, fabsf(f[k][i]) == INFINITY ? 0.f : fabsf(f[k][i]));
        }
        for (int m = (1 << a.lanes_log2) >> 1; m > 0; m >>= 1) top = fmaxf(top, shfl_xor(top, m));
        if (e < n && sub == 0) atomicMax(&sm.top[kv][hi][sm.row_lo[e] / kBlk], __float_as_uint(top));
      }
    });
    __syncthreads();
    for (int i = tid; i < 2 * kHeads * kBlk; i += kThreads) {
      const int kv = i / (kHeads * kBlk), hi = i / kBlk % kHeads, l = i % kBlk;
      if (hi >= nh || sm.state[l] == 0) continue;
      const float need = block_scale(sm.top[kv][hi][l]);
      const float s = (sm.state[l] & 1) != 0 ? need : fmaxf(sm.old[kv][hi][l], need);
      sm.now[kv][hi][l] = s;
      (kv ? b.v_scales : b.k_scales)[(int64_t)sm.lead[l] * a.num_kv_heads + head_of(hi)] = s;
    }
    __syncthreads();
    walk([&](int kv, int group, int e, int share) {
      uint8_t* cache = static_cast<uint8_t*>(kv ? a.vc : a.kc);
      const int l = e < n ? sm.row_lo[e] / kBlk : 0, off = e < n ? sm.row_lo[e] % kBlk : 0;
      const int64_t block = (int64_t)sm.lead[l] * a.num_kv_heads;
      if (!once) angles(kv, e);
#pragma unroll 1
      for (int hi = share; hi < nh; hi += sharing) {
        if (!(once && nh <= sharing)) values(kv, group, e, hi, head_of(hi));  // one head: still in f
        if (e >= n) continue;
        const float s = sm.now[kv][hi][l];
        uint8_t* dst = cache + ((block + head_of(hi)) * kBlk + off) * a.head_dim;
        const uint32_t bits = __float_as_uint(s);
        if ((bits & 0x7fffffu) == 0u && bits >= (1u << 23) && bits < (254u << 23)) {
          const float inv = __uint_as_float((254u << 23) - bits);  // x / 2^k = x 2^-k, exactly
          const Pair r = pair(inv, inv);
#pragma unroll
          for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < 2 * V; i += 2) split(mul2(pair(f[k][i], f[k][i + 1]), r), f[k][i], f[k][i + 1]);
        } else if (s > 0.f) {  // a pool may hold scales that are no powers of two
#pragma unroll
          for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) f[k][i] = __fdiv_rn(f[k][i], s);
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (un[k].has1) store_e4m3<V>(dst + un[k].o1, f[k]);
          if (un[k].has2) store_e4m3<V>(dst + un[k].o2, f[k] + V);
        }
      }
    });
    // blocks whose scale grew under rows that stay: those rows, a warp a block
    for (int i0 = warp * 32; i0 < 2 * kHeads * kBlk; i0 += kThreads) {
      const int i = i0 + lane, kvl = i / (kHeads * kBlk), hil = i / kBlk % kHeads, ll = i % kBlk;
      const bool grew = hil < nh && sm.state[ll] != 0 && (sm.state[ll] & 1) == 0 && sm.now[kvl][hil][ll] > sm.old[kvl][hil][ll];
      uint32_t todo = __ballot_sync(0xffffffffu, grew);
      while (todo != 0u) {
        const int j = i0 + __ffs(todo) - 1;
        todo &= todo - 1u;
        const int kv = j / (kHeads * kBlk), hi = j / kBlk % kHeads, l = j % kBlk;
        const float ratio = sm.old[kv][hi][l] / sm.now[kv][hi][l];
        const int chunks = a.head_dim / 16;
        uint8_t* base = static_cast<uint8_t*>(kv ? a.vc : a.kc) +
                        ((int64_t)sm.lead[l] * a.num_kv_heads + head_of(hi)) * kBlk * a.head_dim;
        for (int c = lane; c < kBlk * chunks; c += 32) {
          if ((sm.state[l] >> (c / chunks)) & 1) continue;
          uint4* p = reinterpret_cast<uint4*>(base) + c;
          float x[16];
          load_widen<__nv_fp8_e4m3, 16>(reinterpret_cast<const __nv_fp8_e4m3*>(p), x);
#pragma unroll
          for (int k = 0; k < 16; ++k) x[k] *= ratio;
          store_e4m3<16>(reinterpret_cast<uint8_t*>(p), x);
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
int sm_count() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 148;
}

// The widest vector (elements) that every address of the call allows: 16
// bytes, 8 (16-bit types), or one element.
int vector_elems(const RopeArgs& a, int eb) {
  auto ok = [&](int v) {
    const int64_t bytes = (int64_t)v * eb;
    auto ptr = [&](const void* p, int64_t al) { return p == nullptr || reinterpret_cast<uintptr_t>(p) % al == 0; };
    auto row = [&](const void* p, int64_t ts, int64_t hs) {
      return p == nullptr || (ptr(p, bytes) && ts * eb % bytes == 0 && hs * eb % bytes == 0);
    };
    const int64_t wb = a.w_f32 ? 16 : bytes;
    return a.head_dim % v == 0 && a.rotary % (2 * v) == 0 && row(a.q, a.q_ts, a.q_hs) && row(a.k, a.k_ts, a.k_hs) &&
           row(a.v, a.v_ts, a.v_hs) && row(a.q_out, a.qo_ts, a.qo_hs) && row(a.k_out, a.ko_ts, a.ko_hs) &&
           ptr(a.q_w, wb) && ptr(a.k_w, wb) && ptr(a.cos_sin, 16) && ptr(a.kc, bytes) && ptr(a.vc, bytes);
  };
  if (ok(16 / eb)) return 16 / eb;
  if (eb == 2 && ok(4)) return 4;
  return 1;
}

// Fills the row layout; K = units per lane (1 or 4).
int row_layout(RopeArgs& a, int v) {
  a.rot_units = a.rotary / (2 * v);
  a.units = a.rot_units + (a.head_dim - a.rotary + 2 * v - 1) / (2 * v);
  const int k = v == 1 ? 4 : 1;
  const int lanes = (a.units + k - 1) / k;
  a.lanes_log2 = 0;
  while ((1 << a.lanes_log2) < lanes) ++a.lanes_log2;
  return k;
}

// Whether every lane of a row has a unit that rotates.
bool full_rows(const RopeArgs& a) { return a.rotary == a.head_dim && a.units == (1 << a.lanes_log2); }

// CTAs of `warps` warps for the row items of `heads` (a count per kind, 0 for
// none), at most `cap`.
unsigned row_ctas(const RopeArgs& a, int u, int warps, int64_t cap, std::initializer_list<int> heads) {
  const int rows = (32 >> a.lanes_log2) * u;
  int64_t items = 0;
  for (int h : heads) items += (h + rows - 1) / rows;
  items *= a.num_tokens;
  const int64_t want = (items + warps - 1) / warps;
  return (unsigned)(want < cap ? want : cap);
}

// Runs as many CTAs as are resident at once: each walks its items with the
// next one's copies in flight (8192 tokens of 64 / 8 heads 60 us, 76 with a
// quarter more CTAs than that, 63 with four times as many).
template <typename T, int V, int K, int U, bool IL, bool kFull>
cf_status launch_rows_kernel(const RopeArgs& a, cudaStream_t stream) {
  static std::atomic<int> resident[64];
  auto kern = rope_rows_kernel<T, V, K, U, IL, kFull>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e);
  int per_sm = dev < 64 ? resident[dev].load(std::memory_order_relaxed) : 0;
  if (per_sm == 0) {
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, kRowThreads, 0);
    if (e != cudaSuccess) return cuda_status(e);
    per_sm = per_sm < 1 ? 1 : per_sm;
    if (dev < 64) resident[dev].store(per_sm, std::memory_order_relaxed);
  }
  const unsigned grid = row_ctas(a, U, kRowWarps, (int64_t)sm_count() * per_sm,
                                 {a.num_heads, a.num_kv_heads, a.dest == kDense ? 0 : a.num_kv_heads});
  kern<<<grid, kRowThreads, 0, stream>>>(a);
  return check_launch();
}

template <typename T, int V, int K, int U>
cf_status launch_rows_u(const RopeArgs& a, bool interleaved, cudaStream_t stream) {
  if constexpr (K == 1) {
    if (full_rows(a))
      return interleaved ? launch_rows_kernel<T, V, K, U, true, true>(a, stream)
                         : launch_rows_kernel<T, V, K, U, false, true>(a, stream);
  }
  return interleaved ? launch_rows_kernel<T, V, K, U, true, false>(a, stream)
                     : launch_rows_kernel<T, V, K, U, false, false>(a, stream);
}

template <typename T, int V, int K>
cf_status launch_rows(const RopeArgs& a, bool interleaved, cudaStream_t stream) {
  if constexpr (K == 1) {
    // Heads per lane group and item: four 16-bit rows (8192 tokens of 64 / 8
    // heads 64 us, 77 with two), two f32 ones (4095 tokens of 32 / 32 heads 29
    // us, 32 with four), one where a call has few items (a token of 32 / 8
    // heads 3.7 us, 4.3 with four).
    constexpr int U = sizeof(T) == 4 ? 2 : 4;
    const unsigned ctas = row_ctas(a, U, kRowWarps, INT32_MAX, {a.num_heads, a.num_kv_heads, a.num_kv_heads});
    return ctas < (unsigned)sm_count() ? launch_rows_u<T, V, K, 1>(a, interleaved, stream)
                                       : launch_rows_u<T, V, K, U>(a, interleaved, stream);
  }
  return launch_rows_u<T, V, K, 1>(a, interleaved, stream);
}

template <typename T>
cf_status launch_rows_type(RopeArgs& a, bool interleaved, cudaStream_t stream) {
  const int v = vector_elems(a, sizeof(T));
  row_layout(a, v);
  if (v == 16 / (int)sizeof(T)) return launch_rows<T, 16 / (int)sizeof(T), 1>(a, interleaved, stream);
  if constexpr (sizeof(T) == 2)
    if (v == 4) return launch_rows<T, 4, 1>(a, interleaved, stream);
  return launch_rows<T, 1, 4>(a, interleaved, stream);
}

// Per kernel instantiation and device: opt in to > 48 KB of dynamic smem.
template <typename T, int V, int K, bool IL, bool kFull>
cf_status launch_block_kernel(const BlockArgs& b, unsigned grid, cudaStream_t stream) {
  static std::once_flag flags[64];
  static cudaError_t errs[64];
  auto kern = rope_block_append_kernel<T, V, K, IL, kFull>;
  constexpr int bytes = kBlockBytes<T, V, K>;
  auto set = [&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); };
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) {
    if (dev >= 0 && dev < 64) {
      std::call_once(flags[dev], [&] { errs[dev] = set(); });
      e = errs[dev];
    } else {
      e = set();
    }
  }
  if (e != cudaSuccess) return cuda_status(e);
  kern<<<grid, kThreads, bytes, stream>>>(b);
  return check_launch();
}

template <typename T, int V, int K>
cf_status launch_block(BlockArgs b, bool interleaved, cudaStream_t stream) {
  const RopeArgs& a = b.r;
  const int windows = (a.num_tokens + kBlk - 1) / kBlk;
  // Two CTAs per SM are resident.  Up to a CTA per SM a window's heads are
  // shared among several.  The Q rows take what the windows leave of one wave
  // as long as a Q CTA is done with them about when the windows are, which
  // take as long as 4 rounds of Q items and 3.7 for each KB of a token's K.
  // Past that they get up to four CTAs per SM among the windows.  Measured,
  // one wave / four per SM: 32 / 8 heads of 128, 2048 tokens 21 / 28 us, 3400
  // (10 rounds) 33 / 36, 3600 (13) 40 / 37, 4096 75 / 40; 64 / 8 heads, 2400 (8)
  // 28 / 37, 3200 (17) 52 / 45; 128 / 8 heads, 1600 (8) 29 / 39, 2368 (16) 51 / 48;
  // 32 / 8 of 256, 3200 (17) 54 / 67, 3600 (25) 76 / 75; 32 / 32, 4200 (32) 81 / 91,
  // 4300 (40) 111 / 94; 12 / 4 of 96, 3600 (6) 24 / 26, 4000 (11) 37 / 27.  Two or
  // eight per SM in place of four: 16384 tokens of 32 / 8 heads 128 and 119 / 117.
  const int sms = sm_count();
  const int split = sms / windows;
  b.head_split = split < 1 ? 1 : (split > a.num_kv_heads ? a.num_kv_heads : split);
  b.kv_ctas = windows * b.head_split;
  const int64_t left = 2 * (int64_t)sms - b.kv_ctas;
  constexpr int U = K == 1 ? 4 : 1;
  const double rounds = 4 + 3.7 / 1024 * a.num_kv_heads * a.head_dim * (double)sizeof(T);
  const bool one_wave = left > 0 && row_ctas(a, U, kWarps, INT32_MAX, {a.num_heads}) <= rounds * left;
  b.q_ctas = a.num_heads > 0 ? (int32_t)row_ctas(a, U, kWarps, one_wave ? left : 4 * (int64_t)sms, {a.num_heads}) : 0;
  const unsigned grid = (unsigned)(b.kv_ctas + b.q_ctas);
  if constexpr (K == 1) {
    if (full_rows(a))
      return interleaved ? launch_block_kernel<T, V, K, true, true>(b, grid, stream)
                         : launch_block_kernel<T, V, K, false, true>(b, grid, stream);
  }
  return interleaved ? launch_block_kernel<T, V, K, true, false>(b, grid, stream)
                     : launch_block_kernel<T, V, K, false, false>(b, grid, stream);
}

template <typename T>
cf_status launch_block_type(BlockArgs& b, bool interleaved, cudaStream_t stream) {
  const int v = vector_elems(b.r, sizeof(T));
  row_layout(b.r, v);
  if (v == 16 / (int)sizeof(T)) return launch_block<T, 16 / (int)sizeof(T), 1>(b, interleaved, stream);
  if constexpr (sizeof(T) == 2)
    if (v == 4) return launch_block<T, 4, 1>(b, interleaved, stream);
  return launch_block<T, 1, 4>(b, interleaved, stream);
}

RopeArgs rope_args(const cf_rope_params& p) {
  RopeArgs a = {};
  a.q = p.query;
  a.k = p.key;
  a.v = p.value;
  a.q_out = p.query_out;
  a.k_out = p.key_out;
  a.q_ts = p.query_stride[0], a.q_hs = p.query_stride[1];
  a.k_ts = p.key_stride[0], a.k_hs = p.key_stride[1];
  a.v_ts = p.value_stride[0], a.v_hs = p.value_stride[1];
  a.qo_ts = p.query_out_stride[0], a.qo_hs = p.query_out_stride[1];
  a.ko_ts = p.key_out_stride[0], a.ko_hs = p.key_out_stride[1];
  a.positions = p.positions;
  a.cos_sin = p.cos_sin;
  a.q_w = p.query_weight;
  a.k_w = p.key_weight;
  a.w_f32 = p.weight_dtype == CF_F32;
  a.eps = p.eps;
  a.inv_dim = 1.f / (float)p.head_dim;
  a.num_tokens = p.num_tokens;
  a.num_heads = p.num_heads;
  a.num_kv_heads = p.num_kv_heads;
  a.head_dim = p.head_dim;
  a.rotary = p.rotary_dim;
  a.max_positions = p.max_positions;
  return a;
}

}  // namespace

cf_status launch_qk_norm_rope(const cf_rope_params& p, cudaStream_t stream) {
  RopeArgs a = rope_args(p);
  a.v = nullptr;
  a.dest = kDense;
  a.num_slots = INT64_MAX;
  const bool il = p.interleaved != 0;
  switch (p.dtype) {
    case CF_F32: return launch_rows_type<float>(a, il, stream);
    case CF_F16: return launch_rows_type<__half>(a, il, stream);
    default: return launch_rows_type<__nv_bfloat16>(a, il, stream);
  }
}

cf_status launch_rope_and_cache(const cf_rope_params& p, void* key_cache, void* value_cache,
                                const int32_t* slot_mapping, int32_t block_size, int64_t num_blocks, bool fp8,
                                float k_scale, float v_scale, cudaStream_t stream) {
  RopeArgs a = rope_args(p);
  a.k_out = nullptr;
  a.dest = fp8 ? kCacheFp8 : kCacheSame;
  a.kc = key_cache;
  a.vc = value_cache;
  a.slots = slot_mapping;
  a.block_size = block_size;
  a.num_slots = num_blocks * block_size;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  const bool il = p.interleaved != 0;
  switch (p.dtype) {
    case CF_F32: return launch_rows_type<float>(a, il, stream);
    case CF_F16: return launch_rows_type<__half>(a, il, stream);
    default: return launch_rows_type<__nv_bfloat16>(a, il, stream);
  }
}

cf_status launch_rope_and_cache_fp8_block(const cf_rope_params& p, void* key_cache, void* value_cache,
                                          float* k_scales, float* v_scales, const int32_t* slot_mapping,
                                          int64_t num_blocks, cudaStream_t stream) {
  const int eb = dtype_bytes(p.dtype);
  for (int64_t t0 = 0; t0 < p.num_tokens; t0 += kPiece) {
    BlockArgs b = {};
    b.r = rope_args(p);
    RopeArgs& a = b.r;
    auto at = [&](const void* base, int64_t stride) -> void* {
      return base == nullptr ? nullptr : const_cast<uint8_t*>(static_cast<const uint8_t*>(base)) + t0 * stride * eb;
    };
    a.q = at(a.q, a.q_ts);
    a.k = at(a.k, a.k_ts);
    a.v = at(a.v, a.v_ts);
    a.q_out = at(a.q_out, a.qo_ts);
    a.k_out = nullptr;
    if (a.positions != nullptr)
      a.positions += t0;
    else
      a.max_positions = 1;  // every token's position counts as 0
    a.num_tokens = (int32_t)(p.num_tokens - t0 < kPiece ? p.num_tokens - t0 : kPiece);
    a.dest = kCacheFp8;
    a.kc = key_cache;
    a.vc = value_cache;
    a.slots = slot_mapping + t0;
    a.block_size = kBlk;
    a.num_slots = num_blocks * kBlk;
    b.k_scales = k_scales;
    b.v_scales = v_scales;
    const bool il = p.interleaved != 0;
    cf_status st;
    switch (p.dtype) {
      case CF_F32: st = launch_block_type<float>(b, il, stream); break;
      case CF_F16: st = launch_block_type<__half>(b, il, stream); break;
      default: st = launch_block_type<__nv_bfloat16>(b, il, stream); break;
    }
    if (st != CF_OK) return st;
  }
  return CF_OK;
}

cf_status rope_read_errors(uint32_t* bits, bool clear) {
  uint32_t v = 0;
  cf_status s = cuda_status(cudaMemcpyFromSymbol(&v, g_rope_errors, sizeof(v)));
  if (s != CF_OK) return s;
  *bits |= v;
  if (clear) {
    const uint32_t zero = 0;
    s = cuda_status(cudaMemcpyToSymbol(g_rope_errors, &zero, sizeof(zero)));
  }
  return s;
}

}  // namespace cfb
