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
// (R floats) is shared by all its heads.
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

template <int V, bool IL>
__device__ __forceinline__ Unit unit_of(const RopeArgs& a, int u) {
  Unit x;
  x.rot = u < a.rot_units;
  x.has1 = u < a.units;
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

template <int V, bool IL>
__device__ __forceinline__ void rotate(float* f, const float* cs, const float* sn) {  // f[0..V) and f[V..2V)
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int ia = IL ? 2 * i : i, ib = IL ? 2 * i + 1 : V + i;
    const float x = f[ia], y = f[ib];
    f[ia] = fmaf(x, cs[i], -(y * sn[i]));
    f[ib] = fmaf(y, cs[i], x * sn[i]);
  }
}

// Sum over the 2^log2 lanes of a row (aligned groups of a warp).
__device__ __forceinline__ float row_sum(float v, int log2) {
  for (int m = (1 << log2) >> 1; m > 0; m >>= 1) v += shfl_xor(v, m);
  return v;
}

// The lane's K units of one row, normed (w not null) and rotated (rot), in
// f32.  Every lane of the warp calls it: the rows of a warp may differ in
// having a weight, and the sum runs across lanes.
template <typename T, int V, int K, bool IL>
__device__ __forceinline__ void norm_rotate(const RopeArgs& a, float (&f)[K][2 * V], const void* w, bool rot,
                                            const Unit (&un)[K], const float (&cs)[K][V], const float (&sn)[K][V]) {
  if (a.q_w != nullptr || a.k_w != nullptr) {
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 2 * V; ++i) ss = fmaf(f[k][i], f[k][i], ss);
    ss = row_sum(ss, a.lanes_log2);
    if (w != nullptr) {
      const float rs = rsqrtf(ss / (float)a.head_dim + a.eps);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float g[V];
        if (un[k].has1) {
          load_weight<T, V>(a, w, un[k].o1, g);
#pragma unroll
          for (int i = 0; i < V; ++i) f[k][i] = f[k][i] * rs * g[i];
        }
        if (un[k].has2) {
          load_weight<T, V>(a, w, un[k].o2, g);
#pragma unroll
          for (int i = 0; i < V; ++i) f[k][V + i] = f[k][V + i] * rs * g[i];
        }
      }
    }
  }
  if (rot) {
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (un[k].rot) rotate<V, IL>(f[k], cs[k], sn[k]);
  }
}

template <int V, int K>
__device__ __forceinline__ void load_angles(const RopeArgs& a, int pos, int lane, const Unit (&un)[K],
                                            float (&cs)[K][V], float (&sn)[K][V]) {
  const float* row = a.cos_sin + (size_t)pos * a.rotary;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (un[k].rot) {
      const int i = (lane + (k << a.lanes_log2)) * V;
      load_f32<V>(row + i, cs[k]);
      load_f32<V>(row + a.rotary / 2 + i, sn[k]);
    }
  }
}

// ---------------------------------------------------------------------------
// Row items.  A warp takes 32 / lanes rows of one token at a time, U times
// over: the token's angles are loaded once for all of them, and their 2U
// loads per lane are in flight together.  Rows: the query heads, then the K
// heads, then (cache destinations) the V heads; `nrows` of them.
// ---------------------------------------------------------------------------
template <typename T, int V, int K, int U, bool IL>
__device__ __forceinline__ void row_items(const RopeArgs& a, int64_t warp, int64_t num_warps, int nrows) {
  const int lane = threadIdx.x & 31;
  const int sub = lane & ((1 << a.lanes_log2) - 1);
  const int per_warp = 32 >> a.lanes_log2;
  const int grp = lane >> a.lanes_log2;
  const int per_token = (nrows + per_warp * U - 1) / (per_warp * U);
  const int64_t items = (int64_t)a.num_tokens * per_token;
  Unit un[K];
#pragma unroll
  for (int k = 0; k < K; ++k) un[k] = unit_of<V, IL>(a, sub + (k << a.lanes_log2));

  for (int64_t item = warp; item < items; item += num_warps) {
    const int64_t t = item / per_token;
    const int row0 = (int)(item - t * per_token) * per_warp * U + grp;
    int pos = 0;
    if (a.positions != nullptr) pos = a.positions[t];
    int64_t slot = -1;
    if (a.slots != nullptr) slot = a.slots[t];
    Raw<T, V> raw[U][K][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = row0 + u * per_warp;
      if (r >= nrows) continue;
      const T* src;
      if (r < a.num_heads)
        src = static_cast<const T*>(a.q) + t * a.q_ts + r * a.q_hs;
      else if (r < a.num_heads + a.num_kv_heads)
        src = static_cast<const T*>(a.k) + t * a.k_ts + (r - a.num_heads) * a.k_hs;
      else
        src = static_cast<const T*>(a.v) + t * a.v_ts + (r - a.num_heads - a.num_kv_heads) * a.v_hs;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (un[k].has1) raw[u][k][0] = *reinterpret_cast<const Raw<T, V>*>(src + un[k].o1);
        if (un[k].has2) raw[u][k][1] = *reinterpret_cast<const Raw<T, V>*>(src + un[k].o2);
      }
    }
    const bool first = row0 - grp == 0 && lane == 0;
    if (a.positions != nullptr) {
      if (pos >= a.max_positions && first) rope_error(CF_DEVERR_POSITION);
      if (pos < 0 || pos >= a.max_positions) continue;  // a padding token, or one without angles: left out whole
    }
    if (slot >= a.num_slots) {
      if (first) rope_error(CF_DEVERR_SLOT);
      slot = -1;
    }
    float cs[K][V], sn[K][V];
    if (a.positions != nullptr) load_angles<V, K>(a, pos, sub, un, cs, sn);
    const int64_t blk = slot >= 0 ? slot / a.block_size : 0;
    const int64_t off = slot - blk * a.block_size;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = row0 + u * per_warp;
      const bool valid = r < nrows;
      const int kind = r < a.num_heads ? 0 : (r < a.num_heads + a.num_kv_heads ? 1 : 2);
      const int head = kind == 0 ? r : (kind == 1 ? r - a.num_heads : r - a.num_heads - a.num_kv_heads);
      float f[K][2 * V];
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) f[k][i] = 0.f;
        if (valid && un[k].has1) unpack<T, V>(raw[u][k][0], f[k]);
        if (valid && un[k].has2) unpack<T, V>(raw[u][k][1], f[k] + V);
      }
      norm_rotate<T, V, K, IL>(a, f, kind == 0 ? a.q_w : (kind == 1 ? a.k_w : nullptr), kind < 2, un, cs, sn);
      if (!valid) continue;
      if (kind > 0 && a.dest != kDense) {
        if (slot < 0) continue;  // a padding row: nothing is appended
        const int64_t row = ((blk * a.num_kv_heads + head) * a.block_size + off) * a.head_dim;
        if (a.dest == kCacheFp8) {
          uint8_t* dst = static_cast<uint8_t*>(kind == 1 ? a.kc : a.vc) + row;
          const float sc = kind == 1 ? a.k_scale : a.v_scale;
#pragma unroll
          for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) f[k][i] = __fdiv_rn(f[k][i], sc);
            if (un[k].has1) store_e4m3<V>(dst + un[k].o1, f[k]);
            if (un[k].has2) store_e4m3<V>(dst + un[k].o2, f[k] + V);
          }
        } else {
          T* dst = static_cast<T*>(kind == 1 ? a.kc : a.vc) + row;
#pragma unroll
          for (int k = 0; k < K; ++k) {
            // V is moved as it is, bit for bit
            if (un[k].has1)
              *reinterpret_cast<Raw<T, V>*>(dst + un[k].o1) = kind == 2 ? raw[u][k][0] : pack<T, V>(f[k]);
            if (un[k].has2)
              *reinterpret_cast<Raw<T, V>*>(dst + un[k].o2) = kind == 2 ? raw[u][k][1] : pack<T, V>(f[k] + V);
          }
        }
      } else {
        T* dst = kind == 0 ? static_cast<T*>(a.q_out) + t * a.qo_ts + head * a.qo_hs
                           : static_cast<T*>(a.k_out) + t * a.ko_ts + head * a.ko_hs;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (un[k].has1) *reinterpret_cast<Raw<T, V>*>(dst + un[k].o1) = pack<T, V>(f[k]);
          if (un[k].has2) *reinterpret_cast<Raw<T, V>*>(dst + un[k].o2) = pack<T, V>(f[k] + V);
        }
      }
    }
  }
}

template <typename T, int V, int K, int U, bool IL>
__global__ void __launch_bounds__(kThreads) rope_rows_kernel(const RopeArgs a) {
  row_items<T, V, K, U, IL>(a, (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5), (int64_t)gridDim.x * kWarps,
                            a.num_heads + a.num_kv_heads * (a.dest == kDense ? 1 : 2));
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

struct BlockArgs {
  RopeArgs r;
  float* k_scales;  // [num_blocks, Hkv]
  float* v_scales;
  int32_t head_split;  // CTAs per window, each with every head_split-th head
  int32_t kv_ctas;     // windows * head_split; the CTAs past them take the Q rows
};

struct BlockSmem {
  int32_t key[kBlk];            // block id of each window token, -1: none
  int32_t lead[kBlk];           // the block this token is the first of in the window, else -1
  int32_t dead[kBlk];           // its first token lies before the window
  int32_t win[kBlk][kBlk];      // token that gives row `off` of block lead[l], -1: none
  uint32_t filter[32];
  int32_t row_tok[kBlk * kBlk]; // the rows to append: token, and l * 16 + off
  int32_t row_lo[kBlk * kBlk];
  int32_t count[kWarps];
  uint32_t top[3][2][kBlk];     // max |x| of each block's rows, as f32 bits (K, V)
  float old[3][2][kBlk];
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

__device__ __forceinline__ float div_scale(float x, float s) {
  // x * 2^-k is exact; a pool may also hold scales that are no powers of two
  const uint32_t b = __float_as_uint(s);
  if ((b & 0x7fffffu) == 0u && b >= (1u << 23) && b < (254u << 23)) return x * __uint_as_float((254u << 23) - b);
  return __fdiv_rn(x, s);
}

template <typename T, int V, int K, bool IL>
__global__ void __launch_bounds__(kThreads) rope_block_append_kernel(const BlockArgs b) {
  const RopeArgs& a = b.r;
  if ((int)blockIdx.x >= b.kv_ctas) {
    row_items<T, V, K, K == 1 ? 4 : 1, IL>(a, (int64_t)(blockIdx.x - b.kv_ctas) * kWarps + (threadIdx.x >> 5),
                                           (int64_t)(gridDim.x - b.kv_ctas) * kWarps, a.num_heads);
    return;
  }
  __shared__ BlockSmem sm;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int window = blockIdx.x / b.head_split;
  const int w0 = window * kBlk;
  const int T_ = a.num_tokens;

  // 1. the window's blocks
  (&sm.win[0][0])[tid] = -1;
  if (tid < 32) sm.filter[tid] = 0u;
  if (tid < 2 * kBlk) {
    sm.top[0][tid / kBlk][tid % kBlk] = 0u;
  }
  int key = -1;
  if (tid < kBlk) {
    if (w0 + tid < T_) {
      const int64_t slot = a.slots[w0 + tid];
      if (slot >= a.num_slots)
        rope_error(CF_DEVERR_SLOT);
      else if (slot >= 0)
        key = (int)(slot / kBlk);
    }
    sm.key[tid] = key;
    sm.dead[tid] = 0;
  }
  __syncthreads();
  bool leads = false;
  if (tid < kBlk) {
    leads = key >= 0;
    for (int j = 0; j < tid; ++j) leads = leads && sm.key[j] != key;
    sm.lead[tid] = leads ? key : -1;
    if (leads) atomicOr(&sm.filter[(key >> 5) & 31], 1u << (key & 31));
  }
  if (__syncthreads_or(leads ? 1 : 0) == 0) return;  // padding only

  // 2. their tokens, wherever they are in the call
  for (int i = tid; i < T_; i += kThreads) {
    const int slot = a.slots[i];
    if (slot < 0) continue;
    const int k = slot / kBlk;
    if (!((sm.filter[(k >> 5) & 31] >> (k & 31)) & 1u)) continue;
    for (int l = 0; l < kBlk; ++l) {
      if (sm.lead[l] != k) continue;
      if (i < w0)
        sm.dead[l] = 1;
      else
        atomicMax(&sm.win[l][slot % kBlk], i);
    }
  }
  __syncthreads();

  // 3. the rows to append, in (block, offset) order
  int n;
  {
    const int l = tid / kBlk, off = tid % kBlk;
    int tok = sm.dead[l] ? -1 : sm.win[l][off];
    if (tok >= 0 && a.positions != nullptr) {
      const int pos = a.positions[tok];
      if (pos < 0 || pos >= a.max_positions) {
        if (pos >= a.max_positions) rope_error(CF_DEVERR_POSITION);
        tok = -1;
      }
    }
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
  }
  __syncthreads();

  // 4. head by head: warps 0-3 take the K rows, warps 4-7 the V rows
  const int kv = warp >= kWarps / 2 ? 1 : 0;
  const int ht = tid & (kThreads / 2 - 1);
  const int sub = lane & ((1 << a.lanes_log2) - 1);
  const int row_in_pass = ht >> a.lanes_log2;
  const int per_pass = (kThreads / 2) >> a.lanes_log2;
  const int passes = (n + per_pass - 1) / per_pass;
  Unit un[K];
#pragma unroll
  for (int k = 0; k < K; ++k) un[k] = unit_of<V, IL>(a, sub + (k << a.lanes_log2));
  float* scales = kv ? b.v_scales : b.k_scales;
  uint8_t* cache = static_cast<uint8_t*>(kv ? a.vc : a.kc);
  const T* src = static_cast<const T*>(kv ? a.v : a.k);
  const int64_t ts = kv ? a.v_ts : a.k_ts, hs = kv ? a.v_hs : a.k_hs;

  float cs[K][V], sn[K][V], f[K][2 * V];
  auto load = [&](int e, int head) {  // row e of the list, normed and rotated
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 2 * V; ++i) f[k][i] = 0.f;
    if (e < n) {
      const T* p = src + (int64_t)sm.row_tok[e] * ts + (int64_t)head * hs;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (un[k].has1) unpack<T, V>(*reinterpret_cast<const Raw<T, V>*>(p + un[k].o1), f[k]);
        if (un[k].has2) unpack<T, V>(*reinterpret_cast<const Raw<T, V>*>(p + un[k].o2), f[k] + V);
      }
    }
    if (kv == 0) norm_rotate<T, V, K, IL>(a, f, a.k_w, e < n && a.positions != nullptr, un, cs, sn);
  };
  auto angles = [&](int e) {
    if (kv == 0 && e < n && a.positions != nullptr)
      load_angles<V, K>(a, a.positions[sm.row_tok[e]], sub, un, cs, sn);
  };
  angles(row_in_pass);
  int buf = 0;
  for (int head = blockIdx.x % b.head_split; head < a.num_kv_heads; head += b.head_split) {
    const int next = buf == 2 ? 0 : buf + 1;
    if (ht < kBlk) {
      const int blk = sm.dead[ht] ? -1 : sm.lead[ht];
      float s = blk >= 0 ? scales[(int64_t)blk * a.num_kv_heads + head] : 0.f;
      sm.old[buf][kv][ht] = s > 0.f && s < INFINITY ? s : 0.f;
      sm.top[next][kv][ht] = 0u;
    }
    for (int p = 0; p < passes; ++p) {
      const int e = p * per_pass + row_in_pass;
      if (passes > 1) angles(e);
      load(e, head);
      float top = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) {
          const float x = fabsf(f[k][i]);
          top = fmaxf(top, x <= 3.402823466e38f ? x : 0.f);
        }
      for (int m = (1 << a.lanes_log2) >> 1; m > 0; m >>= 1) top = fmaxf(top, shfl_xor(top, m));
      if (e < n && sub == 0) atomicMax(&sm.top[buf][kv][sm.row_lo[e] / kBlk], __float_as_uint(top));
    }
    __syncthreads();
    for (int p = 0; p < passes; ++p) {
      const int e = p * per_pass + row_in_pass;
      if (passes > 1) {
        angles(e);
        load(e, head);
      }
      if (e >= n) continue;
      const int l = sm.row_lo[e] / kBlk, off = sm.row_lo[e] % kBlk;
      const float need = block_scale(sm.top[buf][kv][l]);
      const float s = sm.win[l][0] >= 0 ? need : fmaxf(sm.old[buf][kv][l], need);
      uint8_t* dst = cache + (((int64_t)sm.lead[l] * a.num_kv_heads + head) * kBlk + off) * a.head_dim;
      if (s > 0.f) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) f[k][i] = div_scale(f[k][i], s);
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (un[k].has1) store_e4m3<V>(dst + un[k].o1, f[k]);
        if (un[k].has2) store_e4m3<V>(dst + un[k].o2, f[k] + V);
      }
    }
    // the blocks whose scale changed: the scale, and where it grew under
    // rows that stay, those rows
    bool grew = false;
    float s_new = 0.f, s_old = 0.f;
    if (lane < kBlk && !sm.dead[lane] && sm.lead[lane] >= 0) {
      bool any = false;
      for (int j = 0; j < kBlk; ++j) any = any || sm.win[lane][j] >= 0;
      const bool fresh = sm.win[lane][0] >= 0;
      const float need = block_scale(sm.top[buf][kv][lane]);
      s_old = sm.old[buf][kv][lane];
      s_new = fresh ? need : fmaxf(s_old, need);
      grew = any && !fresh && s_new > s_old;
      if (any && ht < 32) scales[(int64_t)sm.lead[lane] * a.num_kv_heads + head] = s_new;
    }
    uint32_t todo = __ballot_sync(0xffffffffu, grew);
    while (todo != 0u) {
      const int l = __ffs(todo) - 1;
      todo &= todo - 1u;
      const float ratio = __shfl_sync(0xffffffffu, s_old, l) / __shfl_sync(0xffffffffu, s_new, l);
      const int chunks = a.head_dim / 16;
      uint8_t* base = cache + ((int64_t)sm.lead[l] * a.num_kv_heads + head) * kBlk * a.head_dim;
      for (int c = ht; c < kBlk * chunks; c += kThreads / 2) {
        if (sm.win[l][c / chunks] >= 0) continue;
        uint4* p = reinterpret_cast<uint4*>(base) + c;
        float x[16];
        load_widen<__nv_fp8_e4m3, 16>(reinterpret_cast<const __nv_fp8_e4m3*>(p), x);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] *= ratio;
        store_e4m3<16>(reinterpret_cast<uint8_t*>(p), x);
      }
    }
    buf = next;
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

template <typename T, int V, int K, int U, bool IL>
cf_status launch_rows(const RopeArgs& a, int nrows, cudaStream_t stream) {
  const int64_t rows = (int64_t)(32 >> a.lanes_log2) * U;
  const int64_t items = (int64_t)a.num_tokens * ((nrows + rows - 1) / rows);
  const int64_t want = (items + kWarps - 1) / kWarps, cap = (int64_t)sm_count() * 32;
  rope_rows_kernel<T, V, K, U, IL><<<(unsigned)(want < cap ? want : cap), kThreads, 0, stream>>>(a);
  return check_launch();
}

template <typename T, int V, int K>
cf_status launch_rows_of(const RopeArgs& a, bool interleaved, cudaStream_t stream) {
  const int nrows = a.num_heads + a.num_kv_heads * (a.dest == kDense ? 1 : 2);
  constexpr int U = K == 1 ? 4 : 1;
  return interleaved ? launch_rows<T, V, K, U, true>(a, nrows, stream)
                     : launch_rows<T, V, K, U, false>(a, nrows, stream);
}

template <typename T>
cf_status launch_rows_type(RopeArgs& a, bool interleaved, cudaStream_t stream) {
  const int v = vector_elems(a, sizeof(T));
  row_layout(a, v);
  if (v == 16 / (int)sizeof(T)) return launch_rows_of<T, 16 / (int)sizeof(T), 1>(a, interleaved, stream);
  if constexpr (sizeof(T) == 2)
    if (v == 4) return launch_rows_of<T, 4, 1>(a, interleaved, stream);
  return launch_rows_of<T, 1, 4>(a, interleaved, stream);
}

template <typename T, int V, int K>
cf_status launch_block_of(BlockArgs b, bool interleaved, cudaStream_t stream) {
  const RopeArgs& a = b.r;
  const int windows = (a.num_tokens + kBlk - 1) / kBlk;
  // about four CTAs per SM: a CTA per (window, head) for decode steps, whole
  // windows once there are enough of them
  const int target = 4 * sm_count();
  int split = (target + windows - 1) / windows;
  b.head_split = split < 1 ? 1 : (split > a.num_kv_heads ? a.num_kv_heads : split);
  b.kv_ctas = windows * b.head_split;
  int64_t q_ctas = 0;
  if (a.num_heads > 0) {
    const int64_t rows = (int64_t)(32 >> a.lanes_log2) * (K == 1 ? 4 : 1);
    const int64_t items = (int64_t)a.num_tokens * ((a.num_heads + rows - 1) / rows);
    const int64_t cap = (int64_t)sm_count() * 32;
    q_ctas = (items + kWarps - 1) / kWarps;
    q_ctas = q_ctas < cap ? q_ctas : cap;
  }
  const unsigned grid = (unsigned)(b.kv_ctas + q_ctas);
  if (interleaved)
    rope_block_append_kernel<T, V, K, true><<<grid, kThreads, 0, stream>>>(b);
  else
    rope_block_append_kernel<T, V, K, false><<<grid, kThreads, 0, stream>>>(b);
  return check_launch();
}

template <typename T>
cf_status launch_block_type(BlockArgs& b, bool interleaved, cudaStream_t stream) {
  const int v = vector_elems(b.r, sizeof(T));
  row_layout(b.r, v);
  if (v == 16 / (int)sizeof(T)) return launch_block_of<T, 16 / (int)sizeof(T), 1>(b, interleaved, stream);
  if constexpr (sizeof(T) == 2)
    if (v == 4) return launch_block_of<T, 4, 1>(b, interleaved, stream);
  return launch_block_of<T, 1, 4>(b, interleaved, stream);
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
    a.positions = a.positions == nullptr ? nullptr : a.positions + t0;
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
