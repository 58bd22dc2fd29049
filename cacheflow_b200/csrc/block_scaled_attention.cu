// block_scaled_attention.cu -- paged decode attention over e4m3 caches with a
// scale for each block of 16 tokens and KV head:
//   out[s, h] = sum_t p_t (vs[b_t] v_t),  p = softmax_t(scale ks[b_t] q . k_t)
// over t < context_lens[s], b_t the block of token t.
//
// A weight p_t vs[b_t] is 2^(x_t) / L with x_t = log2(e) scale ks q.k_t +
// log2 vs[b_t] up to the reference point of the running maximum, so the online
// softmax runs on x: the products with the stored bytes are the ones that
// dominate the output whatever the scales are, and L counts
// 2^(x_t) / vs[b_t].  A block whose vs is 0 adds to L alone.
#include <cmath>
#include <mutex>
#include <type_traits>

#include "cf_device.cuh"
#include "cf_internal.h"

namespace cfb {

__device__ uint32_t g_block_attn_errors;

__device__ __forceinline__ void block_attn_error(uint32_t bits) { atomicOr(&g_block_attn_errors, bits); }

namespace {

constexpr int kBlk = 16;
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
  const void* q;
  const float* ks;
  const float* vs;
  void* out;
  const int32_t* tables;
  const int32_t* lens;
  float* part_max;  // [S, H, P] log2 units; null when unsplit
  float* part_sum;
  float* part_out;  // [S, H, P, D]
  float scale_log2;
  int32_t num_heads, num_kv_heads, group;
  int32_t max_blocks;
  int32_t head_chunks;  // CTAs per KV head
  int32_t part_tokens;  // a multiple of 128
  int32_t num_parts;
  int64_t num_blocks;
  uint64_t wait_limit_ns;      // of every pipeline wait
  int32_t unarm_first_stage;   // test hook (cf_testing_set_pipeline_faults)
};

__device__ __forceinline__ int context_of(const Args& a, int seq, bool report) {
  const int ctx = a.lens[seq];
  const int cap = a.max_blocks * kBlk;
  if (ctx < 0 || ctx > cap) {
    if (report) block_attn_error(CF_DEVERR_CONTEXT_LEN);
    return ctx < 0 ? 0 : cap;
  }
  return ctx;
}

// ---------------------------------------------------------------------------
// The streaming kernel: one CTA per (partition, KV head [x head chunk], row),
// tiles of 128 tokens (8 blocks) of one KV head.
//
// Both products run on the stored bytes, tcgen05 kind::f8f6f4 with f32
// accumulation in tensor memory, the tokens or head dimensions as the 128
// rows of the MMA and the few query heads as its columns:
//   S[128 tokens x N] = K . Q^T      A = K tile (K-major), B = Q
//   O[128 dims   x N] = V^T . P^T    A = V tile (MN-major), B = P
// so no cached byte passes through a register.  Q and P, which e4m3 alone
// would round to 4 bits, are three e4m3 terms each, in three of the N columns
// per head: x = t1 + t2 / 16 + t3 / 256, every term the rounding of 16 times
// what the ones before it leave (13 significant bits; bf16 queries are
// exact).  Q is brought under 448 by a power of two for each head, P lies in
// [0, 256].  The block scales join outside: ks on a token's logit, vs in its
// weight's exponent.
//
// Roles: warp 4 issues the TMA copies (2 KB boxes of 16 tokens x 128 bytes,
// 128-byte swizzle) into a ring of stages, one thread of warp 5 the MMAs, and
// warps 0-3 do the softmax: thread t has token t of each tile, reads its N
// logit terms from tensor memory, and writes its P bytes; as the owner of
// head dimension t it reads the tile's O from tensor memory and adds it to
// f32 registers, rescaled there when the maximum moved.  S, P and O are
// double-buffered: the MMAs of a tile run under the softmax of the next.
// ---------------------------------------------------------------------------
constexpr int kTile = 128;                 // tokens of a tile
constexpr int kTileBlocks = kTile / kBlk;  // 8
constexpr int kBox = kTile * 128;          // 128 rows x 128 bytes
constexpr int kThreads = 192;
constexpr int kProducerWarp = 4;
constexpr int kMmaWarp = 5;
constexpr float kPScale = 256.f;

// e4m3 terms of a query element and of a weight: two hold a bf16's 8
// significant bits, three an f16's 11.
template <typename T>
constexpr int kTerms = std::is_same<T, __half>::value ? 3 : 2;

template <typename T, int D, int HG>
struct Layout {
  static constexpr int kN = (kTerms<T> * HG + 15) / 16 * 16;  // MMA columns
  static constexpr int kBoxes = D / 128;
  static constexpr int kHalf = kBoxes * kBox;         // a tile's K or V
  // K and V have rings of their own: a K stage is free once its QK is done,
  // a V stage an exchange of maxima and a PV later.
  static constexpr bool kThree = D == 128 && kN == 16;  // three CTAs per SM
  static constexpr int kStages = kThree ? 2 : 3;
  static constexpr int kVOff = kStages * kHalf;
  static constexpr int kQOff = 2 * kStages * kHalf;   // Q: kBoxes x [kN rows x 128 B]
  static constexpr int kQBox = kN * 128;
  static constexpr int kPOff = kQOff + kBoxes * kQBox;  // P: 2 x [kN/16 planes x 128 tokens x 16 B]
  static constexpr int kPBytes = kN * 128;
  static constexpr int kBarOff = kPOff + 2 * kPBytes;
  // full, empty of K and of V; s_full, p_full, o_full, top by tile parity; fin
  static constexpr int kNumBars = 4 * kStages + 4 * 2 + 1;
  static constexpr int kMaxOff = kBarOff + (kNumBars * 8 + 15) / 16 * 16;  // [2][4][HG] f32
  static constexpr int kMaxHeads = (HG + 3) / 4 * 4;
  static constexpr int kSumOff = kMaxOff + 2 * 4 * kMaxHeads * 4;          // [4][HG] f32
  static constexpr int kQsOff = kSumOff + 4 * kMaxHeads * 4;               // [HG] f32
  static constexpr int kOkOff = kQsOff + kMaxHeads * 4;                     // [4] int
  static constexpr int kTmemOff = kOkOff + 16;
  static constexpr int kBytes = kTmemOff + 16;
  static constexpr int kAlloc = kBytes + 1024;
  static constexpr int kMinCtas = kThree ? 3 : (D == 128 ? 2 : 1);
  static constexpr int kOCol = 2 * kN;                 // O after the two S buffers
  static constexpr int kCols = 2 * kN + 2 * kBoxes * kN;
  static constexpr uint32_t kTmemCols = kCols <= 64 ? 64 : kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
  static_assert(kAlloc <= 227 * 1024, "shared memory of one CTA");
};

// Instruction descriptor of kind::f8f6f4: f32 accumulation, A and B e4m3,
// A and B K-major (0) or MN-major (1).
__host__ __device__ constexpr uint32_t idesc_f8(uint32_t mn_major, uint32_t n) {
  return (1u << 4) | (mn_major << 15) | (mn_major << 16) | ((n >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}

// Matrix descriptor without a swizzle (version 1, layout type 0).
__device__ __forceinline__ uint64_t smem_desc_plain(uint32_t saddr, uint32_t lbo_bytes, uint32_t sbo_bytes) {
  return (uint64_t)((saddr >> 4) & 0x3fffu) | ((uint64_t)((lbo_bytes >> 4) & 0x3fffu) << 16) |
         ((uint64_t)((sbo_bytes >> 4) & 0x3fffu) << 32) | (1ull << 46);
}

__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float* v) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
      "%13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// Max over the warp; a NaN takes no part.
__device__ __forceinline__ float warp_max(float x) {
  float m;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(x));
  return m;
}

__device__ __forceinline__ uint16_t h2_to_e4m3x2(__half2 h) {
  return (uint16_t)__nv_cvt_halfraw2_to_fp8x2(static_cast<__half2_raw>(h), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ __half2 e4m3x2_to_half2(uint16_t c) {
  return __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)c, __NV_E4M3));
}

// Two f16 values -> kT e4m3 terms each: x = t1 + t2/16 + t3/256, every term
// the rounding of 16 times what the ones before it leave (exact in f16).
template <int kT>
__device__ __forceinline__ void split_terms(__half2 x, uint16_t (&t)[kT]) {
  const __half2 sixteen = __float2half2_rn(16.f);
#pragma unroll
  for (int i = 0; i < kT; ++i) {
    t[i] = h2_to_e4m3x2(x);
    if (i + 1 < kT) x = __hmul2(__hsub2(x, e4m3x2_to_half2(t[i])), sixteen);
  }
}

// The sum of a head's terms: columns h, HG + h, ... of v.
template <int kT, int HG>
__device__ __forceinline__ float join_terms(const float* v, int h) {
  float r = v[(kT - 1) * HG + h];
#pragma unroll
  for (int i = kT - 2; i >= 0; --i) r = fmaf(r, 0.0625f, v[i * HG + h]);
  return r;
}

template <typename T, int D, int HG>
__global__ void __launch_bounds__(kThreads, Layout<T, D, HG>::kMinCtas)
    block_attention_kernel(const Args a, const __grid_constant__ CUtensorMap tmk,
                           const __grid_constant__ CUtensorMap tmv) {
  using L = Layout<T, D, HG>;
  constexpr int N = L::kN, S = L::kStages, kT = kTerms<T>;
  const int part = blockIdx.x, seq = blockIdx.z;
  const int kvh = blockIdx.y / a.head_chunks, chunk = blockIdx.y - kvh * a.head_chunks;
  const int head0 = kvh * a.group + chunk * HG;
  const int nheads = min(HG, a.group - chunk * HG);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ctx = context_of(a, seq, threadIdx.x == 0 && part == 0 && blockIdx.y == 0);
  const int nparts = ctx == 0 ? 1 : (ctx + a.part_tokens - 1) / a.part_tokens;
  if (part >= nparts) return;
  if (part == 0 && nparts > (int)gridDim.x && threadIdx.x == 0 && blockIdx.y == 0)
    block_attn_error(CF_DEVERR_CONTEXT_LEN);  // context_lens exceeds max_context_len
  const bool single = nparts == 1;
  const int t0 = part * a.part_tokens;
  const int ntok = min(a.part_tokens, ctx - t0);  // of this partition; 0 for an empty row
  const int ntiles = (ntok + kTile - 1) / kTile;
  const int nblk = (ntok + kBlk - 1) / kBlk;
  const int32_t* table = a.tables + (size_t)seq * a.max_blocks + t0 / kBlk;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* k_full = bars;
  uint64_t* k_empty = bars + S;
  uint64_t* v_full = bars + 2 * S;
  uint64_t* v_empty = bars + 3 * S;
  uint64_t* s_full = bars + 4 * S;  // [2], by tile parity, as the ones below
  uint64_t* p_full = s_full + 2;
  uint64_t* o_full = p_full + 2;
  uint64_t* top = o_full + 2;
  uint64_t* fin = top + 2;
  float* smax = reinterpret_cast<float*>(smem + L::kMaxOff);
  float* ssum = reinterpret_cast<float*>(smem + L::kSumOff);
  float* sqs = reinterpret_cast<float*>(smem + L::kQsOff);
  int* sok = reinterpret_cast<int*>(smem + L::kOkOff);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kTmemOff);

  int ids = 0, ids_next = 0;  // producer: block ids of this and the next 32 blocks
  auto load_ids = [&](int b) { return b + lane < nblk ? table[b + lane] : 0; };
  int id = 0;
  bool valid_id = false;
  auto produce_k = [&](int j) {  // takes the tile's ids, then copies K
    const int b0 = j * kTileBlocks;
    if ((b0 & 31) == 0) {
      ids = b0 == 0 ? load_ids(0) : ids_next;
      ids_next = load_ids(b0 + 32);
    }
    id = __shfl_sync(0xffffffffu, ids, (b0 & 31) + (lane & 7));
    const bool want = lane < kTileBlocks && b0 + lane < nblk;
    valid_id = want && id >= 0 && (int64_t)id < a.num_blocks;
    if (want && !valid_id) block_attn_error(CF_DEVERR_BLOCK_ID);
  };
  // Copies the tile's K or V: lane k block k, onto the stage's barrier.
  auto copy = [&](int j, const CUtensorMap* map, uint64_t* full, uint8_t* ring) {
    if (a.unarm_first_stage && j == 0) return;  // test hook: the stage never completes
    const uint32_t bar = smem_addr(&full[j % S]);
    const uint32_t mask = __ballot_sync(0xffffffffu, valid_id);
    if (lane == 0) {
      fence_proxy_async_smem();
      if (mask == 0)
        mbar_arrive(bar);
      else
        mbar_arrive_expect_tx(bar, (uint32_t)__popc(mask) * kBlk * D);
    }
    __syncwarp();
    if (valid_id) {
      const int32_t row = (int32_t)(((int64_t)id * a.num_kv_heads + kvh) * kBlk);
      uint8_t* dst = ring + (j % S) * L::kHalf + lane * (kBlk * 128);
#pragma unroll
      for (int b = 0; b < L::kBoxes; ++b) tma_load_2d(smem_addr(dst + b * kBox), map, b * 128, row, bar);
    }
    __syncwarp();
  };
  auto produce = [&](int j) {
    produce_k(j);
    copy(j, &tmk, k_full, smem);
    copy(j, &tmv, v_full, smem + L::kVOff);
  };

  // Set-up: the producer starts copying as soon as the barriers are there;
  // Q's terms and the tensor memory follow beside it.
  int produced = 0;
  if (warp == kProducerWarp) {
    if (lane == 0) {
      for (int s = 0; s < S; ++s) {
        mbar_init(smem_addr(&k_full[s]), 1);
        mbar_init(smem_addr(&k_empty[s]), 1);
        mbar_init(smem_addr(&v_full[s]), 1);
        mbar_init(smem_addr(&v_empty[s]), 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(smem_addr(&s_full[i]), 1);
        mbar_init(smem_addr(&p_full[i]), kTile);
        mbar_init(smem_addr(&o_full[i]), 1);
        mbar_init(smem_addr(&top[i]), 4);
      }
      mbar_init(smem_addr(fin), 1);
      fence_mbar_init();
    }
    __syncwarp();
    for (; produced < ntiles && produced < S; ++produced) produce(produced);
  } else if (warp == kMmaWarp) {
    tmem_alloc(smem_addr(tmem_slot), L::kTmemCols);
    tmem_relinquish();
  } else {
    constexpr int E = D / 32;
    for (int n = warp; n < N; n += 4) {  // rows past the terms
      if (n >= kT * HG)
        for (int b = 0; b < L::kBoxes; ++b)
          reinterpret_cast<uint32_t*>(smem + L::kQOff + b * L::kQBox + n * 128)[lane] = 0u;
    }
    for (int h = warp; h < HG; h += 4) {
      float q[E];
#pragma unroll
      for (int e = 0; e < E; ++e) q[e] = 0.f;
      if (h < nheads)
        load_widen<T, E>(static_cast<const T*>(a.q) + ((size_t)seq * a.num_heads + head0 + h) * D + lane * E, q);
      float mx = 0.f;
      bool bad = false;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const bool fin = fabsf(q[e]) <= 3.402823466e38f;
        bad = bad || !fin;
        mx = fmaxf(mx, fin ? fabsf(q[e]) : 0.f);
      }
      mx = warp_max(mx);
      bad = __any_sync(0xffffffffu, bad);
      // the smallest power of two s with mx <= 448 s (448 = 1.75 * 2^8)
      const uint32_t bits = __float_as_uint(mx);
      int ex = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
      ex = mx == 0.f ? 127 : (ex < 1 ? 1 : ex);
      const float inv = __uint_as_float((uint32_t)(254 - ex) << 23);
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        uint16_t lo[kT], hi[kT];
        split_terms<kT>(__floats2half2_rn(q[e] * inv, q[e + 1] * inv), lo);
        split_terms<kT>(__floats2half2_rn(q[e + 2] * inv, q[e + 3] * inv), hi);
        const int col = lane * E + e;  // byte of the row
#pragma unroll
        for (int t = 0; t < kT; ++t) {
          const int n = t * HG + h;
          uint32_t w = (uint32_t)lo[t] | ((uint32_t)hi[t] << 16);
          if (bad) w = 0x7f7f7f7fu;  // a query that is not finite has no softmax: NaN
          *reinterpret_cast<uint32_t*>(smem + L::kQOff + (col >> 7) * L::kQBox + n * 128 +
                                       ((((col >> 4) & 7) ^ (n & 7)) << 4) + (col & 15)) = w;
        }
      }
      if (lane == 0) sqs[h] = __uint_as_float((uint32_t)ex << 23);
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == kProducerWarp) {
    bool ok = true;
    for (; produced < ntiles; ++produced) {
      const int s = produced % S;
      const uint32_t parity = (uint32_t)(produced / S - 1) & 1u;
      produce_k(produced);
      ok = mbar_wait_bounded(smem_addr(&k_empty[s]), parity, a.wait_limit_ns);
      if (!__all_sync(0xffffffffu, ok)) break;
      copy(produced, &tmk, k_full, smem);
      ok = mbar_wait_bounded(smem_addr(&v_empty[s]), parity, a.wait_limit_ns);
      if (!__all_sync(0xffffffffu, ok)) {
        if (lane == 0) mbar_wait_bounded(smem_addr(&k_full[s]), (uint32_t)(produced / S) & 1u, a.wait_limit_ns);
        break;
      }
      copy(produced, &tmv, v_full, smem + L::kVOff);
    }
    if (!ok) block_attn_error(CF_DEVERR_TIMEOUT);
    // no copy may land after the CTA has left
    if (lane == 0)
      for (int j = produced > S ? produced - S : 0; j < produced; ++j) {
        mbar_wait_bounded(smem_addr(&k_full[j % S]), (uint32_t)(j / S) & 1u, a.wait_limit_ns);
        mbar_wait_bounded(smem_addr(&v_full[j % S]), (uint32_t)(j / S) & 1u, a.wait_limit_ns);
      }
  } else if (warp == kMmaWarp) {
    if (lane == 0) {
      const uint64_t k_desc = smem_desc_sw128(smem_addr(smem), 16, 1024);
      const uint64_t v_desc = smem_desc_sw128(smem_addr(smem + L::kVOff), 16, 1024);
      const uint64_t q_desc = smem_desc_sw128(smem_addr(smem + L::kQOff), 16, 1024);
      // P: 8 tokens x 16 columns per 128 bytes, tokens onward, then planes
      const uint64_t p_desc = smem_desc_plain(smem_addr(smem + L::kPOff), 128, kTile * 16);
      bool ok = true;
      auto issue_qk = [&](int j) {
        const int s = j % S;
        ok = ok && mbar_wait_bounded(smem_addr(&k_full[s]), (uint32_t)(j / S) & 1u, a.wait_limit_ns);
        if (!ok) return;
        tc_fence_after();
        const uint64_t kd = k_desc + (uint64_t)((s * L::kHalf) >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk) {
          const uint64_t ad = kd + (uint64_t)(((kk >> 2) * kBox + (kk & 3) * 32) >> 4);
          const uint64_t bd = q_desc + (uint64_t)(((kk >> 2) * L::kQBox + (kk & 3) * 32) >> 4);
          mma_f8(tmem + (j & 1) * N, ad, bd, idesc_f8(0, N), kk > 0 ? 1u : 0u);
        }
        tc_commit(smem_addr(&s_full[j & 1]));
        tc_commit(smem_addr(&k_empty[s]));
      };
      auto issue_pv = [&](int j) {
        const int s = j % S;
        ok = mbar_wait_bounded(smem_addr(&v_full[s]), (uint32_t)(j / S) & 1u, a.wait_limit_ns);
        if (!ok) return;
        tc_fence_after();
        const uint64_t vd = v_desc + (uint64_t)((s * L::kHalf) >> 4);
        const uint64_t pd = p_desc + (uint64_t)(((j & 1) * L::kPBytes) >> 4);
#pragma unroll
        for (int b = 0; b < L::kBoxes; ++b)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)  // 32 tokens each
            mma_f8(tmem + L::kOCol + ((j & 1) * L::kBoxes + b) * N, vd + (uint64_t)((b * kBox + kk * 4096) >> 4),
                   pd + (uint64_t)((kk * 512) >> 4), idesc_f8(1, N), kk > 0 ? 1u : 0u);
        tc_commit(smem_addr(&o_full[j & 1]));
        tc_commit(smem_addr(&v_empty[s]));
      };
      for (int j = 0; j < 2 && j < ntiles; ++j) issue_qk(j);
      for (int j = 0; j < ntiles && ok; ++j) {
        ok = mbar_wait_bounded(smem_addr(&p_full[j & 1]), (uint32_t)(j >> 1) & 1u, a.wait_limit_ns);
        if (!ok) break;
        tc_fence_after();
        issue_pv(j);
        if (ok && j + 2 < ntiles) issue_qk(j + 2);
      }
      if (!ok) {
        // every MMA issued so far has finished before tensor memory is freed
        block_attn_error(CF_DEVERR_TIMEOUT);
        tc_commit(smem_addr(fin));
        mbar_wait_bounded(smem_addr(fin), 0u, a.wait_limit_ns);
      }
    }
    __syncwarp();
  } else {
    const int tok = threadIdx.x;  // token of the tile; head dimension of O
    const uint32_t trow = tmem + ((uint32_t)(32 * warp) << 16);
    float qsc[HG], m[HG], l[HG], alpha[HG], acc[L::kBoxes][HG];
#pragma unroll
    for (int h = 0; h < HG; ++h) {
      qsc[h] = sqs[h] * a.scale_log2;
      m[h] = -INFINITY;
      l[h] = 0.f;
      alpha[h] = 0.f;
#pragma unroll
      for (int b = 0; b < L::kBoxes; ++b) acc[b][h] = 0.f;
    }
    // The scales of this thread's token, one tile ahead (the id two ahead).
    auto id_of = [&](int j) {
      const int b = j * kTileBlocks + (tok >> 4);
      return b < nblk ? table[b] : -1;
    };
    auto scales_of = [&](int id, float& ks, float& vs) {
      ks = vs = 0.f;
      if (id < 0 || (int64_t)id >= a.num_blocks) return;
      const int64_t u = (int64_t)id * a.num_kv_heads + kvh;
      ks = a.ks[u];
      vs = a.vs[u];
    };
    int id_cur = id_of(0), id_nxt = id_of(1);
    float ks, vs;
    scales_of(id_cur, ks, vs);
    bool ok = true;
    auto add_o = [&](int j) {  // the accumulator takes tile j's O
      ok = mbar_wait_bounded(smem_addr(&o_full[j & 1]), (uint32_t)(j >> 1) & 1u, a.wait_limit_ns);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        return;
      }
      tc_fence_after();
#pragma unroll
      for (int b = 0; b < L::kBoxes; ++b) {
        float o[N];
#pragma unroll
        for (int c = 0; c < N; c += 16) tmem_ld16(trow + L::kOCol + ((j & 1) * L::kBoxes + b) * N + c, &o[c]);
        tmem_wait_ld();
#pragma unroll
        for (int h = 0; h < HG; ++h)
          acc[b][h] = fmaf(acc[b][h], alpha[h], join_terms<kT, HG>(o, h));
      }
    };
    for (int j = 0; j < ntiles; ++j) {
      const bool valid = j * kTile + tok < ntok && id_cur >= 0 && (int64_t)id_cur < a.num_blocks;
      const int id_nn = id_of(j + 2);
      float ks_nxt, vs_nxt;
      scales_of(id_nxt, ks_nxt, vs_nxt);
      const bool vzero = vs == 0.f;
      const float lv = vzero ? 0.f : __log2f(vs);
      const float vinv = vzero ? 1.f : __fdividef(1.f, vs);

      ok = mbar_wait_bounded(smem_addr(&s_full[j & 1]), (uint32_t)(j >> 1) & 1u, a.wait_limit_ns);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tc_fence_after();
      float x[N];
#pragma unroll
      for (int c = 0; c < N; c += 16) tmem_ld16(trow + (j & 1) * N + c, &x[c]);
      tmem_wait_ld();
      float* tops = smax + (j & 1) * 4 * L::kMaxHeads;
#pragma unroll
      for (int h = 0; h < HG; ++h) {
        const float s = join_terms<kT, HG>(x, h);
        x[h] = valid ? fmaf(s, qsc[h] * ks, lv) : -INFINITY;
        const float w = warp_max(x[h]);
        if (lane == 0) tops[warp * L::kMaxHeads + h] = w;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&top[j & 1]));
      ok = mbar_wait_bounded(smem_addr(&top[j & 1]), (uint32_t)(j >> 1) & 1u, a.wait_limit_ns);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      float alpha_new[HG];
#pragma unroll
      for (int h = 0; h < HG; ++h) {
        const float mx = fmaxf(fmaxf(tops[h], tops[L::kMaxHeads + h]),
                               fmaxf(tops[2 * L::kMaxHeads + h], tops[3 * L::kMaxHeads + h]));
        const float mn = fmaxf(m[h], mx);
        const float mu = mn == -INFINITY ? 0.f : mn;
        alpha_new[h] = ex2_approx(m[h] - mu);
        m[h] = mn;
        x[h] = ex2_approx(x[h] - mu);
        l[h] = fmaf(l[h], alpha_new[h], x[h] * vinv);
      }
      // P's bytes: column t HG + h is term t of head h
      uint16_t pairs[N / 2];
#pragma unroll
      for (int i = 0; i < N / 2; ++i) pairs[i] = 0;
      const float ps = vzero ? 0.f : kPScale;
#pragma unroll
      for (int h = 0; h < HG; h += 2) {
        uint16_t t[kT];
        split_terms<kT>(__floats2half2_rn(x[h] * ps, h + 1 < HG ? x[h + 1 < HG ? h + 1 : h] * ps : 0.f), t);
#pragma unroll
        for (int k = 0; k < kT; ++k) {
          const int c = k * HG + h;
          if (HG % 2 == 0)
            pairs[c / 2] = t[k];
          else  // one head: terms in neighbouring columns
            pairs[c / 2] |= (uint16_t)((t[k] & 0xffu) << (8 * (c & 1)));
        }
      }
      uint4* pb = reinterpret_cast<uint4*>(smem + L::kPOff + (j & 1) * L::kPBytes) + tok;
#pragma unroll
      for (int c = 0; c < N / 16; ++c) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = (uint32_t)pairs[c * 8 + 2 * i] | ((uint32_t)pairs[c * 8 + 2 * i + 1] << 16);
        pb[c * kTile] = make_uint4(w[0], w[1], w[2], w[3]);
      }
      if (!valid) {
        // A V row that no token of the row owns (past the context, or a
        // rejected block's) may hold any bytes, and 0 * NaN is not 0.
        mbar_wait_bounded(smem_addr(&v_full[j % S]), (uint32_t)(j / S) & 1u, a.wait_limit_ns);
        uint8_t* v = smem + L::kVOff + (j % S) * L::kHalf + tok * 128;
#pragma unroll
        for (int b = 0; b < L::kBoxes; ++b)
#pragma unroll
          for (int c = 0; c < 8; ++c) reinterpret_cast<uint4*>(v + b * kBox)[c] = make_uint4(0, 0, 0, 0);
      }
      fence_proxy_async_smem();
      tc_fence_before();
      mbar_arrive(smem_addr(&p_full[j & 1]));
      if (j > 0) {
        add_o(j - 1);
        if (!ok) break;
      }
#pragma unroll
      for (int h = 0; h < HG; ++h) alpha[h] = alpha_new[h];
      id_cur = id_nxt;
      id_nxt = id_nn;
      ks = ks_nxt;
      vs = vs_nxt;
    }
    if (ok && ntiles > 0) add_o(ntiles - 1);
    if (!ok && lane == 0) block_attn_error(CF_DEVERR_TIMEOUT);

    // The row's sums over its 128 token threads, then this thread's dimension.
#pragma unroll
    for (int h = 0; h < HG; ++h) {
      float w = l[h];
      for (int i = 16; i > 0; i >>= 1) w += shfl_xor(w, i);
      if (lane == 0) ssum[warp * L::kMaxHeads + h] = w;
    }
    if (lane == 0) sok[warp] = ok ? 1 : 0;
    asm volatile("bar.sync 1, 128;" ::: "memory");  // every softmax warp comes here, with or without a timeout
    if (sok[0] & sok[1] & sok[2] & sok[3]) {  // after a timeout nothing is written
#pragma unroll
      for (int h = 0; h < HG; ++h) {
        if (h >= nheads) continue;
        const float sum = (ssum[h] + ssum[L::kMaxHeads + h]) + (ssum[2 * L::kMaxHeads + h] + ssum[3 * L::kMaxHeads + h]);
        const size_t hq = (size_t)seq * a.num_heads + head0 + h;
        const float inv = sum == 0.f ? 0.f : 1.f / (sum * kPScale);
#pragma unroll
        for (int b = 0; b < L::kBoxes; ++b) {
          const float r = acc[b][h] * inv;
          if (single)
            static_cast<T*>(a.out)[hq * D + b * 128 + tok] = from_float<T>(r);
          else
            a.part_out[(hq * a.num_parts + part) * D + b * 128 + tok] = r;
        }
        if (!single && tok == 0) {
          a.part_max[hq * a.num_parts + part] = m[h];
          a.part_sum[hq * a.num_parts + part] = sum;
        }
      }
    }
  }
  grid_dependency_launch();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) tmem_dealloc(tmem, L::kTmemCols);
}

// Merges a row's partitions, one warp per (query head, row):
// out = sum_p w_p o_p / sum_p w_p, w_p = sum_p 2^(max_p - max).
template <typename T, int D>
__global__ void __launch_bounds__(128) block_attention_merge_kernel(const Args a) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int head = blockIdx.x * 4 + (threadIdx.x >> 5), seq = blockIdx.y;
  if (head >= a.num_heads) return;
  grid_dependency_wait();
  const int ctx = context_of(a, seq, false);
  const int parts = min(a.num_parts, (ctx + a.part_tokens - 1) / a.part_tokens);
  if (parts <= 1) return;  // written by the partition kernel
  const size_t base = ((size_t)seq * a.num_heads + head) * a.num_parts;
  float m = -INFINITY;
  for (int p = lane; p < parts; p += 32) m = fmaxf(m, a.part_max[base + p]);
  for (int i = 16; i > 0; i >>= 1) m = fmaxf(m, shfl_xor(m, i));
  float l = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  if (m != -INFINITY) {
#pragma unroll 4
    for (int p = 0; p < parts; ++p) {
      const float w = a.part_sum[base + p] * exp2f(a.part_max[base + p] - m);
      l += w;
      float x[E];
      load_widen<float, E>(a.part_out + (base + p) * D + lane * E, x);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(w, x[e], o[e]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* out = static_cast<T*>(a.out) + ((size_t)seq * a.num_heads + head) * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) out[e] = from_float<T>(o[e] * inv);
}

// Per kernel instantiation and device: opt in to > 48 KB of dynamic smem.
template <typename T, int D, int HG>
cf_status ensure_smem() {
  static std::once_flag flags[64];
  static cudaError_t errs[64];
  auto kern = block_attention_kernel<T, D, HG>;
  constexpr int bytes = Layout<T, D, HG>::kAlloc;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e);
  if (dev < 0 || dev >= 64)
    return cuda_status(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  std::call_once(flags[dev], [&] {
    errs[dev] = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  });
  return cuda_status(errs[dev]);
}

template <typename T, int D, int HG>
cf_status launch_heads(Args a, const cf_paged_attention_params& p, cudaStream_t stream) {
  a.head_chunks = (a.group + HG - 1) / HG;
  if ((int64_t)p.num_kv_heads * a.head_chunks > 65535) return CF_ERR_UNSUPPORTED;
  CUtensorMap mk, mv;
  const int64_t rows = p.num_blocks * (int64_t)p.num_kv_heads * kBlk;
  if (!kv_tensor_map(&mk, p.key_cache, rows, D, CF_FP8_E4M3) ||
      !kv_tensor_map(&mv, p.value_cache, rows, D, CF_FP8_E4M3))
    return CF_ERR_CUDA;
  cf_status st = ensure_smem<T, D, HG>();
  if (st != CF_OK) return st;
  const dim3 grid((unsigned)a.num_parts, (unsigned)(p.num_kv_heads * a.head_chunks), (unsigned)p.num_seqs);
  block_attention_kernel<T, D, HG><<<grid, kThreads, Layout<T, D, HG>::kAlloc, stream>>>(a, mk, mv);
  return check_launch();
}

template <typename T, int D>
cf_status launch_dim(const Args& a, const cf_paged_attention_params& p, cudaStream_t stream) {
  cf_status st;
  if (a.group == 1)
    st = launch_heads<T, D, 1>(a, p, stream);
  else if (a.group <= 4)
    st = launch_heads<T, D, 4>(a, p, stream);
  else if (a.group <= 8)
    st = launch_heads<T, D, 8>(a, p, stream);
  else
    st = launch_heads<T, D, 16>(a, p, stream);
  if (st != CF_OK || a.part_max == nullptr) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3((unsigned)((a.num_heads + 3) / 4), (unsigned)p.num_seqs);
  cfg.blockDim = dim3(128);
  return cuda_status(cudaLaunchKernelEx(&cfg, block_attention_merge_kernel<T, D>, a));
}

}  // namespace

cf_status launch_block_scaled_attention(const BlockScaledLaunch& l) {
  const cf_paged_attention_params& p = *l.p;
  Args a = {};
  a.q = p.query;
  a.ks = l.k_scales;
  a.vs = l.v_scales;
  a.out = p.output;
  a.tables = p.block_tables;
  a.lens = p.context_lens;
  a.scale_log2 = p.scale * kLog2e;
  a.num_heads = p.num_heads;
  a.num_kv_heads = p.num_kv_heads;
  a.group = p.num_heads / p.num_kv_heads;
  a.max_blocks = p.max_blocks_per_seq;
  a.num_parts = l.num_parts;
  // unsplit: one partition, whole tiles
  a.part_tokens = l.num_parts > 1 ? l.part_tokens : (p.max_blocks_per_seq * kBlk + kTile - 1) / kTile * kTile;
  a.num_blocks = p.num_blocks;
  const int64_t lim = g_test_wait_limit_ns.load(std::memory_order_relaxed);
  a.wait_limit_ns = lim > 0 ? (uint64_t)lim : kWaitLimitNs;
  a.unarm_first_stage = g_test_unarm_first_stage.load(std::memory_order_relaxed);
  if (l.num_parts > 1) {
    a.part_max = l.part_max;
    a.part_sum = l.part_sum;
    a.part_out = l.part_out;
  }
  if (p.dtype == CF_F16)
    return p.head_dim == 128 ? launch_dim<__half, 128>(a, p, l.stream) : launch_dim<__half, 256>(a, p, l.stream);
  return p.head_dim == 128 ? launch_dim<__nv_bfloat16, 128>(a, p, l.stream)
                           : launch_dim<__nv_bfloat16, 256>(a, p, l.stream);
}

cf_status block_scaled_read_errors(uint32_t* bits, bool clear) {
  uint32_t v = 0;
  cf_status s = cuda_status(cudaMemcpyFromSymbol(&v, g_block_attn_errors, sizeof(v)));
  if (s != CF_OK) return s;
  *bits |= v;
  if (clear) {
    const uint32_t zero = 0;
    s = cuda_status(cudaMemcpyToSymbol(g_block_attn_errors, &zero, sizeof(zero)));
  }
  return s;
}

}  // namespace cfb
