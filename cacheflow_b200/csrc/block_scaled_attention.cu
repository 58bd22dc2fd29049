// block_scaled_attention.cu -- paged decode attention over e4m3 caches with a
// scale for each block of 16 tokens and KV head:
//   out[s, h] = sum_t p_t (vs[b_t] v_t),  p = softmax_t(scale ks[b_t] q . k_t)
// over t < context_lens[s], b_t the block of token t.
//
// A weight p_t vs[b_t] is 2^(x_t) / L with x_t = log2(e) scale ks q.k_t +
// log2 vs[b_t] up to a reference point, so the online softmax runs on x: the
// products with the stored bytes are the ones that dominate the output
// whatever the scales are, and L counts 2^(x_t) / vs[b_t].  A tile's weights
// are taken from the tile's own maximum and its sums join the row's in f32, so
// what a weight loses to its 8-bit terms goes by its tile, not by its row.
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

// One launch's work is the tiles (128 tokens) of every (row, KV head [, head
// chunk]) item, rows outermost, laid end to end and cut into equal shares, one
// for each CTA, whatever items they belong to.  Beginning and ending an item
// costs a CTA about 0.7 tiles' time (1.4 us), so an item counts 3 quarters of
// a tile beside its tiles where CTAs have many (without it the CTAs of 256
// rows of 512-8192 tokens that got the short rows ended at 278 us, half of
// them before 228).
struct Args {
  const void* q;
  const float* ks;
  const float* vs;
  void* out;
  const int32_t* tables;
  const int32_t* lens;
  // Results of items that several CTAs share: CTA c's first piece in slot 2c,
  // an item begun but not finished in 2c + 1.  Null: no item is shared, CTA c
  // takes the items that begin in its tiles.
  int4* meta;        // [G]: row, KV head and chunk, last CTA of the item begun (row -1: none)
  float* part_max;   // [2 G, HG] log2 units
  float* part_sum;   // kNoPiece: the CTA could not finish the piece
  float* part_out;   // [2 G, HG, D]
  float scale_log2;
  int32_t num_seqs, num_heads, num_kv_heads, group;
  int32_t max_blocks;
  int32_t head_chunks;  // items per (row, KV head)
  int64_t num_blocks;
  uint64_t wait_limit_ns;     // of every pipeline wait
  int32_t unarm_cta;          // test hook (cf_testing_set_pipeline_faults): a CTA, kEveryCta or kNoCta
};

constexpr int kNoCta = -2, kEveryCta = -1;
constexpr int kTile = 128;                 // tokens of a tile
constexpr int kTileWeight = 4;             // of a tile in the shares
constexpr int kItemWeight = 3;             // of an item's beginning and end
constexpr int kManyTiles = 8;              // per CTA, from which on that counts
constexpr int kTileBlocks = kTile / kBlk;  // 8
constexpr int kBox = kTile * 128;          // 128 rows x 128 bytes

__device__ __forceinline__ int context_of(const Args& a, int seq, bool report) {
  const int ctx = a.lens[seq];
  const int cap = a.max_blocks * kBlk;
  if (ctx < 0 || ctx > cap) {
    if (report) block_attn_error(CF_DEVERR_CONTEXT_LEN);
    return ctx < 0 ? 0 : cap;
  }
  return ctx;
}

// A CTA's way through its tiles, one segment (a run of tiles of one item) at
// a time.  Every role walks its own copy.
struct Cursor {
  int seq, item;  // row; KV head * chunks + chunk
  int ctx, tiles; // of the row
  int tile;       // first tile of the segment
  int left;       // tiles of the CTA from here on
  __device__ __forceinline__ int count() const { return min(left, tiles - tile); }
  __device__ __forceinline__ bool done() const { return left <= 0; }
  __device__ __forceinline__ void next(const Args& a) {
    left -= count();
    tile = 0;
    if (left <= 0) return;
    if (++item == a.num_kv_heads * a.head_chunks) {
      item = 0;
      do {
        ++seq;
        ctx = context_of(a, seq, false);
      } while (ctx == 0);  // left > 0: a row with tiles follows
      tiles = (ctx + kTile - 1) / kTile;
    }
  }
};

// ---------------------------------------------------------------------------
// The streaming kernel, three CTAs per SM (one at head_dim 256) for the whole
// launch.
//
// Both products run on the stored bytes, tcgen05 kind::f8f6f4 with f32
// accumulation in tensor memory, the tokens or head dimensions as the 128
// rows of the MMA and the few query heads as its columns:
//   S[128 tokens x N] = K . Q^T      A = K tile (K-major), B = Q
//   O[128 dims   x N] = V^T . P^T    A = V tile (MN-major), B = P
// so no cached byte passes through a register.  Q and P, which e4m3 alone
// would round to 4 bits, are two or three e4m3 terms each, in as many of the
// N columns per head: x = t1 + t2 / 16 + t3 / 256, every term the rounding of
// 16 times what the ones before it leave.  Q is brought under 448 by a power
// of two for each head, P is 256 at the tile's maximum.  The block scales join
// outside: ks on a token's logit, vs in its weight's exponent.
//
// Rounding: Q's terms hold every bit of a bf16 (an f16 to 2^-12).  P's are
// off by 2^-8 p at most (f16 2^-11) from 2^-14 of the tile's largest on, and
// below by 2^-22 (2^-26) of that one: as much as a P rounded to the rows' type
// but for tokens that next to nothing is left for in their tile.  The sum L
// has the weights before they are rounded.  With the row's running maximum as
// the reference the rest of a row with one dominant token fell under that
// floor as a whole (131072 tokens with at most 1 % of the weight beside one
// whose values are zeros: by its roundings 84 % of the output lost).
//
// Roles: warps 4 and 5 issue the TMA copies of K and of V (2 KB boxes of 16
// tokens x 128 bytes, 128-byte swizzle) into rings of stages, warp 7 stages
// the Q terms of the next segment, one thread of warp 6 issues the MMAs, and
// warps 0-3 do the softmax: thread t has token t of each tile, reads its
// logit terms from tensor memory, and writes its P bytes; as the owner of
// head dimension t it reads the tile's O from tensor memory and adds it to
// f32 registers, both brought to the larger maximum.  The copies run on
// across segments, QK runs two tiles ahead of PV (S is double-buffered), and
// a tile's PV runs under the next tile's logits, whose warps add its O while
// they wait for each other's maxima.
//
// Bound: HBM, the caches' bytes.  Measured, of 6.54 TB/s that a copy reaches:
// 16 rows of 16384-131072 tokens, 32 / 8 heads, bf16, 291 us, 6.37 TB/s; 256
// rows of 512-8192, 64 / 8 heads, 251 us, 5.84 TB/s at 1965 MHz (calls in a row
// and replayed graphs alike; run for seconds, at the card's power cap and 1650-
// 1800 MHz, both take 271-280, since the softmax has half of the issue slots);
// 64 rows of 128-4096, 32 / 32 heads, f16, 103 us, 5.9 TB/s;
// one row of 1001 tokens 10.4 us, the chain of one tile and the join.  What is
// left at many rows is the 8 us to the first tile, shares that end apart, and
// the join.  Groups past 8 heads read K and V once for each chunk: see
// dispatch().
// ---------------------------------------------------------------------------
constexpr int kThreads = 256;  // two warpgroups: softmax, and the rest
constexpr int kKWarp = 4;
constexpr int kVWarp = 5;
constexpr int kMmaWarp = 6;
constexpr int kQWarp = 7;
constexpr float kPScale = 256.f;
constexpr float kNoPiece = -1.f;  // in the place of a sum
constexpr float kNoMax = -3.402823466e38f;  // the maximum over no token: finite, so that differences are
// vs enters the exponent down to 2^-60 and multiplies the weight below (zero
// among it), so that L, which counts weights over their vs, stays in range.
constexpr float kLeastScale = 8.67361737988403547e-19f;

// e4m3 terms of a query element and of a weight: while they are normal, two
// hold a bf16's 8 significant bits, three an f16's 11.  More terms for a weight
// would take its floor down (four bits each) and cost the softmax warps the
// time of f16's third: with 8 heads 62 us against 55 (64 rows of 512-4096, 64 / 8 heads).
template <typename T>
constexpr int kTerms = std::is_same<T, __half>::value ? 3 : 2;

template <typename T, int D, int HG>
struct Layout {
  static constexpr int kN = (kTerms<T> * HG + 15) / 16 * 16;  // MMA columns
  static constexpr int kBoxes = D / 128;
  static constexpr int kHalf = kBoxes * kBox;         // a tile's K or V
  // K and V have rings of their own: a K stage is free once its QK is done,
  // a V stage an exchange of maxima and a PV later.
  static constexpr int kMinCtas = D == 128 ? 3 : 1;  // per SM
  static constexpr int kStages = D == 128 ? 2 : 3;
  // Registers of a softmax thread, and of the others, where the launch's even
  // share of three CTAs per SM is too few: what one warpgroup gives up is at
  // least what the other takes.
  static constexpr bool kSplitRegs = D == 128 && HG == 8;
  static constexpr int kLaunchRegs = 80;
  static constexpr int kSoftmaxRegs = 112;
  static constexpr int kOtherRegs = 48;
  static_assert(kSoftmaxRegs + kOtherRegs <= 2 * kLaunchRegs, "more registers than the block has");
  static constexpr int kVOff = kStages * kHalf;
  static constexpr int kQOff = 2 * kStages * kHalf;   // Q: kBoxes x [kN rows x 128 B]
  static constexpr int kQBox = kN * 128;
  static constexpr int kPOff = kQOff + kBoxes * kQBox;  // P: kN/16 planes x 128 tokens x 16 B
  static constexpr int kBarOff = kPOff + kN * 128;
  // full, empty of K and of V; s_full by tile parity; p_full, o_full, q_full,
  // q_empty, fin
  static constexpr int kNumBars = 4 * kStages + 2 + 5;
  static constexpr int kScaleOff = kBarOff + (kNumBars * 8 + 15) / 16 * 16;  // [stages][ks 8, vs 8] f32
  static constexpr int kMaskOff = kScaleOff + kStages * 2 * kTileBlocks * 4;  // [stages] int
  static constexpr int kFailOff = kMaskOff + 16;                              // [2] int: a wait ran out
  static constexpr int kMaxOff = kFailOff + 16;                               // [2][4][HG] f32
  static constexpr int kMaxHeads = (HG + 3) / 4 * 4;
  static constexpr int kSumOff = kMaxOff + 2 * 4 * kMaxHeads * 4;          // [4][HG] f32
  static constexpr int kQsOff = kSumOff + 4 * kMaxHeads * 4;               // [HG] f32
  static constexpr int kStartOff = (kQsOff + kMaxHeads * 4 + 15) / 16 * 16;  // Cursor
  static constexpr int kSharesOff = (kStartOff + 32 + 15) / 16 * 16;        // Shares
  static constexpr int kScanOff = kSharesOff + 64;                          // [8 warps] int64
  static constexpr int kTmemOff = kScanOff + 64;
  static constexpr int kBytes = kTmemOff + 16;
  static constexpr int kAlloc = kBytes + 1024;
  static constexpr int kOCol = 2 * kN;                 // O after the two S buffers
  static constexpr int kCols = 2 * kN + kBoxes * kN;
  static constexpr uint32_t kTmemCols = kCols <= 64 ? 64 : kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
  static_assert(kStages <= 4, "mask words");
  static_assert(kMinCtas * (kAlloc + 1024) <= 228 * 1024 && kMinCtas * kTmemCols <= 512, "CTAs per SM");
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

// Waits for phase `parity` of *bar, at most limit_ns (false then).  Roles with
// time to spare sleep kSleep ns between their tries and leave the issue slots
// to the softmax.
template <int kSleep = 0>
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, uint64_t limit_ns) {
  const uint32_t b = smem_addr(bar);
  if (mbar_try_wait(b, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 32; ++i) {
      if (kSleep > 0) __nanosleep(kSleep);
      if (mbar_try_wait(b, parity)) return true;
    }
    if (global_timer_ns() - t0 > limit_ns) return false;
  }
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

// What the CTAs' shares are made from.
struct Shares {
  int64_t weight;  // of all items
  int64_t ctas;    // that take part
  int64_t first;   // weight before the item that the CTA's first tile belongs to
  int64_t tile[2]; // tiles before each end of the CTA's share
  int item;        // weight of an item beside its tiles
};

// The CTA's first tile and how many it has, found by all threads: prefix sums
// of the rows' tiles, then the threads whose rows hold the two ends of the
// CTA's share walk them.
template <typename L>
__device__ __forceinline__ Cursor find_start(const Args& a, uint8_t* smem) {
  Cursor* start = reinterpret_cast<Cursor*>(smem + L::kStartOff);
  Shares* sh = reinterpret_cast<Shares*>(smem + L::kSharesOff);
  int64_t* scan = reinterpret_cast<int64_t*>(smem + L::kScanOff);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t items = (int64_t)a.num_kv_heads * a.head_chunks;
  const int per = (a.num_seqs + kThreads - 1) / kThreads;
  const int s0 = min(a.num_seqs, (int)threadIdx.x * per), s1 = min(a.num_seqs, s0 + per);
  // tiles, and rows that have any above bit 40
  constexpr int64_t kRow = (int64_t)1 << 40;
  int64_t sum = 0;
  for (int s = s0; s < s1; ++s) {
    const int n = (context_of(a, s, blockIdx.x == 0) + kTile - 1) / kTile;
    sum += n + (n > 0 ? kRow : 0);
  }
  int64_t incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) scan[warp] = incl;
  __syncthreads();
  int64_t before = incl - sum, total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += scan[w];
    total += scan[w];
  }
  const int64_t tiles = (total & (kRow - 1)) * items;
  // no more CTAs than tiles take part, so each of them has at least one
  const int64_t G = tiles < gridDim.x ? (tiles > 0 ? tiles : 1) : gridDim.x;
  const int wi = tiles >= kManyTiles * G ? kItemWeight : 0;
  auto weight = [&](int64_t v) { return items * (kTileWeight * (v & (kRow - 1)) + wi * (v >> 40)); };
  const int64_t W = weight(total);
  const bool whole = a.meta == nullptr;  // items are not shared: both ends move on to where one begins
  if (threadIdx.x == 0) {
    *start = Cursor{0, 0, 0, 0, 0, 0};
    *sh = Shares{W, G, 0, {tiles, tiles}, wi};
  }
  __syncthreads();
#pragma unroll 1
  for (int e = 0; e < 2; ++e) {
    const int64_t b = blockIdx.x + e < G ? W * (blockIdx.x + e) / G : W;
    if (b < weight(before) || b >= weight(before + sum)) continue;
    int64_t at = before;
    for (int s = s0; s < s1; ++s) {
      const int ctx = context_of(a, s, false);
      const int n = (ctx + kTile - 1) / kTile;
      const int64_t row = n > 0 ? n + kRow : 0;
      if (b < weight(at + row)) {
        const uint32_t w = kTileWeight * n + wi;
        const uint64_t off64 = (uint64_t)(b - weight(at));
        uint32_t item, tile;
        if (off64 >> 32 == 0) {  // (a 64-bit division is a slow one)
          item = (uint32_t)off64 / w;
          tile = (uint32_t)off64 % w;
        } else {
          item = (uint32_t)(off64 / w);
          tile = (uint32_t)(off64 % w);
        }
        tile = (tile + kTileWeight - 1) / kTileWeight;
        if ((whole && tile > 0) || tile >= (uint32_t)n) {
          tile = 0;
          ++item;
        }
        sh->tile[e] = items * (at & (kRow - 1)) + (int64_t)item * n + tile;
        if (e == 0) {
          *start = Cursor{s, (int)item, ctx, n, (int)tile, 0};
          sh->first = weight(at) + (int64_t)item * w;
        }
        break;
      }
      at += row;
    }
  }
  __syncthreads();
  Cursor c = *start;
  c.left = (int)(sh->tile[1] - sh->tile[0]);
  if (c.left > 0 && c.item == items) {  // moved on past the row's last item
    c.item = 0;
    do {
      ++c.seq;
      c.ctx = context_of(a, c.seq, false);
    } while (c.ctx == 0);
    c.tiles = (c.ctx + kTile - 1) / kTile;
  }
  return c;
}

template <typename T, int D, int HG>
__global__ void __launch_bounds__(kThreads, Layout<T, D, HG>::kMinCtas)
    block_attention_kernel(const __grid_constant__ Args a, const __grid_constant__ CUtensorMap tmk,
                           const __grid_constant__ CUtensorMap tmv) {
  using L = Layout<T, D, HG>;
  constexpr int N = L::kN, S = L::kStages, kT = kTerms<T>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* k_full = bars;
  uint64_t* k_empty = bars + S;
  uint64_t* v_full = bars + 2 * S;
  uint64_t* v_empty = bars + 3 * S;
  uint64_t* s_full = bars + 4 * S;  // [2], by tile parity
  uint64_t* p_full = s_full + 2;
  uint64_t* o_full = p_full + 1;
  uint64_t* q_full = o_full + 1;
  uint64_t* q_empty = q_full + 1;
  uint64_t* fin = q_empty + 1;
  float* scales = reinterpret_cast<float*>(smem + L::kScaleOff);
  int* masks = reinterpret_cast<int*>(smem + L::kMaskOff);
  volatile int* fail = reinterpret_cast<int*>(smem + L::kFailOff);  // of a softmax warp, before a meeting of either kind
  float* smax = reinterpret_cast<float*>(smem + L::kMaxOff);
  float* ssum = reinterpret_cast<float*>(smem + L::kSumOff);
  float* sqs = reinterpret_cast<float*>(smem + L::kQsOff);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kTmemOff);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(smem_addr(&k_full[s]), 1);
      mbar_init(smem_addr(&k_empty[s]), 1);
      mbar_init(smem_addr(&v_full[s]), 1 + 2 * kTileBlocks);  // V's bytes, and 16 lanes' scales
      mbar_init(smem_addr(&v_empty[s]), 1);
    }
    for (int i = 0; i < 2; ++i) mbar_init(smem_addr(&s_full[i]), 1);
    mbar_init(smem_addr(p_full), kTile);
    mbar_init(smem_addr(o_full), 1);
    mbar_init(smem_addr(q_full), 32);
    mbar_init(smem_addr(q_empty), 1 + 4);  // its last QK, and the softmax warps' reads of the scales
    mbar_init(smem_addr(fin), 1);
    fail[0] = fail[1] = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_addr(tmem_slot), L::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  // What the launch before this one wrote is read from here on; the join may
  // be set up beside this kernel.
  grid_dependency_wait();
  grid_dependency_launch();
  Cursor cur = find_start<L>(a, smem);  // synchronises the block
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t ntiles = (uint32_t)cur.left;  // of this CTA (its share of all tiles is far below 2^31)

  // Rows without a context: zeros, dealt to the CTAs in turn.
  for (int s = blockIdx.x; s < a.num_seqs; s += gridDim.x)
    if (context_of(a, s, false) == 0) {
      T* o = static_cast<T*>(a.out) + (size_t)s * a.num_heads * D;
      for (int i = threadIdx.x; i < a.num_heads * D; i += kThreads) o[i] = from_float<T>(0.f);
    }

  if (warp >= 4) {
    if constexpr (L::kSplitRegs) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kOtherRegs));
    if (warp == kKWarp || warp == kVWarp) {
      // ---------------- copies of K, or of V with the scales ----------------
      const bool is_k = warp == kKWarp;
      uint64_t* fulls = is_k ? k_full : v_full;
      uint64_t* empties = is_k ? k_empty : v_empty;
      uint8_t* ring = smem + (is_k ? 0 : L::kVOff);
      const CUtensorMap* map = is_k ? &tmk : &tmv;
      bool ok = true;
      uint32_t j = 0;  // tiles begun
      // Block ids come 32 (four tiles) at a time, a group ahead of their use:
      // `ahead` stands at the group whose ids are in `ids_next`.
      Cursor ahead = cur;
      int at = 0;  // tile of `ahead`'s segment
      auto fetch = [&]() {
        if (ahead.done()) return 0;
        const int b = (ahead.tile + at) * kTileBlocks + lane;
        const int last = min((ahead.ctx + kBlk - 1) / kBlk, (ahead.tile + ahead.count()) * kTileBlocks);
        return b < last ? a.tables[(size_t)ahead.seq * a.max_blocks + b] : 0;
      };
      auto step = [&]() {
        at += 4;
        if (at >= ahead.count()) {
          at = 0;
          ahead.next(a);
        }
      };
      int ids_next = fetch();
      for (; !cur.done() && ok; cur.next(a)) {
        const int cnt = cur.count(), nblk = (cur.ctx + kBlk - 1) / kBlk;
        const int kvh = cur.item / a.head_chunks;
        int ids = 0;
        for (int i = 0; i < cnt; ++i, ++j) {
          if ((i & 3) == 0) {
            ids = ids_next;
            step();
            ids_next = fetch();
          }
          const int s = (int)(j % S);
          const int k = lane & 7;
          const int id = __shfl_sync(0xffffffffu, ids, (i & 3) * kTileBlocks + k);
          const bool want = (cur.tile + i) * kTileBlocks + k < nblk;
          const bool valid = want && id >= 0 && (int64_t)id < a.num_blocks;
          if (want && !valid && lane < kTileBlocks) block_attn_error(CF_DEVERR_BLOCK_ID);
          const uint32_t mask = __ballot_sync(0xffffffffu, valid) & 0xffu;
          if (j >= S) {
            ok = wait_bar<64>(&empties[s], (j / S - 1) & 1u, a.wait_limit_ns);
            if (!__all_sync(0xffffffffu, ok)) {
              ok = false;
              break;
            }
          }
          if (j == 0 && (a.unarm_cta == kEveryCta || a.unarm_cta == (int)blockIdx.x))
            continue;  // test hook: the stage never completes
          const uint32_t bar = smem_addr(&fulls[s]);
          if (lane == 0) {
            if (!is_k) masks[s] = (int)mask;
            fence_proxy_async_smem();
            if (mask == 0)
              mbar_arrive(bar);
            else
              mbar_arrive_expect_tx(bar, (uint32_t)__popc(mask) * kBlk * D);
          }
          __syncwarp();
          if (valid && lane < kTileBlocks) {  // lane k copies block k
            const int32_t row = (int32_t)(((int64_t)id * a.num_kv_heads + kvh) * kBlk);
            uint8_t* dst = ring + s * L::kHalf + lane * (kBlk * 128);
#pragma unroll
            for (int b = 0; b < L::kBoxes; ++b) tma_load_2d(smem_addr(dst + b * kBox), map, b * 128, row, bar);
          }
          if (!is_k && lane < 2 * kTileBlocks) {  // lanes 0-7 a block's ks, 8-15 its vs
            if (valid)
              cp_async4(smem_addr(&scales[s * 2 * kTileBlocks + lane]),
                        (lane < kTileBlocks ? a.ks : a.vs) + (int64_t)id * a.num_kv_heads + kvh);
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
          }
          __syncwarp();
        }
      }
      if (!ok) block_attn_error(CF_DEVERR_TIMEOUT);
      // no copy may land after the CTA has left
      cp_async_wait_all();
      if (lane == 0)
        for (uint32_t i = j > S ? j - S : 0; i < j; ++i) wait_bar(&fulls[i % S], (i / S) & 1u, a.wait_limit_ns);
    } else if (warp == kQWarp) {
      // ---------------- Q's terms, a segment at a time ----------------
      constexpr int E = D / 32;
      constexpr int kBatch = HG < 8 ? HG : 8;  // heads whose loads run before the wait
      for (int n = kT * HG; n < N; ++n)  // rows past the terms
        for (int b = 0; b < L::kBoxes; ++b)
          reinterpret_cast<uint32_t*>(smem + L::kQOff + b * L::kQBox + n * 128)[lane] = 0u;
      bool ok = true;
      for (int seg = 0; !cur.done() && ok; cur.next(a), ++seg) {
        const int kvh = cur.item / a.head_chunks, chunk = cur.item - kvh * a.head_chunks;
        const int head0 = kvh * a.group + chunk * HG, nheads = min(HG, a.group - chunk * HG);
        const T* src = static_cast<const T*>(a.q) + ((size_t)cur.seq * a.num_heads + head0) * D + lane * E;
#pragma unroll
        for (int h0 = 0; h0 < HG; h0 += kBatch) {
          uint32_t raw[kBatch][E / 2];
#pragma unroll
          for (int h = 0; h < kBatch; ++h)
#pragma unroll
            for (int e = 0; e < E / 2; ++e)
              raw[h][e] = h0 + h < nheads ? reinterpret_cast<const uint32_t*>(src + (size_t)(h0 + h) * D)[e] : 0u;
          if (h0 == 0 && seg > 0) {
            ok = wait_bar<256>(q_empty, (uint32_t)(seg - 1) & 1u, a.wait_limit_ns);
            if (!__all_sync(0xffffffffu, ok)) {
              ok = false;
              break;
            }
          }
#pragma unroll
          for (int hb = 0; hb < kBatch; ++hb) {
            const int h = h0 + hb;
            float q[E];
            float mx = 0.f;
            bool bad = false;
#pragma unroll
            for (int e = 0; e < E / 2; ++e) unpack_word<T>(raw[hb][e], q + 2 * e);
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
        }
        if (!ok) break;
        fence_proxy_async_smem();
        mbar_arrive(smem_addr(q_full));
      }
      if (!ok) block_attn_error(CF_DEVERR_TIMEOUT);
    } else if (lane == 0) {
      // ---------------- MMA issuer ----------------
      const uint64_t k_desc = smem_desc_sw128(smem_addr(smem), 16, 1024);
      const uint64_t v_desc = smem_desc_sw128(smem_addr(smem + L::kVOff), 16, 1024);
      const uint64_t q_desc = smem_desc_sw128(smem_addr(smem + L::kQOff), 16, 1024);
      // P: 8 tokens x 16 columns per 128 bytes, tokens onward, then planes
      const uint64_t p_desc = smem_desc_plain(smem_addr(smem + L::kPOff), 128, kTile * 16);
      bool ok = true;
      int seg = 0, i = 0;  // segment and its next tile, of the next QK
      auto issue_qk = [&](uint32_t j) {
        const int s = (int)(j % S);
        ok = ok && (i > 0 || wait_bar<32>(q_full, (uint32_t)seg & 1u, a.wait_limit_ns)) &&
             wait_bar<32>(&k_full[s], (j / S) & 1u, a.wait_limit_ns);
        if (!ok) return;
        tc_fence_after();
        const uint64_t kd = k_desc + (uint64_t)((s * L::kHalf) >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk) {
          const uint64_t ad = kd + (uint64_t)(((kk >> 2) * kBox + (kk & 3) * 32) >> 4);
          const uint64_t bd = q_desc + (uint64_t)(((kk >> 2) * L::kQBox + (kk & 3) * 32) >> 4);
          mma_f8(tmem + (int)(j & 1) * N, ad, bd, idesc_f8(0, N), kk > 0 ? 1u : 0u);
        }
        tc_commit(smem_addr(&s_full[j & 1]));
        tc_commit(smem_addr(&k_empty[s]));
        if (++i == cur.count()) {
          tc_commit(smem_addr(q_empty));
          i = 0;
          ++seg;
          cur.next(a);
        }
      };
      for (uint32_t j = 0; j < 2 && j < ntiles; ++j) issue_qk(j);
      for (uint32_t j = 0; j < ntiles && ok; ++j) {
        const int s = (int)(j % S);
        ok = wait_bar<32>(p_full, (uint32_t)j & 1u, a.wait_limit_ns) &&
             wait_bar<32>(&v_full[s], (j / S) & 1u, a.wait_limit_ns);
        if (!ok) break;
        tc_fence_after();
        const uint64_t vd = v_desc + (uint64_t)((s * L::kHalf) >> 4);
#pragma unroll
        for (int b = 0; b < L::kBoxes; ++b)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)  // 32 tokens each
            mma_f8(tmem + L::kOCol + b * N, vd + (uint64_t)((b * kBox + kk * 4096) >> 4),
                   p_desc + (uint64_t)((kk * 512) >> 4), idesc_f8(1, N), kk > 0 ? 1u : 0u);
        tc_commit(smem_addr(o_full));
        tc_commit(smem_addr(&v_empty[s]));
        if (j + 2 < ntiles) issue_qk(j + 2);
      }
      if (!ok) {
        // every MMA issued so far has finished before tensor memory is freed
        block_attn_error(CF_DEVERR_TIMEOUT);
        tc_commit(smem_addr(fin));
        wait_bar(fin, 0u, a.wait_limit_ns);
      }
    }
    __syncwarp();
  } else {
    // ---------------- softmax ----------------
    if constexpr (L::kSplitRegs) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::kSoftmaxRegs));
    const int tok = threadIdx.x;  // token of the tile; head dimension of O
    const uint32_t trow = tmem + ((uint32_t)(32 * warp) << 16);
    bool begun = false;
    uint32_t j = 0;
    const Shares& sh = *reinterpret_cast<const Shares*>(smem + L::kSharesOff);
    int64_t at = sh.first;  // weight before the segment's item
    // Warp 0 waits for the others, which sleep at a hardware barrier: polling
    // warps would take the issue slots of the other CTAs' softmax.  A wait that
    // runs out sets fail[] of the next meeting, and every warp reads it there
    // and leaves.  Meetings alternate between two kinds (0 and 1), so nobody
    // sets one's flag before the others have read it at the last of its kind:
    // the four warps leave at the same one.  (A barrier that reduces a
    // predicate, the other way to this, takes 267 us against 250 at 256 rows.)
    auto meet = [&](int kind) {
      asm volatile("bar.sync 1, 128;" ::: "memory");
      return fail[kind] == 0;
    };
    bool ok = true;
    for (int seg = 0; !cur.done(); cur.next(a), ++seg) {
      const int cnt = cur.count();
      const int kvh = cur.item / a.head_chunks, chunk = cur.item - kvh * a.head_chunks;
      float qsc[HG], m[HG], l[HG], beta[HG], acc[L::kBoxes][HG];
      if (warp == 0) {
        if (!wait_bar(q_full, (uint32_t)seg & 1u, a.wait_limit_ns)) fail[0] = 1;
        __syncwarp();  // lanes may have given up at different tries; a warp meets as one
      }
      ok = meet(0);
      if (!ok) break;
#pragma unroll
      for (int h = 0; h < HG; ++h) {
        qsc[h] = sqs[h] * a.scale_log2;
        m[h] = kNoMax;
        l[h] = 0.f;
#pragma unroll
        for (int b = 0; b < L::kBoxes; ++b) acc[b][h] = 0.f;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(q_empty));
      // the accumulator takes tile t's O, before a meeting of this kind
      auto add_o = [&](uint32_t t, int kind) {
        if (!wait_bar(o_full, t & 1u, a.wait_limit_ns)) fail[kind] = 1;
        __syncwarp();
        tc_fence_after();
#pragma unroll
        for (int b = 0; b < L::kBoxes; ++b) {
          float o[N];
#pragma unroll
          for (int c = 0; c < N; c += 16) tmem_ld16(trow + L::kOCol + b * N + c, &o[c]);
          tmem_wait_ld();
#pragma unroll
          for (int h = 0; h < HG; ++h) acc[b][h] = fmaf(join_terms<kT, HG>(o, h), beta[h], acc[b][h]);
        }
      };
      for (int i = 0; i < cnt; ++i, ++j) {
        const int par = (int)(j & 1), s = (int)(j % S);
        if (warp == 0) {
          if (!(wait_bar(&v_full[s], (j / S) & 1u, a.wait_limit_ns) &&
                wait_bar(&s_full[par], (j >> 1) & 1u, a.wait_limit_ns)))
            fail[1] = 1;
          __syncwarp();
        }
        ok = meet(1);
        if (!ok) break;
        tc_fence_after();
        const bool valid =
            (cur.tile + i) * kTile + tok < cur.ctx && ((masks[s] >> (tok / kBlk)) & 1) != 0;
        const float ks = scales[s * 2 * kTileBlocks + tok / kBlk];
        const float vs = valid ? scales[s * 2 * kTileBlocks + kTileBlocks + tok / kBlk] : 1.f;
        const float vf = vs < kLeastScale ? kLeastScale : vs;
        const float lv = __log2f(vf);
        const float vinv = __fdividef(1.f, vf);
        float x[N];
#pragma unroll
        for (int c = 0; c < N; c += 16) tmem_ld16(trow + par * N + c, &x[c]);
        tmem_wait_ld();
        float* tops = smax + par * 4 * L::kMaxHeads;
#pragma unroll
        for (int h = 0; h < HG; ++h) {
          const float r = join_terms<kT, HG>(x, h);
          x[h] = valid ? fmaf(r, qsc[h] * ks, lv) : -INFINITY;
          const float w = warp_max(x[h]);
          if (lane == 0) tops[warp * L::kMaxHeads + h] = w;
        }
        // The last tile's O, while the other warps' maxima come in.  After it
        // P and O are free: this tile's PV may write them.
        if (i > 0) add_o(j - 1, 0);
        ok = meet(0);
        if (!ok) break;
#pragma unroll
        for (int h = 0; h < HG; ++h) {
          const float mx = fmaxf(fmaxf(fmaxf(tops[h], tops[L::kMaxHeads + h]), kNoMax),
                                 fmaxf(tops[2 * L::kMaxHeads + h], tops[3 * L::kMaxHeads + h]));
          // of 2^(m - max) and 2^(mx - max), which bring the row's sums and the
          // tile's to the larger of the two maxima, one is 1
          const float d = m[h] - mx, r = ex2_approx(-fabsf(d));
          const float alpha = d < 0.f ? r : 1.f;
          beta[h] = d < 0.f ? 1.f : r;
          m[h] = fmaxf(m[h], mx);
          x[h] = ex2_approx(x[h] - mx);
          l[h] = fmaf(x[h] * vinv, beta[h], l[h] * alpha);
#pragma unroll
          for (int b = 0; b < L::kBoxes; ++b) acc[b][h] *= alpha;
        }
        // P's bytes: column t HG + h is term t of head h
        uint16_t pairs[N / 2];
#pragma unroll
        for (int k = 0; k < N / 2; ++k) pairs[k] = 0;
        const float ps = vs < kLeastScale ? vs * (kPScale / kLeastScale) : kPScale;
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
        uint4* pb = reinterpret_cast<uint4*>(smem + L::kPOff) + tok;
#pragma unroll
        for (int c = 0; c < N / 16; ++c) {
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            w[k] = (uint32_t)pairs[c * 8 + 2 * k] | ((uint32_t)pairs[c * 8 + 2 * k + 1] << 16);
          pb[c * kTile] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        if (!valid) {
          // A V row that no token of the row owns (past the context, or a
          // rejected block's) may hold any bytes, and 0 * NaN is not 0.
          uint8_t* v = smem + L::kVOff + s * L::kHalf + tok * 128;
#pragma unroll
          for (int b = 0; b < L::kBoxes; ++b)
#pragma unroll
            for (int c = 0; c < 8; ++c) reinterpret_cast<uint4*>(v + b * kBox)[c] = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(smem_addr(p_full));
      }
      if (!ok) break;
      add_o(j - 1, 1);

      // The segment's sums over its 128 token threads, then its result.
#pragma unroll
      for (int h = 0; h < HG; ++h) {
        float w = l[h];
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) w += shfl_xor(w, k);
        if (lane == 0) ssum[warp * L::kMaxHeads + h] = w;
      }
      ok = meet(1);
      if (!ok) break;
      const bool whole = cur.tile == 0 && cnt == cur.tiles;
      const int slot = 2 * blockIdx.x + (cur.tile == 0 ? 1 : 0);
      const int head0 = kvh * a.group + chunk * HG, nheads = min(HG, a.group - chunk * HG);
#pragma unroll
      for (int h = 0; h < HG; ++h) {
        if (h >= nheads) continue;
        const float sum = (ssum[h] + ssum[L::kMaxHeads + h]) + (ssum[2 * L::kMaxHeads + h] + ssum[3 * L::kMaxHeads + h]);
        const float inv = sum == 0.f ? 0.f : 1.f / (sum * kPScale);
#pragma unroll
        for (int b = 0; b < L::kBoxes; ++b) {
          const float r = acc[b][h] * inv;
          if (whole)
            static_cast<T*>(a.out)[((size_t)cur.seq * a.num_heads + head0 + h) * D + b * 128 + tok] = from_float<T>(r);
          else
            a.part_out[((size_t)slot * HG + h) * D + b * 128 + tok] = r;
        }
        if (!whole && tok == 0) {
          a.part_max[slot * HG + h] = m[h];
          a.part_sum[slot * HG + h] = sum;
        }
      }
      if (!whole && cur.tile == 0 && tok == 0) {
        // An item begun here.  CTA c's share begins at c W / G: the last one
        // to begin at the item's last tile or before has that tile.
        const int64_t last = at + (int64_t)kTileWeight * (cur.tiles - 1);
        a.meta[blockIdx.x] = make_int4(cur.seq, cur.item, (int)(((last + 1) * sh.ctas - 1) / sh.weight), 0);
        begun = true;
      }
      at += (int64_t)kTileWeight * cur.tiles + sh.item;
    }
    if (!ok && lane == 0) block_attn_error(CF_DEVERR_TIMEOUT);
    // The CTA that began this item may have told the join of this piece.
    if (!ok && a.meta != nullptr && cur.tile > 0 && tok < HG) a.part_sum[2 * blockIdx.x * HG + tok] = kNoPiece;
    if (a.meta != nullptr && tok == 0 && !begun) a.meta[blockIdx.x] = make_int4(-1, 0, 0, 0);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) tmem_dealloc(tmem, L::kTmemCols);
}

// Joins the items that several CTAs share, one CTA per CTA c of the streaming
// kernel: the item that c began, its later pieces in the first slots of CTAs
// c + 1 .. last.  With few pieces a warp takes a head, with many (a few rows
// over all CTAs) the warps share each head's; a lane has the maximum and sum
// of one of 32 pieces, then its columns of all.
// out = sum_p w_p o_p / sum_p w_p, w_p = sum_p 2^(max_p - max).  An item with
// a piece that its CTA could not finish (CF_DEVERR_TIMEOUT) is left unwritten.
// Latency-bound: three dependent loads (the CTA's entry, the sums, the
// pieces' outputs) behind a launch that overlaps the streaming kernel's end.
constexpr int kJoinWarps = 8;
constexpr int kFewPieces = 8;

template <typename T, int D, int HG>
__global__ void __launch_bounds__(kJoinWarps * 32) block_attention_join_kernel(const __grid_constant__ Args a) {
  constexpr int E = D / 32;
  __shared__ float sm[kJoinWarps], sl[kJoinWarps];
  __shared__ __align__(16) float so[kJoinWarps][D];
  grid_dependency_wait();
  const int c = blockIdx.x;
  const int4 meta = a.meta[c];
  if (meta.x < 0) return;
  const int kvh = meta.y / a.head_chunks, chunk = meta.y - kvh * a.head_chunks;
  const int nheads = min(HG, a.group - chunk * HG);
  const int pieces = meta.z - c + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  T* out = static_cast<T*>(a.out) + ((size_t)meta.x * a.num_heads + kvh * a.group + chunk * HG) * D;
  float m, l, o[E];
  bool lost;  // a piece
  auto collect = [&](int h, int first, int stride) {  // pieces first, first + stride, ... of head h
    auto slot = [&](int p) { return (size_t)(p == 0 ? 2 * c + 1 : 2 * (c + p)) * HG + h; };
    m = -INFINITY;
    l = 0.f;
    lost = false;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    for (int p0 = first; p0 < pieces; p0 += stride * 32) {
      const int mine = p0 + stride * lane;
      const float sum = mine < pieces ? a.part_sum[slot(mine)] : 0.f;
      const float top = mine < pieces ? a.part_max[slot(mine)] : -INFINITY;
      lost |= __any_sync(0xffffffffu, sum == kNoPiece) != 0;
      // a piece without a readable token has sum 0
      const float mn = fmaxf(m, warp_max(top));
      const float mu = mn == -INFINITY ? 0.f : mn;
      const float alpha = exp2f(m - mu);
      m = mn;
      const float w = sum == 0.f ? 0.f : sum * exp2f(top - mu);
      float ws = w;
#pragma unroll
      for (int i = 16; i > 0; i >>= 1) ws += shfl_xor(ws, i);
      l = l * alpha + ws;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] *= alpha;
      const int n = min(32, (pieces - p0 + stride - 1) / stride);
#pragma unroll 4
      for (int i = 0; i < n; ++i) {
        const float wp = __shfl_sync(0xffffffffu, w, i);
        float x[E];
        load_widen<float, E>(a.part_out + slot(p0 + stride * i) * D + lane * E, x);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(wp, x[e], o[e]);
      }
    }
  };
  if (pieces <= kFewPieces) {
    for (int h = warp; h < nheads; h += kJoinWarps) {
      collect(h, 0, 1);
      if (lost) return;
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int e = 0; e < E; ++e) out[h * D + lane * E + e] = from_float<T>(o[e] * inv);
    }
    return;
  }
  for (int h = 0; h < nheads; ++h) {
    collect(h, warp, kJoinWarps);
    if (lane == 0) {
      sm[warp] = m;
      sl[warp] = lost ? kNoPiece : l;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) so[warp][lane * E + e] = o[e];
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) m = fmaxf(m, sm[w]);
    const float mu = m == -INFINITY ? 0.f : m;
    float scale[kJoinWarps];
    l = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) {
      if (sl[w] == kNoPiece) return;  // for the whole block
      scale[w] = exp2f(sm[w] - mu);
      l = fmaf(sl[w], scale[w], l);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    for (int d = threadIdx.x; d < D; d += kJoinWarps * 32) {
      float r = 0.f;
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) r = fmaf(so[w][d], scale[w], r);
      out[h * D + d] = from_float<T>(r * inv);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
// Streaming CTAs that are resident at once on the current device.
template <typename T, int D, int HG>
int resident_ctas() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) == cudaSuccess)
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  else
    cudaGetLastError();
  return (n > 0 ? n : 148) * Layout<T, D, HG>::kMinCtas;
}

struct Workspace {
  size_t meta, max, sum, out, bytes;
};

Workspace workspace_of(int ctas, int hg, int d) {
  auto round = [](size_t b) { return (b + 255) / 256 * 256; };
  const size_t rows = (size_t)2 * ctas * hg;
  Workspace w;
  w.meta = 0;
  w.max = round((size_t)ctas * sizeof(int4));
  w.sum = w.max + round(rows * 4);
  w.out = w.sum + round(rows * 4);
  w.bytes = w.out + round(rows * d * 4);
  return w;
}

// Per kernel instantiation and device: opt in to > 48 KB of dynamic smem.
template <typename T, int D, int HG>
cf_status ensure_smem() {
  static std::once_flag flags[64];
  static cudaError_t errs[64];
  auto set = [] {
    auto kern = block_attention_kernel<T, D, HG>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<T, D, HG>::kAlloc);
    if (Layout<T, D, HG>::kSplitRegs && e == cudaSuccess) {
      // a build with fewer registers than the split shares out must not run
      cudaFuncAttributes fa;
      e = cudaFuncGetAttributes(&fa, kern);
      if (e == cudaSuccess && fa.numRegs < Layout<T, D, HG>::kLaunchRegs) e = cudaErrorInvalidConfiguration;
    }
    return e;
  };
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e);
  if (dev < 0 || dev >= 64) return cuda_status(set());
  std::call_once(flags[dev], [&] { errs[dev] = set(); });
  return cuda_status(errs[dev]);
}

template <typename T, int D, int HG>
cf_status launch_heads(Args a, const BlockScaledLaunch& l) {
  const cf_paged_attention_params& p = *l.p;
  a.head_chunks = (a.group + HG - 1) / HG;
  CUtensorMap mk, mv;
  const int64_t rows = p.num_blocks * (int64_t)p.num_kv_heads * kBlk;
  if (!kv_tensor_map(&mk, p.key_cache, rows, D, CF_FP8_E4M3) ||
      !kv_tensor_map(&mv, p.value_cache, rows, D, CF_FP8_E4M3))
    return CF_ERR_CUDA;
  cf_status st = ensure_smem<T, D, HG>();
  if (st != CF_OK) return st;
  const int ctas = resident_ctas<T, D, HG>();
  const int64_t items = (int64_t)p.num_seqs * p.num_kv_heads * a.head_chunks;
  const int64_t tiles = p.max_context_len > kTile ? (p.max_context_len + kTile - 1) / kTile : 1;
  const Workspace w = workspace_of(ctas, HG, D);
  const bool share = tiles > 1 && l.workspace != nullptr && l.workspace_bytes >= w.bytes;
  if (share) {
    uint8_t* base = static_cast<uint8_t*>(l.workspace);
    a.meta = reinterpret_cast<int4*>(base + w.meta);
    a.part_max = reinterpret_cast<float*>(base + w.max);
    a.part_sum = reinterpret_cast<float*>(base + w.sum);
    a.part_out = reinterpret_cast<float*>(base + w.out);
  }
  const int64_t want = share ? items * tiles : items;
  const unsigned grid = (unsigned)(want < ctas ? want : ctas);
  // Both launches may begin under the end of what is before them in the
  // stream; each waits for it before it touches memory.
  cudaLaunchConfig_t cfg = {};
  cfg.stream = l.stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Layout<T, D, HG>::kAlloc;
  st = cuda_status(cudaLaunchKernelEx(&cfg, block_attention_kernel<T, D, HG>, a, mk, mv));
  if (st != CF_OK || !share) return st;
  cfg.dynamicSmemBytes = 0;
  cfg.blockDim = dim3(kJoinWarps * 32);
  return cuda_status(cudaLaunchKernelEx(&cfg, block_attention_join_kernel<T, D, HG>, a));
}

// Calls f with the kernel's types as template arguments: HG query heads of a
// KV head per item, larger groups in chunks of 8.  Chunks are items of their
// own, so each reads the KV head's K and V: from L2 where they are still
// there (64 rows of 1024-8192 tokens, 4 KV heads, 16 heads each, 83 us; 89 as
// one item, which leaves room for two CTAs per SM), from HBM where rows are
// long and many (64 rows of 8192 tokens, 8 KV heads: 2.18 GB read with 16
// heads each, 1.09 GB with 8; 256 such rows 1321 and 662 us).
template <typename F>
auto dispatch(const cf_paged_attention_params& p, F&& f) {
  const int group = p.num_heads / p.num_kv_heads;
  auto heads = [&](auto t, auto d) {
    using Tp = decltype(t);
    constexpr int D = decltype(d)::value;
    if (group == 1) return f.template operator()<Tp, D, 1>();
    if (group <= 4) return f.template operator()<Tp, D, 4>();
    return f.template operator()<Tp, D, 8>();
  };
  using D128 = std::integral_constant<int, 128>;
  using D256 = std::integral_constant<int, 256>;
  if (p.dtype == CF_F16) return p.head_dim == 128 ? heads(__half{}, D128{}) : heads(__half{}, D256{});
  return p.head_dim == 128 ? heads(__nv_bfloat16{}, D128{}) : heads(__nv_bfloat16{}, D256{});
}

struct SizeOf {
  template <typename T, int D, int HG>
  size_t operator()() const {
    return workspace_of(resident_ctas<T, D, HG>(), HG, D).bytes;
  }
};

struct Launch {
  const Args& a;
  const BlockScaledLaunch& l;
  template <typename T, int D, int HG>
  cf_status operator()() const {
    return launch_heads<T, D, HG>(a, l);
  }
};

}  // namespace

size_t block_scaled_workspace(const cf_paged_attention_params& p) {
  return p.num_seqs > 0 && p.max_context_len > kTile ? dispatch(p, SizeOf{}) : 0;
}

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
  a.num_seqs = p.num_seqs;
  a.num_heads = p.num_heads;
  a.num_kv_heads = p.num_kv_heads;
  a.group = p.num_heads / p.num_kv_heads;
  a.max_blocks = p.max_blocks_per_seq;
  a.num_blocks = p.num_blocks;
  const int64_t lim = g_test_wait_limit_ns.load(std::memory_order_relaxed);
  a.wait_limit_ns = lim > 0 ? (uint64_t)lim : kWaitLimitNs;
  a.unarm_cta = g_test_unarm_first_stage.load(std::memory_order_relaxed) != 0
                    ? g_test_unarm_cta.load(std::memory_order_relaxed)
                    : kNoCta;
  return dispatch(p, Launch{a, l});
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
