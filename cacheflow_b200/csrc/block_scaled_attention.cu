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
  const uint8_t* kc;
  const uint8_t* vc;
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
  int32_t part_tokens;
  int32_t num_parts;
  int64_t num_blocks;
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

// One warp per (query head, row, partition); a lane holds D/32 columns.
template <typename T, int D>
__global__ void __launch_bounds__(128) block_attention_simple_kernel(const Args a) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int head = blockIdx.y * 4 + (threadIdx.x >> 5), seq = blockIdx.z, part = blockIdx.x;
  if (head >= a.num_heads) return;
  const int ctx = context_of(a, seq, lane == 0 && head == 0 && part == 0);
  const int t0 = part * a.part_tokens, t1 = min(ctx, t0 + a.part_tokens);
  if (part > 0 && t0 >= ctx) return;
  const int kvh = head / a.group;
  float q[E], o[E], m = -INFINITY, l = 0.f;
  load_widen<T, E>(static_cast<const T*>(a.q) + ((size_t)seq * a.num_heads + head) * D + lane * E, q);
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  const int32_t* table = a.tables + (size_t)seq * a.max_blocks;
  for (int t = t0; t < t1; ++t) {
    const int64_t blk = table[t / kBlk];
    if (blk < 0 || blk >= a.num_blocks) {
      if (lane == 0) block_attn_error(CF_DEVERR_BLOCK_ID);
      continue;
    }
    const int64_t unit = blk * a.num_kv_heads + kvh;
    const int64_t at = (unit * kBlk + t % kBlk) * D + lane * E;
    float k[E], v[E];
    load_widen<__nv_fp8_e4m3, E>(reinterpret_cast<const __nv_fp8_e4m3*>(a.kc + at), k);
    load_widen<__nv_fp8_e4m3, E>(reinterpret_cast<const __nv_fp8_e4m3*>(a.vc + at), v);
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(q[e], k[e], s);
    for (int i = 16; i > 0; i >>= 1) s += shfl_xor(s, i);
    const float vs = a.vs[unit];
    const bool zero = vs == 0.f;
    const float x = s * (a.scale_log2 * a.ks[unit]) + (zero ? 0.f : log2f(vs));
    const float mn = fmaxf(m, x);
    const float alpha = exp2f(m - mn), p = exp2f(x - mn);
    m = mn;
    l = l * alpha + (zero ? p : p / vs);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * alpha + (zero ? 0.f : p * v[e]);
  }
  const size_t hq = (size_t)seq * a.num_heads + head;
  const float inv = l > 0.f ? 1.f / l : 0.f;
  if (a.part_max == nullptr) {
#pragma unroll
    for (int e = 0; e < E; ++e) static_cast<T*>(a.out)[hq * D + lane * E + e] = from_float<T>(o[e] * inv);
    return;
  }
  const size_t pi = hq * a.num_parts + part;
#pragma unroll
  for (int e = 0; e < E; ++e) a.part_out[pi * D + lane * E + e] = o[e] * inv;
  if (lane == 0) {
    a.part_max[pi] = m;
    a.part_sum[pi] = l;
  }
}

// Merges a row's partitions, one warp per (query head, row):
// out = sum_p w_p o_p / sum_p w_p, w_p = sum_p 2^(max_p - max).
template <typename T, int D>
__global__ void __launch_bounds__(128) block_attention_merge_kernel(const Args a) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int head = blockIdx.x * 4 + (threadIdx.x >> 5), seq = blockIdx.y;
  if (head >= a.num_heads) return;
  const int ctx = context_of(a, seq, false);
  const int parts = ctx == 0 ? 1 : min(a.num_parts, (ctx + a.part_tokens - 1) / a.part_tokens);
  const size_t base = ((size_t)seq * a.num_heads + head) * a.num_parts;
  float m = -INFINITY;
  for (int p = lane; p < parts; p += 32) m = fmaxf(m, a.part_max[base + p]);
  for (int i = 16; i > 0; i >>= 1) m = fmaxf(m, shfl_xor(m, i));
  float l = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  if (m != -INFINITY) {
    for (int p = 0; p < parts; ++p) {
      const float w = a.part_sum[base + p] * exp2f(a.part_max[base + p] - m);
      l += w;
      float x[E];
      load_widen<float, E>(a.part_out + (base + p) * D + lane * E, x);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(w, x[e], o[e]);
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  T* out = static_cast<T*>(a.out) + ((size_t)seq * a.num_heads + head) * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) out[e] = from_float<T>(o[e] * inv);
}

template <typename T, int D>
cf_status launch_typed(const Args& a, int num_seqs, cudaStream_t stream) {
  const unsigned groups = (unsigned)((a.num_heads + 3) / 4);
  block_attention_simple_kernel<T, D><<<dim3((unsigned)a.num_parts, groups, (unsigned)num_seqs), 128, 0, stream>>>(a);
  cf_status st = check_launch();
  if (st != CF_OK || a.part_max == nullptr) return st;
  block_attention_merge_kernel<T, D><<<dim3(groups, (unsigned)num_seqs), 128, 0, stream>>>(a);
  return check_launch();
}

}  // namespace

cf_status launch_block_scaled_attention(const BlockScaledLaunch& l) {
  const cf_paged_attention_params& p = *l.p;
  Args a = {};
  a.q = p.query;
  a.kc = static_cast<const uint8_t*>(p.key_cache);
  a.vc = static_cast<const uint8_t*>(p.value_cache);
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
  a.part_tokens = l.num_parts > 1 ? l.part_tokens : p.max_blocks_per_seq * kBlk;
  a.num_blocks = p.num_blocks;
  if (l.num_parts > 1) {
    a.part_max = l.part_max;
    a.part_sum = l.part_sum;
    a.part_out = l.part_out;
  }
  if (p.dtype == CF_F16)
    return p.head_dim == 128 ? launch_typed<__half, 128>(a, p.num_seqs, l.stream)
                             : launch_typed<__half, 256>(a, p.num_seqs, l.stream);
  return p.head_dim == 128 ? launch_typed<__nv_bfloat16, 128>(a, p.num_seqs, l.stream)
                           : launch_typed<__nv_bfloat16, 256>(a, p.num_seqs, l.stream);
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
