// Attention over the 4-bit paged KV cache: one CTA per (row, kv head), its four warps taking every
// fourth token with one online softmax each, merged at the end.
#include "kv4.cuh"

namespace hk {
namespace {

using kv4::Unit;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxGroup = 16;

template <int HD>
__global__ void __launch_bounds__(128) kv4_attn_kernel(Kv4AttnArgs a) {
  using U = Unit<HD>;
  constexpr int NV = HD < 128 ? 1 : HD / 128, LG = HD < 128 ? HD / 4 : 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, G = a.nh / a.nkv;
  __shared__ float so[4][HD];
  __shared__ float sm[4], sl[4];
  pdl_wait();
  const int r = blockIdx.y, kh = blockIdx.x / G, h = blockIdx.x;
  const int seq = a.row_seq[r];
  const bool ok = seq >= 0 && seq < a.table_rows;
  if (!ok && threadIdx.x == 0) set_error(a.status, HK_ERR_BAD_ARG);
  const int ctx = ok ? (int)min((int64_t)max(a.row_ctx[r], 0), (int64_t)a.max_blocks * a.block_size) : 0;
  const bool on = lane < LG;
  float q[NV][4] = {}, o[NV][4] = {};
  for (int j = 0; j < NV && on; ++j)
    for (int e = 0; e < 4; ++e) q[j][e] = bf2f(a.q[r * a.q_stride + (int64_t)h * HD + 128 * j + 4 * lane + e]);
  float m = -INFINITY, l = 0.f;
  const float sl2 = a.scale * kLog2e;
  for (int t = warp; t < ctx; t += 4) {
    const int64_t blk = a.block_tables[(int64_t)seq * a.max_blocks + t / a.block_size];
    if (blk < 0 || blk >= a.cache_blocks) {
      set_error(a.status, HK_ERR_BAD_ARG);
      continue;
    }
    const int off = t % a.block_size, tok = off & 15;
    const uint8_t* u = a.cache + ((blk * a.nkv + kh) * (a.block_size / 16) + off / 16) * U::kBytes;
    float s = 0.f, v[NV][4];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int d = 128 * j + 4 * (on ? lane : 0);
      const uint32_t kw = *reinterpret_cast<const uint32_t*>(u + U::key_word(tok, d & ~7)) >> ((d & 4) * 2);
      const uint32_t vw = *reinterpret_cast<const uint16_t*>(u + U::value_half(tok, d));
      const float2 kp = __half22float2(*reinterpret_cast<const __half2*>(u + U::pair(false, tok, d >> 6)));
      const float2 vp = __half22float2(*reinterpret_cast<const __half2*>(u + U::pair(true, tok, d >> 6)));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (on) s += q[j][e] * fmaf(kp.x, (float)((int)(kw >> ((e >> 1) * 4 + (e & 1) * 16) & 15u) - 8), kp.y);
        v[j][e] = fmaf(vp.x, (float)((int)(vw >> (4 * e) & 15u) - 8), vp.y);
      }
    }
    s = warp_sum(s) * sl2;
    const float mn = fmaxf(m, s), corr = exp2f(m - mn), p = exp2f(s - mn);
    m = mn;
    l = l * corr + p;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[j][e] = o[j][e] * corr + p * v[j][e];
  }
  for (int j = 0; j < NV && on; ++j)
    for (int e = 0; e < 4; ++e) so[warp][128 * j + 4 * lane + e] = o[j][e];
  if (lane == 0) sm[warp] = m, sl[warp] = l;
  __syncthreads();
  float mt = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  if (a.sinks) mt = fmaxf(mt, a.sinks[h] * kLog2e);
  const float mb = mt == -INFINITY ? 0.f : mt;
  float lt = a.sinks ? exp2f(a.sinks[h] * kLog2e - mb) : 0.f;
  for (int w = 0; w < 4; ++w) lt += sl[w] * exp2f(sm[w] - mb);
  for (int d = threadIdx.x; d < HD; d += 128) {
    float x = 0.f;
    for (int w = 0; w < 4; ++w) x += so[w][d] * exp2f(sm[w] - mb);
    x = ctx > 0 ? x / lt : 0.f;
    if (a.out_bf16) a.out_bf16[r * a.out_stride + h * HD + d] = __bfloat16_as_ushort(__float2bfloat16(x));
    if (a.out) a.out[r * a.outf_stride + h * HD + d] = x;
  }
  pdl_launch();
}

void launch_any(const Kv4AttnArgs& a, cudaStream_t s, bool pdl) {
  if (a.R <= 0) return;
  const dim3 grid(a.nh, a.R);
  switch (a.hd) {
    case 64: launch(kv4_attn_kernel<64>, grid, dim3(128), 0, s, pdl, a); break;
    case 128: launch(kv4_attn_kernel<128>, grid, dim3(128), 0, s, pdl, a); break;
    case 256: launch(kv4_attn_kernel<256>, grid, dim3(128), 0, s, pdl, a); break;
    default: throw std::runtime_error("kv4 attention: head_dim 64, 128 or 256");
  }
}

}  // namespace

void kv4_attention_prefill_launch(const Kv4AttnArgs& a, cudaStream_t s, bool pdl) { launch_any(a, s, pdl); }

}  // namespace hk
