// The 4-bit paged KV cache's bookkeeping: a step's rows, slots and new blocks from the request
// lengths, RoPE + quantise + append, and the gather of tokens back to 16-bit rows.
#include "kv4.cuh"

namespace hk {
namespace {

using kv4::Unit;

// ---- rows, slots and blocks of a step ------------------------------------------------------------
// With start = exclusive scan of the new tokens and base = exclusive scan of the blocks that each
// request still needs, row r belongs to the last request i with start[i] <= r, its position is
// cached[i] + r - start[i], and block j of the step goes to the last request with base[j'] <= j.
constexpr int kPlanThreads = 512;
constexpr int kPlanRows = 2048;    // rows per CTA
constexpr int kPlanMaxSeqs = 8192;  // both scans in shared memory

// index of the last entry of the non-decreasing a[0..n) that is <= v (a[0] == 0)
__device__ __forceinline__ int last_not_above(const int* a, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= v) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) kv4_plan_kernel(Kv4PlanArgs a) {
  extern __shared__ int plan_smem[];
  int* start = plan_smem;         // [S]
  int* base = plan_smem + a.S;    // [S]
  __shared__ long long warp_rows[kPlanThreads / 32], warp_need[kPlanThreads / 32];
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int bs = a.block_size;
  const int per = (a.S + kPlanThreads - 1) / kPlanThreads;
  const int i0 = min(a.S, tid * per), i1 = min(a.S, i0 + per);
  const long long room = (long long)a.max_blocks * bs;
  bool bad = false;
  long long rows = 0, need = 0;  // this thread's requests
  for (int i = i0; i < i1; ++i) {
    int n = a.fresh[i];
    const int c = a.cached[i], seq = a.seq_rows[i];
    // a request that cannot be laid out gets no rows
    if (n < 0 || c < 0 || seq < 0 || seq >= a.table_rows || (long long)c + n > room) n = 0, bad = true;
    const int nd = n > 0 ? (c + n + bs - 1) / bs - (c + bs - 1) / bs : 0;
    start[i] = n;
    base[i] = nd;
    rows += n;
    need += nd;
  }
  long long ir = rows, in = need;  // inclusive scan over the warp
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long r = __shfl_up_sync(0xffffffffu, ir, o), d = __shfl_up_sync(0xffffffffu, in, o);
    if (lane >= o) ir += r, in += d;
  }
  if (lane == 31) warp_rows[warp] = ir, warp_need[warp] = in;
  const int any_bad = __syncthreads_or(bad);
  long long r0 = ir - rows, d0 = in - need, total = 0, total_need = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w < warp) r0 += warp_rows[w], d0 += warp_need[w];
    total += warp_rows[w];
    total_need += warp_need[w];
  }
  const long long kTop = 0x7fffffff;
  for (int i = i0; i < i1; ++i) {
    const int n = start[i], nd = base[i];
    start[i] = (int)min(r0, kTop);
    base[i] = (int)min(d0, kTop);
    r0 += n;
    d0 += nd;
  }
  __syncthreads();
  const bool take = a.free_blocks != nullptr;
  const int n_rows = (int)min(total, (long long)a.cap);
  for (int r = blockIdx.x * kPlanThreads + tid; r < a.cap; r += gridDim.x * kPlanThreads) {
    int pos = 0, seq = 0, ctx = 0, slot = -1;
    if (r < n_rows) {
      const int i = last_not_above(start, a.S, r);
      const int c = a.cached[i];
      seq = a.seq_rows[i];
      pos = c + r - start[i];
      ctx = pos + 1;
      const int col = pos / bs, b0 = (c + bs - 1) / bs;
      int blk;
      if (take && col >= b0) {
        const long long j = (long long)base[i] + col - b0;
        blk = j < a.n_free ? a.free_blocks[j] : -1;
      } else {
        blk = a.tables[(int64_t)seq * a.max_blocks + col];
      }
      slot = blk < 0 ? -1 : blk * bs + pos % bs;
    }
    a.positions[r] = pos;
    a.row_seq[r] = seq;
    a.row_ctx[r] = ctx;
    a.slots[r] = slot;
  }
  if (take) {
    const int n = (int)min(total_need, (long long)a.n_free);
    for (int j = blockIdx.x * kPlanThreads + tid; j < n; j += gridDim.x * kPlanThreads) {
      const int i = last_not_above(base, a.S, j);
      a.tables[(int64_t)a.seq_rows[i] * a.max_blocks + (a.cached[i] + bs - 1) / bs + j - base[i]] = a.free_blocks[j];
    }
  }
  if (blockIdx.x == 0 && tid == 0) {
    const bool over = total > a.cap || (take && total_need > a.n_free);
    if (a.taken) *a.taken = take ? (int)min(total_need, (long long)a.n_free) : 0;
    if (any_bad || over) set_error(a.status, HK_ERR_BAD_ARG);
  }
}

// ---- RoPE + quantise + append ----------------------------------------------------------------------
// One warp per head row (two heads per warp at HD 64): every lane holds 4 consecutive dims of each
// 128 (or 64), so that 16 lanes hold the 64 dims of a quantisation group. Products and sums of the
// rotation are rounded one by one and the codes use exact divisions, so the bytes written do not
// depend on how the compiler contracts them.
struct Vec4 {
  float v[4];
};
__device__ __forceinline__ Vec4 ld4(const float* p) {
  const float4 f = *reinterpret_cast<const float4*>(p);
  return {{f.x, f.y, f.z, f.w}};
}

template <int HD>
__global__ void __launch_bounds__(256) kv4_append_kernel(Kv4AppendArgs a) {
  constexpr int LG = HD < 128 ? HD / 4 : 32;  // lanes of one head
  constexpr int HPW = 32 / LG;                // heads per warp
  constexpr int NV = HD / (4 * LG);           // vectors of 4 dims per lane
  using U = Unit<HD>;
  pdl_wait();
  const int lane = threadIdx.x & 31, sl = lane % LG;
  const int heads = a.nh + 2 * a.nkv, per_row = (heads + HPW - 1) / HPW;
  const int64_t unit = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (unit >= (int64_t)a.R * per_row) return;
  const int r = (int)(unit / per_row);
  const int h = (int)(unit % per_row) * HPW + lane / LG;
  const bool live = h < heads;
  const int hc = live ? h : heads - 1;  // lanes without a head compute on the last one and store nothing
  const int pos = a.positions[r];
  if (pos < 0 || pos >= a.rope_rows) return;  // the whole warp
  const int kind = hc < a.nh ? 0 : (hc < a.nh + a.nkv ? 1 : 2);  // q, k, v
  const float* src = a.qkv + (int64_t)r * a.qkv_stride + (int64_t)hc * HD;
  const float* bias = a.bias ? a.bias + (int64_t)hc * HD : nullptr;
  const float* nw = kind == 0 ? a.q_norm : (kind == 1 ? a.k_norm : nullptr);
  Vec4 x[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    x[j] = ld4(src + 128 * j + 4 * sl);
    if (bias) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[j].v[e] += bias[128 * j + 4 * sl + e];
    }
  }
  float inv = 1.f;
  {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) ss += x[j].v[e] * x[j].v[e];
#pragma unroll
    for (int o = LG / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (nw) inv = rsqrtf(ss / HD + a.eps);
  }
  if (nw) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[j].v[e] = __fmul_rn(__fmul_rn(x[j].v[e], inv), nw[128 * j + 4 * sl + e]);
  }
  if (kind < 2) {
    const int half = a.rot_dim / 2;
    const float* rope = a.rope + (int64_t)pos * a.rot_dim;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int d0 = 128 * j + 4 * sl;
      if (a.rope_style == 0) {  // pairs (d, d + 1)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          if (d0 + e < a.rot_dim) {
            const float2 cs = *reinterpret_cast<const float2*>(rope + d0 + e);
            const float p = x[j].v[e], q = x[j].v[e + 1];
            x[j].v[e] = __fsub_rn(__fmul_rn(p, cs.x), __fmul_rn(q, cs.y));
            x[j].v[e + 1] = __fadd_rn(__fmul_rn(p, cs.y), __fmul_rn(q, cs.x));
          }
        }
      } else {  // pairs (d, d + half): the partner is read again (an L1 hit), normalised alike
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = d0 + e;
          if (d < a.rot_dim) {
            const bool first = d < half;
            const int o = first ? d + half : d - half;
            float y = src[o] + (bias ? bias[o] : 0.f);
            if (nw) y = __fmul_rn(__fmul_rn(y, inv), nw[o]);
            const float2 cs = *reinterpret_cast<const float2*>(rope + 2 * (first ? d : o));
            x[j].v[e] = first ? __fsub_rn(__fmul_rn(x[j].v[e], cs.x), __fmul_rn(y, cs.y))
                              : __fadd_rn(__fmul_rn(y, cs.y), __fmul_rn(x[j].v[e], cs.x));
          }
        }
      }
    }
  }
  if (kind == 0 && live) {
    uint16_t* dst = a.q_out + (int64_t)r * a.q_stride + (int64_t)h * HD;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const __nv_bfloat162 lo = __floats2bfloat162_rn(x[j].v[0], x[j].v[1]);
      const __nv_bfloat162 hi = __floats2bfloat162_rn(x[j].v[2], x[j].v[3]);
      *reinterpret_cast<uint2*>(dst + 128 * j + 4 * sl) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
  }
  if (!__any_sync(0xffffffffu, kind != 0)) return;
  int64_t slot = -1;
  if (a.slots) {
    slot = a.slots[r];
  } else {
    const int seq = a.row_seq[r], col = pos / a.block_size;
    if (seq >= 0 && seq < a.table_rows && col < a.max_blocks)
      slot = (int64_t)a.block_tables[(int64_t)seq * a.max_blocks + col] * a.block_size + pos % a.block_size;
  }
  const bool store = live && kind != 0 && slot >= 0 && slot < a.cache_blocks * a.block_size;
  const int kh = kind == 1 ? hc - a.nh : hc - a.nh - a.nkv;
  const int64_t blk = store ? slot / a.block_size : 0;
  const int off = store ? (int)(slot % a.block_size) : 0, tok = off & 15;
  uint8_t* u = a.cache + ((blk * a.nkv + (store ? kh : 0)) * (a.block_size / 16) + off / 16) * U::kBytes;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    bool odd = false;  // a NaN or an infinity in the group
    float lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float& t = x[j].v[e];
      odd |= !(fabsf(t) < INFINITY);
      t = fminf(fmaxf(t, -kv4::kMaxValue), kv4::kMaxValue);
      lo = fminf(lo, t);
      hi = fmaxf(hi, t);
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    odd = (__ballot_sync(0xffffffffu, odd) >> (lane & 16) & 0xffffu) != 0;
    __half sh = __float2half_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f));
    const float s = __half2float(sh);
    __half ch = __float2half_rn(__fadd_rn(lo, __fmul_rn(8.f, s)));
    const float c = __half2float(ch);
    uint32_t code[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float q = s > 0.f ? __fadd_rn(rintf(__fdiv_rn(__fsub_rn(x[j].v[e], c), s)), 8.f) : 8.f;
      code[e] = odd ? 8u : (uint32_t)fminf(fmaxf(q, 0.f), 15.f);
    }
    if (odd) sh = ch = __ushort_as_half(0x7fff);  // such a group reads back as NaN
    // key words hold 8 dims: two lanes' parts
    uint32_t w = code[0] | code[1] << 16 | code[2] << 4 | code[3] << 20;
    w <<= (lane & 1) * 8;
    w |= __shfl_xor_sync(0xffffffffu, w, 1);
    if (store) {
      const int d = 128 * j + 4 * sl;
      if (kind == 1) {
        if ((lane & 1) == 0) *reinterpret_cast<uint32_t*>(u + U::key_word(tok, d)) = w;
      } else {
        *reinterpret_cast<uint16_t*>(u + U::value_half(tok, d)) =
            (uint16_t)(code[0] | code[1] << 4 | code[2] << 8 | code[3] << 12);
      }
      if ((lane & 15) == 0) *reinterpret_cast<__half2*>(u + U::pair(kind == 2, tok, d >> 6)) = __halves2half2(sh, ch);
    }
  }
  pdl_launch();
}

// ---- gather ----------------------------------------------------------------------------------------
// 4 dims of one token's head per thread (K and V): 8-byte stores, coalesced over the dims.
template <int HD>
__global__ void __launch_bounds__(256) kv4_gather_kernel(Kv4GatherArgs a) {
  using U = Unit<HD>;
  pdl_wait();
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t total = (int64_t)a.N * a.nkv * (HD / 4);
  if (i >= total) return;
  const int d = (int)(i % (HD / 4)) * 4;
  const int64_t th = i / (HD / 4);
  const int h = (int)(th % a.nkv);
  const int64_t slot = a.slots[th / a.nkv];
  float k[4] = {}, v[4] = {};
  if (slot >= 0 && slot < a.cache_blocks * a.block_size) {
    const int off = (int)(slot % a.block_size), tok = off & 15;
    const uint8_t* u =
        a.cache + (((slot / a.block_size) * a.nkv + h) * (a.block_size / 16) + off / 16) * U::kBytes;
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(u + U::key_word(tok, d & ~7)) >> ((d & 4) * 2);
    const uint32_t vw = *reinterpret_cast<const uint16_t*>(u + U::value_half(tok, d));
    const float2 kp = __half22float2(*reinterpret_cast<const __half2*>(u + U::pair(false, tok, d >> 6)));
    const float2 vp = __half22float2(*reinterpret_cast<const __half2*>(u + U::pair(true, tok, d >> 6)));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      k[e] = fmaf(kp.x, (float)((int)(kw >> ((e >> 1) * 4 + (e & 1) * 16) & 15u) - 8), kp.y);
      v[e] = fmaf(vp.x, (float)((int)(vw >> (4 * e) & 15u) - 8), vp.y);
    }
  }
  auto put = [&](uint16_t* dst, const float (&x)[4]) {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(x[0], x[1]), hi = __floats2bfloat162_rn(x[2], x[3]);
    *reinterpret_cast<uint2*>(dst + th * HD + d) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
  };
  if (a.k) put(a.k, k);
  if (a.v) put(a.v, v);
  pdl_launch();
}

}  // namespace

void kv4_plan_launch(const Kv4PlanArgs& a, cudaStream_t s, bool pdl) {
  if (a.S > kPlanMaxSeqs) throw std::runtime_error("kv4 plan: at most 8192 requests");
  const size_t smem = (size_t)2 * a.S * sizeof(int);
  static bool configured = false;
  if (!configured) {
    HK_CUDA_CHECK(cudaFuncSetAttribute(kv4_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       2 * kPlanMaxSeqs * (int)sizeof(int)));
    configured = true;
  }
  const int grid = std::max(1, std::min(148, (a.cap + kPlanRows - 1) / kPlanRows));
  launch(kv4_plan_kernel, dim3(grid), dim3(kPlanThreads), smem, s, pdl, a);
}

void kv4_append_launch(const Kv4AppendArgs& a, cudaStream_t s, bool pdl) {
  if (a.R <= 0) return;
  const int hpw = a.hd == 64 ? 2 : 1, heads = a.nh + 2 * a.nkv;
  const int64_t units = (int64_t)a.R * ((heads + hpw - 1) / hpw);
  const dim3 grid((unsigned)((units + 7) / 8));
  switch (a.hd) {
    case 64: launch(kv4_append_kernel<64>, grid, dim3(256), 0, s, pdl, a); break;
    case 128: launch(kv4_append_kernel<128>, grid, dim3(256), 0, s, pdl, a); break;
    case 256: launch(kv4_append_kernel<256>, grid, dim3(256), 0, s, pdl, a); break;
    default: throw std::runtime_error("kv4 append: head_dim 64, 128 or 256");
  }
}

void kv4_gather_launch(const Kv4GatherArgs& a, cudaStream_t s, bool pdl) {
  if (a.N <= 0) return;
  const int64_t n = (int64_t)a.N * a.nkv * (a.hd / 4);
  const dim3 grid((unsigned)((n + 255) / 256));
  switch (a.hd) {
    case 64: launch(kv4_gather_kernel<64>, grid, dim3(256), 0, s, pdl, a); break;
    case 128: launch(kv4_gather_kernel<128>, grid, dim3(256), 0, s, pdl, a); break;
    case 256: launch(kv4_gather_kernel<256>, grid, dim3(256), 0, s, pdl, a); break;
    default: throw std::runtime_error("kv4 gather: head_dim 64, 128 or 256");
  }
}

}  // namespace hk
