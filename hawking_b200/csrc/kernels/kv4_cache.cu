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
// Latency bounds it: 64 requests of one token take 6 us, 512 requests of which 64 bring 16 to 1024 tokens 10 us with
// cold caches, for two scans and three dependent reads. So every CTA scans all requests by itself, and a launch has no
// second phase.
constexpr int kPlanThreads = 512;
constexpr int kPlanRows = 2048;    // rows per CTA
constexpr int kPlanMaxSeqs = 8192;  // both scans in shared memory

// blocks that n >= 0 tokens take (n may be near 2^31: no n + bs - 1)
__device__ __forceinline__ int blocks_of(int n, int bs) { return n / bs + (n % bs != 0); }

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
    const int nd = n > 0 ? blocks_of(c + n, bs) - blocks_of(c, bs) : 0;
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
      const int col = pos / bs, b0 = blocks_of(c, bs);
      int blk;
      if (take && col >= b0) {
        const long long j = (long long)base[i] + col - b0;
        blk = j < a.n_free ? a.free_blocks[j] : -1;
      } else {
        blk = a.tables[(int64_t)seq * a.max_blocks + col];
      }
      // no block, or one whose slots no int32 holds: the row's keys and values have no place
      const long long at = (long long)blk * bs + pos % bs;
      if (blk >= 0 && at <= kTop) slot = (int)at;
      else set_error(a.status, HK_ERR_BAD_ARG);
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
      a.tables[(int64_t)a.seq_rows[i] * a.max_blocks + blocks_of(a.cached[i], bs) + j - base[i]] = a.free_blocks[j];
    }
  }
  if (blockIdx.x == 0 && tid == 0) {
    const bool over = total > a.cap || (take && total_need > a.n_free);
    if (a.taken) *a.taken = take ? (int)min(total_need, (long long)a.n_free) : 0;
    if (any_bad || over) set_error(a.status, HK_ERR_BAD_ARG);
  }
}

// ---- RoPE + quantise + append ----------------------------------------------------------------------
// A warp takes HB heads of one row (HB pairs of heads at HD 64), so that the position's rotation is read once
// for them and all their loads are in flight together: at 2048 rows of 48 heads of 128 in the L2 cache HB = 4 took
// 17 us, 2 took 21, 1 took 31. A few rows keep one head per warp (the launch needs warps more than the warps work).
// 2048 rows of 32 / 8 heads of 128 took 20 us (70 MB: 11): issue slots 63 % busy, the ALU 45 %, and 30 % of a warp's time
// waiting for loads that nothing overlaps, at the half occupancy of 60 registers.
// An instance per rotation style, with and without bias and norms: deciding both in the kernel took 25 us instead of 17
// in the L2 cache. Codes come from a reciprocal, with the exact division only near half-way between two codes.
// Every lane holds 4 consecutive dims of each 128 (or 64), 16 lanes the 64 dims of a quantisation group.
// Sums, products and divisions are rounded one by one, the norm's sum of squares in a fixed order,
// so the bytes written do not depend on how the compiler contracts them.
struct Vec4 {
  float v[4];
};
__device__ __forceinline__ Vec4 ld4(const float* p) {
  const float4 f = *reinterpret_cast<const float4*>(p);
  return {{f.x, f.y, f.z, f.w}};
}

// minimum and maximum that keep a NaN
__device__ __forceinline__ float min_nan(float x, float y) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float max_nan(float x, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <int HD, int HB, int STYLE, bool EXTRA>
__global__ void __launch_bounds__(128) kv4_append_kernel(Kv4AppendArgs a) {
  constexpr int LG = HD < 128 ? HD / 4 : 32;  // lanes of one head
  constexpr int HPW = 32 / LG;                // heads side by side in a warp
  constexpr int NV = HD / (4 * LG);           // vectors of 4 dims per lane
  using U = Unit<HD>;
  pdl_wait();
  const int lane = threadIdx.x & 31, sl = lane % LG;
  const int heads = a.nh + 2 * a.nkv, per_row = (heads + HPW * HB - 1) / (HPW * HB);
  const int r = blockIdx.x, unit = (gridDim.y - 1 - blockIdx.y) * 4 + (threadIdx.x >> 5);
  if (unit >= per_row) return;  // (the last heads, keys and values, first: they take longest)
  const int h0 = unit * (HPW * HB) + lane / LG;
  const float* row = a.qkv + (int64_t)r * a.qkv_stride;
  Vec4 x[HB][NV];
#pragma unroll
  for (int b = 0; b < HB; ++b)
#pragma unroll
    for (int j = 0; j < NV; ++j)  // (lanes without a head compute on the last one and store nothing)
      x[b][j] = ld4(row + (int64_t)min(h0 + b * HPW, heads - 1) * HD + 128 * j + 4 * sl);
  const int pos = a.positions[r];
  if (pos < 0 || pos >= a.rope_rows) return;  // the whole warp
  int64_t slot = -1;
  if (__any_sync(0xffffffffu, h0 + (HB - 1) * HPW >= a.nh)) {  // keys or values among the heads
    if (a.slots) {
      slot = a.slots[r];
    } else {
      const int seq = a.row_seq[r], col = pos / a.block_size;
      if (seq >= 0 && seq < a.table_rows && col < a.max_blocks)
        slot = (int64_t)a.block_tables[(int64_t)seq * a.max_blocks + col] * a.block_size + pos % a.block_size;
    }
  }
  const bool keep = slot >= 0 && slot < a.cache_blocks * a.block_size;
  int blk = 0, off = 0;
  if (keep) {
    blk = (int)slot / a.block_size;  // (the pool holds less than 2^31 tokens)
    off = (int)slot - blk * a.block_size;
  }
  const int tok = off & 15;
  // this lane's rotations: adjacent pairs, or halves (cos, sin of dims d and, with the sign, their partners)
  const int half = a.rot_dim / 2;
  const float* rope = a.rope + (int64_t)pos * a.rot_dim;
  float cs[NV][4], sn[NV][4];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = 128 * j + 4 * sl + e;
      cs[j][e] = 1.f;
      sn[j][e] = 0.f;
      if (d < a.rot_dim) {
        const int i = STYLE == 0 ? d >> 1 : (d < half ? d : d - half);
        const float2 t = *reinterpret_cast<const float2*>(rope + 2 * i);
        cs[j][e] = t.x;
        sn[j][e] = t.y;
      }
    }
#pragma unroll
  for (int b = 0; b < HB; ++b) {
    const int h = h0 + b * HPW;
    const bool live = h < heads;
    const int hc = min(h, heads - 1);
    const int kind = hc < a.nh ? 0 : (hc < a.nh + a.nkv ? 1 : 2);  // q, k, v
    const float* src = row + (int64_t)hc * HD;
    const float* bias = EXTRA && a.bias ? a.bias + (int64_t)hc * HD : nullptr;
    const float* nw = !EXTRA ? nullptr : kind == 0 ? a.q_norm : (kind == 1 ? a.k_norm : nullptr);
    Vec4(&v)[NV] = x[b];
    if (bias) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[j].v[e] = __fadd_rn(v[j].v[e], bias[128 * j + 4 * sl + e]);
    }
    float inv = 1.f;
    if (EXTRA && (a.q_norm || a.k_norm)) {  // (the same for the warp)
      float ss[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ss[e] = __fmul_rn(v[0].v[e], v[0].v[e]);
#pragma unroll
        for (int j = 1; j < NV; ++j) ss[e] = __fadd_rn(ss[e], __fmul_rn(v[j].v[e], v[j].v[e]));
      }
      // 64 dims in halves all the way down, more dims four in a row and then in halves
      float sum;
      if (HD == 64) {
#pragma unroll
        for (int o = LG / 2; o > 0; o >>= 1)
#pragma unroll
          for (int e = 0; e < 4; ++e) ss[e] = __fadd_rn(ss[e], __shfl_xor_sync(0xffffffffu, ss[e], o));
        sum = __fadd_rn(__fadd_rn(ss[0], ss[2]), __fadd_rn(ss[1], ss[3]));
      } else {
        sum = __fadd_rn(__fadd_rn(__fadd_rn(ss[0], ss[1]), ss[2]), ss[3]);
#pragma unroll
        for (int o = LG / 2; o > 0; o >>= 1) sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, o));
      }
      if (nw) {
        inv = rsqrtf(__fadd_rn(__fmul_rn(sum, 1.f / HD), a.eps));
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[j].v[e] = __fmul_rn(__fmul_rn(v[j].v[e], inv), nw[128 * j + 4 * sl + e]);
      }
    }
    if (STYLE == 1 && a.rot_dim == HD) {  // pairs (d, d + half), in two lanes or in two vectors of one
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float y[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j)  // (the two heads of a warp may be of two kinds: all lanes shuffle)
          y[j] = NV == 1 ? __shfl_xor_sync(0xffffffffu, v[0].v[e], LG / 2) : v[NV - 1 - j].v[e];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const float p = __fmul_rn(v[j].v[e], cs[j][e]), q = __fmul_rn(y[j], sn[j][e]);
          if (kind < 2) v[j].v[e] = 128 * j + 4 * sl < half ? __fsub_rn(p, q) : __fadd_rn(q, p);
        }
      }
    } else if (kind < 2) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int d0 = 128 * j + 4 * sl;
        if (STYLE == 0) {  // pairs (d, d + 1)
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            if (d0 + e < a.rot_dim) {
              const float p = v[j].v[e], q = v[j].v[e + 1];
              v[j].v[e] = __fsub_rn(__fmul_rn(p, cs[j][e]), __fmul_rn(q, sn[j][e]));
              v[j].v[e + 1] = __fadd_rn(__fmul_rn(p, sn[j][e]), __fmul_rn(q, cs[j][e]));
            }
          }
        } else {  // pairs (d, d + half): the partner is read again (an L1 hit), normalised alike
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int d = d0 + e;
            if (d < a.rot_dim) {
              const bool first = d < half;
              const int o = first ? d + half : d - half;
              float y = src[o];
              if (bias) y = __fadd_rn(y, bias[o]);
              if (nw) y = __fmul_rn(__fmul_rn(y, inv), nw[o]);
              v[j].v[e] = first ? __fsub_rn(__fmul_rn(v[j].v[e], cs[j][e]), __fmul_rn(y, sn[j][e]))
                                : __fadd_rn(__fmul_rn(y, sn[j][e]), __fmul_rn(v[j].v[e], cs[j][e]));
            }
          }
        }
      }
    }
    if (kind == 0 && live) {
      uint16_t* dst = a.q_out + (int64_t)r * a.q_stride + (int64_t)h * HD;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(v[j].v[0], v[j].v[1]);
        const __nv_bfloat162 hi = __floats2bfloat162_rn(v[j].v[2], v[j].v[3]);
        *reinterpret_cast<uint2*>(dst + 128 * j + 4 * sl) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
      }
    }
    if (!__any_sync(0xffffffffu, kind != 0 && live && keep)) continue;
    const bool store = live && kind != 0 && keep;
    const int kh = kind == 0 ? 0 : (kind == 1 ? hc - a.nh : hc - a.nh - a.nkv);
    uint8_t* u = a.cache + (((int64_t)blk * a.nkv + kh) * (a.block_size / 16) + off / 16) * U::kBytes;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float lo = min_nan(min_nan(v[j].v[0], v[j].v[1]), min_nan(v[j].v[2], v[j].v[3]));
      float hi = max_nan(max_nan(v[j].v[0], v[j].v[1]), max_nan(v[j].v[2], v[j].v[3]));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      }
      const bool odd = !(lo > -INFINITY && hi < INFINITY);  // a NaN or an infinity in the group
      if (lo < -kv4::kMaxValue || hi > kv4::kMaxValue) {
        lo = fminf(fmaxf(lo, -kv4::kMaxValue), kv4::kMaxValue);
        hi = fminf(fmaxf(hi, -kv4::kMaxValue), kv4::kMaxValue);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[j].v[e] = fminf(fmaxf(v[j].v[e], -kv4::kMaxValue), kv4::kMaxValue);
      }
      __half sh = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f));
      const float s = __half2float(sh);
      __half ch = __float2half_rn(__fadd_rn(lo, __fmul_rn(8.f, s)));
      const float c = __half2float(ch);
      // round((x - c) / s): by the reciprocal, whose product is off by less than 3e-6 where it matters (up to 8), and by
      // the division where that product is within 1e-5 of a half. Adding kRound leaves code = round + 8 in the last bits.
      constexpr float kRound = 12582912.f + 8.f;
      const float rs = s > 0.f ? rcp(s) : 0.f;
      uint32_t code[4];
      bool half_way = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float q = fminf(fmaxf(__fmul_rn(__fsub_rn(v[j].v[e], c), rs), -8.f), 7.f);
        const float t = __fadd_rn(q, kRound);
        half_way |= fabsf(__fsub_rn(q, __fsub_rn(t, kRound))) > 0.49999f;
        code[e] = __float_as_uint(t) & 15u;
      }
      if (half_way) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          code[e] = __float_as_uint(__fadd_rn(fminf(fmaxf(__fdiv_rn(__fsub_rn(v[j].v[e], c), s), -8.f), 7.f), kRound)) & 15u;
      }
      if (odd) sh = ch = __ushort_as_half(0x7fff);  // such a group reads back as NaN, its codes as 8
      // key words hold 8 dims: two lanes' parts
      uint32_t w = odd ? 0x00880088u : code[0] | code[1] << 16 | code[2] << 4 | code[3] << 20;
      const uint32_t vw = odd ? 0x8888u : code[0] | code[1] << 4 | code[2] << 8 | code[3] << 12;
      w <<= (lane & 1) * 8;
      w |= __shfl_xor_sync(0xffffffffu, w, 1);
      if (store) {
        const int d = 128 * j + 4 * sl;
        if (kind == 1) {
          if ((lane & 1) == 0) *reinterpret_cast<uint32_t*>(u + U::key_word(tok, d)) = w;
        } else {
          *reinterpret_cast<uint16_t*>(u + U::value_half(tok, d)) = (uint16_t)vw;
        }
        if ((lane & 15) == 0) *reinterpret_cast<__half2*>(u + U::pair(kind == 2, tok, d >> 6)) = __halves2half2(sh, ch);
      }
    }
  }
  pdl_launch();
}

// ---- gather ----------------------------------------------------------------------------------------
// A warp takes 16 slots of one head. Where they are the 16 tokens of a unit in order, as a sequence's slots
// are, it reads the unit whole, in its own order: a lane's 16 bytes of key codes are 4 x 8 dims of a token, its
// 16 bytes of value codes 2 x 4 dims of four tokens, so loads and stores are whole sectors. 65536 slots of 8 heads
// of 128 (344 MB, most of it written) took 60 us this way, 5.7 TB/s and bound by the memory; token by token, 4 dims
// per lane, as any other slots go, 128 us.
__device__ __forceinline__ uint32_t bf16_pair(uint32_t codes, float2 p) {  // centred codes (float16 pair), (s, c)
  const float2 n = __half22float2(*reinterpret_cast<const __half2*>(&codes));
  const __nv_bfloat162 v = __floats2bfloat162_rn(fmaf(p.x, n.x, p.y), fmaf(p.x, n.y, p.y));
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <int HD>
__global__ void __launch_bounds__(256) kv4_gather_kernel(Kv4GatherArgs a) {
  using U = Unit<HD>;
  constexpr int GR = HD / 64;
  pdl_wait();
  const int lane = threadIdx.x & 31;
  if (blockIdx.y == 0) a.v = nullptr;  // keys and values by different warps: short lists are a matter of latency
  else a.k = nullptr;
  const int64_t task = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int64_t groups = (a.N + 15) / 16;
  if (task >= groups * a.nkv) return;
  const int64_t i0 = task / a.nkv * 16;
  const int h = (int)(task % a.nkv), n = (int)min((int64_t)16, a.N - i0);
  const int64_t pool = a.cache_blocks * a.block_size;
  const int mine = lane < n ? a.slots[i0 + lane] : -1;
  const int first = __shfl_sync(0xffffffffu, mine, 0);
  const bool run = __all_sync(0xffffffffu, lane >= n || mine == first + lane) && n == 16 && first >= 0 &&
                   (first & 15) == 0 && first < pool;
  if (run) {
    const int blk = first / a.block_size, off = first - blk * a.block_size;
    const uint8_t* u = a.cache + (((int64_t)blk * a.nkv + h) * (a.block_size / 16) + off / 16) * U::kBytes;
    const int64_t out = (i0 * a.nkv + h) * HD;
    const int64_t step = (int64_t)a.nkv * HD;  // to the next token's row
    if (a.k) {
      constexpr int W = HD < 128 ? 2 : 4;  // words of a token in a plane
#pragma unroll
      for (int pl = 0; pl < (HD + 127) / 128; ++pl)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int tok = 8 * x + (lane >> 2), t = lane & 3;
          const uint8_t* src = u + pl * 16 * U::kRow + tok * U::kRow + t * (U::kRow / 4);
          uint32_t w[4];
          if (W == 4) {
            const uint4 y = __ldg(reinterpret_cast<const uint4*>(src));
            w[0] = y.x, w[1] = y.y, w[2] = y.z, w[3] = y.w;
          } else {
            const uint2 y = __ldg(reinterpret_cast<const uint2*>(src));
            w[0] = y.x, w[1] = y.y;
          }
#pragma unroll
          for (int i = 0; i < W; ++i) {
            const int grp = pl * 2 + i / 2;
            const float2 p = __half22float2(__ldg(reinterpret_cast<const __half2*>(u + U::pair(false, tok, grp))));
            uint4 v;
            v.x = bf16_pair(kv4::centre_even(w[i]), p);
            v.y = bf16_pair(kv4::centre_odd(w[i]), p);
            v.z = bf16_pair(kv4::centre_even(w[i] >> 8), p);
            v.w = bf16_pair(kv4::centre_odd(w[i] >> 8), p);
            *reinterpret_cast<uint4*>(a.k + out + tok * step + pl * 128 + 32 * i + 8 * t) = v;
          }
        }
    }
    if (a.v) {
      const int g = lane >> 2, t = lane & 3;
#pragma unroll
      for (int grp = 0; grp < GR; ++grp) {
        const uint4 y = __ldg(reinterpret_cast<const uint4*>(u + U::kCodes + grp * 512 + lane * 16));
        const uint32_t w[2][2] = {{y.x, y.y}, {y.z, y.w}};  // [32 dims][8 tokens]
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int tok = 8 * hh + 2 * t;
          const float2 p0 = __half22float2(__ldg(reinterpret_cast<const __half2*>(u + U::pair(true, tok, grp))));
          const float2 p1 = __half22float2(__ldg(reinterpret_cast<const __half2*>(u + U::pair(true, tok + 1, grp))));
#pragma unroll
          for (int il = 0; il < 2; ++il) {
            uint32_t c[4] = {kv4::centre_even(w[il][hh]), kv4::centre_odd(w[il][hh]), kv4::centre_even(w[il][hh] >> 8),
                             kv4::centre_odd(w[il][hh] >> 8)};  // dims 0 .. 3 of both tokens
            uint16_t* dst = a.v + out + tok * step + grp * 64 + 32 * il + 4 * g;
            *reinterpret_cast<uint2*>(dst) =
                make_uint2(bf16_pair(__byte_perm(c[0], c[1], 0x5410), p0), bf16_pair(__byte_perm(c[2], c[3], 0x5410), p0));
            *reinterpret_cast<uint2*>(dst + step) =
                make_uint2(bf16_pair(__byte_perm(c[0], c[1], 0x7632), p1), bf16_pair(__byte_perm(c[2], c[3], 0x7632), p1));
          }
        }
      }
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      const int64_t slot = __shfl_sync(0xffffffffu, mine, i);
      const int64_t out = ((i0 + i) * a.nkv + h) * HD;
#pragma unroll 1
      for (int d = 4 * lane; d < HD; d += 128) {
        uint2 k = make_uint2(0u, 0u), v = k;
        if (slot >= 0 && slot < pool) {
          const int off = (int)(slot % a.block_size), tok = off & 15;
          const uint8_t* u =
              a.cache + (((slot / a.block_size) * a.nkv + h) * (a.block_size / 16) + off / 16) * U::kBytes;
          const uint32_t kw = *reinterpret_cast<const uint32_t*>(u + U::key_word(tok, d & ~7)) >> ((d & 4) * 2);
          const uint32_t vw = *reinterpret_cast<const uint16_t*>(u + U::value_half(tok, d));
          const float2 kp = __half22float2(*reinterpret_cast<const __half2*>(u + U::pair(false, tok, d >> 6)));
          const float2 vp = __half22float2(*reinterpret_cast<const __half2*>(u + U::pair(true, tok, d >> 6)));
          k = make_uint2(bf16_pair(kv4::centre_even(kw), kp), bf16_pair(kv4::centre_odd(kw), kp));
          const uint32_t c[4] = {kv4::centre_even(vw), kv4::centre_odd(vw), kv4::centre_even(vw >> 8), kv4::centre_odd(vw >> 8)};
          v = make_uint2(bf16_pair(__byte_perm(c[0], c[1], 0x5410), vp), bf16_pair(__byte_perm(c[2], c[3], 0x5410), vp));
        }
        if (a.k) *reinterpret_cast<uint2*>(a.k + out + d) = k;
        if (a.v) *reinterpret_cast<uint2*>(a.v + out + d) = v;
      }
    }
  }
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

template <int HD, int HB>
static void launch_append(const Kv4AppendArgs& a, cudaStream_t s, bool pdl) {
  const int per_warp = (HD == 64 ? 2 : 1) * HB, warps = (a.nh + 2 * a.nkv + per_warp - 1) / per_warp;
  const bool extra = a.bias || a.q_norm || a.k_norm;
  const auto kernel = a.rope_style == 0 ? (extra ? kv4_append_kernel<HD, HB, 0, true> : kv4_append_kernel<HD, HB, 0, false>)
                                        : (extra ? kv4_append_kernel<HD, HB, 1, true> : kv4_append_kernel<HD, HB, 1, false>);
  launch(kernel, dim3(a.R, (warps + 3) / 4), dim3(128), 0, s, pdl, a);
}

void kv4_append_launch(const Kv4AppendArgs& a, cudaStream_t s, bool pdl) {
  if (a.R <= 0) return;
  // several heads per warp once one head each would make 80 warps per SM: 256 rows of 48 heads of 128 took 6.5 us with 4
  // heads per warp and 6.6 with one, 384 rows 6.5 and 8.6, 128 rows 6.4 and 5.9
  const bool many = (int64_t)a.R * (a.nh + 2 * a.nkv) >= 148 * 80;
  switch (a.hd) {
    case 64: many ? launch_append<64, 4>(a, s, pdl) : launch_append<64, 1>(a, s, pdl); break;
    case 128: many ? launch_append<128, 4>(a, s, pdl) : launch_append<128, 1>(a, s, pdl); break;
    case 256: many ? launch_append<256, 2>(a, s, pdl) : launch_append<256, 1>(a, s, pdl); break;
    default: throw std::runtime_error("kv4 append: head_dim 64, 128 or 256");
  }
}

void kv4_gather_launch(const Kv4GatherArgs& a, cudaStream_t s, bool pdl) {
  if (a.N <= 0) return;
  const int64_t tasks = (int64_t)((a.N + 15) / 16) * a.nkv;
  const dim3 grid((unsigned)((tasks + 7) / 8), 2);
  switch (a.hd) {
    case 64: launch(kv4_gather_kernel<64>, grid, dim3(256), 0, s, pdl, a); break;
    case 128: launch(kv4_gather_kernel<128>, grid, dim3(256), 0, s, pdl, a); break;
    case 256: launch(kv4_gather_kernel<256>, grid, dim3(256), 0, s, pdl, a); break;
    default: throw std::runtime_error("kv4 gather: head_dim 64, 128 or 256");
  }
}

}  // namespace hk
