// Decode attention over the 4-bit paged KV cache on the tensor cores.
//
// Mathematics. With keys k = ck + sk (n - 8) and values v = cv + sv (m - 8) (codes n, m; one pair
// (s, c) per token and 64 dims), a row's score is
//     S = sum over groups [ sk (q . n) + (ck - 8 sk) sum(q) ]
// and its output, with p = exp(S - R) for a running reference R,
//     o = [ 2^E sum_t (p sv 2^-E) (m - 8) + sum_t p cv ] / sum_t p.
// So the matrix instructions multiply the codes themselves. Keys: the nibbles of a word, masked, are
// the float16 subnormals n 2^-24 (and 16 n 2^-24 for the odd nibbles, against a query divided by
// 16): exact, one AND per pair of operands. Values: centred codes m - 8 are exact float16, so that
// long sums do not carry a bias. The query is float16 after an exact power-of-two scaling of each
// head; the weights p sv 2^-E are rounded to float16 (E: the largest exponent of sv so far, so they
// stay below 2^8); everything else is fp32.
//
// Layout. Scores are computed transposed, S^T = K Q^T (mma.m16n8k16: 16 tokens x 8 heads), so the
// up to 8 query heads of a kv head fill the narrow side and one instruction takes 256 codes; the
// weights become the operand of O^T = V^T P^T by movmatrix. The running reference moves only when a
// score exceeds it by 2^7 (weights of up to 128 are fine in float16): one vote per tile instead of a
// reduction, and every lane sums its own tokens' weights until the end of a segment.
//
// Work. The (row, kv head) pairs' units of 16 tokens form one sequence that is cut into equal ranges,
// one per CTA (at least kMinUnits long), and each range into equal parts, one per warp: ragged batches
// and single long rows load every warp alike, and a warp needs nobody inside its part. A pair that lies
// in one part is written out by its warp; one that spans warps is merged in shared memory at the end
// of the CTA; one that spans CTAs leaves partials (reference, sum, output), merged in CTA order by the
// last CTA to arrive (groups of kTree CTAs first, where there are many).
#include "kv4.cuh"
#include "sm100.cuh"

namespace hk {
namespace {

using kv4::Unit;
using sm100::smem_u32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kStages = 2;     // tiles in a warp's ring
constexpr int kTree = 8;       // CTAs whose partials are merged first
constexpr float kHead = 7.f;   // log2 of how far a score may exceed the reference

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8 x 8 transpose of 16-bit elements held as rows of the fragment layout
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// centred codes of the even (0x000f000f) and odd (0x00f000f0) nibbles as float16 pairs
__device__ __forceinline__ uint32_t centre_even(uint32_t w) {
  const uint32_t x = (w & 0x000f000fu) | 0x64006400u;  // 1024 + m
  const uint32_t k = 0xe408e408u;                      // -1032
  const __half2 r = __hadd2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&k));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t centre_odd(uint32_t w) {
  const uint32_t x = (w & 0x00f000f0u) | 0x64006400u;              // 1024 + 16 m
  const uint32_t s = 0x2c002c00u, k = 0xd480d480u;                 // 1 / 16, -72
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&s),
                            *reinterpret_cast<const __half2*>(&k));
  return *reinterpret_cast<const uint32_t*>(&r);
}

struct DecodeArgs {
  Kv4AttnArgs a;
  int heads_per_item, splits;  // query heads of one item, items per kv head
  int upb_shift;               // log2 of the units per block, or -1
  float* part;                 // [grid][2][heads_per_item * (HD + 4)]
  int* counters;               // [3 * grid], zero between launches
};

constexpr int kMaxRows = 512;  // rows of one launch

template <int HD, int NT>
struct DecodeShape {
  static constexpr int kWarps = NT == 1 && HD <= 128 ? 8 : 4;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kPerSm = NT == 1 && HD <= 128 ? 2 : HD * NT <= 256 ? 3 : 2;  // CTAs, by registers
  static constexpr int kTile = 256 / HD;                                           // units per stage (4608 bytes)
  static constexpr int kStageBytes = kTile * Unit<HD>::kBytes;
  static constexpr int kRow = HD + 4;  // floats of one head's partial: output, reference, sum
  static constexpr int kRing = kStages * kStageBytes;
  // per warp: the ring (whose place the part's last partial takes) and the first partial
  static size_t warp_bytes(int heads) { return kRing + (size_t)heads * kRow * 4; }
  static size_t smem(int heads) { return kWarps * warp_bytes(heads); }
  static_assert(8 * NT * kRow * 4 <= kRing, "the last partial fits the ring");
};

// One partial of a pair: the CTA's own in shared memory, a CTA's in global memory.
struct Part {
  int row, item, u0, u1;  // row < 0: none
};

template <int HD, int NT>
__global__ void __launch_bounds__(DecodeShape<HD, NT>::kThreads, DecodeShape<HD, NT>::kPerSm)
    kv4_decode_kernel(DecodeArgs g_) {
  using U = Unit<HD>;
  using Sh = DecodeShape<HD, NT>;
  constexpr int GR = HD / 64, KT = HD / 16, TU = Sh::kTile, kWarps = Sh::kWarps, kThreads = Sh::kThreads;
  constexpr int kMinUnits = kWarps;
  const Kv4AttnArgs& a = g_.a;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[kWarps][kStages];
  __shared__ long long before[kMaxRows + 1];  // units of the rows before each row
  __shared__ long long wsum[kWarps];
  __shared__ Part parts[2 * kWarps];
  __shared__ int last_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int fg = lane >> 2, ft = lane & 3;
  const int G = a.nh / a.nkv, items = a.nkv * g_.splits, HPI = g_.heads_per_item;
  const int upb = a.block_size / 16;
  const int wbytes = Sh::kRing + HPI * Sh::kRow * 4;
  uint8_t* ring = smem + warp * wbytes;
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) sm100::mbar_init(&full[warp][s], 1);
    sm100::fence_barrier_init();
    parts[2 * warp].row = parts[2 * warp + 1].row = -1;
  }
  pdl_wait();

  // ---- work: scan of the rows' units ----
  const auto row_len = [&](int r, bool report) {
    const int seq = a.row_seq[r], ctx = a.row_ctx[r];
    if (seq < 0 || seq >= a.table_rows) {
      if (report) set_error(a.status, HK_ERR_BAD_ARG);
      return 0;
    }
    return min(max(ctx, 0), a.max_blocks * a.block_size);
  };
  {
    const int per = (a.R + kThreads - 1) / kThreads;
    const int r0 = min(a.R, tid * per), r1 = min(a.R, r0 + per);
    long long sum = 0;
    for (int r = r0; r < r1; ++r) {
      const int n = (row_len(r, blockIdx.x == 0) + 15) >> 4;
      before[r + 1] = n;
      sum += n;
    }
    long long inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) wsum[warp] = inc;
    if (tid == 0) before[0] = 0;
    __syncthreads();
    long long base = inc - sum;
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
      if (w < warp) base += wsum[w];
    for (int r = r0; r < r1; ++r) {
      base += before[r + 1];
      before[r + 1] = base;
    }
    __syncthreads();
  }
  const long long total = before[a.R] * items;
  const int N = (int)min((long long)gridDim.x, max(1ll, (total + kMinUnits - 1) / kMinUnits));
  const int cta = blockIdx.x;
  // rows without context
  for (int r = cta; r < a.R; r += gridDim.x)
    if (before[r + 1] == before[r])
      for (int i = tid; i < a.nh * HD; i += kThreads) {
        if (a.out_bf16) a.out_bf16[r * a.out_stride + i] = 0;
        if (a.out) a.out[r * a.outf_stride + i] = 0.f;
      }
  if (cta >= N || total == 0) return;
  const long long w0 = total * cta / N, w1 = total * (cta + 1) / N;
  const long long p0 = w0 + (w1 - w0) * warp / kWarps, p1 = w0 + (w1 - w0) * (warp + 1) / kWarps;

  // ---- cursor over the pairs of this warp's part [p0, p1) ----
  struct Cursor {
    int row, item, u, units;
    long long left;  // units of the part still to come
  };
  Cursor cc;
  {
    int lo = 0, hi = a.R;  // last row with before * items <= p0
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (before[mid] * items <= p0) lo = mid;
      else hi = mid;
    }
    cc.row = lo;
    cc.units = (int)(before[lo + 1] - before[lo]);
    const long long off = p0 - before[lo] * items;
    cc.item = cc.units ? (int)(off / cc.units) : 0;
    cc.u = (int)(off - (long long)cc.item * cc.units);
    cc.left = p1 - p0;
  }
  const auto next_pair = [&](Cursor& c) {  // only while units are left
    c.u = 0;
    if (++c.item == items) {
      c.item = 0;
      do ++c.row;
      while (before[c.row + 1] == before[c.row]);
      c.units = (int)(before[c.row + 1] - before[c.row]);
    }
  };

  // ---- producer: the part's tiles in order, kStages ahead ----
  Cursor pc = cc;
  int p_stage = 0, blk = 0, pos = 0;  // this lane's block and unit in the block, of the next tile
  const uint8_t* p_head = nullptr;    // the pair's kv head in block 0
  const int* p_table = nullptr;
  const int64_t blk_bytes = (int64_t)a.nkv * upb * U::kBytes;
  const auto pair_base = [&]() {
    p_head = a.cache + (int64_t)(pc.item / g_.splits) * upb * U::kBytes;
    p_table = a.block_tables + (int64_t)a.row_seq[pc.row] * a.max_blocks;
  };
  const auto fetch = [&]() {  // block ids of the next tile's units, one per lane
    const int u = pc.u + lane;
    if (lane < TU && u < pc.units) {
      const int b = g_.upb_shift >= 0 ? u >> g_.upb_shift : u / upb;
      pos = u - b * upb;
      blk = p_table[b];
    }
  };
  const auto produce = [&]() {
    if (pc.left <= 0) return;
    uint8_t* dst = ring + p_stage * Sh::kStageBytes + lane * U::kBytes;
    uint64_t* bar = &full[warp][p_stage];
    const int n = (int)min((long long)min(TU, pc.units - pc.u), pc.left);
    const bool mine = lane < n, good = mine && blk >= 0 && blk < a.cache_blocks;
    const unsigned m = __ballot_sync(0xffffffffu, good);
    if (mine && !good) {  // a block outside the cache reads as zeros
      set_error(a.status, HK_ERR_BAD_ARG);
      for (int i = 0; i < U::kBytes; i += 16) *reinterpret_cast<uint4*>(dst + i) = make_uint4(0u, 0u, 0u, 0u);
      sm100::fence_proxy_async_smem();
    }
    if (lane == 0) sm100::mbar_arrive_expect_tx(bar, __popc(m) * U::kBytes);
    __syncwarp();
    if (good) sm100::bulk_g2s(dst, p_head + blk * blk_bytes + pos * U::kBytes, U::kBytes, bar);
    p_stage = p_stage + 1 == kStages ? 0 : p_stage + 1;
    pc.u += n;
    pc.left -= n;
    if (pc.left > 0) {
      if (pc.u == pc.units) {
        next_pair(pc);
        pair_base();
      }
      fetch();
    }
  };
  if (pc.left > 0) {
    pair_base();
    fetch();
  }
#pragma unroll
  for (int s = 0; s < kStages; ++s) produce();

  // ---- consumer ----
  int c_stage = 0, c_phase = 0;
  bool first_pair = true;
  while (cc.left > 0) {
    const int u_first = cc.u, kvh = cc.item / g_.splits, h0 = kvh * G + (cc.item % g_.splits) * HPI;
    const int heads = min(HPI, kvh * G + G - h0);
    const int len = row_len(cc.row, false);
    // queries: B fragments (dims x 8 heads), float16 after a power-of-two scaling of each head
    uint32_t qf[NT][KT][2];
    float mult[NT][2], qsum[NT][2][GR];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      uint4 raw[HD / 32];
      const int h = nt * 8 + fg;
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) {
        raw[i] = make_uint4(0u, 0u, 0u, 0u);
        if (h < heads)
          raw[i] = *reinterpret_cast<const uint4*>(a.q + cc.row * a.q_stride + (int64_t)(h0 + h) * HD + 32 * i + 8 * ft);
      }
      float mx = 0.f, qs[GR];
#pragma unroll
      for (int grp = 0; grp < GR; ++grp) qs[grp] = 0.f;
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) {
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float lo = __uint_as_float(w[j] << 16), hi = __uint_as_float(w[j] & 0xffff0000u);
          mx = fmaxf(mx, fmaxf(fabsf(lo), fabsf(hi)));
          qs[i / 2] += lo + hi;
        }
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      // 2^-e with 1 <= mx 2^-e < 2 (1 for a zero, subnormal or non-finite head)
      const int ex = (int)(__float_as_uint(mx) >> 23);
      const float down = ex > 0 && ex < 254 ? __uint_as_float((uint32_t)(254 - ex) << 23) : 1.f;
      // 2^24 of the subnormal codes, less the 16 of the query
      const float up = (ex > 0 && ex < 254 ? __uint_as_float((uint32_t)ex << 23) : 1.f) * (a.scale * kLog2e * 1048576.f);
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) {
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float lo = __uint_as_float(w[j] << 16) * down, hi = __uint_as_float(w[j] & 0xffff0000u) * down;
          const float f = j & 1 ? 1.f : 16.f;  // the odd nibbles' codes come 16 times larger
          qf[nt][2 * i + j / 2][j & 1] = pack_f16(lo * f, hi * f);
        }
      }
#pragma unroll
      for (int grp = 0; grp < GR; ++grp) {
        qs[grp] += __shfl_xor_sync(0xffffffffu, qs[grp], 1);
        qs[grp] += __shfl_xor_sync(0xffffffffu, qs[grp], 2);
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        mult[nt][c] = __shfl_sync(0xffffffffu, up, (2 * ft + c) * 4);
#pragma unroll
        for (int grp = 0; grp < GR; ++grp)
          qsum[nt][c][grp] = __shfl_sync(0xffffffffu, qs[grp], (2 * ft + c) * 4) * a.scale * kLog2e;
      }
    }
    float o[NT][KT][4], ref[NT][2], l[NT][2], oc[NT][2][GR];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int m = 0; m < KT; ++m) o[nt][m][0] = o[nt][m][1] = o[nt][m][2] = o[nt][m][3] = 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        ref[nt][c] = -INFINITY;
        l[nt][c] = 0.f;
#pragma unroll
        for (int grp = 0; grp < GR; ++grp) oc[nt][c][grp] = 0.f;
      }
    }
    float sdown = 16777216.f;  // 2^-E
    while (cc.left > 0 && cc.u < cc.units) {
      const int n = (int)min((long long)min(TU, cc.units - cc.u), cc.left);
      const uint8_t* base = ring + c_stage * Sh::kStageBytes;
      sm100::mbar_wait(&full[warp][c_stage], c_phase, a.status);
      float s[TU][NT][4];
      __half2 vp[TU][2][GR];
      // scores and value pairs of the tile
#pragma unroll
      for (int j = 0; j < TU; ++j) {
        if (j < n) {
          const uint8_t* un = base + j * U::kBytes;
          float acc[NT][GR][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int grp = 0; grp < GR; ++grp) acc[nt][grp][0] = acc[nt][grp][1] = acc[nt][grp][2] = acc[nt][grp][3] = 0.f;
#pragma unroll
          for (int pl = 0; pl < (HD + 127) / 128; ++pl) {
            constexpr int W = HD < 128 ? 2 : 4;
            uint32_t wa[W], wb[W];
            const uint8_t* ka = un + pl * 1024 + fg * U::kRow + ft * (U::kRow / 4);
            if (W == 4) {
              const uint4 x = *reinterpret_cast<const uint4*>(ka), y = *reinterpret_cast<const uint4*>(ka + 8 * U::kRow);
              wa[0] = x.x, wa[1] = x.y, wa[W - 2] = x.z, wa[W - 1] = x.w;
              wb[0] = y.x, wb[1] = y.y, wb[W - 2] = y.z, wb[W - 1] = y.w;
            } else {
              const uint2 x = *reinterpret_cast<const uint2*>(ka), y = *reinterpret_cast<const uint2*>(ka + 8 * U::kRow);
              wa[0] = x.x, wa[1] = x.y;
              wb[0] = y.x, wb[1] = y.y;
            }
#pragma unroll
            for (int i = 0; i < W; ++i) {
              const int grp = pl * 2 + i / 2, k = pl * 8 + 2 * i;
              const uint32_t x = wa[i], y = wb[i], x8 = x >> 8, y8 = y >> 8;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma_f16(acc[nt][grp], x & 0x000f000fu, y & 0x000f000fu, x & 0x00f000f0u, y & 0x00f000f0u, qf[nt][k][0],
                        qf[nt][k][1]);
                mma_f16(acc[nt][grp], x8 & 0x000f000fu, y8 & 0x000f000fu, x8 & 0x00f000f0u, y8 & 0x00f000f0u,
                        qf[nt][k + 1][0], qf[nt][k + 1][1]);
              }
            }
          }
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float x[NT][2], y[NT][2];
#pragma unroll
            for (int grp = 0; grp < GR; ++grp) {
              vp[j][half][grp] = *reinterpret_cast<const __half2*>(un + U::pair(true, fg + 8 * half, grp));
              const float2 p = __half22float2(*reinterpret_cast<const __half2*>(un + U::pair(false, fg + 8 * half, grp)));
              const float b = fmaf(-8.f, p.x, p.y);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                  x[nt][c] = grp ? fmaf(p.x, acc[nt][grp][2 * half + c], x[nt][c]) : p.x * acc[nt][grp][2 * half + c];
                  y[nt][c] = grp ? fmaf(b, qsum[nt][c][grp], y[nt][c]) : b * qsum[nt][c][grp];
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int c = 0; c < 2; ++c) s[j][nt][2 * half + c] = fmaf(x[nt][c], mult[nt][c], y[nt][c]);
          }
        } else {
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int grp = 0; grp < GR; ++grp) vp[j][half][grp] = __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[j][nt][e] = -INFINITY;
        }
      }
      if ((cc.u + n) * 16 > len) {  // the last unit's tokens past the context hold stale bytes: whatever they are
#pragma unroll
        for (int j = 0; j < TU; ++j)
#pragma unroll
          for (int half = 0; half < 2; ++half)
            if ((cc.u + j) * 16 + fg + 8 * half >= len) {
#pragma unroll
              for (int grp = 0; grp < GR; ++grp) vp[j][half][grp] = __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) s[j][nt][2 * half] = s[j][nt][2 * half + 1] = -INFINITY;
            }
      }
      // the tile's largest scale and scores: move the references where they are passed
      float top_s;
      {
        __half2 t = __habs2(vp[0][0][0]);
#pragma unroll
        for (int j = 0; j < TU; ++j)
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int grp = 0; grp < GR; ++grp) t = __hmax2(t, __habs2(vp[j][half][grp]));
        top_s = __low2float(t);
      }
      bool move = top_s * sdown > 1.f;
      float mx[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          mx[nt][c] = fmaxf(s[0][nt][c], s[0][nt][2 + c]);
#pragma unroll
          for (int j = 1; j < TU; ++j) mx[nt][c] = fmaxf(mx[nt][c], fmaxf(s[j][nt][c], s[j][nt][2 + c]));
          move |= mx[nt][c] > ref[nt][c] + kHead;
        }
      if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) top_s = fmaxf(top_s, __shfl_xor_sync(0xffffffffu, top_s, off));
        // 2^-E with E the exponent above the largest scale so far
        const float need = top_s > 0.f ? __uint_as_float((uint32_t)(253 - (int)(__float_as_uint(top_s) >> 23)) << 23) : sdown;
        const float nd = fminf(sdown, need), fall = nd / sdown;
        sdown = nd;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float m = fmaxf(ref[nt][c], mx[nt][c]);
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
            const float corr = m > -INFINITY ? ex2(ref[nt][c] - m) : 1.f;
            ref[nt][c] = m;
            l[nt][c] *= corr;
#pragma unroll
            for (int grp = 0; grp < GR; ++grp) oc[nt][c][grp] *= corr;
            const float f = corr * fall;
#pragma unroll
            for (int k = 0; k < KT; ++k) {
              o[nt][k][c] *= f;
              o[nt][k][2 + c] *= f;
            }
          }
      }
      // weights and values
#pragma unroll
      for (int j = 0; j < TU; ++j) {
        if (j < n) {
          uint32_t pb[NT][GR][2];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float sv[GR], vc[GR];
#pragma unroll
            for (int grp = 0; grp < GR; ++grp) {
              sv[grp] = __low2float(vp[j][half][grp]) * sdown;
              vc[grp] = __high2float(vp[j][half][grp]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const float w0_ = ex2(s[j][nt][2 * half] - fmaxf(ref[nt][0], -1e30f));
              const float w1_ = ex2(s[j][nt][2 * half + 1] - fmaxf(ref[nt][1], -1e30f));
              l[nt][0] += w0_;
              l[nt][1] += w1_;
#pragma unroll
              for (int grp = 0; grp < GR; ++grp) {
                oc[nt][0][grp] = fmaf(w0_, vc[grp], oc[nt][0][grp]);
                oc[nt][1][grp] = fmaf(w1_, vc[grp], oc[nt][1][grp]);
                pb[nt][grp][half] = transpose8(pack_f16(w0_ * sv[grp], w1_ * sv[grp]));
              }
            }
          }
          const uint8_t* vb = base + j * U::kBytes + U::kCodes + lane * 16;
#pragma unroll
          for (int grp = 0; grp < GR; ++grp) {
            const uint4 x = *reinterpret_cast<const uint4*>(vb + grp * 512);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};  // [32-dim half][tokens 8 h ..]
#pragma unroll
            for (int il = 0; il < 2; ++il) {
              const uint32_t lo = w[2 * il], hi = w[2 * il + 1], lo8 = lo >> 8, hi8 = hi >> 8;
              const uint32_t a0 = centre_even(lo), a1 = centre_odd(lo), a2 = centre_even(hi), a3 = centre_odd(hi);
              const uint32_t b0 = centre_even(lo8), b1 = centre_odd(lo8), b2 = centre_even(hi8), b3 = centre_odd(hi8);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma_f16(o[nt][4 * grp + 2 * il], a0, a1, a2, a3, pb[nt][grp][0], pb[nt][grp][1]);
                mma_f16(o[nt][4 * grp + 2 * il + 1], b0, b1, b2, b3, pb[nt][grp][0], pb[nt][grp][1]);
              }
            }
          }
        }
      }
      cc.u += n;
      cc.left -= n;
      if (++c_stage == kStages) c_stage = 0, c_phase ^= 1;
      __syncwarp();
      produce();  // into the stage whose last operands the instructions above have taken
    }

    // ---- the pair's result in this part ----
    const float sup = 1.f / sdown;
    const bool whole = u_first == 0 && cc.u == cc.units;
    const int slot = first_pair ? 0 : 1;
    float* dst0 = reinterpret_cast<float*>(ring + (slot ? 0 : Sh::kRing));
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int h = nt * 8 + 2 * ft + c;
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], off);
#pragma unroll
          for (int grp = 0; grp < GR; ++grp) oc[nt][c][grp] += __shfl_xor_sync(0xffffffffu, oc[nt][c][grp], off);
        }
        if (h < heads) {
          float f = 1.f;
          if (whole) {
            float lt = l[nt][c], e = 1.f;
            if (a.sinks) {
              const float sk = a.sinks[h0 + h] * kLog2e, m = fmaxf(sk, ref[nt][c]), mb = fmaxf(m, -1e30f);
              e = ex2(ref[nt][c] - mb);
              lt = fmaf(lt, e, ex2(sk - mb));
            }
            f = e / lt;
          }
#pragma unroll
          for (int k = 0; k < KT; k += 2) {
            const int d = (k >> 2) * 64 + ((k >> 1) & 1) * 32 + 4 * fg;
            float4 v = make_float4(fmaf(o[nt][k][c], sup, oc[nt][c][k >> 2]), fmaf(o[nt][k][2 + c], sup, oc[nt][c][k >> 2]),
                                   fmaf(o[nt][k + 1][c], sup, oc[nt][c][k >> 2]),
                                   fmaf(o[nt][k + 1][2 + c], sup, oc[nt][c][k >> 2]));
            if (whole) {
              v.x *= f, v.y *= f, v.z *= f, v.w *= f;
              const int64_t at = (int64_t)(h0 + h) * HD + d;
              if (a.out_bf16) {
                const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
                *reinterpret_cast<uint2*>(a.out_bf16 + cc.row * a.out_stride + at) =
                    make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
              }
              if (a.out) *reinterpret_cast<float4*>(a.out + cc.row * a.outf_stride + at) = v;
            } else {
              *reinterpret_cast<float4*>(dst0 + h * Sh::kRow + d) = v;
            }
          }
          if (!whole && fg == 0) {
            dst0[h * Sh::kRow + HD] = ref[nt][c];
            dst0[h * Sh::kRow + HD + 1] = l[nt][c];
          }
        }
      }
    if (!whole && lane == 0) parts[2 * warp + slot] = Part{cc.row, cc.item, u_first, cc.u};
    first_pair = false;
    if (cc.left > 0) next_pair(cc);
  }

  // ---- pairs that span warps or CTAs ----
  __syncthreads();
  const int pstride = HPI * Sh::kRow;
  const auto local = [&](int i) {  // partial i of the CTA
    return reinterpret_cast<const float*>(smem + (i >> 1) * wbytes + (i & 1 ? 0 : Sh::kRing));
  };
  const auto emit4 = [&](int row, int h, int d, float4 v, float f) {
    v.x *= f, v.y *= f, v.z *= f, v.w *= f;
    if (a.out_bf16) {
      const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
      *reinterpret_cast<uint2*>(a.out_bf16 + row * a.out_stride + (int64_t)h * HD + d) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
    if (a.out) *reinterpret_cast<float4*>(a.out + row * a.outf_stride + (int64_t)h * HD + d) = v;
  };
  const auto sink_of = [&](int h) { return a.sinks ? a.sinks[h] * kLog2e : -INFINITY; };
  for (int i = 0; i < 2 * kWarps;) {
    const Part p = parts[i];
    if (p.row < 0) {
      ++i;
      continue;
    }
    unsigned set = 0;  // the pair's partials in this CTA
    int end = p.u1, j = i;
    for (; j < 2 * kWarps; ++j) {
      const Part q = parts[j];
      if (q.row < 0) continue;
      if (q.row != p.row || q.item != p.item) break;
      set |= 1u << j;
      end = q.u1;
    }
    i = j;
    const int units = (int)(before[p.row + 1] - before[p.row]);
    const bool done = p.u0 == 0 && end == units;
    const long long i0 = before[p.row] * items + (long long)p.item * units, i1 = i0 + units;
    const int kvh = p.item / g_.splits, h0 = kvh * G + (p.item % g_.splits) * HPI;
    const int heads = min(HPI, kvh * G + G - h0);
    const int my_slot = i0 + p.u0 == w0 ? 0 : 1;
    float* mine = g_.part + ((int64_t)cta * 2 + my_slot) * pstride;
    for (int x = tid; x < heads * (HD / 4); x += kThreads) {
      const int h = x / (HD / 4), d = x % (HD / 4) * 4;
      const float sk = done ? sink_of(h0 + h) : -INFINITY;
      float m = sk;
      for (unsigned b = set; b; b &= b - 1) m = fmaxf(m, local(__ffs(b) - 1)[h * Sh::kRow + HD]);
      const float mb = fmaxf(m, -1e30f);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      float lt = ex2(sk - mb);
      for (unsigned b = set; b; b &= b - 1) {
        const float* q = local(__ffs(b) - 1) + h * Sh::kRow;
        const float e = ex2(q[HD] - mb);
        const float4 t = *reinterpret_cast<const float4*>(q + d);
        v.x = fmaf(t.x, e, v.x), v.y = fmaf(t.y, e, v.y), v.z = fmaf(t.z, e, v.z), v.w = fmaf(t.w, e, v.w);
        lt = fmaf(q[HD + 1], e, lt);
      }
      if (done) {
        emit4(p.row, h0 + h, d, v, 1.f / lt);
      } else {
        __stcg(reinterpret_cast<float4*>(mine + h * Sh::kRow + d), v);
        if (d == 0) __stcg(reinterpret_cast<float2*>(mine + h * Sh::kRow + HD), make_float2(m, lt));
      }
    }
    if (done) continue;
    // partials of several CTAs: c0 .. c1 in order, the first of them in slot 1 unless the pair begins it
    const int c0 = (int)(((i0 + 1) * N - 1) / total), c1 = (int)((i1 * N - 1) / total);
    const int first_slot = total * c0 / N < i0 ? 1 : 0;
    const auto part_of = [&](int c) { return g_.part + ((int64_t)c * 2 + (c == c0 ? first_slot : 0)) * pstride; };
    // true in the last of `n` CTAs to come here (its reads see the others' writes)
    const auto arrive_last = [&](int* counter, int n) {
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        const int got = atomicAdd(counter, 1);
        last_s = got == n - 1;
        if (last_s) *counter = 0;
      }
      __syncthreads();
      const bool last = last_s;
      __syncthreads();
      if (last) __threadfence();
      return last;
    };
    // sum of the partials from, from + step, .. < to, to the row's output or to dst (with its reference and
    // sum two places on: others still read the first). `ml`: where the partials' reference and sum are
    const auto merge = [&](int from, int to, int step, int ml_at, float* dst) {
      for (int x = tid; x < heads * (HD / 4); x += kThreads) {
        const int h = x / (HD / 4), d = x % (HD / 4) * 4;
        const float sk = dst ? -INFINITY : sink_of(h0 + h);
        float m = sk;
#pragma unroll 8
        for (int c = from; c < to; c += step) m = fmaxf(m, __ldcg(part_of(c) + h * Sh::kRow + ml_at));
        const float mb = fmaxf(m, -1e30f);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float lt = ex2(sk - mb);
#pragma unroll 8
        for (int c = from; c < to; c += step) {
          const float* q = part_of(c) + h * Sh::kRow;
          const float2 ml = __ldcg(reinterpret_cast<const float2*>(q + ml_at));
          const float4 t = __ldcg(reinterpret_cast<const float4*>(q + d));
          const float e = ex2(ml.x - mb);
          v.x = fmaf(t.x, e, v.x), v.y = fmaf(t.y, e, v.y), v.z = fmaf(t.z, e, v.z), v.w = fmaf(t.w, e, v.w);
          lt = fmaf(ml.y, e, lt);
        }
        if (dst) {
          __stcg(reinterpret_cast<float4*>(dst + h * Sh::kRow + d), v);
          if (d == 0) __stcg(reinterpret_cast<float2*>(dst + h * Sh::kRow + HD + 2), make_float2(m, lt));
        } else {
          emit4(p.row, h0 + h, d, v, 1.f / lt);
        }
      }
    };
    const int n = c1 - c0 + 1;
    if (n <= 2 * kTree) {
      if (arrive_last(g_.counters + c0, n)) merge(c0, c1 + 1, 1, HD, nullptr);
    } else {
      const int grp = (cta - c0) / kTree, g0 = c0 + grp * kTree, g1 = min(g0 + kTree, c1 + 1);
      if (arrive_last(g_.counters + gridDim.x + 2 * g0 + (g0 == c0 ? first_slot : 0), g1 - g0)) {
        merge(g0, g1, 1, HD, part_of(g0));
        if (arrive_last(g_.counters + c0, (n + kTree - 1) / kTree)) merge(c0, c1 + 1, kTree, HD + 2, nullptr);
      }
    }
  }
  pdl_launch();
}

template <int HD, int NT>
void launch_decode(const DecodeArgs& d, int sms, cudaStream_t s, bool pdl) {
  using Sh = DecodeShape<HD, NT>;
  const size_t smem = Sh::smem(d.heads_per_item);
  static int per_sm[8 * NT + 1] = {};  // by heads per item; per instantiation, one device per process
  int& resident = per_sm[d.heads_per_item];
  if (!resident) {
    HK_CUDA_CHECK(cudaFuncSetAttribute(kv4_decode_kernel<HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)Sh::smem(8 * NT)));
    int n = 0;
    HK_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kv4_decode_kernel<HD, NT>, Sh::kThreads, smem));
    if (n < 1) throw std::runtime_error("kv4 attention decode: the kernel does not fit on an SM");
    resident = n < 4 ? n : 4;
  }
  launch(kv4_decode_kernel<HD, NT>, dim3(sms * resident), dim3(Sh::kThreads), smem, s, pdl, d);
}

}  // namespace

void kv4_attention_decode_launch(const Kv4AttnArgs& args, const Kv4Workspace& ws, cudaStream_t s, bool pdl) {
  const int G = args.nh / args.nkv;
  for (int r0 = 0; r0 < args.R; r0 += kMaxRows) {
    DecodeArgs d{};
    d.a = args;
    d.a.R = args.R - r0 < kMaxRows ? args.R - r0 : kMaxRows;
    d.a.q += r0 * args.q_stride;
    d.a.row_seq += r0;
    d.a.row_ctx += r0;
    if (d.a.out) d.a.out += r0 * args.outf_stride;
    if (d.a.out_bf16) d.a.out_bf16 += r0 * args.out_stride;
    d.part = ws.part;
    d.counters = ws.counters;
    const bool wide = G > 8 && args.hd <= 128;  // two tiles of 8 heads share each key and value
    d.heads_per_item = wide ? G : (G < 8 ? G : 8);
    d.splits = (G + d.heads_per_item - 1) / d.heads_per_item;
    const int upb = args.block_size / 16;
    d.upb_shift = (upb & (upb - 1)) ? -1 : __builtin_ctz(upb);
    if (args.hd == 64) wide ? launch_decode<64, 2>(d, ws.sms, s, pdl) : launch_decode<64, 1>(d, ws.sms, s, pdl);
    else if (args.hd == 128) wide ? launch_decode<128, 2>(d, ws.sms, s, pdl) : launch_decode<128, 1>(d, ws.sms, s, pdl);
    else if (args.hd == 256) launch_decode<256, 1>(d, ws.sms, s, pdl);
    else throw std::runtime_error("kv4 attention: head_dim 64, 128 or 256");
  }
}

}  // namespace hk
