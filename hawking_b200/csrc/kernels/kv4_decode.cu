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
// More than 8 query heads per kv head make two items of it. (One item of two narrow tiles, which unpacks every code
// once, was 7 % faster for 64 rows of 8000 tokens and 16 heads, but its registers halve the warps: 28 us against 20
// for 8 such rows.)
//
// Work. The (row, item) pairs' units of 16 tokens form one sequence that is cut into equal ranges,
// one per CTA (at least kMinUnits long), and each range into equal parts, one per warp: ragged batches
// and single long rows load every warp alike, and a warp needs nobody inside its part. A pair that lies
// in one part is written out by its warp; one that spans warps is merged in shared memory at the end
// of the CTA; one that spans CTAs leaves partials (reference, sum, output), merged in CTA order by the
// last CTA to arrive (groups of kTree CTAs first, where there are many). One CTA per SM; a warp of it
// only issues the copies for all others (bulk copies of whole units, a ring of tiles per warp).
//
// What bounds it, on one B200. 64 rows of 200 to 8192 tokens, 32 / 8 heads of 128 (163 MB of cache): 45 us. About 32 us
// of them stream at 5 TB/s, 0.77 of the memory's measured rate, with issue slots 56 % and the ALU 51 % busy: four warps
// per scheduler do not cover the latency of unpacking. The first data are there after 4.7 us; merging and stragglers
// take 8. Two rows of 30 and 60 thousand tokens, 16 / 2 heads of 256 (52 MB): 29 us, 12 for the bytes, the rest the
// merges of 37 CTAs per pair. One row of 2048 tokens (2.4 MB): 10 us, all of it latency.
#include <algorithm>

#include "kv4.cuh"
#include "sm100.cuh"

namespace hk {
namespace {

using kv4::centre_even;
using kv4::centre_odd;
using kv4::Unit;
using sm100::smem_u32;
constexpr float kLog2e = 1.4426950408889634f;
// CTAs whose partials are merged first where a pair has more than kFlat: two rows over 37 CTAs per pair took 31.1 us
// with 8, 32.0 with 6, 32.7 with 12.
constexpr int kTree = 8;
constexpr int kFlat = 24;
constexpr int kMaxCtas = 32 * kTree;  // (a lane per partial)
// Units (and visits) of a warp below which fewer CTAs work: one row of 2048 tokens took 12.6 us with 3, 14.6 with 8.
constexpr int kMinUnits = 3;
// What a pair costs a warp besides its units, in units: the 64 ragged rows above took 53.5 us with 0, 48.9 with 4, 47.3
// with 8, 49.3 with 12.
constexpr int kVisit = 8;
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
// Loads past the L1 cache, of shared or global memory, that may be in flight together.
__device__ __forceinline__ float2 fresh2(const float* p) {
  float2 v;
  asm volatile("ld.relaxed.gpu.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ float4 fresh4(const float* p) {
  float4 v;
  asm volatile("ld.relaxed.gpu.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
  return v;
}

struct DecodeArgs {
  Kv4AttnArgs a;
  int heads_per_item, split;   // query heads of one item, log2 of the items per kv head (0 or 1)
  int upb_shift;               // log2 of the units per block, or -1
  float* part;                 // [grid][2 + kWarps][heads_per_item * (HD + 4)]: the CTAs', then the warps' first
  int* counters;               // [3 * grid], zero between launches
};

constexpr int kMaxRows = 512;  // rows of one launch

template <int HD>
struct DecodeShape {
  // one CTA per SM (fewer partials to merge than several smaller ones), its warps by the registers:
  // 128 a thread, or 168
  static constexpr int kWarps = HD <= 128 ? 15 : 11;  // and one that issues the copies
  static constexpr int kThreads = (kWarps + 1) * 32;
  static_assert(2 * kWarps <= 32, "one lane per partial");
  static constexpr int kStages = HD <= 128 ? 3 : 4;                     // tiles in a warp's ring
  static constexpr int kTile = 256 / HD;                                           // units per stage (4608 bytes)
  static constexpr int kStageBytes = kTile * Unit<HD>::kBytes;
  static constexpr int kRow = HD + 4;  // floats of one head's partial: output, reference, sum
  static constexpr int kRing = kStages * kStageBytes;
  static constexpr int kSmem = kWarps * kRing;  // the ring's place takes the part's last partial
  static_assert(kSmem + 10 * 1024 <= 227 * 1024, "shared memory of an SM");
  static_assert(kKv4ItemHeads * kRow * 4 <= kRing, "the last partial fits the ring");
  static_assert((2 + kWarps) * kKv4ItemHeads * kRow <= kKv4PartFloatsPerSm, "a CTA's partials fit the workspace");
};

// A warp's partial in shared memory: units [u0, u1) of a pair.
struct Part {
  int row, item, u0, u1;  // row < 0: none
};

// Where a merged head goes: the output in either type, or a partial with its reference and sum at ml. Addresses,
// so that nothing of the arguments is read again on the way.
struct MergeTo {
  float* part;
  float2* ml;
  uint16_t* out16;
  float* out;
};

// One head of the sum of n <= 32 partials and of a sink of log2 weight m, if any, by a warp: lane k has the address of
// partial k, in shared or global memory, where the head is `at` floats on and its reference and sum at `ml_at`. A lane
// without a partial (live: false) has partial 0's address and weight 0. Every lane weighs one partial and sums 4 dims of
// each 128. A few warps do this once, so what bounds it is the latency of its instructions, not the bytes: 11 partials of
// 8 heads of 256 in shared memory took 4.4 us when a thread per 4 dims weighed all partials itself, 1.3 this way.
template <int HD, int FLY>
__device__ __noinline__ void merge_parts(const float* from, bool live, int n, int at, int ml_at, float m, const MergeTo to) {
  constexpr int NV = (HD + 127) / 128;  // vectors of a lane; FLY: partials in flight
  const int lane = threadIdx.x & 31;
  const bool mine = HD >= 128 || lane < HD / 4;
  float2 ml = make_float2(-INFINITY, 0.f);
  if (live) ml = fresh2(from + ml_at);
  const unsigned long long base = reinterpret_cast<unsigned long long>(from + at);
  const int d0 = HD >= 128 ? 4 * lane : 4 * (lane % (HD / 4));
  float4 v[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
  float e = 0.f, lt = 0.f;
#pragma unroll 1
  for (int k0 = 0; k0 < n; k0 += FLY) {
    float4 t[FLY][NV];
#pragma unroll
    for (int k = 0; k < FLY; ++k) {
      const float* q = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, base, k0 + k)) + d0;
#pragma unroll
      for (int j = 0; j < NV; ++j) t[k][j] = fresh4(q + 128 * j);
    }
    if (k0 == 0) {
      float top = fmaxf(m, ml.x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float mb = fmaxf(top, -1e30f);
      e = ex2(ml.x - mb);
      lt = ml.y * e;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) lt += __shfl_xor_sync(0xffffffffu, lt, o);
      lt += ex2(m - mb);  // the sink
      m = top;
    }
#pragma unroll
    for (int k = 0; k < FLY; ++k) {
      const float w = __shfl_sync(0xffffffffu, e, k0 + k);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        v[j].x = fmaf(t[k][j].x, w, v[j].x), v[j].y = fmaf(t[k][j].y, w, v[j].y);
        v[j].z = fmaf(t[k][j].z, w, v[j].z), v[j].w = fmaf(t[k][j].w, w, v[j].w);
      }
    }
  }
  if (to.part) {
    if (mine)
#pragma unroll
      for (int j = 0; j < NV; ++j) __stcg(reinterpret_cast<float4*>(to.part + 4 * lane + 128 * j), v[j]);
    if (lane == 0) __stcg(to.ml, make_float2(m, lt));
    return;
  }
  if (!mine) return;
  const float f = 1.f / lt;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int d = 4 * lane + 128 * j;
    const float4 z = make_float4(v[j].x * f, v[j].y * f, v[j].z * f, v[j].w * f);
    if (to.out16) {
      const __nv_bfloat162 lo = __floats2bfloat162_rn(z.x, z.y), hi = __floats2bfloat162_rn(z.z, z.w);
      *reinterpret_cast<uint2*>(to.out16 + d) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
    if (to.out) *reinterpret_cast<float4*>(to.out + d) = z;
  }
}

template <int HD>
__global__ void __launch_bounds__(DecodeShape<HD>::kThreads, 1)
    kv4_decode_kernel(const __grid_constant__ DecodeArgs g_) {
  using U = Unit<HD>;
  using Sh = DecodeShape<HD>;
  static_assert(kFlat <= 32 && kTree <= 32, "one lane per partial");
  constexpr int GR = HD / 64, KT = HD / 16, TU = Sh::kTile, kWarps = Sh::kWarps, kThreads = Sh::kThreads,
                kStages = Sh::kStages;
  const Kv4AttnArgs& a = g_.a;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[kWarps][kStages], empty[kWarps][kStages];
  __shared__ int before[kMaxRows + 1];  // work (units x items) of the rows before each row
  __shared__ int2 rows[kMaxRows];        // block-table row and context of each row
  __shared__ int wsum[kWarps + 1];
  __shared__ Part parts[2 * kWarps];
  __shared__ int last_s[2];
  __shared__ volatile int gave_up;       // a wait of this CTA ran out
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int fg = lane >> 2, ft = lane & 3;
  const int G = a.nh / a.nkv, items = a.nkv << g_.split, HPI = g_.heads_per_item;
  const int upb = a.block_size / 16;
  uint8_t* ring = smem + warp * Sh::kRing;
  // query heads of an item
  const auto head_of = [&](int item) { return (item >> g_.split) * G + (item & g_.split) * HPI; };
  const auto heads_of = [&](int item) { return min(HPI, G - (item & g_.split) * HPI); };
  if (warp == kWarps && lane < kWarps) {
    for (int s = 0; s < kStages; ++s) {
      sm100::mbar_init(&full[lane][s], 1);
      sm100::mbar_init(&empty[lane][s], 1);
    }
    sm100::fence_barrier_init();
    parts[2 * lane].row = parts[2 * lane + 1].row = -1;
  }
  pdl_wait();

  // ---- work: scan of the rows' units (the host sees to it that the sum fits 32 bits) ----
  {
    const int per = (a.R + kThreads - 1) / kThreads;
    const int r0 = min(a.R, tid * per), r1 = min(a.R, r0 + per);
    int sum = 0;
#pragma unroll 1
    for (int r = r0; r < r1; ++r) {
      int seq = a.row_seq[r];
      const int len = min(max(a.row_ctx[r], 0), a.max_blocks * a.block_size);
      if (seq < 0 || seq >= a.table_rows) {  // reads as zeros, and leaves the other rows' parts as they are
        seq = -1;
        if (blockIdx.x == 0) set_error(a.status, HK_ERR_BAD_ARG);
      }
      rows[r] = make_int2(seq, len);
      const int n = len ? (((len + 15) >> 4) + kVisit) * items : 0;
      before[r + 1] = n;
      sum += n;
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) wsum[warp] = inc;
    if (tid == 0) before[0] = gave_up = 0;
    __syncthreads();
    int base = inc - sum;
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
      if (w < warp) base += wsum[w];
#pragma unroll 1
    for (int r = r0; r < r1; ++r) {
      base += before[r + 1];
      before[r + 1] = base;
    }
    __syncthreads();
  }
  const int total = before[a.R];
  // CTAs and warps at work. A warp's part takes time, and so does each partial in its CTA's merge: with u units for a
  // CTA, u / W + W is least at W = sqrt(u). (8 rows of 8000 tokens of two kv heads: 20.6 us, with sqrt(1.5 u) 22.8.)
  const int W = min(kWarps, max(1, (int)ceilf(sqrtf((float)total / (float)gridDim.x))));
  const int N = min((int)gridDim.x, (total + W * kMinUnits - 1) / (W * kMinUnits));
  const int cta = blockIdx.x;
  // rows without context
#pragma unroll 1
  for (int r = cta; r < a.R; r += gridDim.x)
    if (rows[r].y == 0)
#pragma unroll 1
      for (int i = tid; i < a.nh * HD; i += kThreads) {
        if (a.out_bf16) a.out_bf16[r * a.out_stride + i] = 0;
        if (a.out) a.out[r * a.outf_stride + i] = 0.f;
      }
  if (cta >= N) return;
  // part i of N * W begins at i * each + min(i, more)
  const int each = total / (N * W), more = total - each * (N * W);
  const auto part_begin = [&](int i) { return i * each + min(i, more); };
  const auto part_of = [&](int x) { return x < more * (each + 1) ? x / (each + 1) : more + (x - more * (each + 1)) / each; };
  const int w0 = part_begin(cta * W);
  // a warp has its part; in the copying warp lane w has warp w's
  const bool copies = warp == kWarps;
  const int who = copies ? lane : warp;
  const int p0 = part_begin(cta * W + min(who, W)), p1 = part_begin(cta * W + min(who + 1, W));

  // ---- cursor over the pairs of the part [p0, p1) ----
  struct Cursor {
    int row, item, u, units;
    int at;  // place of the pair's unit 0: units [u, min(units, p1 - at)) are this part's
  };
  Cursor cc;
  {
    int lo = 0, hi = a.R;  // last row with before <= p0
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (before[mid] <= p0) lo = mid;
      else hi = mid;
    }
    cc.row = lo;
    cc.units = (rows[lo].y + 15) >> 4;
    cc.item = cc.units ? (p0 - before[lo]) / (cc.units + kVisit) : 0;
    cc.at = before[lo] + cc.item * (cc.units + kVisit) + kVisit;
    cc.u = max(0, p0 - cc.at);
  }
  const auto more_in = [&](const Cursor& c) { return c.at + c.u < p1; };
  const auto next_pair = [&](Cursor& c) {  // to the next pair (which may lie past the part)
    c.u = 0;
    c.at += c.units + kVisit;
    if (++c.item == items) {
      c.item = 0;
      do ++c.row;
      while (c.row < a.R && rows[c.row].y == 0);
      c.units = c.row < a.R ? (rows[c.row].y + 15) >> 4 : 0;
    }
  };

  int c_stage = 0, c_phase = 0;  // next stage of the ring: to read, or (in the copying warp) to fill
  // ---- the copying warp: every lane fetches one warp's tiles, kStages ahead, so that the cursors and
  // addresses of all warps cost one warp's instructions ----
  if (copies) {
    const uint8_t* head = nullptr;  // the pair's kv head in block 0
    const int* table = nullptr;
    const int64_t blk_bytes = (int64_t)a.nkv * upb * U::kBytes;
    int blk_last = 0;  // block of the last tile's last unit
    int blk[TU], at = 0;  // blocks of the next tile's units, and the first unit's place in its block
    const auto lookup = [&](bool pair) {
      if (pair) {
        head = a.cache + (int64_t)(cc.item >> g_.split) * upb * U::kBytes;
        const int seq = rows[cc.row].x;
        table = seq < 0 ? nullptr : a.block_tables + (int64_t)seq * a.max_blocks;
      }
      const int b0 = g_.upb_shift >= 0 ? cc.u >> g_.upb_shift : cc.u / upb;
      at = cc.u - b0 * upb;
      const bool kept = !pair && at > 0;  // the tile begins in the last one's block
      int b = b0, k = at;
#pragma unroll
      for (int i = 0; i < TU; ++i) {
        if (i > 0 && ++k == upb) k = 0, ++b;
        if (i == 0 && kept) blk[0] = blk_last;
        else if (i > 0 && b == b0) blk[i] = blk[0];
        else if (cc.u + i < cc.units) blk[i] = table ? table[b] : -1;
      }
    };
    uint8_t* const my_ring = smem + lane * Sh::kRing;
    int st = 0, ph = 1;
    unsigned idle = 0;  // turns in a row in which no lane had a free stage (the same for the warp, as its ways out)
    bool more = lane < W && more_in(cc);
    if (more) lookup(true);
#pragma unroll 1
    while (__any_sync(0xffffffffu, more)) {
      const bool go = more && sm100::mbar_try_wait(&empty[lane][st], ph);
      if (go) {
        const int n = min(TU, min(cc.units, p1 - cc.at) - cc.u);
        uint8_t* dst = my_ring + st * Sh::kStageBytes;
        uint64_t* bar = &full[lane][st];
        int good = 0;
#pragma unroll
        for (int i = 0; i < TU; ++i) {
          if (i < n) {
            if (blk[i] >= 0 && blk[i] < a.cache_blocks) {
              ++good;
            } else {  // a block outside the cache reads as zeros
              set_error(a.status, HK_ERR_BAD_ARG);
#pragma unroll 1
              for (int x = 0; x < U::kBytes; x += 16)
                *reinterpret_cast<uint4*>(dst + i * U::kBytes + x) = make_uint4(0u, 0u, 0u, 0u);
              sm100::fence_proxy_async_smem();
            }
            blk_last = blk[i];
          }
        }
        sm100::mbar_arrive_expect_tx(bar, good * U::kBytes);
        int k = at;  // one copy for the units of one block
#pragma unroll
        for (int i = 0; i < TU; ++i) {
          if (i < n && (i == 0 || k == 0) && blk[i] >= 0 && blk[i] < a.cache_blocks)
            sm100::bulk_g2s(dst + i * U::kBytes, head + blk[i] * blk_bytes + k * U::kBytes,
                            min(n - i, upb - k) * U::kBytes, bar);
          if (++k == upb) k = 0;
        }
        if (++st == kStages) st = 0, ph ^= 1;
        cc.u += n;
        const bool pair = cc.u == cc.units;
        if (pair) next_pair(cc);
        more = more_in(cc);
        if (more) lookup(pair);
      }
      if (__any_sync(0xffffffffu, go)) {
        idle = 0;
      } else {
        const bool over = ++idle > a.wait_polls;  // warps that never free a stage
        if (__any_sync(0xffffffffu, over || gave_up)) {
          if (over) kv4::timed_out(a.status);
          gave_up = 1;
          break;
        }
        __nanosleep(64);
      }
    }
    c_stage = st;
    c_phase = ph;
  }

  // ---- the other warps: one pair after the other. A pair's part goes out (if it is the whole pair) or to a
  // partial: the first of the warp's to global memory (its ring is in use), the last to the ring's place ----
  const int pstride = HPI * Sh::kRow;
  float* const firsts = g_.part + ((int64_t)gridDim.x * 2 + (int64_t)cta * kWarps) * pstride;
  bool ok = true;  // the same for the warp
  while (!copies && ok && more_in(cc)) {
    const int u_first = cc.u, h0 = head_of(cc.item), heads = heads_of(cc.item);
    const int len = rows[cc.row].y;
    // queries: B fragments (dims x 8 heads), float16 after a power-of-two scaling of each head
    uint32_t qf[KT][2];
    float mult[2], qsum[2][GR];
    uint4 raw[HD / 32];
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
      raw[i] = make_uint4(0u, 0u, 0u, 0u);
      if (fg < heads)
        raw[i] = *reinterpret_cast<const uint4*>(a.q + cc.row * a.q_stride + (int64_t)(h0 + fg) * HD + 32 * i + 8 * ft);
    }
    __nv_bfloat162 top = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
      const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) top = __hmax2(top, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[j])));
    }
    float mx = fmaxf(__low2float(top), __high2float(top));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    // 2^-e with 1 <= mx 2^-e < 2 (1 for a zero, subnormal or non-finite head), exact in bf16
    const int ex = (int)(__float_as_uint(mx) >> 23);
    const bool norm = ex > 4 && ex < 254;
    const uint32_t dn = norm ? (uint32_t)(254 - ex) << 7 : 0x3f80u, dn16 = dn + (4u << 7);
    const uint32_t d1 = dn | dn << 16, d16 = dn16 | dn16 << 16;
    // 2^24 of the subnormal codes, less the 16 of the query
    const float un = norm ? __uint_as_float((uint32_t)ex << 23) : 1.f, up = un * (a.scale * kLog2e * 1048576.f);
    float qs[GR];
#pragma unroll
    for (int grp = 0; grp < GR; ++grp) qs[grp] = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
      const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // the odd nibbles' codes come 16 times larger
        const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w[j]),
                                         *reinterpret_cast<const __nv_bfloat162*>(j & 1 ? &d1 : &d16));
        const float lo = __low2float(y), hi = __high2float(y);
        qf[2 * i + j / 2][j & 1] = pack_f16(lo, hi);
        qs[i / 2] = fmaf(lo + hi, j & 1 ? 1.f : 0.0625f, qs[i / 2]);
      }
    }
#pragma unroll
    for (int grp = 0; grp < GR; ++grp) {
      qs[grp] += __shfl_xor_sync(0xffffffffu, qs[grp], 1);
      qs[grp] += __shfl_xor_sync(0xffffffffu, qs[grp], 2);
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      mult[c] = __shfl_sync(0xffffffffu, up, (2 * ft + c) * 4);
#pragma unroll
      for (int grp = 0; grp < GR; ++grp)
        qsum[c][grp] = __shfl_sync(0xffffffffu, qs[grp] * un, (2 * ft + c) * 4) * (a.scale * kLog2e);
    }
    float o[KT][4], ref[2], l[2], oc[2][GR];
#pragma unroll
    for (int m = 0; m < KT; ++m) o[m][0] = o[m][1] = o[m][2] = o[m][3] = 0.f;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      ref[c] = 0.f;
      l[c] = 0.f;
#pragma unroll
      for (int grp = 0; grp < GR; ++grp) oc[c][grp] = 0.f;
    }
    float log2_s = -24.f;  // E
    bool first = true;     // no reference yet
    const int u_last = min(cc.units, p1 - cc.at);
    while (cc.u < u_last) {
      const int n = min(TU, u_last - cc.u);
      const uint8_t* base = ring + c_stage * Sh::kStageBytes;
      if (!(ok = kv4::warp_wait(&full[warp][c_stage], c_phase, a.status, a.wait_polls))) break;
      float s[TU][4];
      __half2 vp[TU][2][GR];
      // scores and value pairs of the tile
#pragma unroll
      for (int j = 0; j < TU; ++j) {
        {
          const uint8_t* un = base + j * U::kBytes;
          float acc[GR][4];
#pragma unroll
          for (int grp = 0; grp < GR; ++grp) acc[grp][0] = acc[grp][1] = acc[grp][2] = acc[grp][3] = 0.f;
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
              mma_f16(acc[grp], x & 0x000f000fu, y & 0x000f000fu, x & 0x00f000f0u, y & 0x00f000f0u, qf[k][0],
                      qf[k][1]);
              mma_f16(acc[grp], x8 & 0x000f000fu, y8 & 0x000f000fu, x8 & 0x00f000f0u, y8 & 0x00f000f0u,
                      qf[k + 1][0], qf[k + 1][1]);
            }
          }
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float x[2], y[2];
#pragma unroll
            for (int grp = 0; grp < GR; ++grp) {
              vp[j][half][grp] = *reinterpret_cast<const __half2*>(un + U::pair(true, fg + 8 * half, grp));
              const float2 p = __half22float2(*reinterpret_cast<const __half2*>(un + U::pair(false, fg + 8 * half, grp)));
              const float b = fmaf(-8.f, p.x, p.y);
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                x[c] = grp ? fmaf(p.x, acc[grp][2 * half + c], x[c]) : p.x * acc[grp][2 * half + c];
                y[c] = fmaf(b, qsum[c][grp], grp ? y[c] : -ref[c]);
              }
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) s[j][2 * half + c] = fmaf(x[c], mult[c], y[c]);
          }
        }
      }
      const int lim = min(len, (cc.u + n) * 16);
      if (lim < (cc.u + TU) * 16) {  // past the tile or the context: stale bytes, whatever they hold
#pragma unroll
        for (int j = 0; j < TU; ++j)
#pragma unroll
          for (int half = 0; half < 2; ++half)
            if ((cc.u + j) * 16 + fg + 8 * half >= lim) {
#pragma unroll
              for (int grp = 0; grp < GR; ++grp) vp[j][half][grp] = __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
              s[j][2 * half] = s[j][2 * half + 1] = -INFINITY;
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
      const float bound = kHead - log2_s;  // scores are relative to ref = R + E
      bool move = first || top_s > ex2(log2_s);
      float mx[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        mx[c] = fmaxf(s[0][c], s[0][2 + c]);
#pragma unroll
        for (int j = 1; j < TU; ++j) mx[c] = fmaxf(mx[c], fmaxf(s[j][c], s[j][2 + c]));
        move |= mx[c] > bound;
      }
      if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) top_s = fmaxf(top_s, __shfl_xor_sync(0xffffffffu, top_s, off));
        // E: at least the exponent above the largest scale so far
        const float e_new = fmaxf(log2_s, (float)((int)(__float_as_uint(top_s) >> 23) - 126));
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float m = mx[c];
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
          m += log2_s;  // the tile's largest score, relative to R
          const float rise = m > -INFINITY && (first || m > 0.f) ? m : 0.f;
          const float up_to = rise + (e_new - log2_s), corr = first ? 1.f : ex2(-up_to);
          ref[c] += up_to;
          l[c] *= corr;
#pragma unroll
          for (int grp = 0; grp < GR; ++grp) oc[c][grp] *= corr;
#pragma unroll
          for (int k = 0; k < KT; ++k) {
            o[k][c] *= corr;
            o[k][2 + c] *= corr;
          }
#pragma unroll
          for (int j = 0; j < TU; ++j) s[j][c] -= up_to, s[j][2 + c] -= up_to;
        }
        log2_s = e_new;
        first = false;
      }
      // weights and values
#pragma unroll
      for (int j = 0; j < TU; ++j) {
        {
          uint32_t pb[GR][2];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float sv[GR], vc[GR];
#pragma unroll
            for (int grp = 0; grp < GR; ++grp) {
              sv[grp] = __low2float(vp[j][half][grp]);
              vc[grp] = __high2float(vp[j][half][grp]);
            }
            const float w0_ = ex2(s[j][2 * half]), w1_ = ex2(s[j][2 * half + 1]);
            l[0] += w0_;
            l[1] += w1_;
#pragma unroll
            for (int grp = 0; grp < GR; ++grp) {
              oc[0][grp] = fmaf(w0_, vc[grp], oc[0][grp]);
              oc[1][grp] = fmaf(w1_, vc[grp], oc[1][grp]);
              pb[grp][half] = transpose8(pack_f16(w0_ * sv[grp], w1_ * sv[grp]));
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
              mma_f16(o[4 * grp + 2 * il], a0, a1, a2, a3, pb[grp][0], pb[grp][1]);
              mma_f16(o[4 * grp + 2 * il + 1], b0, b1, b2, b3, pb[grp][0], pb[grp][1]);
            }
          }
        }
      }
      cc.u += n;
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(&empty[warp][c_stage]);
      if (++c_stage == kStages) c_stage = 0, c_phase ^= 1;
    }

    if (!ok) {  // its stage is not freed: the copying warp ends too
      gave_up = 1;
      break;
    }
    // ---- the pair's result in this part ----
    const bool whole = u_first == 0 && cc.u == cc.units;
    const int slot = cc.at + cc.units + kVisit >= p1 ? 1 : 0;  // the part's last pair: its ring is done
    float* mine = slot ? reinterpret_cast<float*>(ring) : firsts + warp * pstride;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int h = 2 * ft + c;
      float lt = l[c], f = 1.f;
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        lt += __shfl_xor_sync(0xffffffffu, lt, off);
#pragma unroll
        for (int grp = 0; grp < GR; ++grp) oc[c][grp] += __shfl_xor_sync(0xffffffffu, oc[c][grp], off);
      }
      if (h < heads) {
        float* to = mine + h * Sh::kRow + 4 * fg;  // fp32: the partial, or the output itself
        uint16_t* to16 = nullptr;
        if (whole) {
          const int64_t at = (int64_t)(h0 + h) * HD + 4 * fg;
          if (a.sinks) lt += ex2(kv4::sink_over(a.sinks[h0 + h], ref[c]));
          f = __frcp_rn(lt);
          to = a.out ? a.out + cc.row * a.outf_stride + at : nullptr;
          to16 = a.out_bf16 ? a.out_bf16 + cc.row * a.out_stride + at : nullptr;
        } else if (fg == 0) {
          *reinterpret_cast<float2*>(mine + h * Sh::kRow + HD) = make_float2(ref[c], lt);
        }
#pragma unroll
        for (int k = 0; k < KT; k += 2) {
          const int d = (k >> 2) * 64 + ((k >> 1) & 1) * 32;
          const float z = oc[c][k >> 2];
          const float4 v = make_float4((o[k][c] + z) * f, (o[k][2 + c] + z) * f, (o[k + 1][c] + z) * f,
                                       (o[k + 1][2 + c] + z) * f);
          if (to) *reinterpret_cast<float4*>(to + d) = v;
          if (to16) {
            const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
            *reinterpret_cast<uint2*>(to16 + d) =
                make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
          }
        }
      }
    }
    if (!whole && lane == 0) parts[2 * warp + slot] = Part{cc.row, cc.item, u_first, cc.u};
    next_pair(cc);
  }

  const auto sink_of = [&](const float* dst, int item, int h) {
    return !dst && a.sinks ? kv4::sink_log2(a.sinks[head_of(item) + h]) : -INFINITY;
  };
  const auto merge_to = [&](float* dst, int row, int item, int h, int ml_at) {
    const int64_t at = (int64_t)(head_of(item) + h) * HD;
    return MergeTo{dst ? dst + h * Sh::kRow : nullptr, reinterpret_cast<float2*>(dst + h * Sh::kRow + ml_at),
                   a.out_bf16 ? a.out_bf16 + row * a.out_stride + at : nullptr,
                   a.out ? a.out + row * a.outf_stride + at : nullptr};
  };
  // ---- pairs that span warps or CTAs (rolled loops: this code runs once per CTA, cold) ----
  __syncthreads();
  if (gave_up) {  // nothing is merged; the CTA's memory stays until its copies have arrived
    if (copies && lane < W)
      for (int s = 0; s < kStages; ++s) kv4::drain(&full[lane][s], s < c_stage ? c_phase ^ 1 : c_phase);
    return;
  }
  // the CTA's pairs that reach into others: at most one at its begin (0) and one at its end (1)
  __shared__ int span[2][5];  // row (-1: none), item, CTAs c0 .. c1, slot of c0's partial (the others' are 0)
  if (tid < 2) span[tid][0] = -1;
  __syncthreads();
  {
    const Part p = lane < 2 * kWarps ? parts[lane] : Part{-1, 0, 0, 0};
    const unsigned valid = __ballot_sync(0xffffffffu, p.row >= 0);
    const unsigned below = valid & ((1u << lane) - 1);
    const int prev = below ? 31 - __clz(below) : lane;
    const int prow = __shfl_sync(0xffffffffu, p.row, prev), pitem = __shfl_sync(0xffffffffu, p.item, prev);
    const unsigned begins = __ballot_sync(0xffffffffu, p.row >= 0 && (!below || prow != p.row || pitem != p.item));
    // all pairs at once: a warp takes one head of one pair, or finds the CTAs that a pair spans
    const int pairs = __popc(begins), work = pairs * HPI;
#pragma unroll 1
    for (int x = warp; x < work + pairs; x += kThreads / 32) {
      const bool merges = x < work;
      const int g = merges ? x / HPI : x - work, h = x - g * HPI;
      unsigned left = begins;
#pragma unroll 1
      for (int i = g; i > 0; --i) left &= left - 1;
      const int i0 = __ffs(left) - 1;
      const unsigned rest = left & (left - 1);
      const unsigned set = valid & ~((1u << i0) - 1) & (rest ? (rest & -rest) - 1 : ~0u);
      const int i1 = 31 - __clz(set);
      const Part f = parts[i0];
      const int u1 = parts[i1].u1, units = (rows[f.row].y + 15) >> 4;
      const bool done = f.u0 == 0 && u1 == units;
      const int at0 = before[f.row] + f.item * (units + kVisit) + kVisit;  // place of its unit 0
      const int slot = at0 + f.u0 <= w0 ? 0 : 1;
      if (merges && h < heads_of(f.item)) {
        float* dst = done ? nullptr : g_.part + ((int64_t)cta * 2 + slot) * pstride;
        // a pair begins with its first warp's last partial and goes on in the next warps' last ones, the last
        // warp's may be a first one; or it has but a first one
        int i = i0 + 2 * lane;
        if (i == i1 + 1) i = i1;
        const bool live = i <= i1 && (set >> i & 1);
        if (!live) i = i0;
        const float* from = i & 1 ? reinterpret_cast<const float*>(smem + (i >> 1) * Sh::kRing) : firsts + (i >> 1) * pstride;
        merge_parts<HD, 4>(from, live, ((i1 | 1) - i0) / 2 + 1, h * Sh::kRow, h * Sh::kRow + HD, sink_of(dst, f.item, h),
                           merge_to(dst, f.row, f.item, h, HD));
      } else if (!merges && !done && lane == 0) {
        const int c0 = part_of(at0) / W;
        span[slot][1] = f.item;
        span[slot][2] = c0;
        span[slot][3] = part_of(at0 + units - 1) / W;
        span[slot][4] = part_begin(c0 * W) < at0 ? 1 : 0;
        span[slot][0] = f.row;
      }
    }
  }
  // Round 0: the last CTA of a pair to arrive sums its partials; where there are many, the last of each
  // kTree CTAs sums theirs, and in round 1 the last of these sums the sums.
#pragma unroll 1
  for (int round = 0; round < 2; ++round) {
    __threadfence();
    __syncthreads();
    if (span[0][0] < 0 && span[1][0] < 0) break;
    if (tid < 2) {
      int last = 0;
      const int* sp = span[tid];
      if (sp[0] >= 0) {
        const int n = sp[3] - sp[2] + 1, g0 = (cta - sp[2]) / kTree * kTree;
        const bool deep = n > kFlat;
        int* counter = g_.counters + sp[2];
        int want = n;
        if (deep && round == 0) {
          counter = g_.counters + gridDim.x + 2 * (sp[2] + g0) + (g0 == 0 ? sp[4] : 0);
          want = min(kTree, n - g0);
        } else if (deep) {
          want = (n + kTree - 1) / kTree;
        }
        last = atomicAdd(counter, 1) == want - 1;
        if (last) *counter = 0;
      }
      last_s[tid] = last;
    }
    __syncthreads();
    __threadfence();
    bool again = false;
#pragma unroll 1
    for (int x = warp; x < 2 * HPI; x += kThreads / 32) {
      const int s = x >= HPI ? 1 : 0;
      if (!last_s[s]) continue;
      const int row = span[s][0], item = span[s][1], c0 = span[s][2], n = span[s][3] - c0 + 1, first = span[s][4];
      const bool deep = n > kFlat, inner = deep && round == 0;
      const int g0 = inner ? (cta - c0) / kTree * kTree : 0, step = deep && round ? kTree : 1;
      const int cnt = inner ? min(kTree, n - g0) : deep ? (n + kTree - 1) / kTree : n;
      float* part = g_.part + (int64_t)(c0 + g0) * 2 * pstride;
      const int off = g0 == 0 ? first * pstride : 0;
      const bool live = lane < cnt;
      const float* from = part + (live && lane ? lane * 2 * step * pstride : off);
      const int h = x - s * HPI;
      if (h < heads_of(item)) {  // a sum's reference and sum go beside the first partial's: others still read those
        float* dst = inner ? part + off : nullptr;
        merge_parts<HD, 8>(from, live, cnt, h * Sh::kRow, h * Sh::kRow + (deep && round ? HD + 2 : HD), sink_of(dst, item, h),
                        merge_to(dst, row, item, h, HD + 2));
      }
    }
    for (int s = 0; s < 2; ++s) again |= last_s[s] && round == 0 && span[s][3] - span[s][2] + 1 > kFlat;
    if (!again) break;
    // only the spans summed in this round arrive in the next
    __syncthreads();
    if (tid < 2 && !(last_s[tid] && span[tid][3] - span[tid][2] + 1 > kFlat)) span[tid][0] = -1;
  }
  pdl_launch();
}

template <int HD>
void launch_decode(const DecodeArgs& d, int sms, cudaStream_t s, bool pdl) {
  using Sh = DecodeShape<HD>;
  static bool configured = false;  // per instantiation; one device per process
  if (!configured) {
    HK_CUDA_CHECK(cudaFuncSetAttribute(kv4_decode_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       Sh::kSmem));
    configured = true;
  }
  launch(kv4_decode_kernel<HD>, dim3(std::min(sms, kMaxCtas)), dim3(Sh::kThreads), Sh::kSmem, s, pdl, d);
}

}  // namespace

void kv4_attention_decode_launch(const Kv4AttnArgs& args, const Kv4Workspace& ws, cudaStream_t s, bool pdl) {
  const int G = args.nh / args.nkv;
  // rows of a launch: the sum of their units and visits x items stays below 2^31 by more than the kernel adds to it
  const int64_t most = ((int64_t)args.max_blocks * (args.block_size / 16) + kVisit) * args.nkv * 2;
  const int chunk = (int)std::min<int64_t>(kMaxRows, ((int64_t(1) << 31) - (1 << 20)) / most);
  if (chunk < 1) throw std::runtime_error("kv4 attention decode: context x kv heads too large");
  for (int r0 = 0; r0 < args.R; r0 += chunk) {
    DecodeArgs d{};
    d.a = args;
    d.a.R = args.R - r0 < chunk ? args.R - r0 : chunk;
    d.a.q += r0 * args.q_stride;
    d.a.row_seq += r0;
    d.a.row_ctx += r0;
    if (d.a.out) d.a.out += r0 * args.outf_stride;
    if (d.a.out_bf16) d.a.out_bf16 += r0 * args.out_stride;
    d.part = ws.part;
    d.counters = ws.counters;
    d.heads_per_item = G < kKv4ItemHeads ? G : kKv4ItemHeads;
    d.split = G > kKv4ItemHeads ? 1 : 0;
    const int upb = args.block_size / 16;
    d.upb_shift = (upb & (upb - 1)) ? -1 : __builtin_ctz(upb);
    if (args.hd == 64) launch_decode<64>(d, ws.sms, s, pdl);
    else if (args.hd == 128) launch_decode<128>(d, ws.sms, s, pdl);
    else if (args.hd == 256) launch_decode<256>(d, ws.sms, s, pdl);
    else throw std::runtime_error("kv4 attention: head_dim 64, 128 or 256");
  }
}

}  // namespace hk
