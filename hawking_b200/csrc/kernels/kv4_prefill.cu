// Prefill attention over the 4-bit paged KV cache on the 5th-generation tensor cores.
//
// Mathematics: o = softmax(scale q K^T) V per query row over its first row_ctx tokens, with one pass over
// the keys, a running reference and sum per row, float16 operands and fp32 accumulators in tensor
// memory. Keys and values enter as c + s (code - 8) rounded once to float16, the query as float16 after an
// exact power-of-two scaling of its row, the weights p as float16 (p <= 2^8: the reference moves only when a
// score passes it by more, so the output accumulator is rescaled rarely).
//
// A CTA owns 256 (query row, query head) pairs of one kv head, two tiles of 128, so that every key and value
// it unpacks serves 256 rows whatever the number of heads per kv head. 512 threads:
//   warps 0-3, 4-7   softmax of tile 0 and 1: one thread per row reads its 128 scores from tensor memory,
//                    writes the weights back over them and, at the end, the output
//   warps 8-11       unpack 128 tokens at a time from global memory (registers one tile ahead) to two shared
//                    memory stages of keys and of values
//   warps 13-15      fetch the query rows by bulk copies at the begin
//   warp 12          issues the matrix instructions: S_t = Q_t K^T (both operands in shared memory) and
//                    O_t += P_t V (P from tensor memory), the two tiles alternating so that one tile's
//                    products run during the other's softmax
// Token order. The unpackers hold 8 tokens of a head dim in a thread as their nibbles lie in a value word;
// the keys of a tile are written in that order too, so scores, weights and values agree: column
// 32 v + 8 t + 4 b + 2 h + e of a tile is token 32 v + 16 b + 8 h + 2 t + e.
//
// Rows of different sequences may share a CTA: it goes through their runs one after the other. Where there are
// fewer CTAs than SMs the keys are split over blockIdx.z; the last CTA of a tile to arrive adds the parts.
// One block of 512 threads per SM: the tiles fill the tensor memory (2 x 128 columns of scores, 2 x HD of output) and the
// softmax threads need 168 registers, which the unpackers (112) and the issuing warpgroup (64) give up. Four unpacking
// warps keep ahead of the products; with eight, in 640 threads, the softmax threads spilled and it was slower.
//
// What bounds it, on one B200, 32 / 8 heads of 128. 2048 rows after 6144 tokens: 299 us, 0.8 PFLOP/s, 0.49 of the
// measured bf16 rate. 256 equal CTAs on 148 SMs take two turns where 1.73 would do; within a CTA 128 keys take 2.8 us,
// the exchange of scores and weights through tensor memory 48 % busy and issue slots 47 %: the softmax of a tile, not
// the products (1.8 us by themselves), paces the loop. A CTA's begin (queries fetched and scaled, first keys unpacked) takes 6 us and its
// end (output read and written) 3.6, so 2048 rows from an empty cache, 8.5 tiles of keys on average, take 59 us. Loads of
// the query rows by a thread per row, 32 lines with every load, made that 64; 16 lanes per row with the maximum by
// shuffles, and 8 lanes per row for the output, 70. Fewer CTAs than SMs: 256 rows after 4096 tokens took 66 us with the keys split
// over blockIdx.z and 102 without.
// A value group that holds NaN is unpacked as zeros and noted: rows that see the token get NaN in its 64
// dims at the end (a weight of zero times NaN would reach every row of the tile).
#include <algorithm>

#include "kv4.cuh"
#include "sm100.cuh"

namespace hk {
namespace {

using namespace sm100;
using kv4::Unit;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRows = 256;     // (row, head) pairs per CTA
constexpr int kKeys = 128;     // tokens per tile
constexpr int kThreads = 512;
// Registers a thread: at launch, then by role (softmax two warpgroups, unpack and matrix instructions one
// each). An increase waits for registers that the other roles gave up, so the shares must fit the launch's total.
constexpr int kRegsLaunch = 128, kRegsSoftmax = 168, kRegsUnpack = 112, kRegsIssue = 64;
static_assert(2 * 128 * kRegsSoftmax + 128 * kRegsUnpack + 128 * kRegsIssue <= kThreads * kRegsLaunch &&
                  kRegsUnpack <= kRegsLaunch && kRegsIssue <= kRegsLaunch && kRegsSoftmax >= kRegsLaunch,
              "setmaxnreg shares exceed the block's registers");
constexpr float kHead = 8.f;   // log2 of how far a score may exceed the reference
constexpr int kMaxRuns = kRows + 1;

struct PrefillArgs {
  Kv4AttnArgs a;
  int splits;        // parts of the keys (grid.z)
  int upb_shift;     // log2 of the units per block, or -1
  float* part;       // [grid.x * grid.y * splits][256][HD + 4]
  int* counters;     // [grid.x * grid.y], zero between launches
};

template <int HD>
struct PrefillShape {
  static constexpr int kAtom = 128 * 128;                 // 128 rows of 64 float16
  static constexpr int kQTile = (HD / 64) * kAtom;        // one tile of queries
  static constexpr int kKStage = (HD / 64) * kAtom;       // 128 keys
  static constexpr int kVStage = 2 * HD * 128;            // HD rows (dims) of 128 tokens
  static constexpr int kOffK = 2 * kQTile;
  static constexpr int kOffV = kOffK + 2 * kKStage;
  static constexpr int kSmem = kOffV + 2 * kVStage + 1024;  // + alignment
  static_assert(kRows * (HD + 4) <= kKv4PartFloatsPerSm, "a CTA's part fits the workspace");
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ __half2 as_h2(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
// (code - 8) s + c of the even and odd nibble pairs of w
__device__ __forceinline__ uint32_t value_even(uint32_t w, __half2 s, __half2 c) {
  return as_u32(__hfma2(as_h2(kv4::centre_even(w)), s, c));
}
__device__ __forceinline__ uint32_t value_odd(uint32_t w, __half2 s, __half2 c) {
  return as_u32(__hfma2(as_h2(kv4::centre_odd(w)), s, c));
}

#define HK_R4(r, i) "=r"((r)[i]), "=r"((r)[i + 1]), "=r"((r)[i + 2]), "=r"((r)[i + 3])
#define HK_V4(r, i) "r"((r)[i]), "r"((r)[i + 1]), "r"((r)[i + 2]), "r"((r)[i + 3])
// 32 columns of this thread's lane
__device__ __forceinline__ void tmem_ld_x32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : HK_R4(r, 0), HK_R4(r, 4), HK_R4(r, 8), HK_R4(r, 12), HK_R4(r, 16), HK_R4(r, 20), HK_R4(r, 24), HK_R4(r, 28)
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld_x16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : HK_R4(r, 0), HK_R4(r, 4), HK_R4(r, 8), HK_R4(r, 12)
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st_x16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::HK_V4(r, 0),
      HK_V4(r, 4), HK_V4(r, 8), HK_V4(r, 12), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// The matrix instructions are issued by one elected lane of a converged warp (their operands then stay in
// uniform registers).
__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void commit_elected(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem desc]^T, float16 operands
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b_desc), "r"(idesc), "r"(acc)
      : "memory");
}
// float16 A and B (K major), fp32 D
__host__ __device__ constexpr uint32_t idesc_f16_f32(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
template <int N>
__device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ void sts16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 ldg16(const uint8_t* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }

template <int HD>
__global__ void __launch_bounds__(kThreads, 1) kv4_prefill_kernel(const __grid_constant__ PrefillArgs g_) {
  using U = Unit<HD>;
  using Sh = PrefillShape<HD>;
  constexpr int GR = HD / 64;
  const Kv4AttnArgs& a = g_.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_ready[2], p_ready[2], o_done[2], q_raw, q_ready, ended;
  __shared__ uint32_t tmem_s;
  __shared__ int seq_s[kMaxRuns], ctx_s[kMaxRuns], run_at[kMaxRuns + 1], run_kv[kMaxRuns];
  __shared__ int nan_at[kMaxRuns][GR];  // first token of a run whose value group holds NaN
  __shared__ int n_runs_s, kv_top_s, last_s;
  __shared__ volatile int gave_up;      // a wait of this CTA ran out
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wg = tid >> 7;
  const int G = a.nh / a.nkv, kvh = blockIdx.x, tile = gridDim.y - 1 - blockIdx.y;  // longest rows first
  const int m0 = tile * kRows, m_end = min(m0 + kRows, a.R * G);  // flat (row, head) pairs
  const int row0 = m0 / G, nrows = (m_end - 1) / G - row0 + 1;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 128);
      mbar_init(&v_full[i], 128);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_ready[i], 1);
      mbar_init(&p_ready[i], 128);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(&q_raw, 1);
    mbar_init(&q_ready, 256);
    mbar_init(&ended, 1);
    fence_barrier_init();
    kv_top_s = gave_up = 0;
  }
  pdl_wait();
  if (warp == 12) {  // (not before: a CTA of the previous launch may still need its columns to finish)
    tmem_alloc(&tmem_s, 512);
    tmem_relinquish();
  }
  // ---- runs of rows of one sequence ----
  for (int i = tid; i < nrows; i += kThreads) {
    const int seq = a.row_seq[row0 + i];
    int ctx = min(max(a.row_ctx[row0 + i], 0), a.max_blocks * a.block_size);
    if (seq < 0 || seq >= a.table_rows) {
      ctx = 0;
      set_error(a.status, HK_ERR_BAD_ARG);
    }
    seq_s[i] = seq;
    ctx_s[i] = ctx;
    run_kv[i] = 0;
#pragma unroll
    for (int g = 0; g < GR; ++g) nan_at[i][g] = 0x7fffffff;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) {
    int n = 0;
    for (int b = 0; b < nrows; b += 32) {
      const int i = b + lane;
      const bool live = i < nrows, begin = live && (i == 0 || seq_s[i] != seq_s[i - 1]);
      const unsigned m = __ballot_sync(0xffffffffu, begin);
      const int id = n + __popc(m & (0xffffffffu >> (31 - lane))) - 1;
      if (begin) run_at[id] = i;
      if (live) {
        atomicMax(&run_kv[id], ctx_s[i]);
        atomicMax(&kv_top_s, ctx_s[i]);
      }
      n += __popc(m);
    }
    if (lane == 0) {
      run_at[n] = nrows;
      n_runs_s = n;
    }
  }
  __syncthreads();
  const uint32_t tmem = tmem_s;
  const int n_runs = n_runs_s;
  // parts of the keys: at least two tiles each
  const int top_tiles = (kv_top_s + kKeys - 1) / kKeys;
  const int Z = min(g_.splits, max(1, top_tiles / 2)), z = blockIdx.z;
  const auto tiles_of = [&](int run, int& t0, int& t1) {
    const int n = (run_kv[run] + kKeys - 1) / kKeys;
    t0 = n * z / Z;
    t1 = n * (z + 1) / Z;
  };
  bool ok = true;  // the same for a warp
  const auto wait = [&](uint64_t* bar, uint32_t parity) {
    return ok = kv4::warp_wait(bar, parity, a.status, a.wait_polls);
  };
  const uint32_t smem_q = smem_u32(smem), smem_k = smem_q + Sh::kOffK, smem_v = smem_q + Sh::kOffV;
  if (z < Z) {
    if (wg < 2) {
      // ================================ softmax ================================
      regs_up<kRegsSoftmax>();
      const int t = wg, i = tid & 127, m = m0 + t * 128 + i;
      const int my_row = m < m_end ? m / G - row0 : -1;  // row of the CTA
      const int head = kvh * G + (m < m_end ? m % G : 0);
      const uint32_t lane_at = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t s_at = tmem + lane_at + t * 128, o_at = tmem + lane_at + 256 + t * 128;
      // this thread's query row: float16 after an exact scaling, from the raw rows into the swizzled tile (both for all
      // runs). The chunk that is read in step c, c ^ x i in GF(8), takes all banks in turn on both sides
      float mult;
      {
        if (!(ok = __all_sync(0xffffffffu, kv4::drain(&q_raw, 0)))) {  // (the CTA's memory stays until they have arrived)
          kv4::timed_out(a.status);
        }
        const int turn = ((i << 1) & 6) ^ (i & 4 ? 3 : 0);
        uint4 qr[HD / 8];
#pragma unroll
        for (int c = 0; c < HD / 8; ++c) {
          qr[c] = make_uint4(0u, 0u, 0u, 0u);
          if (m < m_end) qr[c] = *reinterpret_cast<const uint4*>(smem + (t * 128 + i) * HD * 2 + 16 * (c ^ turn));
        }
        asm volatile("bar.sync %0, 128;" ::"r"(1 + t) : "memory");  // the tile lies where its raw rows did
        __nv_bfloat162 top = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < HD / 8; ++c) {
          const uint32_t w[4] = {qr[c].x, qr[c].y, qr[c].z, qr[c].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) top = __hmax2(top, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[k])));
        }
        const float mx = fmaxf(__low2float(top), __high2float(top));
        const int ex = (int)(__float_as_uint(mx) >> 23);
        const bool norm = ex > 0 && ex < 254;  // 2^-e with 1 <= mx 2^-e < 2
        const uint32_t dn = norm ? (uint32_t)(254 - ex) << 7 : 0x3f80u, dn2 = dn | dn << 16;
        mult = (norm ? __uint_as_float((uint32_t)ex << 23) : 1.f) * (a.scale * kLog2e);
#pragma unroll
        for (int c = 0; c < HD / 8; ++c) {
          uint32_t w[4] = {qr[c].x, qr[c].y, qr[c].z, qr[c].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w[k]),
                                             *reinterpret_cast<const __nv_bfloat162*>(&dn2));
            w[k] = pack_f16(__low2float(y), __high2float(y));
          }
          const int chunk = c ^ turn;
          *reinterpret_cast<uint4*>(smem + t * Sh::kQTile + (chunk >> 3) * Sh::kAtom + sw128_offset(i, chunk & 7)) =
              make_uint4(w[0], w[1], w[2], w[3]);
        }
        fence_proxy_async_smem();
      }
      int s_phase = 0, o_phase = 0;
      for (int run = 0; run < n_runs && ok; ++run) {
        int t0, t1;
        tiles_of(run, t0, t1);
        const bool mine = my_row >= run_at[run] && my_row < run_at[run + 1];
        const int ctx = mine ? ctx_s[my_row] : 0;
        float ref = -INFINITY, l = 0.f;
        if (t1 > t0) {
          mbar_arrive(&q_ready);
          for (int j = t0; j < t1; ++j) {
            if (!wait(&s_ready[t], s_phase)) break;
            s_phase ^= 1;
            tc_fence_after();
            const int left = ctx - j * kKeys;  // tokens of the tile that the row sees
            // 64 scores, those that the row does not see at -infinity, and the largest of them
            uint32_t s[2][32];
            const bool edge = __any_sync(0xffffffffu, left < kKeys);
            const auto fetch = [&](int half) {
              tmem_ld_x32(s_at + 64 * half, s[0]);
              tmem_ld_x32(s_at + 64 * half + 32, s[1]);
              tmem_wait_ld();
              if (edge) {
#pragma unroll
                for (int c = 0; c < 64; ++c) {
                  const int tok = (c & 32) + ((c >> 2) & 1) * 16 + ((c >> 1) & 1) * 8 + ((c >> 3) & 3) * 2 + (c & 1);
                  if (64 * half + tok >= left) s[c >> 5][c & 31] = 0xff800000u;
                }
              }
            };
            const auto largest = [&](float top) {
              float t4[4] = {top, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
              for (int c = 0; c < 64; c += 2)
                t4[(c >> 1) & 3] = max3(t4[(c >> 1) & 3], __uint_as_float(s[c >> 5][c & 31]), __uint_as_float(s[c >> 5][(c & 31) + 1]));
              return fmaxf(max3(t4[0], t4[1], t4[2]), t4[3]);
            };
            fetch(1);
            const float top = largest(-INFINITY);
            fetch(0);
            const float mx = largest(top) * mult;
            const bool move = mx > ref + kHead;
            if (__any_sync(0xffffffffu, move)) {
              const float corr = move ? (ref > -INFINITY ? ex2(ref - mx) : 0.f) : 1.f;
              if (move) ref = mx;
              l *= corr;
              if (j > t0) {  // the products before this tile's scores are complete: rescale their sum
#pragma unroll 1
                for (int c = 0; c < HD; c += 16) {
                  uint32_t o[16];
                  tmem_ld_x16(o_at + c, o);
                  tmem_wait_ld();
#pragma unroll
                  for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * corr);
                  tmem_st_x16(o_at + c, o);
                }
              }
            }
            const float base = ref > -INFINITY ? -ref : 0.f;
            const uint64_t mult2 = pack2(mult, mult), base2 = pack2(base, base);
            uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              if (half == 1) fetch(1);  // (the first half's weights lie over its own scores)
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                uint32_t p[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                  float lo, hi;
                  unpack2(fma2(pack2(__uint_as_float(s[q][2 * k]), __uint_as_float(s[q][2 * k + 1])), mult2, base2), lo, hi);
                  lo = ex2(lo);
                  hi = ex2(hi);
                  sum2[k & 1] = add2(sum2[k & 1], pack2(lo, hi));
                  p[k] = pack_f16(lo, hi);
                }
                tmem_st_x16(s_at + 32 * half + 16 * q, p);
              }
            }
            float s0, s1;
            unpack2(add2(sum2[0], sum2[1]), s0, s1);
            l += s0 + s1;
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&p_ready[t]);
          }
          if (ok && wait(&o_done[t], o_phase)) {
            o_phase ^= 1;
            tc_fence_after();
          }
        }
        // the rows' outputs (or partials)
        const bool any = t1 > t0 && ok;
        float* part = g_.part + (((int64_t)z * gridDim.y + tile) * gridDim.x + kvh) * kRows * (HD + 4) +
                      (int64_t)(t * 128 + i) * (HD + 4);
        float f = 0.f;
        if (Z == 1 && any) {
          float lt = l;
          if (a.sinks) lt += ex2(kv4::sink_over(a.sinks[head], ref > -INFINITY ? ref : 0.f));
          f = ctx > 0 ? __frcp_rn(lt) : 0.f;
        } else if (any) {
          f = 1.f;
        }
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
          uint32_t o[32];
          __syncwarp();  // (rows that are not of this run skip the rest of the turn)
          if (any) {  // (the same for the whole warp)
            tmem_ld_x32(o_at + c, o);
            tmem_wait_ld();
          }
          if (!mine) continue;
          const bool bad = any && ctx > nan_at[run][c >> 6];
          float v[32];
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            v[k] = any && ctx > 0 ? __uint_as_float(o[k]) * f : 0.f;
            if (bad) v[k] = __uint_as_float(0x7fffffffu);
          }
          if (Z > 1) {
#pragma unroll
            for (int k = 0; k < 32; k += 4)
              __stcg(reinterpret_cast<float4*>(part + c + k), make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]));
            if (c == 0) __stcg(reinterpret_cast<float2*>(part + HD), make_float2(any && ctx > 0 ? ref : -INFINITY, l));
            continue;
          }
          const int64_t row = row0 + my_row, col = (int64_t)head * HD + c;
          if (a.out_bf16) {
#pragma unroll
            for (int k = 0; k < 32; k += 8) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const __nv_bfloat162 h2 = __floats2bfloat162_rn(v[k + 2 * e], v[k + 2 * e + 1]);
                w[e] = *reinterpret_cast<const uint32_t*>(&h2);
              }
              *reinterpret_cast<uint4*>(a.out_bf16 + row * a.out_stride + col + k) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
          if (a.out) {
#pragma unroll
            for (int k = 0; k < 32; k += 4)
              *reinterpret_cast<float4*>(a.out + row * a.outf_stride + col + k) =
                  make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
          }
        }
        tc_fence_before();  // (the next run's products overwrite what was read here: q_ready orders them)
      }
    } else if (wg == 2) {
      // ================================ unpack ================================
      regs_down<kRegsUnpack>();
      const int w = warp & 3;  // tokens 32 w .. of the tile: units 2 w, 2 w + 1
      const int upb = a.block_size / 16;
      int n_done = 0;
      const int* table = nullptr;
      int units = 0;
      // block of unit u (-1 past the sequence's end), and the unit's bytes; a block outside the cache reads as zeros
      const auto block_of = [&](int u) {
        return u < units ? table[g_.upb_shift >= 0 ? u >> g_.upb_shift : u / upb] : -1;
      };
      const auto unit_at = [&](int u, int blk) -> const uint8_t* {
        if (blk < 0 || blk >= a.cache_blocks) {
          if (u < units) set_error(a.status, HK_ERR_BAD_ARG);
          return nullptr;
        }
        const int in = g_.upb_shift >= 0 ? u & (upb - 1) : u % upb;
        return a.cache + (((int64_t)blk * a.nkv + kvh) * upb + in) * U::kBytes;
      };
      // keys: a thread has 16 bytes (HD 64: 8) of tokens 4 i + kx of unit 2 w + b
      const int b = (lane >> 2) & 1, kt = lane & 3, kx = lane >> 3;
      // values: 16 bytes of both units, tokens 8 h + 2 vt, + 1 of dims 4 vg .. of each 32
      const int vt = lane & 3, vg = lane >> 2;
      {
        for (int run = 0; run < n_runs && ok; ++run) {
          int t0, t1;
          tiles_of(run, t0, t1);
          if (t1 <= t0) continue;
          const int kv_len = run_kv[run];
          units = (kv_len + 15) >> 4;
          table = a.block_tables + (int64_t)seq_s[run_at[run]] * a.max_blocks;
          uint4 kr[4];
          uint2 kp[4];
          const auto load_k = [&](const uint8_t* ku) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              kr[i] = make_uint4(0u, 0u, 0u, 0u);
              kp[i] = make_uint2(0u, 0u);
              if (ku) {
                const int tok = 4 * i + kx;
                if (HD == 64) {
                  const uint2 x = __ldg(reinterpret_cast<const uint2*>(ku + tok * U::kRow + kt * 8));
                  kr[i].x = x.x, kr[i].y = x.y;
                  kp[i].x = __ldg(reinterpret_cast<const uint32_t*>(ku + U::pair(false, tok, 0)));
                } else {
                  kr[i] = ldg16(ku + tok * U::kRow + kt * 16);
                  kp[i] = __ldg(reinterpret_cast<const uint2*>(ku + U::pair(false, tok, 0)));
                }
              }
            }
          };
          uint4 vr[2][GR];  // values of units 2 w, 2 w + 1
          uint4 vp[2][2];   // pairs of tokens 8 h + 2 vt, + 1
          const auto load_v = [&](int x, const uint8_t* vu) {
#pragma unroll
            for (int g = 0; g < GR; ++g) {
              vr[x][g] = make_uint4(0u, 0u, 0u, 0u);
              if (vu) vr[x][g] = ldg16(vu + U::kCodes + g * 512 + lane * 16);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              vp[x][h] = make_uint4(0u, 0u, 0u, 0u);
              if (vu) {
                const int tok = 8 * h + 2 * vt;
                if (HD == 64) {
                  const uint2 y = __ldg(reinterpret_cast<const uint2*>(vu + U::pair(true, tok, 0)));
                  vp[x][h].x = y.x, vp[x][h].z = y.y;
                } else {
                  vp[x][h] = ldg16(vu + U::pair(true, tok, 0));
                }
              }
            }
          };
          const auto load = [&](int u, int blk0, int blk1) {
            const uint8_t *u0 = unit_at(u, blk0), *u1 = unit_at(u + 1, blk1);
            load_k(b ? u1 : u0);
            load_v(0, u0);
            load_v(1, u1);
          };
          int u = 8 * t0 + 2 * w;
          load(u, block_of(u), block_of(u + 1));
          int blk0 = block_of(u + 8), blk1 = block_of(u + 9);  // of the tile after the loaded one
          for (int j = t0; j < t1; ++j, ++n_done) {
            const int st = n_done & 1;
            if (!wait(&k_empty[st], ((n_done >> 1) & 1) ^ 1)) break;
            const uint32_t ks = smem_k + st * Sh::kKStage + (32 * w + (kx >> 1) * 8 + b * 4 + (kx & 1)) * 128;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              // row 32 w + 8 (2 (i & 1) + (kx >> 1)) + 4 b + 2 (i >> 1) + (kx & 1) of the tile
              const int r = (2 * (i & 1)) * 8 + (i >> 1) * 2;
              const uint32_t x[4] = {kr[i].x, kr[i].y, kr[i].z, kr[i].w};
#pragma unroll
              for (int k = 0; k < HD / 32; ++k) {
                const __half2 p = as_h2(k < 2 ? kp[i].x : kp[i].y);
                const __half2 s = __low2half2(p), c = __high2half2(p);
                const int chunk = (4 * (k & 1) + kt) ^ (4 * b + 2 * (i >> 1) + (kx & 1));
                sts16(ks + (k >> 1) * Sh::kAtom + r * 128 + chunk * 16, value_even(x[k], s, c), value_odd(x[k], s, c),
                      value_even(x[k] >> 8, s, c), value_odd(x[k] >> 8, s, c));
              }
            }
            fence_proxy_async_smem();
            mbar_arrive(&k_full[st]);
            // scales and centres of the token pairs [unit][half][group]
            uint32_t s2[2][2][GR], c2[2][2][GR];
            __half2 odd = __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
            const __half2 zero = odd;
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int g = 0; g < GR; ++g) {
                  const uint32_t p0 = g ? vp[x][h].y : vp[x][h].x, p1 = g ? vp[x][h].w : vp[x][h].z;
                  s2[x][h][g] = __byte_perm(p0, p1, 0x5410);
                  c2[x][h][g] = __byte_perm(p0, p1, 0x7632);
                  odd = __hfma2(as_h2(s2[x][h][g]), zero, __hfma2(as_h2(c2[x][h][g]), zero, odd));
                }
            // the sequence's last tokens hold stale bytes past its end; NaN is noted: both become zeros
            const bool end = (j + 1) * kKeys > kv_len;
            if (end || (as_u32(odd) & 0x7fff7fffu)) {
#pragma unroll
              for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                  for (int g = 0; g < GR; ++g) {
                    const int tok = j * kKeys + 32 * w + 16 * x + 8 * h + 2 * vt;
                    const uint32_t sv = s2[x][h][g], cv = c2[x][h][g];
                    const bool odd0 = (~sv & 0x7c00u) == 0 || (~cv & 0x7c00u) == 0;
                    const bool odd1 = (~sv & 0x7c000000u) == 0 || (~cv & 0x7c000000u) == 0;
                    const bool end0 = tok >= kv_len, end1 = tok + 1 >= kv_len;
                    if (odd0 && !end0) atomicMin(&nan_at[run][g], tok);
                    if (odd1 && !end1) atomicMin(&nan_at[run][g], tok + 1);
                    const uint32_t keep = (odd0 || end0 ? 0u : 0xffffu) | (odd1 || end1 ? 0u : 0xffff0000u);
                    s2[x][h][g] = sv & keep;
                    c2[x][h][g] = cv & keep;
                  }
            }
            if (!wait(&v_empty[st], ((n_done >> 1) & 1) ^ 1)) break;
            const uint32_t vs = smem_v + st * Sh::kVStage + (w >> 1) * HD * 128 + 4 * vg * 128;
#pragma unroll
            for (int g = 0; g < GR; ++g)
#pragma unroll
              for (int il = 0; il < 2; ++il) {
                uint32_t x[2][2];
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                  x[y][0] = il ? vr[y][g].z : vr[y][g].x;
                  x[y][1] = il ? vr[y][g].w : vr[y][g].y;
                }
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                  uint32_t o[4];
#pragma unroll
                  for (int y = 0; y < 4; ++y) {
                    const int xx = y >> 1, h = y & 1;
                    const uint32_t v = p < 2 ? x[xx][h] : x[xx][h] >> 8;
                    o[y] = p & 1 ? value_odd(v, as_h2(s2[xx][h][g]), as_h2(c2[xx][h][g]))
                                 : value_even(v, as_h2(s2[xx][h][g]), as_h2(c2[xx][h][g]));
                  }
                  // row 64 g + 32 il + 4 vg + p
                  const int chunk = (4 * (w & 1) + vt) ^ (4 * (vg & 1) + p);
                  sts16(vs + (64 * g + 32 * il + p) * 128 + chunk * 16, o[0], o[1], o[2], o[3]);
                }
              }
            fence_proxy_async_smem();
            mbar_arrive(&v_full[st]);
            if (j + 1 < t1) {
              u += 8;
              load(u, blk0, blk1);
              blk0 = block_of(u + 8);
              blk1 = block_of(u + 9);
            }
          }
        }
      }
    } else {
      // ================================ matrix instructions ================================
      regs_down<kRegsIssue>();
      if (warp == 12) {
        constexpr uint32_t id_s = idesc_f16_f32(128, kKeys), id_o = idesc_f16_f32(128, HD);
        int n_k = 0, n_v = 0, p_phase = 0, q_phase = 0;
        // (descriptor addresses count 16 bytes)
        const uint64_t dq = sdesc_k_sw128(smem_q), dk = sdesc_k_sw128(smem_k), dv = sdesc_k_sw128(smem_v);
        const auto scores = [&](int t, int st) {
          const uint64_t q0 = dq + t * (Sh::kQTile >> 4), k0 = dk + st * (Sh::kKStage >> 4);
#pragma unroll 1
          for (int at = 0; at < HD / 64; ++at)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t off = at * (Sh::kAtom >> 4) + k * 2;
              umma_f16_ss(tmem + t * 128, q0 + off, k0 + off, id_s, (at | k) > 0);
            }
          commit_elected(&s_ready[t]);
        };
        const auto output = [&](int t, int st, bool more) {
          const uint64_t v0 = dv + st * (Sh::kVStage >> 4);
#pragma unroll 1
          for (int at = 0; at < kKeys / 64; ++at)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + at * 32 + 8 * k, v0 + at * (HD * 128 >> 4) + k * 2, id_o,
                          more || (at | k) > 0);
        };
        for (int run = 0; run < n_runs && ok; ++run) {
          int t0, t1;
          tiles_of(run, t0, t1);
          if (t1 <= t0) continue;
          if (!wait(&q_ready, q_phase) || !wait(&k_full[n_k & 1], (n_k >> 1) & 1)) break;
          q_phase ^= 1;
          tc_fence_after();
          scores(0, n_k & 1);
          scores(1, n_k & 1);
          commit_elected(&k_empty[n_k & 1]);
          ++n_k;
          for (int j = t0; j < t1 && ok; ++j, ++n_v) {
            const int vst = n_v & 1, kst = n_k & 1;
            const bool more = j + 1 < t1;
            wait(&v_full[vst], (n_v >> 1) & 1);
#pragma unroll 1
            for (int t = 0; t < 2; ++t) {
              if (ok) wait(&p_ready[t], p_phase);
              if (ok && more && t == 0) wait(&k_full[kst], (n_k >> 1) & 1);
              if (!ok) break;
              tc_fence_after();
              output(t, vst, j > t0);
              if (t == 1) commit_elected(&v_empty[vst]);
              if (more) scores(t, kst);
              else commit_elected(&o_done[t]);
              if (more && t == 1) commit_elected(&k_empty[kst]);
            }
            if (more) ++n_k;
            p_phase ^= 1;
          }
        }
      } else {  // the query rows, as they lie, to the tiles' place: a row's heads of the kv head in one copy
        if (tid == 13 * 32) mbar_arrive_expect_tx(&q_raw, (m_end - m0) * HD * 2);
        for (int i = tid - 13 * 32; i < nrows; i += 3 * 32) {
          const int b = max(m0, (row0 + i) * G), e = min(m_end, (row0 + i + 1) * G);
          bulk_g2s(smem + (b - m0) * HD * 2,
                   a.q + (int64_t)(row0 + i) * a.q_stride + (int64_t)(kvh * G + b - (row0 + i) * G) * HD, (e - b) * HD * 2,
                   &q_raw);
        }
      }
    }
    if (!ok) gave_up = 1;
  }
  __syncthreads();
  tc_fence_after();
  if (warp == 12) {
    __syncwarp();
    if (gave_up) {  // products may be under way
      commit_elected(&ended);
      kv4::drain(&ended, 0);
      __syncwarp();
    }
    tmem_dealloc(tmem, 512);
  }
  if (z >= Z || Z == 1 || gave_up) return;
  // ---- parts of the keys: the last CTA of the tile adds them, in order ----
  __threadfence();
  __syncthreads();
  if (tid == 0) {
    int* counter = g_.counters + tile * gridDim.x + kvh;
    last_s = atomicAdd(counter, 1) == Z - 1;
    if (last_s) *counter = 0;
  }
  __syncthreads();
  if (!last_s) return;
  __threadfence();
  const int64_t step = (int64_t)gridDim.y * gridDim.x * kRows * (HD + 4);
  const float* first = g_.part + ((int64_t)tile * gridDim.x + kvh) * kRows * (HD + 4);
  for (int x = tid; x < (m_end - m0) * (HD / 4); x += kThreads) {
    const int i = x / (HD / 4), d = x % (HD / 4) * 4, m = m0 + i;
    const int row = m / G, head = kvh * G + m % G;
    const float* p = first + (int64_t)i * (HD + 4);
    float r = a.sinks ? kv4::sink_log2(a.sinks[head]) : -INFINITY;
    float lt = a.sinks ? 1.f : 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = 0; k0 < Z; k0 += 4) {
      float2 ml[4];
      float4 o[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        ml[k] = make_float2(-INFINITY, 0.f);
        o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (k0 + k < Z) {
          ml[k] = __ldcg(reinterpret_cast<const float2*>(p + (k0 + k) * step + HD));
          o[k] = __ldcg(reinterpret_cast<const float4*>(p + (k0 + k) * step + d));
        }
      }
      float top = r;
#pragma unroll
      for (int k = 0; k < 4; ++k) top = fmaxf(top, ml[k].x);
      const float base = fmaxf(top, -1e30f), f = ex2(r - base);
      r = top;
      lt *= f;
      v.x *= f, v.y *= f, v.z *= f, v.w *= f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float e = ex2(ml[k].x - base);
        v.x = fmaf(o[k].x, e, v.x), v.y = fmaf(o[k].y, e, v.y), v.z = fmaf(o[k].z, e, v.z), v.w = fmaf(o[k].w, e, v.w);
        lt = fmaf(ml[k].y, e, lt);
      }
    }
    const float f = ctx_s[row - row0] > 0 ? __frcp_rn(lt) : 0.f;
    v.x *= f, v.y *= f, v.z *= f, v.w *= f;
    const int64_t col = (int64_t)head * HD + d;
    if (a.out_bf16) {
      const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
      *reinterpret_cast<uint2*>(a.out_bf16 + row * a.out_stride + col) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
    if (a.out) *reinterpret_cast<float4*>(a.out + row * a.outf_stride + col) = v;
  }
}

template <int HD>
void launch_prefill(const PrefillArgs& p, dim3 grid, cudaStream_t s, bool pdl) {
  static bool configured = false;  // per instantiation; one device per process
  if (!configured) {
    HK_CUDA_CHECK(cudaFuncSetAttribute(kv4_prefill_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       PrefillShape<HD>::kSmem));
    cudaFuncAttributes at;
    HK_CUDA_CHECK(cudaFuncGetAttributes(&at, kv4_prefill_kernel<HD>));
    // (the register shares count on it: a smaller allocation would leave the increases waiting)
    if (at.numRegs != kRegsLaunch) throw std::runtime_error("kv4 attention prefill: built with another register count");
    configured = true;
  }
  launch(kv4_prefill_kernel<HD>, grid, dim3(kThreads), PrefillShape<HD>::kSmem, s, pdl, p);
}

}  // namespace

void kv4_attention_prefill_launch(const Kv4AttnArgs& args, const Kv4Workspace& ws, cudaStream_t s, bool pdl) {
  if (args.R <= 0) return;
  const int64_t pairs = (int64_t)args.R * (args.nh / args.nkv), tiles = (pairs + kRows - 1) / kRows;
  if (pairs >= (int64_t(1) << 31) - kRows || tiles > 65535) throw std::runtime_error("kv4 attention prefill: too many rows");
  PrefillArgs p{};
  p.a = args;
  p.part = ws.part;
  p.counters = ws.counters;
  // with fewer CTAs than SMs the keys are split over the rest (256 rows after 4096 tokens: 66 us against 102; three short
  // prompts of 64-wide heads, where there is little to split, 29.2 against 28.8)
  const int upb = args.block_size / 16;
  p.upb_shift = (upb & (upb - 1)) ? -1 : __builtin_ctz(upb);
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(32, ws.sms / (tiles * args.nkv)));
  const dim3 grid(args.nkv, (unsigned)tiles, p.splits);
  if (args.hd == 64) launch_prefill<64>(p, grid, s, pdl);
  else if (args.hd == 128) launch_prefill<128>(p, grid, s, pdl);
  else throw std::runtime_error("kv4 attention prefill: head_dim 64 or 128");
}

}  // namespace hk
