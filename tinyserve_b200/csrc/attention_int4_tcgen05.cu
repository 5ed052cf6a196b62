// Attention of prompt portions over a paged cache in 4 bits, on the 5th-generation tensor cores: bfloat16 queries, head size 64 or 128
// (-DTS_HEAD_DIM).  The mathematics and the use of tensor memory are those of attention_tcgen05.cu (two tiles of 128 rows = (query, head) of one
// key head take turns on the tensor core, S = Q K^T, P written over S, O += P V, one softmax thread a row, maxima that move by
// more than 2^8 only); keys and values come differently.  Four warps make them: a thread reads a key's row of codes (64 bytes at 128
// columns) and its pair, and writes the row as 16-bit numbers into the swizzled tile that the tensor core reads: a code becomes the number
// 1 + c / 16 (one shift, one AND-OR for two codes), times 16 scale, plus zero - 16 scale (rounded once for the row; the value once more).  That is
// 400 instructions a thread for a tile of 128 keys, while the tensor core takes 2,000 cycles for the tile's four products.
// Nothing is expanded in memory: a portion of any length behind a context of any length needs no scratch.
//
// The 16 bits are those of half precision (11 significant bits, where bfloat16 has 8): the codes' values, the queries and the probabilities lose
// nothing that shows behind the rounding of the output (2,048 queries over 4,096 keys, 32 heads of 128 on 8, relative error of the output:
// in bfloat16 4.4e-3, so 1.7e-3, which is that rounding alone; exact codes, with scales and zeros applied to every score and probability, came
// to 2.3e-3 and took 271 us instead of 131).  Its range is short, so powers of two keep everything inside: one a row for the queries, one a tile for the keys,
// and one for the values of all tiles so far, with which the sums in tensor memory are rescaled when it grows.  (From the
// pairs of the tile at hand: a look at all of a block's pairs beforehand took 30 us.)  Half precision holds 2^26 that way: where the
// keys of a tile or the values of a block lie further apart than 2^24, whoever sees them, the makers say so and the block's rows are made again in 32
// bits, by one warp each.  (That takes 35 ms for the portion above, and no model's cache is like that; without it, a key that only later queries see
// could take the bits of the others' values.  Looking for it costs 1 us of 131.)
//
// That portion takes 132 us, 0.78 PFLOP/s.  What bounds it is the chain of a query tile's steps: 2,000 cycles from its scores to its last
// probabilities, 900 until the issuing thread has put P V and the next scores in the pipe, 600 until these are seen, with the other tile's chain beside
// it (with one matrix instruction a product, tiles made twice only and hardly any softmax still 88 us).  Then come the start of a block (22 us for
// 256 blocks of one tile) and the makers (11 us).  The subtraction of 1024 that an earlier form of the makers had cost 10 us; pairs of 32-bit operations in
// the softmax save 5; probabilities in one part or in four instead of two took 143 us,
// steps of 64 keys with the scores of two steps in tensor memory 168, two softmax threads a row 217 (what they wait for one another
// weighs more than what overlaps).
//
// A key whose pair is not finite becomes a key of NaN with a value of zeros: who sees it gets NaN, who does not is not touched (its
// probability of 0 would not survive a NaN in V).
//
// 512 threads: warp 0 loads the queries, warp 1 issues, warps 4-7 and 8-11 are the softmax of the two tiles (168 registers), 12-15 make keys and
// values.  Blocks find their request themselves (a scan over the query offsets), so that no list is cut on the host and a captured graph
// serves any step of its shape.  Every wait is bounded; a block that gives up raises ts_attention_int4_tcgen05_error.
#include <cuda_fp16.h>

#include "entry.cuh"
#include "pairs.cuh"
#include "softcap.cuh"
#include "tcgen05.cuh"

#ifndef TS_HEAD_DIM
#error "compile with -DTS_HEAD_DIM=64 or 128"
#endif

TS_DEFINE_LAST_ERROR()

namespace {

using bf16 = __nv_bfloat16;
constexpr int D = TS_HEAD_DIM;
static_assert(D == 64 || D == 128, "the tcgen05 prefill kernel takes head sizes 64 and 128");
constexpr int BM = 128;                      // rows of a query tile
constexpr int BN = 128;                      // keys of a tile
constexpr int GROUPS = 2;                    // query tiles of a block
constexpr int P_PARTS = 2;                   // the probabilities of a key tile are handed over in this many parts
constexpr int SOFTMAX_WARP0 = 4, MAKER_WARP0 = 12, THREADS = 512;
constexpr int K_STAGES = 2, V_STAGES = 2;
constexpr int DCH = D / 64;                  // 64-column chunks of a head
constexpr int CHUNK_BYTES = 128 * 128;       // 128 rows of 128 bytes
constexpr int Q_BYTES = DCH * CHUNK_BYTES;
constexpr int KV_BYTES = DCH * CHUNK_BYTES;  // one of K or V of a tile
constexpr int TMEM_COLS = 512;               // S_0, S_1: 128 columns each (P_g over the first 64 of S_g); O_0 at 256, O_1 at 384
constexpr int W4 = D / 32;                   // 16-byte pieces of a row of codes
constexpr size_t SMEM = 1024 + GROUPS * Q_BYTES + (K_STAGES + V_STAGES) * KV_BYTES + 512;
constexpr int RANGES = 4;                    // tiles whose exponents are kept
constexpr float P_UP = 7.f;                  // probabilities are written times 2^7: up to 2^15, so that those of long rows stay above 2^-24
// scores up to this many powers of two: beyond, score * scale - maximum in one rounding is off by the half step that the maximum was rounded by,
// which as a power of two passes half precision, and in the end 32 bits
constexpr float FAR = 65536.f;
constexpr int HIGHEST = 12;                  // the largest of what is scaled goes to 2^12 .. 2^13 (half precision ends at 65,504)
constexpr float LOG2E = 1.4426950408889634f;

struct Params {
  bf16* out;                // [T, H, D]
  const uint4 *kc, *vc;     // codes
  const uint32_t *kp, *vp;  // pairs
  const int* block_table;   // [B, table_stride]
  const int* cu_q;          // [B + 1]
  const int* kv_lens;       // [B]
  int T, B, H, Hkv, page_shift, max_blocks, table_stride, num_pages;
  int heads_per_tile, queries_per_tile, head_tiles;     // of one query tile
  int few;                  // requests of up to this many queries are somebody else's
  int window;
  const float* sinks;       // [H] or null
  float scale_log2;
  float cap2, cap_in;       // a soft cap c > 0: c log2(e) and scale / c
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t halves2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// columns 2 E and 2 E + 1 of a word's eight, as scale * c + zero
template <int E>
__device__ __forceinline__ uint32_t values2(uint32_t word, __half2 scale, __half2 zero) {
  const uint32_t moved = E < 2 ? word << (6 - 4 * E) : word >> (4 * E - 6);
  uint32_t two;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(two) : "r"(moved), "r"(0x03c003c0u), "r"(0x3c003c00u));
  const __half2 v = __hfma2(*reinterpret_cast<const __half2*>(&two), scale, zero);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// instruction descriptor of kind::f16 with half precision on both sides (make_idesc has bfloat16)
__host__ __device__ constexpr uint32_t idesc_half(int M, int N, bool b_mn_major) { return make_idesc(M, N, b_mn_major) & ~((1u << 7) | (1u << 10)); }
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(min(max(e, -126), 127) + 127) << 23); }
// the exponent that the largest magnitude (as bits) has; for 0 and what is not finite HIGHEST, so that nothing is scaled for them
__device__ __forceinline__ int exponent_of(uint32_t bits) { return bits == 0 || bits >= 0x7f800000u ? HIGHEST : max((int)(bits >> 23) - 127, -100); }
__device__ __forceinline__ float pair_scale(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float pair_zero(uint32_t pair) { return __uint_as_float(pair & 0xffff0000u); }
constexpr int WIDEST = 24;                   // powers of two between the largest and the least magnitude that half precision is trusted with
// `least`: a magnitude but 0, as bits, less one (so that 0, all ones, is never the least)
__device__ __forceinline__ bool too_wide(int exponent, uint32_t least) { return exponent + 127 - (int)(least >> 23) > WIDEST; }
__device__ __forceinline__ bool finite_pair(uint32_t pair) {
  return (pair & 0x7f80u) != 0x7f80u && (pair & 0x7f800000u) != 0x7f800000u;
}

// A row (query, head) by one warp in 32 bits, for the blocks whose keys or values are too far apart for half precision (see `wide`; what a row does
// not see, or gives no weight, must not cost the others their bits) and for scores beyond FAR.  Lanes are 32 keys for the scores, and D / 32 columns each for their sum.
__device__ __noinline__ void whole_row(const Params& p, const char* q_tile, int r, float q_down, const int* bt, int kvh, int from, int pos, float sink, bf16* out, int lane) {
  constexpr int W = D / 8, SHARE = 32 / W, CPL = D / 32;          // words of a row, lanes of a word, columns of a lane
  const uint32_t* kc = reinterpret_cast<const uint32_t*>(p.kc);
  const uint32_t* vc = reinterpret_cast<const uint32_t*>(p.vc);
  auto unit = [&](int u) { return *reinterpret_cast<const uint4*>(q_tile + r * 128 + (u / 8) * CHUNK_BYTES + (((u % 8) ^ (r & 7)) << 4)); };
  auto halves = [](uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); };
  float o[CPL] = {}, m = -INFINITY, l = 0.f;
  for (int j0 = from; j0 <= pos; j0 += 32) {
    const int j = j0 + lane;
    const bool seen = j <= pos;
    int page = seen ? bt[j >> p.page_shift] : 0;
    if ((unsigned)page >= (unsigned)p.num_pages) page = 0;          // (reported when the tile was made)
    const size_t row = (((size_t)page * p.Hkv + kvh) << p.page_shift) + (j & ((1 << p.page_shift) - 1));
    const uint32_t k_pair = seen ? p.kp[row] : 0u, v_pair = seen ? p.vp[row] : 0u;
    float dot = 0.f, sum = 0.f;
#pragma unroll 4
    for (int u = 0; u < W; ++u) {
      const uint4 q8 = unit(u);
      const uint32_t w = seen ? kc[row * W + u] : 0u;
      const uint32_t q2[4] = {q8.x, q8.y, q8.z, q8.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 x = halves(q2[e]);
        dot = fmaf(x.x, (float)(int)(w >> (4 * e) & 15u) - 8.f, fmaf(x.y, (float)(int)(w >> (4 * e + 16) & 15u) - 8.f, dot));
        sum += x.x + x.y;
      }
    }
    const float ks = pair_scale(k_pair);
    float s = fmaf(ks, dot * q_down, fmaf(8.f, ks, pair_zero(k_pair)) * (sum * q_down));
    s = p.cap2 > 0.f ? p.cap2 * tanhf(s * p.cap_in) : s * p.scale_log2;
    if (!finite_pair(k_pair) || !finite_pair(v_pair)) s = __int_as_float(0x7fc00000);
    if (!seen) s = -INFINITY;
    float top = s;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float m_new = fmaxf(m, top), base = m_new == -INFINITY ? 0.f : m_new, alpha = exp2f(m - base), weight = exp2f(s - base);
    float total = weight;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    l = fmaf(l, alpha, total);
    m = m_new;
#pragma unroll
    for (int e = 0; e < CPL; ++e) o[e] *= alpha;
    // (a key behind the row's last has weight 0, pair 0 and stands in page 0; a pair that is not finite made the weight a NaN, which l has)
#pragma unroll 8
    for (int k = 0; k < 32; ++k) {
      const float w = __shfl_sync(0xffffffffu, weight, k);
      const uint32_t pair = __shfl_sync(0xffffffffu, v_pair, k), word = vc[__shfl_sync(0xffffffffu, (unsigned long long)row, k) * W + lane / SHARE];
      const float vs = finite_pair(pair) ? pair_scale(pair) : 0.f, vz = finite_pair(pair) ? pair_zero(pair) : 0.f;
#pragma unroll
      for (int e = 0; e < CPL; ++e) {
        const int i = lane % SHARE * CPL + e;
        o[e] = fmaf(w, fmaf((float)(int)(word >> ((i >> 1) * 4 + (i & 1) * 16) & 15u), vs, vz), o[e]);
      }
    }
  }
  const float sink2 = sink * LOG2E, m_new = fmaxf(m, sink2), base = m_new == -INFINITY ? 0.f : m_new, alpha = exp2f(m - base);
  l = fmaf(l, alpha, exp2f(sink2 - base));
#pragma unroll
  for (int e = 0; e < CPL; ++e) out[lane * CPL + e] = __float2bfloat16_rn(l == 0.f ? 0.f : o[e] * alpha / l);
}

// CAPPED: with a soft cap, whose code in the loop would cost the calls without one (2,048 queries over 4,096 keys 130.5 us, in one kernel
// for both 133; with a cap 270)
template <bool CAPPED>
__global__ void __launch_bounds__(THREADS, 1)
int4_prefill_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ Params p) {
  extern __shared__ char smem_raw[];
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  char* Qs = smem;                               // [GROUPS][Q_BYTES]
  char* Ks = Qs + GROUPS * Q_BYTES;              // [K_STAGES][KV_BYTES]
  char* Vs = Ks + K_STAGES * KV_BYTES;           // [V_STAGES][KV_BYTES]
  uint64_t* bars = reinterpret_cast<uint64_t*>(Vs + V_STAGES * KV_BYTES);
  uint64_t* q_full = bars;                       // 1: the queries have landed
  uint64_t* q_ready = q_full + 1;                // the softmax warps: ... and are in half precision
  uint64_t* seen = q_ready + 1;                  // the makers' four warps have seen the tile's pairs
  uint64_t* range = seen + 1;                    // [RANGES] the exponents of a tile's keys and values are known (a place is free when it
                                                 // comes up again: keys four tiles on need the scores of two tiles on, which come
                                                 // behind the probabilities of one tile on)
  uint64_t* k_full = range + RANGES;             // [K_STAGES] the makers' four warps
  uint64_t* k_empty = k_full + K_STAGES;         // [K_STAGES] both tiles' scores of the stage's keys are computed
  uint64_t* v_full = k_empty + K_STAGES;         // [V_STAGES]
  uint64_t* v_empty = v_full + V_STAGES;         // [V_STAGES] the stage's values are added to both O
  uint64_t* s_full = v_empty + V_STAGES;         // [GROUPS] S_g holds the scores of a key tile
  uint64_t* p_full = s_full + GROUPS;            // [GROUPS][P_PARTS] the part of P_g is in tensor memory, O_g is rescaled
  uint64_t* o_ready = p_full + GROUPS * P_PARTS; // [GROUPS] O_g holds the sum over the key tiles so far
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_ready + GROUPS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint32_t* largest = tmem_slot + 2;             // [2][8]: largest magnitudes of a tile's keys and values, by maker warp
  int2* exponents = reinterpret_cast<int2*>(largest + 16);       // [RANGES]
  volatile int* wide = reinterpret_cast<volatile int*>(exponents + RANGES);      // a tile's keys, or the values so far, are too far apart for half precision

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(q_full), 1);
    mbar_init(smem_u32(q_ready), GROUPS * 4);
    mbar_init(smem_u32(seen), 4);
    for (int s = 0; s < RANGES; ++s) mbar_init(smem_u32(&range[s]), 1);
    for (int s = 0; s < K_STAGES; ++s) {
      mbar_init(smem_u32(&k_full[s]), 4);
      mbar_init(smem_u32(&k_empty[s]), 1);
    }
    for (int s = 0; s < V_STAGES; ++s) {
      mbar_init(smem_u32(&v_full[s]), 4);
      mbar_init(smem_u32(&v_empty[s]), 1);
    }
    for (int g = 0; g < GROUPS; ++g) {
      mbar_init(smem_u32(&s_full[g]), 1);
      for (int h = 0; h < P_PARTS; ++h) mbar_init(smem_u32(&p_full[g * P_PARTS + h]), 4);
      mbar_init(smem_u32(&o_ready[g]), 1);
    }
    *abort_flag = *wide = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n"
                 ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // This block holds all of the SM's tensor memory now: only now may a dependent kernel start.
  pdl_wait();
  pdl_trigger();

  // block x from the last: the tiles of all requests in a row, the latest queries (the most keys) first
  const int QPT = p.queries_per_tile, GT = p.heads_per_tile, per_block = GROUPS * QPT;
  const int G = p.H / p.Hkv;
  int b = -1, q0 = 0, q_begin = 0, q_len = 0, held = 0;
  {
    int total = 0;
    for (int at = 0; at < p.B; at += 32) {
      const int n = at + lane < p.B ? min(p.cu_q[at + lane + 1], p.T) - p.cu_q[at + lane] : 0;
      if (at + lane < p.B) asm volatile("prefetch.global.L1 [%0];" ::"l"(p.kv_lens + at + lane));
      total += n > p.few ? (n + per_block - 1) / per_block : 0;
    }
    total = __reduce_add_sync(0xffffffffu, total);
    const int want = total - 1 - (int)blockIdx.x;
    int before = 0;
    for (int at = 0; at < p.B && want >= 0 && b < 0; at += 32) {
      const int from = at + lane < p.B ? p.cu_q[at + lane] : 0, n = at + lane < p.B ? min(p.cu_q[at + lane + 1], p.T) - from : 0;
      const int kv = at + lane < p.B ? p.kv_lens[at + lane] : 0;
      const int tiles = n > p.few ? (n + per_block - 1) / per_block : 0;
      int upto = tiles;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += y;
      }
      const uint32_t here = __ballot_sync(0xffffffffu, before + upto > want);
      if (here != 0) {
        const int who = __ffs(here) - 1;
        b = at + who;
        q0 = (want - before - __shfl_sync(0xffffffffu, upto - tiles, who)) * per_block;
        q_begin = __shfl_sync(0xffffffffu, from, who);
        q_len = __shfl_sync(0xffffffffu, n, who);
        held = __shfl_sync(0xffffffffu, kv, who);
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  const int kvh = blockIdx.y / p.head_tiles, head_tile = blockIdx.y % p.head_tiles;
  const int kv_len = (int)min((long long)held, (long long)p.max_blocks << p.page_shift);
  const int g0 = head_tile * GT;
  const int nq_all = max(0, min(per_block, q_len - q0));
  const int groups = nq_all > QPT ? 2 : 1;       // query tiles of this block that hold queries
  const int pos0 = kv_len - q_len + q0;
  const int j_hi = max(0, min(kv_len, pos0 + nq_all));
  const int j_lo = p.window > 0 ? max(0, pos0 - p.window + 1) : 0;
  const int first_tile = j_lo / BN;
  // (a block whose rows see no key at all still walks one tile, of which nothing is visible)
  const int n_tiles = nq_all > 0 ? max(1, (j_hi + BN - 1) / BN - first_tile) : 0;

  if (warp < SOFTMAX_WARP0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;\n");
    if (warp == 0 && lane == 0 && n_tiles > 0) {
      // queries: rows (query, head) with the head fastest; one box per 64 columns and query tile
      const uint32_t qbar = smem_u32(q_full);
      mbar_expect_tx(qbar, groups * DCH * 64 * 2 * GT * QPT);
      for (int g = 0; g < groups; ++g)
        for (int c = 0; c < DCH; ++c)
          tma_load_3d(smem_u32(Qs + g * Q_BYTES + c * CHUNK_BYTES), &map_q, qbar, c * 64, kvh * G + g0, q_begin + q0 + g * QPT);
    } else if (warp == 1 && n_tiles > 0 && elect_one()) {
      constexpr uint32_t idesc_qk = idesc_half(BM, BN, false);
      constexpr uint32_t idesc_pv = idesc_half(BM, D, true);
      constexpr int QK_STEPS = D / 16, PV_STEPS = BN / 16 / P_PARTS;
      const uint64_t q_desc = smem_desc(smem_u32(Qs)), k_desc = smem_desc(smem_u32(Ks));
      const uint64_t v_desc = smem_desc_mn(smem_u32(Vs), CHUNK_BYTES);
      // S_g = Q_g K^T of key tile t (the P V of tile g's previous key tile, which reads P_g from S_g's
      // columns, is in the pipe before it)
      auto scores = [&](int g, int t) -> bool {
        const int s = t % K_STAGES;
        if (!mbar_spin_wait(smem_u32(&k_full[s]), (t / K_STAGES) & 1, abort_flag)) return false;
        tcgen05_fence_after();
        const uint64_t qd = q_desc + g * (Q_BYTES >> 4), kd = k_desc + s * (KV_BYTES >> 4);
#pragma unroll
        for (int k = 0; k < QK_STEPS; ++k) {
          const uint64_t off = ((k / 4) * CHUNK_BYTES + (k % 4) * 32) >> 4;
          umma(tmem_base + g * BN, qd + off, kd + off, idesc_qk, k > 0 ? 1u : 0u);
        }
        tcgen05_commit(smem_u32(&s_full[g]));
        if (g == groups - 1) tcgen05_commit(smem_u32(&k_empty[s]));
        return true;
      };
      // O_g += P_g V of key tile t, a part of the keys at a time
      auto values = [&](int g, int t) -> bool {
        const int s = t % V_STAGES;
        if (!mbar_spin_wait(smem_u32(&v_full[s]), (t / V_STAGES) & 1, abort_flag)) return false;
        const uint64_t vd = v_desc + s * (KV_BYTES >> 4);
        const uint32_t o_addr = tmem_base + 2 * BN + g * 128, p_addr = tmem_base + g * BN;
#pragma unroll
        for (int h = 0; h < P_PARTS; ++h) {
          if (!mbar_spin_wait(smem_u32(&p_full[g * P_PARTS + h]), t & 1, abort_flag)) return false;
          tcgen05_fence_after();
#pragma unroll
          for (int i = 0; i < PV_STEPS; ++i) {
            const int k = h * PV_STEPS + i;
            umma_ts(o_addr, p_addr + k * 8, vd + ((k * 16 * 128) >> 4), idesc_pv, t > 0 || k > 0 ? 1u : 0u);
          }
        }
        tcgen05_commit(smem_u32(&o_ready[g]));
        if (g == groups - 1) tcgen05_commit(smem_u32(&v_empty[s]));
        return true;
      };
      bool ok = mbar_spin_wait(smem_u32(q_ready), 0, abort_flag);
      tcgen05_fence_after();
      for (int g = 0; ok && g < groups; ++g) ok = scores(g, 0);
      for (int t = 0; ok && t < n_tiles; ++t)
        for (int g = 0; ok && g < groups; ++g) {
          ok = values(g, t);
          if (ok && t + 1 < n_tiles) ok = scores(g, t + 1);
        }
    }
  } else if (warp >= MAKER_WARP0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;\n");
    // thread r makes row r of every tile
    const int r = threadIdx.x - MAKER_WARP0 * 32;
    const int* bt = p.block_table + (size_t)max(b, 0) * p.table_stride;
    struct Row { uint4 codes[W4]; uint32_t pair; };
    struct Where { size_t row; bool live; };
    // the row of the cache that tile t's key r stands in; live: it belongs to the block's range
    auto find = [&](int t) -> Where {
      const int j = (first_tile + t) * BN + r;
      const bool live = t < n_tiles && j >= j_lo && j < j_hi;
      int page = live ? bt[j >> p.page_shift] : 0;
      if ((unsigned)page >= (unsigned)p.num_pages) {
        ts_raise_status(TS_STATUS_BOUNDS, TS_BAD_PAGE);
        page = 0;
      }
      return {(((size_t)page * p.Hkv + kvh) << p.page_shift) + (j & ((1 << p.page_shift) - 1)), live};
    };
    auto read = [&](const uint4* codes, const Where& w, Row& row) {
#pragma unroll
      for (int i = 0; i < W4; ++i) row.codes[i] = w.live ? codes[w.row * W4 + i] : make_uint4(0u, 0u, 0u, 0u);
    };
    auto write = [&](char* tile, const Row& row, uint32_t pair, float factor) {
      const float s16 = 16.f * factor * pair_scale(pair);
      const __half2 scale = __float2half2_rn(s16), zero = __float2half2_rn(fmaf(pair_zero(pair), factor, -s16));
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const uint32_t w = i % 4 == 0 ? row.codes[i / 4].x : i % 4 == 1 ? row.codes[i / 4].y : i % 4 == 2 ? row.codes[i / 4].z : row.codes[i / 4].w;
        *reinterpret_cast<uint4*>(tile + (i / 8) * CHUNK_BYTES + r * 128 + (((i % 8) ^ (r & 7)) << 4)) =
            make_uint4(values2<0>(w, scale, zero), values2<1>(w, scale, zero), values2<2>(w, scale, zero), values2<3>(w, scale, zero));
      }
    };
    constexpr uint32_t NAN_PAIR = 0x7fc07fc0u;
    // the largest magnitude that a pair's codes can stand for
    auto reach = [](uint32_t pair) -> uint32_t {
      if (!finite_pair(pair)) return 0u;
      const float zero = pair_zero(pair), end = fmaf(15.f, pair_scale(pair), zero);
      return min(__float_as_uint(fmaxf(fabsf(zero), fabsf(end))), 0x7f7fffffu);
    };
    uint32_t top_v = 0, least_v = ~0u;          // of all tiles so far: the block's largest, this thread's least
    bool ok = true;
    // the next tile's keys are on their way while this tile's values are made, and these while its keys are
    Where at_k = find(0);
    Row k, v;
    read(p.kc, at_k, k);
    uint32_t k_pair = at_k.live ? p.kp[at_k.row] : 0u, v_pair = at_k.live ? p.vp[at_k.row] : 0u;
    auto hand_over = [&](uint64_t* full) {
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(full));
    };
    auto room = [&](uint64_t* empty, int round) -> bool {
      const bool got = mbar_wait(smem_u32(empty), (round & 1) ^ 1, abort_flag);
      return __all_sync(0xffffffffu, got);
    };
    for (int t = 0; ok && t < n_tiles; ++t) {
      read(p.vc, at_k, v);
      const Where next_k = find(t + 1);
      const bool good = finite_pair(k_pair) && finite_pair(v_pair);
      uint32_t* of_tile = largest + (t & 1) * 8;
      const uint32_t k_reach = reach(k_pair), v_reach = reach(v_pair);
      const uint32_t k_of_warp = __reduce_max_sync(0xffffffffu, k_reach), v_of_warp = __reduce_max_sync(0xffffffffu, v_reach);
      if (lane == 0) {
        of_tile[warp - MAKER_WARP0] = k_of_warp;
        of_tile[4 + warp - MAKER_WARP0] = v_of_warp;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(seen));
      ok = mbar_wait(smem_u32(seen), t & 1, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      top_v = max(top_v, max(max(of_tile[4], of_tile[5]), max(of_tile[6], of_tile[7])));
      const int k_exponent = exponent_of(max(max(of_tile[0], of_tile[1]), max(of_tile[2], of_tile[3]))), v_exponent = exponent_of(top_v);
      least_v = min(least_v, v_reach - 1u);
      if (too_wide(k_exponent, k_reach - 1u) || too_wide(v_exponent, least_v)) *wide = 1;          // (before the values are handed over)
      const float k_factor = power_of_two(HIGHEST - k_exponent), v_factor = power_of_two(HIGHEST - v_exponent);
      ok = room(&k_empty[t % K_STAGES], t / K_STAGES);
      if (!ok) break;
      if (r == 0) {
        exponents[t % RANGES] = make_int2(k_exponent, v_exponent);
        mbar_arrive(smem_u32(&range[t % RANGES]));
      }
      const uint32_t pair_of_v = good ? v_pair : 0u;
      write(Ks + (t % K_STAGES) * KV_BYTES, k, good ? k_pair : NAN_PAIR, k_factor);
      hand_over(&k_full[t % K_STAGES]);
      read(p.kc, next_k, k);
      k_pair = next_k.live ? p.kp[next_k.row] : 0u;
      v_pair = next_k.live ? p.vp[next_k.row] : 0u;
      ok = room(&v_empty[t % V_STAGES], t / V_STAGES);
      if (!ok) break;
      write(Vs + (t % V_STAGES) * KV_BYTES, v, pair_of_v, v_factor);
      hand_over(&v_full[t % V_STAGES]);
      at_k = next_k;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;\n");
    // one thread per row of query tile g
    const int g = (warp - SOFTMAX_WARP0) >> 2;
    if (g >= groups && lane == 0) mbar_arrive(smem_u32(q_ready));
    if (g < groups && n_tiles > 0) {
      const int q4 = warp & 3;
      const int r = q4 * 32 + lane;
      const int qg = q0 + g * QPT;                       // the tile's first query
      const int nq = min(QPT, q_len - qg);
      const int n_valid = QPT > 1 ? nq * GT : min(GT, G - g0);
      const bool valid = r < n_valid;
      const int qi = QPT > 1 ? r / GT : 0, gg = QPT > 1 ? r % GT : r;
      const int pos = valid ? kv_len - q_len + qg + qi : -1;
      const int lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
      const uint32_t lane_addr = static_cast<uint32_t>(q4 * 32) << 16;
      const uint32_t tmem_s = tmem_base + g * BN, tmem_o = tmem_base + 2 * BN + g * 128;
      float m = -INFINITY, l = 0.f;
      bool far = false;
      bool ok = mbar_wait(smem_u32(q_full), 0, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      // this thread's row of queries in half precision, its largest element at 2^12 .. 2^13 (rows behind the last are whatever lay there)
      char* mine = Qs + g * Q_BYTES + r * 128;
      auto unit = [&](int u) { return reinterpret_cast<uint4*>(mine + (u / 8) * CHUNK_BYTES + (((u % 8) ^ (r & 7)) << 4)); };
      uint32_t top = 0;
#pragma unroll
      for (int u = 0; u < D / 8; ++u) {
        const uint4 x = *unit(u);
        top = __vmaxu2(__vmaxu2(__vmaxu2(top, x.x & 0x7fff7fffu), x.y & 0x7fff7fffu), __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
      }
      const int q_exponent = exponent_of(max(top << 16, top & 0xffff0000u));
      const float up = power_of_two(HIGHEST - q_exponent);
#pragma unroll 4
      for (int u = 0; u < D / 8; ++u) {
        const uint4 x = *unit(u);
        auto both = [&](uint32_t w) { return halves2(__uint_as_float(w << 16) * up, __uint_as_float(w & 0xffff0000u) * up); };
        *unit(u) = make_uint4(both(x.x), both(x.y), both(x.z), both(x.w));
      }
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(q_ready));
      const float down = power_of_two(q_exponent - HIGHEST);           // of this row's scores
      int v_exponent = 0;
      for (int t = 0; ok && t < n_tiles; ++t) {
        const int j0 = (first_tile + t) * BN;
        ok = mbar_wait(smem_u32(&range[t % RANGES]), (t / RANGES) & 1, abort_flag) && mbar_wait(smem_u32(&s_full[g]), t & 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tcgen05_fence_after();
        const int2 of_tile = exponents[t % RANGES];
        const float k_down = down * power_of_two(of_tile.x - HIGHEST), grown = t > 0 ? power_of_two(v_exponent - of_tile.y) : 1.f;
        v_exponent = of_tile.y;
        const bool all_visible = j0 + BN - 1 <= pos && j0 >= lo;
        float sv[BN];
#pragma unroll
        for (int c = 0; c < BN; c += 32) tmem_load32_nowait(tmem_s + lane_addr + c, sv + c);
        tmem_load_wait();
        float sc = p.scale_log2 * k_down;
        if constexpr (CAPPED) {
          if (!all_visible) {
            // (a key that the row does not see has no say in how the others are capped)
#pragma unroll
            for (int e = 0; e < BN; ++e)
              if (j0 + e > pos || j0 + e < lo) sv[e] = 0.f;
          }
          // the usual case: every score of the row's tile is small against the cap
          const float w = p.cap_in * k_down;
          float big = 0.f;
#pragma unroll
          for (int e = 0; e < BN; ++e) {
            sv[e] *= w;
            big = fmaxf(big, fabsf(sv[e]));
          }
          if (big <= TANH_SMALL) {
#pragma unroll
            for (int e = 0; e < BN; ++e) {
              const float t = sv[e] * sv[e];
              sv[e] *= p.cap2 * fmaf(fmaf(fmaf(fmaf(TANH_P4, t, TANH_P3), t, TANH_P2), t, TANH_P1), t, TANH_P0);
            }
          } else {
#pragma unroll
            for (int e = 0; e < BN; ++e) sv[e] = p.cap2 * (1.f - __fdividef(2.f, ex2(sv[e] * (2.f * LOG2E)) + 1.f));
          }
          sc = 1.f;
        }
        if (!all_visible) {
#pragma unroll
          for (int e = 0; e < BN; ++e) {
            const int j = j0 + e;
            if (!(j <= pos && j >= lo)) sv[e] = -INFINITY;
          }
        }
        // the row's maximum, four independent chains
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < BN; e += 4) {
          mx4[0] = fmaxf(mx4[0], sv[e]);
          mx4[1] = fmaxf(mx4[1], sv[e + 1]);
          mx4[2] = fmaxf(mx4[2], sv[e + 2]);
          mx4[3] = fmaxf(mx4[3], sv[e + 3]);
        }
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
        // the reference maximum only moves when the row's maximum has grown by more than 2^8: until then the probabilities are taken
        // against the old reference and O needs no rescaling
        const float m_cand = fmaxf(m, mx * sc);
        const float m_new = (m_cand - m <= 8.f) ? m : m_cand;      // -inf - -inf: moves (to -inf), harmless
        const float m_safe = m_new == -INFINITY ? 0.f : m_new;
        far |= fabsf(m_safe) > FAR;
        const float alpha = ex2(m - m_safe), from = m_safe - P_UP;
        // probabilities -> tensor memory, pairs of half precision over the first 64 columns of S_g, handed over in P_PARTS parts
        F2 sum2[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
        const F2 sc2 = f2(sc, sc), from2 = f2(-from, -from);
#pragma unroll
        for (int h = 0; h < P_PARTS; ++h) {
#pragma unroll
          for (int c = h * (BN / P_PARTS); c < (h + 1) * (BN / P_PARTS); c += 32) {
            float packed[16];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              float p0, p1;
              f2_out(f2_fma(f2(sv[c + e], sv[c + e + 1]), sc2, from2), p0, p1);
              p0 = ex2(p0);        // -inf gives 0
              p1 = ex2(p1);
              sum2[(e / 2) & 1] = f2_add(sum2[(e / 2) & 1], f2(p0, p1));
              packed[e / 2] = __uint_as_float(halves2(p0, p1));
            }
            tmem_store16(tmem_s + lane_addr + c / 2, packed);
          }
          if (h == 0 && t > 0 && !__all_sync(0xffffffffu, alpha * grown == 1.f)) {
            // O_g is rescaled once half of the scores have left their registers, 32 columns at a time
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              float v[32];
              tmem_load32(tmem_o + lane_addr + c, v);
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] *= alpha * grown;
              tmem_store32(tmem_o + lane_addr + c, v);
            }
          }
          tmem_store_wait();
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&p_full[g * P_PARTS + h]));
        }
        float sum_a, sum_b;
        f2_out(f2_add(sum2[0], sum2[1]), sum_a, sum_b);
        l = l * alpha + (sum_a + sum_b);
        m = m_new;
      }
      if (ok) {
        // (the values' barrier for what the makers say in `wide`)
        ok = mbar_wait(smem_u32(&o_ready[g]), (n_tiles - 1) & 1, abort_flag) && mbar_wait(smem_u32(&v_full[(n_tiles - 1) % V_STAGES]), (n_tiles - 1) / V_STAGES & 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
      }
      if (ok && (__any_sync(0xffffffffu, far) || *wide)) {
        // row by row
        for (int i = 0; i < 32; ++i) {
          const int at = __shfl_sync(0xffffffffu, pos, i), from = __shfl_sync(0xffffffffu, lo, i);
          const int head = kvh * G + g0 + __shfl_sync(0xffffffffu, gg, i), token = q_begin + qg + __shfl_sync(0xffffffffu, qi, i);
          const float q_down = __shfl_sync(0xffffffffu, down, i);
          if (__shfl_sync(0xffffffffu, (int)valid, i))
            whole_row(p, Qs + g * Q_BYTES, q4 * 32 + i, q_down, p.block_table + (size_t)b * p.table_stride, kvh, from, at,
                      p.sinks != nullptr ? p.sinks[head] : -INFINITY, p.out + ((size_t)token * p.H + head) * D, lane);
        }
      } else if (ok) {
        tcgen05_fence_after();
        float alpha = 1.f;
        if (p.sinks && valid) {       // (log2 domain, like the running maximum; O is scaled on its way out)
          const float sk = p.sinks[kvh * G + g0 + gg] * LOG2E;
          const float top = fmaxf(m, sk), from = top == -INFINITY ? 0.f : top;          // (neither keys nor a sink)
          alpha = exp2f(m - from);
          l = l * alpha + exp2f(sk - from + P_UP);
        }
        const float inv = l == 0.f ? 0.f : alpha / l * power_of_two(v_exponent - HIGHEST);
        bf16* dst = p.out + ((size_t)(q_begin + qg + qi) * p.H + kvh * G + g0 + gg) * D;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          float v[32];
          tmem_load32(tmem_o + lane_addr + c, v);
          if (valid) {
#pragma unroll
            for (int e = 0; e < 32; e += 8)
              *reinterpret_cast<uint4*>(dst + c + e) =
                  make_uint4(pack2(v[e] * inv, v[e + 1] * inv), pack2(v[e + 2] * inv, v[e + 3] * inv),
                             pack2(v[e + 4] * inv, v[e + 5] * inv), pack2(v[e + 6] * inv, v[e + 7] * inv));
          }
        }
      }
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"((uint32_t)TMEM_COLS) : "memory");
  }
}

template <bool CAPPED>
int launch(const CUtensorMap& mq, const Params& p, dim3 grid, cudaStream_t stream) {
  static SmemSet set;
  const cudaError_t sized = set.to(int4_prefill_kernel<CAPPED>, (int)SMEM);
  if (sized != cudaSuccess) return ts_fail("int4_attention_tcgen05: %s", cudaGetErrorString(sized));
  TS_LAUNCH("int4_attention_tcgen05", int4_prefill_kernel<CAPPED>, grid, dim3(THREADS), SMEM, stream, mq, p);
  return 0;
}

}  // namespace

TS_EXPORT int ts_attention_int4_tcgen05_error() {
  int flag = 0;
  if (cudaMemcpyFromSymbol(&flag, g_error_flag, sizeof(int)) != cudaSuccess) return -1;
  return flag;
}

// q [T, H, D] (strides in elements, of 16 bytes), out [T, H, D]; codes and pairs as for ts_int4_attention.  Requests of up to `few` queries are left
// alone.
static int int4_attention_tcgen05(const void* q, long long q_row, long long q_head, void* out, const void* k_codes, const void* k_pairs,
                                  const void* v_codes, const void* v_pairs, const int* block_table, const int* cu_q, const int* kv_lens,
                                  int T, int B, int H, int Hkv, int page_size, int max_blocks, int table_stride, int num_pages, float scale,
                                  int window, float softcap, const float* sinks, int few, cudaStream_t stream) {
  int shift = 0;
  while (shift < 20 && (1 << shift) < page_size) ++shift;
  TS_REQUIRE(T > 0 && B > 0 && Hkv > 0 && H > 0 && H % Hkv == 0 && page_size == 1 << shift && num_pages > 0 && max_blocks > 0 && few >= 0,
             "int4_attention_tcgen05: %d tokens of %d requests, %d heads on %d, pages of %d", T, B, H, Hkv, page_size);
  TS_REQUIRE((((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_codes | (uintptr_t)v_codes) & 15) == 0 && ((uintptr_t)k_pairs | (uintptr_t)v_pairs) % 4 == 0 &&
                 (q_row * 2) % 16 == 0 && (q_head * 2) % 16 == 0 && q_row > 0 && q_head > 0, "int4_attention_tcgen05: operands must be 16-byte aligned");
  const int G = H / Hkv;
  Params p = {};
  p.out = (bf16*)out; p.kc = (const uint4*)k_codes; p.vc = (const uint4*)v_codes; p.kp = (const uint32_t*)k_pairs; p.vp = (const uint32_t*)v_pairs;
  p.block_table = block_table; p.cu_q = cu_q; p.kv_lens = kv_lens;
  p.T = T; p.B = B; p.H = H; p.Hkv = Hkv; p.page_shift = shift; p.max_blocks = max_blocks; p.table_stride = table_stride; p.num_pages = num_pages;
  p.few = few; p.window = window; p.sinks = sinks;
  p.scale_log2 = scale * LOG2E;
  p.cap2 = softcap > 0.f ? softcap * LOG2E : 0.f;
  p.cap_in = softcap > 0.f ? scale / softcap : 0.f;
  p.heads_per_tile = G < BM ? G : BM;
  p.queries_per_tile = G < BM ? BM / G : 1;
  p.head_tiles = (G + p.heads_per_tile - 1) / p.heads_per_tile;
  const long long gy = (long long)Hkv * p.head_tiles;
  TS_REQUIRE(gy <= 65535, "int4_attention_tcgen05: too many head tiles");
  // every request may end in a block that is not full; one of up to `few` queries has none
  const int per_block = GROUPS * p.queries_per_tile;
  const int with_tiles = T / (few + 1) < B ? T / (few + 1) : B;
  const int blocks = T / per_block + with_tiles;
  TS_REQUIRE(blocks > 0, "int4_attention_tcgen05: %d tokens hold no request of more than %d queries", T, few);
  CUtensorMap mq;
  {
    EncodeTiledFn fn = encode_tiled();
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)H, (cuuint64_t)T};
    const cuuint64_t strides[2] = {(cuuint64_t)q_head * 2, (cuuint64_t)q_row * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)p.heads_per_tile, (cuuint32_t)p.queries_per_tile}, elem[3] = {1, 1, 1};
    TS_REQUIRE(fn && fn(&mq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS,
               "int4_attention_tcgen05: tensor map of q failed");
  }
  return softcap > 0.f ? launch<true>(mq, p, dim3(blocks, (unsigned)gy), stream) : launch<false>(mq, p, dim3(blocks, (unsigned)gy), stream);
}
TS_ENTRY(int4_attention_tcgen05)
