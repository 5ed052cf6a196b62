// A paged cache held in 4 bits: the write of a step's keys and values, and attention over it.
//
// A key or value head of a token is D codes of 4 bits and a pair (scale, zero) of bfloat16: with everything in 32 bits,
//   zero = bfloat16(min x), scale = bfloat16((max x - zero) / 15), code = round((x - zero) / scale), halves to even, within 0 .. 15;
// a code stands for zero + code * scale.  The codes are taken against the rounded pair, so that the pair's own rounding costs
// at most a clamped end of the range.  A row that holds an infinity or a NaN, or whose range passes the largest
// 32-bit number, gets a pair of NaN: whoever attends to it gets NaN, as from a cache of whole numbers.
//
// Eight codes fill a 32-bit word: even columns in its lower half, odd ones in its upper half, the first in the lowest bits.
// One shift and one AND-OR then make a pair of neighbouring columns as two numbers in half precision (see `codes2` below).
// Codes [page, kv head, slot, D / 2] bytes, pairs [page, kv head, slot, 2]: one head's share of a page is one run of memory, 68 bytes
// a token for heads of 128 where bfloat16 takes 256.
#include <cuda_fp16.h>

#include "entry.cuh"
#include "rounding.cuh"
#include "tcgen05.cuh"

#ifndef TS_HEAD_DIM
#error "compile with -DTS_HEAD_DIM=<head size, a multiple of 16 up to 512>"
#endif

TS_DEFINE_LAST_ERROR()

namespace {

using bf16 = __nv_bfloat16;
constexpr int D = TS_HEAD_DIM;
static_assert(D % 16 == 0 && D >= 16 && D <= 512, "head sizes are multiples of 16 up to 512");
constexpr int W = D / 8;                     // words of a row
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float pair_scale(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float pair_zero(uint32_t pair) { return __uint_as_float(pair & 0xffff0000u); }
// where column i of a word's eight stands
__host__ __device__ constexpr int shift_of(int i) { return (i >> 1) * 4 + (i & 1) * 16; }

// ------------------------------------------------------------------------------------------ write
struct WriteParams {
  const void *k, *v;                         // [T, Hkv, D], columns contiguous
  long long k_row, k_head, v_row, v_head;    // strides in elements
  uint32_t *kc, *vc;                         // codes, W words a row
  uint32_t *kp, *vp;                         // pairs
  const int* slot_mapping;                   // [T]: page * page_size + slot, < 0: not written
  int T, Hkv, page_shift;
  long long slots;                           // of the pool
};
// a row's lanes, a power of two: of a word each for few tokens, of two for many, where a division and a reduction serve twice as much (8 heads
// of 128, 4,095 tokens 10.3 us by words, 7.4 by two, 7.3 by four; 64 tokens 1.7 / 1.8 / 2.6; with norm and rotation of 32 heads too, 2,048 tokens 20.9 /
// 17.3 / 20.2, 64 tokens 2.6 / 2.9 / 3.8)
constexpr int FEW_LANES = W > 16 ? 32 : (W > 8 ? 16 : (W > 4 ? 8 : (W > 2 ? 4 : 2)));
constexpr int MANY_LANES = W > 32 ? 32 : (W > 16 ? 16 : (W > 8 ? 8 : (W > 4 ? 4 : 2)));
constexpr int MANY_TOKENS = 256;
__host__ __device__ constexpr int words_of(int lanes) { return (W + lanes - 1) / lanes; }            // words of a lane
constexpr int WRITE_THREADS = 128;

template <typename T>
__device__ __forceinline__ void load8_any(const T* p, float (&x)[8], bool vec) {
  if (vec) {
    load8<T>(p, x);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32<T>(p[i]);
  }
}

// The least and the largest element of a row that LANES lanes have; a NaN if there is one
__device__ __forceinline__ float least(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float largest(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
template <int LANES>
struct RowRange {
  float lo = INFINITY, hi = -INFINITY;
  __device__ __forceinline__ void add(const float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      lo = least(least(lo, x[i]), x[i + 1]);
      hi = largest(largest(hi, x[i]), x[i + 1]);
    }
  }
  __device__ __forceinline__ void join() {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
      lo = least(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = largest(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
  }
};

__device__ __noinline__ float divided_code(float y, float scale) { return fminf(fmaxf(rintf(__fdiv_rn(y, scale)), 0.f), 15.f); }

// eight neighbouring columns as a word of codes.  The quotient rounded to 32 bits decides; a division is only made where the reciprocal could
// overflow.  Adding 1.5 2^23 rounds to a whole number, halves to even; four codes 4 bits apart are a sum of exact products below 2^16.
__device__ __forceinline__ uint32_t word_of(const float (&x)[8], float zero, float scale, bool outside) {
  constexpr float ROUNDER = 12582912.f;
  const float inverse = 1.f / scale;
  const F2 inv = f2(inverse, inverse), minus = f2(-scale, -scale), low = f2(-zero, -zero), up = f2(ROUNDER, ROUNDER), down = f2(-ROUNDER, -ROUNDER);
  F2 n[4];
  if (scale > 1e-30f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) n[i] = f2_quotient(f2_add(f2(x[2 * i], x[2 * i + 1]), low), minus, inv);
    if (outside) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float r0, r1;
        f2_out(n[i], r0, r1);
        n[i] = f2(fminf(fmaxf(r0, 0.f), 15.f), fminf(fmaxf(r1, 0.f), 15.f));
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) n[i] = f2_add(f2_add(n[i], up), down);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) n[i] = f2(divided_code(__fsub_rn(x[2 * i], zero), scale), divided_code(__fsub_rn(x[2 * i + 1], zero), scale));
  }
  const F2 step = f2(16.f, 16.f), four = f2_fma(f2_fma(f2_fma(n[3], step, n[2]), step, n[1]), step, n[0]);
  float even, odd;
  f2_out(f2_add(four, f2(8388608.f, 8388608.f)), even, odd);          // (2^23: the whole number is the low bits)
  return __byte_perm(__float_as_uint(even), __float_as_uint(odd), 0x5410);
}

// a row that its LANES lanes hold, to the slot of its token
template <int LANES>
__device__ __forceinline__ void store_row(const WriteParams& p, const float (&x)[words_of(LANES)][8], const RowRange<LANES>& r, int which, int head, int slot, int lane) {
  if (slot < 0) return;
  if (slot >= p.slots) {
    if (lane == 0) ts_raise_status(TS_STATUS_BOUNDS, TS_BAD_CACHE_SLOT);
    return;
  }
  const bf16 zero16 = __float2bfloat16_rn(r.lo);
  const float zero = __bfloat162float(zero16);
  const bf16 scale16 = __float2bfloat16_rn(__fdiv_rn(__fsub_rn(r.hi, zero), 15.f));
  const float scale = __bfloat162float(scale16);
  // (an infinity or a NaN in the row is one of its ends, and then the pair is not finite)
  const bool bad = !(fabsf(scale) <= 3.402823466e38f) || !(fabsf(zero) <= 3.402823466e38f);
  // the pair's rounding may leave ends of the row outside the codes: rarely, so that only such rows are clamped
  const bool outside = !(__fsub_rn(r.lo, zero) >= -0.4f * scale && __fsub_rn(r.hi, zero) <= 15.4f * scale);
  const size_t at = (((size_t)(slot >> p.page_shift) * p.Hkv + head) << p.page_shift) + (slot & ((1 << p.page_shift) - 1));
#pragma unroll
  for (int w = 0; w < words_of(LANES); ++w) {
    const int word = lane + w * LANES;
    if (word < W) (which ? p.vc : p.kc)[at * W + word] = !bad && scale > 0.f ? word_of(x[w], zero, scale, outside) : 0u;
  }
  if (lane == 0) {
    const uint32_t s = bad ? 0x7fc0u : (scale > 0.f ? __bfloat16_as_ushort(scale16) : 0u), z = bad ? 0x7fc0u : __bfloat16_as_ushort(zero16);
    (which ? p.vp : p.kp)[at] = s | z << 16;
  }
}

// LANES lanes bring one row (token, key or value, head) to its slot; a block's x is the token
template <typename T, int LANES>
__global__ void __launch_bounds__(WRITE_THREADS) int4_kvwrite_kernel(WriteParams p, bool vec) {
  constexpr int WORDS = words_of(LANES);
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x, row = blockIdx.y * (blockDim.x / LANES) + threadIdx.x / LANES, lane = threadIdx.x % LANES;
  const bool live = row < 2 * p.Hkv;
  const int which = row >= p.Hkv ? 1 : 0, head = row - which * p.Hkv;
  const int slot = p.slot_mapping[t];
  const T* src = which ? static_cast<const T*>(p.v) + t * p.v_row + head * p.v_head : static_cast<const T*>(p.k) + t * p.k_row + head * p.k_head;
  float x[WORDS][8];
  RowRange<LANES> r;
#pragma unroll
  for (int w = 0; w < WORDS; ++w) {
    const int word = lane + w * LANES;
    if (live && word < W) {
      load8_any<T>(src + word * 8, x[w], vec);
      r.add(x[w]);
    }
  }
  r.join();
  if (live) store_row(p, x, r, which, head, slot, lane);
}

// The same behind a fused projection: qkv [T, (H + 2 Hkv) D] -> q [T, H, D] and the cache.  Heads of q and k are divided by their root
// mean square (with weights; has_norm) and turned to their token's position; keys are rounded to T, as a cache
// of T would hold them, and then brought to 4 bits.
struct RopeParams {
  const void* qkv;
  void* q;
  const int* positions;
  const float *cos, *sin;                    // [positions, rot / 2]; null: no rotation
  int rot, interleaved;
  VecParam qw, kw;
  int has_norm;
  float eps;
  int H;
  // rows of q, k, v, weights and angles come in eights that begin on 16 bytes (halves of the rotation are whole eights too)
  bool vec, vec_weights, vec_angles;
};

template <typename T, int LANES>
__global__ void __launch_bounds__(WRITE_THREADS) int4_rope_kvwrite_kernel(WriteParams p, RopeParams rp) {
  constexpr int WORDS = words_of(LANES);
  __shared__ __align__(16) float stage[WRITE_THREADS / LANES][D];
  pdl_trigger();
  const int t = blockIdx.x, heads = rp.H + 2 * p.Hkv, head = blockIdx.y * (blockDim.x / LANES) + threadIdx.x / LANES, lane = threadIdx.x % LANES;
  const bool live = head < heads, is_q = head < rp.H, is_v = head >= rp.H + p.Hkv;
  const bool turned = live && !is_v;
  // (weights are nobody's output: they are on their way during the wait)
  float wt[WORDS][8];
  if (rp.has_norm) {
    const VecParam w8 = is_q ? rp.qw : rp.kw;
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
      const int word = lane + w * LANES;
      if (turned && word < W) {
        if (rp.vec_weights) {
          if (w8.is_f32) load8<float>(static_cast<const float*>(w8.ptr) + word * 8, wt[w]);
          else load8<bf16>(static_cast<const bf16*>(w8.ptr) + word * 8, wt[w]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) wt[w][i] = w8[word * 8 + i];
        }
      }
    }
  }
  pdl_wait();
  const T* src = static_cast<const T*>(rp.qkv) + ((size_t)t * heads + head) * D;
  const int slot = p.slot_mapping != nullptr ? p.slot_mapping[t] : -1;
  const int half = rp.rot >> 1;
  const size_t angles = rp.cos != nullptr ? (size_t)rp.positions[t] * half : 0;
  float x[WORDS][8], sum = 0.f;
#pragma unroll
  for (int w = 0; w < WORDS; ++w) {
    const int word = lane + w * LANES;
    if (live && word < W) {
      load8_any<T>(src + word * 8, x[w], rp.vec);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fmaf(x[w][i], x[w][i], sum);
    }
  }
  if (rp.has_norm) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float rstd = rsqrtf(sum / (float)D + rp.eps);
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
      if (turned && lane + w * LANES < W) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[w][i] = x[w][i] * rstd * wt[w][i];
      }
    }
  }
  if (rp.cos != nullptr) {
    float* mine = stage[threadIdx.x / LANES];
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
      const int word = lane + w * LANES;
      if (turned && word < W) store8<float>(mine + word * 8, x[w]);
    }
    __syncwarp();
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
      const int word = lane + w * LANES, d0 = word * 8;
      if (!turned || word >= W || d0 >= rp.rot) continue;
      if (rp.vec_angles) {
        // eight columns of one half with the eight of the other
        const bool first = d0 < half;
        const int j = first ? d0 : d0 - half;
        float mate[8], c[8], s[8];
        load8<float>(mine + (first ? d0 + half : d0 - half), mate);
        load8<float>(rp.cos + angles + j, c);
        load8<float>(rp.sin + angles + j, s);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[w][i] = first ? x[w][i] * c[i] - mate[i] * s[i] : x[w][i] * c[i] + mate[i] * s[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int d = d0 + i;
          if (d >= rp.rot) continue;
          const int j = rp.interleaved ? d >> 1 : (d < half ? d : d - half);
          const bool first = rp.interleaved ? (d & 1) == 0 : d < half;
          const float mate = mine[rp.interleaved ? d ^ 1 : (first ? d + half : d - half)];
          const float c = rp.cos[angles + j], s = rp.sin[angles + j];
          x[w][i] = first ? x[w][i] * c - mate * s : x[w][i] * c + mate * s;
        }
      }
    }
  }
  RowRange<LANES> r;
#pragma unroll
  for (int w = 0; w < WORDS; ++w) {
    const int word = lane + w * LANES;
    if (live && word < W) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[w][i] = to_f32<T>(from_f32<T>(x[w][i]));
      if (is_q) store8<T>(static_cast<T*>(rp.q) + ((size_t)t * rp.H + head) * D + word * 8, x[w]);
      else r.add(x[w]);
    }
  }
  r.join();
  if (live && !is_q) store_row(p, x, r, is_v ? 1 : 0, is_v ? head - rp.H - p.Hkv : head - rp.H, slot, lane);
}

// tokens x groups of a token's rows
struct RowGrid { dim3 grid, block; };
RowGrid row_grid(int tokens, int rows, int lanes) {
  const int threads = rows * lanes < WRITE_THREADS ? (rows * lanes + 31) / 32 * 32 : WRITE_THREADS;
  return {dim3(tokens, (rows + threads / lanes - 1) / (threads / lanes)), dim3(threads)};
}
template <typename T, int LANES>
int launch_write(const WriteParams& p, bool vec, cudaStream_t stream) {
  const RowGrid g = row_grid(p.T, 2 * p.Hkv, LANES);
  TS_REQUIRE(g.grid.y <= 65535, "int4_kvwrite: too many heads");
  TS_LAUNCH("int4_kvwrite", (int4_kvwrite_kernel<T, LANES>), g.grid, g.block, 0, stream, p, vec);
  return 0;
}
template <typename T, int LANES>
int launch_rope_write(const WriteParams& p, const RopeParams& rp, cudaStream_t stream) {
  const RowGrid g = row_grid(p.T, rp.H + 2 * p.Hkv, LANES);
  TS_REQUIRE(g.grid.y <= 65535, "int4_rope_kvwrite: too many heads");
  TS_LAUNCH("int4_rope_kvwrite", (int4_rope_kvwrite_kernel<T, LANES>), g.grid, g.block, 0, stream, p, rp);
  return 0;
}

// ------------------------------------------------------------------------------------------ attention
struct Int4Params {
  const void* q;                             // [T, H, D], columns contiguous
  long long q_row, q_head;                   // strides in elements
  void* out;                                 // [T, H, D]
  const uint32_t *kc, *vc;                   // codes
  const uint32_t *kp, *vp;                   // pairs
  const int* block_table;                    // [B, table_stride], max_blocks used
  const int* cu_q;                           // [B + 1]
  const int* kv_lens;                        // [B]
  int T, B, H, Hkv, page_shift, max_blocks, table_stride, num_pages;
  float scale;
  int window;
  float softcap;
  const float* sinks;                        // [H] or null: one more term exp(sinks[h]) in head h's sum
  int splits;                                // key ranges; > 1: partial results for the combine kernel
  float unit;                                // powers of two in a unit of the partial results' maxima
  int most;                                  // > 0: requests with more queries are somebody else's
  int ordered;                               // != 0: blocks take the requests by length, the longest first
  float *part_o, *part_ml;                   // [T * H][splits][D], [T * H][splits][2] (maximum, sum)
};

// the request that row t belongs to: the first b with cu_q[b + 1] > t (requests may be empty), -1 behind the last
__device__ __forceinline__ int request_of(const int* cu_q, int B, int t) {
  if (t >= cu_q[B]) return -1;
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu_q[mid + 1] > t) hi = mid; else lo = mid + 1;
  }
  return lo;
}
// row of key j of a request in the cache; a page number outside the pool is reported and read as page 0
__device__ __forceinline__ size_t cache_row(const Int4Params& p, int page, int kvh, int j) {
  if ((unsigned)page >= (unsigned)p.num_pages) {
    ts_raise_status(TS_STATUS_BOUNDS, TS_BAD_PAGE);
    page = 0;
  }
  return (((size_t)page * p.Hkv + kvh) << p.page_shift) + (j & ((1 << p.page_shift) - 1));
}
__device__ __forceinline__ float capped(const Int4Params& p, float s) { return p.softcap > 0.f ? p.softcap * tanhf(s / p.softcap) : s; }

// code i of a word as the 32-bit number 2^23 + c (adding or subtracting whole numbers to it is exact)
constexpr float CODE_BASE = 8388608.f;
__device__ __forceinline__ float code_above(uint32_t word, int i) { return __uint_as_float(0x4b000000u | (word >> shift_of(i) & 15u)); }

// The 32-bit form (and head sizes that the tensor-core kernel does not take): a block is one token's heads of one key head, up to eight
// at a time, and a range of its keys.  A thread makes the scores of one key of a tile of 128 for all its heads, so that a
// row of codes is read once; for P V a thread holds eight columns of all heads and walks every KG-th key.
// With a pair (s, z) of the key, q.k = s sum q (c - 8) + (z + 8 s) sum q: around the middle of the codes the two terms are small and little of
// them cancels.  Scores are exponentiated as 2^((score - maximum) log2 e): rounding the product instead of the score
// costs nothing where the score is large.
constexpr int SIMT_THREADS = 128, SIMT_KEYS = 128, SIMT_HEADS = 8, KG = SIMT_THREADS / W;

template <typename T>
__global__ void __launch_bounds__(SIMT_THREADS) int4_attend_kernel(Int4Params p) {
  __shared__ __align__(16) float qs[SIMT_HEADS][D];
  __shared__ float qsum[SIMT_HEADS], alpha[SIMT_HEADS], ml[SIMT_HEADS][2];
  __shared__ float prob[SIMT_HEADS][SIMT_KEYS];
  __shared__ size_t key_row[SIMT_KEYS];
  __shared__ uint32_t v_pair[SIMT_KEYS];
  __shared__ __align__(16) float red[SIMT_THREADS * 8];
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = p.H / p.Hkv, head_tiles = (G + SIMT_HEADS - 1) / SIMT_HEADS;
  const int kvh = blockIdx.y / head_tiles, g0 = blockIdx.y % head_tiles * SIMT_HEADS, split = blockIdx.z;
  const int nh = min(SIMT_HEADS, G - g0), h0 = kvh * G + g0;
  const int b = request_of(p.cu_q, p.B, t);
  if (b < 0) return;
  const int kv_len = (int)min((long long)p.kv_lens[b], (long long)p.max_blocks << p.page_shift);
  const int pos = kv_len - (p.cu_q[b + 1] - t);
  const int j_lo = p.window > 0 ? max(0, pos - p.window + 1) : 0, j_hi = max(pos + 1, j_lo);
  const int tiles = (j_hi - j_lo + SIMT_KEYS - 1) / SIMT_KEYS, per = (tiles + p.splits - 1) / p.splits;
  const int* bt = p.block_table + (size_t)b * p.table_stride;

  for (int i = tid; i < SIMT_HEADS * D; i += SIMT_THREADS) {
    const int h = i / D, d = i % D;
    qs[h][d] = h < nh ? to_f32<T>(static_cast<const T*>(p.q)[t * p.q_row + (h0 + h) * p.q_head + d]) : 0.f;
  }
  if (tid < SIMT_HEADS) { ml[tid][0] = -INFINITY; ml[tid][1] = 0.f; }
  __syncthreads();
  for (int h = warp; h < SIMT_HEADS; h += 4) {
    float s = 0.f;
    for (int d = lane; d < D; d += 32) s += qs[h][d];
    s = warp_sum(s);
    if (lane == 0) qsum[h] = s;
  }
  float o[SIMT_HEADS][8];
#pragma unroll
  for (int h = 0; h < SIMT_HEADS; ++h)
#pragma unroll
    for (int i = 0; i < 8; ++i) o[h][i] = 0.f;
  const int word = tid % W, kg = tid / W;
  __syncthreads();

  for (int tile = split * per; tile < min(tiles, (split + 1) * per); ++tile) {
    const int j0 = j_lo + tile * SIMT_KEYS, j = j0 + tid, n = min(SIMT_KEYS, j_hi - j0);
    if (tid < n) {
      const size_t row = cache_row(p, bt[j >> p.page_shift], kvh, j);
      key_row[tid] = row;
      v_pair[tid] = p.vp[row];
      const uint32_t kpair = p.kp[row];
      const float ks = pair_scale(kpair), kz = fmaf(8.f, ks, pair_zero(kpair));
      float acc[SIMT_HEADS] = {};
      constexpr int AHEAD = W % 16 == 0 ? 16 : W % 12 == 0 ? 12 : W % 8 == 0 ? 8 : W % 4 == 0 ? 4 : 2;      // words of the row that are on their way at once
#pragma unroll 1
      for (int w0 = 0; w0 < W; w0 += AHEAD) {
        uint32_t bits[AHEAD];
        if constexpr (AHEAD % 4 == 0) {
#pragma unroll
          for (int w = 0; w < AHEAD; w += 4) *reinterpret_cast<uint4*>(bits + w) = *reinterpret_cast<const uint4*>(p.kc + row * W + w0 + w);
        } else {
#pragma unroll
          for (int w = 0; w < AHEAD; ++w) bits[w] = p.kc[row * W + w0 + w];
        }
#pragma unroll
        for (int w = 0; w < AHEAD; ++w) {
          float c[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) c[i] = code_above(bits[w], i) - (CODE_BASE + 8.f);
#pragma unroll
          for (int h = 0; h < SIMT_HEADS; ++h)
            if (h < nh) {
              const float4 a = *reinterpret_cast<const float4*>(&qs[h][(w0 + w) * 8]), e = *reinterpret_cast<const float4*>(&qs[h][(w0 + w) * 8 + 4]);
              acc[h] += fmaf(a.x, c[0], fmaf(a.y, c[1], fmaf(a.z, c[2], a.w * c[3]))) + fmaf(e.x, c[4], fmaf(e.y, c[5], fmaf(e.z, c[6], e.w * c[7])));
            }
        }
      }
#pragma unroll
      for (int h = 0; h < SIMT_HEADS; ++h) prob[h][tid] = capped(p, fmaf(ks, acc[h], kz * qsum[h]) * p.scale);
    }
    __syncthreads();
    for (int h = warp; h < nh; h += 4) {
      float s[SIMT_KEYS / 32], m = -INFINITY, sum = 0.f;
#pragma unroll
      for (int i = 0; i < SIMT_KEYS / 32; ++i) {
        s[i] = lane + 32 * i < n ? prob[h][lane + 32 * i] : -INFINITY;
        m = fmaxf(m, s[i]);
      }
      const float before = ml[h][0];
      m = fmaxf(warp_max(m), before);
      const float base = m == -INFINITY ? 0.f : m;          // (every score -infinity or NaN: nothing to subtract)
#pragma unroll
      for (int i = 0; i < SIMT_KEYS / 32; ++i) {
        s[i] = exp2f((s[i] - base) * LOG2E);
        sum += s[i];
        prob[h][lane + 32 * i] = s[i];
      }
      sum = warp_sum(sum);
      if (lane == 0) {
        const float a = exp2f((before - base) * LOG2E);
        alpha[h] = a;
        ml[h][0] = m;
        ml[h][1] = ml[h][1] * a + sum;
      }
    }
    __syncthreads();
    if (kg < KG) {
#pragma unroll
      for (int h = 0; h < SIMT_HEADS; ++h)
        if (h < nh) {
          const float a = alpha[h];
#pragma unroll
          for (int i = 0; i < 8; ++i) o[h][i] *= a;
        }
#pragma unroll 4
      for (int key = kg; key < n; key += KG) {
        const uint32_t bits = p.vc[key_row[key] * W + word];
        const float vs = pair_scale(v_pair[key]), vz = pair_zero(v_pair[key]);
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fmaf(code_above(bits, i) - CODE_BASE, vs, vz);
#pragma unroll
        for (int h = 0; h < SIMT_HEADS; ++h)
          if (h < nh) {
            const float pr = prob[h][key];
#pragma unroll
            for (int i = 0; i < 8; ++i) o[h][i] = fmaf(pr, v[i], o[h][i]);
          }
      }
    }
    __syncthreads();
  }

  for (int h = 0; h < nh; ++h) {
    // (o[h] with a constant h: registers)
    if (kg < KG) {
#pragma unroll
      for (int hh = 0; hh < SIMT_HEADS; ++hh)
        if (hh == h) {
#pragma unroll
          for (int i = 0; i < 8; ++i) red[kg * D + word * 8 + i] = o[hh][i];
        }
    }
    __syncthreads();
    const size_t row = (size_t)t * p.H + h0 + h;
    float m = ml[h][0], l = ml[h][1], a = 1.f;
    if (p.splits == 1 && p.sinks != nullptr) {
      const float sink = p.sinks[h0 + h], top = fmaxf(m, sink), from = top == -INFINITY ? 0.f : top;          // (neither keys nor a sink)
      a = exp2f((m - from) * LOG2E);
      l = l * a + exp2f((sink - from) * LOG2E);
    }
    for (int d = tid; d < D; d += SIMT_THREADS) {
      float sum = 0.f;
      for (int k = 0; k < KG; ++k) sum += red[k * D + d];
      if (p.splits == 1) {
        static_cast<T*>(p.out)[row * D + d] = from_f32<T>(l == 0.f ? 0.f : sum * a / l);
      } else {
        p.part_o[(row * p.splits + split) * D + d] = sum;
      }
    }
    if (p.splits > 1 && tid == 0) {
      p.part_ml[(row * p.splits + split) * 2] = m;
      p.part_ml[(row * p.splits + split) * 2 + 1] = l;
    }
    __syncthreads();
  }
}

// out[row] = sum_s f_s o_s / sum_s f_s l_s with f_s = 2^((m_s - m) unit) over the key ranges of a row (token, head)
template <typename T>
__global__ void int4_combine_kernel(Int4Params p) {
  pdl_trigger();
  pdl_wait();
  const size_t row = blockIdx.x;
  if ((int)(row / p.H) >= p.cu_q[p.B]) return;
  if (p.most > 0) {
    const int b = request_of(p.cu_q, p.B, (int)(row / p.H));
    if (p.cu_q[b + 1] - p.cu_q[b] > p.most) return;
  }
  const float* ml = p.part_ml + row * p.splits * 2;
  float m = p.sinks ? p.sinks[row % p.H] * (LOG2E / p.unit) : -INFINITY;
  const float sink = m;
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, ml[2 * s]);
  const float base = m == -INFINITY ? 0.f : m;
  float l = p.sinks ? exp2f((sink - base) * p.unit) : 0.f;
  for (int s = 0; s < p.splits; ++s) l += exp2f((ml[2 * s] - base) * p.unit) * ml[2 * s + 1];
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float sum = 0.f;
    for (int s = 0; s < p.splits; ++s) sum += exp2f((ml[2 * s] - base) * p.unit) * p.part_o[(row * p.splits + s) * D + d];
    static_cast<T*>(p.out)[row * D + d] = from_f32<T>(l == 0.f ? 0.f : sum / l);
  }
}

#if TS_HEAD_DIM % 32 == 0 && TS_HEAD_DIM <= 256
#define TS_INT4_MMA 1
// ------------------------------------------------------------------------------------------ attention on the tensor cores
// bfloat16 queries.  A block is up to 8 NT columns = (query, head) pairs of one key head, and a range of its keys; every warp walks keys of its
// own, 32 at a time, through a ring of shared memory that nobody else touches (bulk copies by runs of a page, no block barriers in the loop):
//   S^T = K Q^T with the keys as the rows, P^T brought to the next operand's layout by movmatrix, O^T += V^T P^T with the columns of the
//   values as rows.  What bounds it is the instructions that unpack codes, so they are few:
//   K  an AND makes four codes of a word an operand register of 8-bit integers (m16n8k32).  The queries are split for it: a row's elements in
//      units of 2^-14 of its largest one's power of two, 16 bits, are 256 hi + lo, hi signed and lo not; sums are whole numbers, exact.
//      (bfloat16 has 8 significant bits: elements down to 2^-7 of the largest keep all of theirs, smaller ones are
//      rounded to 2^-15 of it, far below what the projection's own rounding left.  Eight-bit floating point would hold a code without
//      any change, but its mma.sync is made of conversions to 16 bits: 827 instructions a step of 32 keys, as it is 635.)
//   V  keys run along K there, two of one column side by side, which bytes would need a transposition for: a code enters as the number
//      16 + c in half precision, one shift and one AND-OR for two of them.
//   Scales and zeros are per key, so they stay outside: with a pair (s, z) of the key, q.k = s (q.c) + z sum(q); for the values, with p' =
//   half(p s), sum p v = sum p' (c - 8) + sum p (z + 8 s), and sum p' (c - 8) = sum p' (16 + c) - 24 sum p', which is one more MMA, with
//   ones for V, so that the 24 cancels whatever p' was rounded to.  A factor for each column keeps p' within half precision: it follows the column's
//   largest p s so far, as the maximum follows the scores.  (Not the largest s: a key that has no weight, or that the column does not see, must not
//   push the others out of the format's range, whatever its values are.)  (64 requests of 2,000 to 8,192 keys, relative error of the output, of which its
//   own rounding makes 1.7e-3: with p' in bfloat16 2.3e-3, around code 0 instead of 8 3.3e-3.)
// Values of 2^110 and more may overflow these sums, as probabilities reach 2^8 in them.
// 64 requests of 2,000 to 8,192 keys, 32 heads of 128 on 8 (366 MB): 90 us, 4.1 TB/s; fetching alone takes 62.  The integer pipe is busiest (two thirds of its
// rate while a block walks), then the fixed 5 us of a block, of which an SM holds two.  Requests in the order of their numbers instead of by length:
// 108 us, for the blocks that come last run alone.  Shifts as multiplications on the other pipe 91 and 99 us, three blocks an SM
// with 80 registers a thread 123.
constexpr int STEP = 32, RING = 3;
constexpr int ROW_BYTES = D / 2, KW = D / 32, UNITS = D / 32;      // words of K a thread holds of a row; 16-bit units of V
constexpr int STAGE_BYTES = 2 * STEP * ROW_BYTES + 2 * STEP * 4;   // codes of K and V, pairs of K and V
constexpr float MIDDLE = 8.f, ABOVE = 16.f + MIDDLE;               // of the codes; what a code's number 16 + c is above c - MIDDLE
constexpr int MERGE_ROW = D + 4;                                   // floats of a column's partial result: the four columns of a quad meet other banks

template <int NT, int WARPS> struct MmaCfg {
  static constexpr int NC = 8 * NT, MAX_CLUSTER = 8;
  static constexpr int Q_BYTES = KW * NT * 32 * 16 + NC * 8;       // operands; (factor, sum) of every column
  static constexpr int RING_BYTES = WARPS * RING * STAGE_BYTES;
  static constexpr int MERGE_BYTES = WARPS * NC * (MERGE_ROW + 3) * 4;
  static constexpr int WORK_BYTES = RING_BYTES > MERGE_BYTES ? RING_BYTES : MERGE_BYTES;
  // what the blocks of a cluster send each other: with n of them [sender][column / n rounded up][D + 4]
  static constexpr int BOX_BYTES = WARPS == 8 ? (NC + MAX_CLUSTER) * MERGE_ROW * 4 : 0;
  static constexpr int SMEM = Q_BYTES + WORK_BYTES + BOX_BYTES;
  static constexpr bool Q_REGS = NT == 1 && D <= 128;              // the queries' operands stay in registers
  static constexpr int BLOCKS = Q_REGS ? 16 / WARPS : 1;          // of an SM
};

// bytes (a multiple of 16) of global memory to shared memory, counted by a barrier
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void mma_half(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
  uint32_t b;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(b) : "r"(a));
  return b;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// four codes of a word as bytes: of columns 0, 4, 1, 5 and, shifted, 2, 6, 3, 7
__device__ __forceinline__ uint32_t codes4(uint32_t word) { return word & 0x0f0f0f0fu; }
// (the first MMA of a chain adds to zeros that are no registers)
__device__ __forceinline__ void mma_hi_first(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
               : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ void mma_lo_first(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
               : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ void mma_hi(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_lo(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// codes number e (0 .. 3) of both halves of a word as two numbers 16 + c in half precision
template <int E>
__device__ __forceinline__ uint32_t codes2(uint32_t word) {
  const uint32_t moved = E < 2 ? word << (6 - 4 * E) : word >> (4 * E - 6);
  uint32_t two;
  // (written out: the compiler makes two instructions of an AND and an OR with constants, and these pipes bound the kernel)
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(two) : "r"(moved), "r"(0x03c003c0u), "r"(0x4c004c00u));
  return two;
}
// Where a running maximum starts: below every score, and finite, so that nothing subtracts infinities.  It moves only when a score passes it by
// more than SLACK (a power of two): probabilities up to 2^SLACK do no harm in 32-bit sums, and most steps then rescale nothing.
constexpr float LOWEST = -3e38f, SLACK = 8.f;
constexpr float UNIT = 6.f, MAX_UNIT = 112.f;                      // 2^(UNIT + SLACK) is within half precision; p <= 2^SLACK times 2^MAX_UNIT within 32 bits
constexpr uint32_t ONES = 0x3c003c00u;                             // two in half precision
// Row r of the 16 that an MMA reads of K is this key of the group: thread t of a quad then finds its columns of V^T (rows 2t, 2t + 1, 2t + 8,
// 2t + 9) in keys t, t + 4, t + 8, t + 12, and the eight lanes whose reads of K meet read neighbouring keys' halves of a bank line
__device__ __forceinline__ int key_of_row(int r) { return (r & 8) | (r >> 1 & 3) | (r & 1) << 2; }

// The request with the n-th longest cache, of up to 256; `lens` is as many integers of shared memory.  Blocks come in the order of their
// index, and a long one that comes last runs alone.
constexpr int MAX_ORDERED = 256;
template <int THREADS>
__device__ __forceinline__ int nth_longest(const Int4Params& p, int n, int* lens) {
#pragma unroll
  for (int i = threadIdx.x; i < MAX_ORDERED; i += THREADS) lens[i] = i < p.B ? p.kv_lens[i] : -1;
  __syncthreads();
  int found = -1;
#pragma unroll
  for (int i = threadIdx.x; i < MAX_ORDERED; i += THREADS) {
    const int len = lens[i];
    int before = 0;
    if (i < p.B) {
      for (int j = 0; j < p.B; j += 4) {
        const int4 x = *reinterpret_cast<const int4*>(lens + j);
        before += (x.x > len || (x.x == len && j < i)) + (x.y > len || (x.y == len && j + 1 < i)) + (x.z > len || (x.z == len && j + 2 < i)) + (x.w > len || (x.w == len && j + 3 < i));
      }
      if (before == n) found = i;
    }
  }
  __syncthreads();
  if (found >= 0) lens[0] = found;
  __syncthreads();
  return lens[0];
}

template <int NT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, MmaCfg<NT, WARPS>::BLOCKS) int4_mma_kernel(Int4Params p) {
  using C = MmaCfg<NT, WARPS>;
  extern __shared__ __align__(16) char smem[];
  __shared__ uint64_t full[WARPS][RING];
  __shared__ volatile int abort_flag;
  uint4* qf_s = reinterpret_cast<uint4*>(smem);                    // [KW][NT][32 lanes]: high and low bytes of eight columns
  float2* q_stat = reinterpret_cast<float2*>(smem + KW * NT * 32 * 16);       // [NC]
  char* work = smem + C::Q_BYTES;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (lane < RING) mbar_init(smem_u32(&full[warp][lane]), 1);
  if (threadIdx.x == 0) abort_flag = 0;
  asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  __syncthreads();
  pdl_trigger();
  // Beside portions (`most`) too: that this kernel's inputs were complete when the portions' kernel began does not make them visible here; only
  // this grid's own wait does.  (64 requests over 800 keys beside a portion of 448: 60 us; 47 without the wait.)
  pdl_wait();
  const int G = p.H / p.Hkv, split = blockIdx.x, col_tiles = gridDim.y / p.Hkv;
  const int kvh = blockIdx.y / col_tiles, c0 = blockIdx.y % col_tiles * C::NC;
  const int b = p.ordered ? nth_longest<WARPS * 32>(p, blockIdx.z, reinterpret_cast<int*>(work)) : blockIdx.z;
  if (p.ordered) {
    // (its memory is the ring's: bulk copies come behind ordinary stores and loads there)
    fence_async_shared();
    __syncthreads();
  }
  const int q_begin = p.cu_q[b], q_len = min(p.cu_q[b + 1], p.T) - q_begin;
  const int nc = min(C::NC, q_len * G - c0);                       // columns of this block (and of its cluster: they leave together)
  if (nc <= 0 || (p.most > 0 && q_len > p.most)) return;
  const bool clustered = WARPS == 8 && p.splits > 1 && p.part_o == nullptr;
  if (clustered) cluster_arrive();                                 // this block runs: peers may write to its memory
  const int kv_len = (int)min((long long)p.kv_lens[b], (long long)p.max_blocks << p.page_shift);
  const int pos0 = kv_len - q_len;                                 // position of the request's first query of this step
  const int* bt = p.block_table + (size_t)b * p.table_stride;
  const int first = pos0 + c0 / G, last = pos0 + (c0 + nc - 1) / G;
  const int j_lo = p.window > 0 ? max(0, first - p.window + 1) : 0, j_hi = max(last + 1, 0);
  const int step0 = j_lo / STEP, steps = max(0, (j_hi + STEP - 1) / STEP - step0), per = (steps + p.splits - 1) / p.splits;
  const int s_end = min(steps, (split + 1) * per);

  char* ring = work + warp * RING * STAGE_BYTES;
  // A step's 32 keys lie in whole or in runs of a page; every run is four copies (codes of K and V, pairs of K and V), each by a lane of its
  // own: eight runs of four keys are all 32 lanes.  A run that starts behind the last key is not fetched, and what its place holds is masked.
  const int run_shift = min(p.page_shift, 5), run = lane >> 2 << run_shift;
  const char* base = reinterpret_cast<const char*>(lane & 2 ? (lane & 1 ? p.vp : p.kp) : (lane & 1 ? p.vc : p.kc));
  const uint32_t row_bytes = lane & 2 ? 4 : ROW_BYTES, run_bytes = row_bytes << run_shift;
  const uint32_t run_at = smem_u32(ring) + (lane & 2 ? 2 * STEP * ROW_BYTES : 0) + ((lane & 1) * STEP + run) * row_bytes;
  const int last_run = run < STEP ? j_hi - run : 0;                // a step that starts in front of it has keys for this lane
  int page_ahead = 0;          // of this lane's run of the step that is fetched next: read a step before it is needed
  auto look = [&](int s) {
    const int j = (step0 + s) * STEP;
    if (s < s_end && j < last_run) page_ahead = bt[(j + run) >> p.page_shift];
  };
  auto fetch = [&](int s, int stage) {
    const int j = (step0 + s) * STEP;
    const bool mine = j < last_run;
    const uint32_t bar = smem_u32(&full[warp][stage]);
    const uint32_t n = __popc(__ballot_sync(0xffffffffu, mine)) >> 2;
    if (lane == 0) mbar_expect_tx(bar, n * (STAGE_BYTES >> (5 - run_shift)));
    __syncwarp();
    if (mine) {
      if ((unsigned)page_ahead >= (unsigned)p.num_pages) {
        ts_raise_status(TS_STATUS_BOUNDS, TS_BAD_PAGE);
        page_ahead = 0;
      }
      // (a pool of this kernel has fewer than 2^31 rows: one multiplication a copy)
      const uint32_t row = (((uint32_t)page_ahead * p.Hkv + kvh) << p.page_shift) + ((j + run) & ((1 << p.page_shift) - 1));
      bulk_copy(run_at + stage * STAGE_BYTES, base + (unsigned long long)row * row_bytes, run_bytes, bar);
    }
    look(s + WARPS);
  };
  const int mine = split * per + warp;
  look(mine);
#pragma unroll
  for (int i = 0; i < RING - 1; ++i)
    if (mine + i * WARPS < s_end) fetch(mine + i * WARPS, i);

  // the queries as B operands: a warp makes a column, a lane a word's eight columns: word t KW + i goes to step i, thread t of the column's quad
  for (int c = warp; c < C::NC; c += WARPS) {
    float x[8] = {};
    if (lane < W && c < nc) {
      const int r = c0 + c;
      const bf16* src = static_cast<const bf16*>(p.q) + (q_begin + r / G) * p.q_row + (kvh * G + r % G) * p.q_head + lane * 8;
      if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) load8<bf16>(src, x);
      else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __bfloat162float(src[e]);
      }
    }
    float top = 0.f, sum = 0.f;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      top = fmaxf(top, fabsf(x[e]));
      sum += x[e];
      bad |= !(fabsf(x[e]) <= 3.402823466e38f);
    }
    top = warp_max(top);
    sum = warp_sum(sum);
    bad = __any_sync(0xffffffffu, bad);
    // the row's largest element goes to 2^14 .. 2^15
    const int ex = min(max((int)(__float_as_uint(top) >> 23) - 127, -112), 127);
    const float up = __uint_as_float((uint32_t)(14 - ex + 127) << 23);
    uint32_t hi[2] = {0u, 0u}, lo[2] = {0u, 0u};
    constexpr int COLUMN[8] = {0, 4, 1, 5, 2, 6, 3, 7};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int whole = bad ? 0 : __float2int_rn(x[COLUMN[e]] * up);
      hi[e >> 2] |= (uint32_t)(whole >> 8 & 255) << (8 * (e & 3));
      lo[e >> 2] |= (uint32_t)(whole & 255) << (8 * (e & 3));
    }
    if (lane < W) qf_s[((lane % KW) * NT + (c >> 3)) * 32 + (c & 7) * 4 + lane / KW] = make_uint4(hi[0], hi[1], lo[0], lo[1]);
    if (lane == 0) q_stat[c] = make_float2(bad ? __int_as_float(0x7fc00000) : 1.f / up, sum);
  }
  __syncthreads();
  uint4 qf[C::Q_REGS ? KW : 1];
  F2 factor[NT], qsum[NT];                                         // of columns 2t and 2t + 1
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    if (C::Q_REGS) {
#pragma unroll
      for (int i = 0; i < KW; ++i) qf[C::Q_REGS ? i : 0] = qf_s[i * 32 + lane];
    }
    const float2 a = q_stat[nt * 8 + 2 * t], b = q_stat[nt * 8 + 2 * t + 1];
    factor[nt] = f2(a.x, b.x);
    qsum[nt] = f2(a.y, b.y);
  }
  int pos[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = nt * 8 + 2 * t + i;
      pos[nt][i] = c < nc ? pos0 + (c0 + c) / G : -1;
    }
  const int all_from = p.window > 0 ? max(0, last - p.window + 1) : 0;       // keys from here to `first` are seen by every column
  const float scale2 = p.scale * LOG2E;

  float o[D / 16][NT][4], m[NT][2], ps[NT][4];                     // ps: sum p' of columns 2t and 2t + 1 (and the same again)
  F2 l[NT], z[NT];
  // a column's largest log2(p s) so far, which moves as m does, and the factor that brings p s there to 2^UNIT.  (Against m and not by
  // itself: beside scores of 10^8 a sum would have no bits left for the scale.)
  float top_v[NT][2], unit[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][nt][e] = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) ps[nt][e] = 0.f;
    m[nt][0] = m[nt][1] = top_v[nt][0] = top_v[nt][1] = LOWEST;
    unit[nt][0] = unit[nt][1] = 1.f;
    l[nt] = z[nt] = f2(0.f, 0.f);
  }

  int stage = 0, waits = 0;
  bool ok = true;
#pragma unroll 1
  for (int s = mine; s < s_end; s += WARPS) {
    ok = mbar_wait(smem_u32(&full[warp][stage]), waits & 1, &abort_flag);
    ok = __all_sync(0xffffffffu, ok);          // (and everybody has read what the stage before this one held)
    if (!ok) break;
    {
      const int ahead = s + (RING - 1) * WARPS;
      if (ahead < s_end) fetch(ahead, stage == 0 ? RING - 1 : stage - 1);
    }
    const char* ks = ring + stage * STAGE_BYTES;
    const char* vs = ks + STEP * ROW_BYTES;
    const uint32_t* kp = reinterpret_cast<const uint32_t*>(vs + STEP * ROW_BYTES) + key_of_row(g);
    const uint32_t* vp = kp + STEP;
    if (stage == RING - 1) { stage = 0; ++waits; } else ++stage;
    const int j0 = (step0 + s) * STEP;

    float sc[2][NT][4];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const uint32_t* r0 = reinterpret_cast<const uint32_t*>(ks + (kb * 16 + key_of_row(g)) * ROW_BYTES) + t * KW;
      const uint32_t* r1 = r0 + 8 * ROW_BYTES / 4;
      uint32_t w0[KW], w1[KW];
      if constexpr (KW % 4 == 0) {
#pragma unroll
        for (int i = 0; i < KW; i += 4) {
          *reinterpret_cast<uint4*>(w0 + i) = *reinterpret_cast<const uint4*>(r0 + i);
          *reinterpret_cast<uint4*>(w1 + i) = *reinterpret_cast<const uint4*>(r1 + i);
        }
      } else if constexpr (KW % 2 == 0) {
#pragma unroll
        for (int i = 0; i < KW; i += 2) {
          *reinterpret_cast<uint2*>(w0 + i) = *reinterpret_cast<const uint2*>(r0 + i);
          *reinterpret_cast<uint2*>(w1 + i) = *reinterpret_cast<const uint2*>(r1 + i);
        }
      } else {
#pragma unroll
        for (int i = 0; i < KW; ++i) { w0[i] = r0[i]; w1[i] = r1[i]; }
      }
      int part[2][NT][4];
#pragma unroll
      for (int i = 0; i < KW; ++i) {
        const uint32_t a0 = codes4(w0[i]), a1 = codes4(w1[i]), a2 = codes4(w0[i] >> 4), a3 = codes4(w1[i] >> 4);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const uint4 q = C::Q_REGS ? qf[C::Q_REGS ? i : 0] : qf_s[(i * NT + nt) * 32 + lane];
          if (i == 0) {
            mma_hi_first(part[0][nt], a0, a1, a2, a3, q.x, q.y);
            mma_lo_first(part[1][nt], a0, a1, a2, a3, q.z, q.w);
          } else {
            mma_hi(part[0][nt], a0, a1, a2, a3, q.x, q.y);
            mma_lo(part[1][nt], a0, a1, a2, a3, q.z, q.w);
          }
        }
      }
      // scores; this thread's keys are those of rows g and g + 8
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t kpair = kp[kb * 16 + 8 * h];
        const float a = pair_scale(kpair) * scale2, b = pair_zero(kpair) * scale2;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const F2 sum = f2((float)(part[0][nt][2 * h] * 256 + part[1][nt][2 * h]), (float)(part[0][nt][2 * h + 1] * 256 + part[1][nt][2 * h + 1]));
          f2_out(f2_fma(f2(a, a), f2_mul(sum, factor[nt]), f2_mul(f2(b, b), qsum[nt])), sc[kb][nt][2 * h], sc[kb][nt][2 * h + 1]);
        }
      }
    }
    float vscale[2][2], vzero[2][2], top[NT][2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t vpair = vp[kb * 16 + 8 * h];
        vscale[kb][h] = pair_scale(vpair);
        vzero[kb][h] = fmaf(MIDDLE, pair_scale(vpair), pair_zero(vpair));
      }
    if (p.softcap > 0.f) {
      const float in = 1.f / (p.softcap * LOG2E), out = p.softcap * LOG2E;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[kb][nt][e] = out * tanhf(sc[kb][nt][e] * in);
    }
    if (j0 < all_from || j0 + STEP - 1 > first) {
      // the ends of somebody's range: hidden keys have no score, and nothing of their values
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int j = j0 + kb * 16 + key_of_row(g) + 8 * h;
          // a probability of 0 must not meet a NaN, of a slot that is not this request's or of a key that only some columns see:
          // the pair becomes 0, and who sees the key gets the NaN through its score
          const bool finite = fabsf(vscale[kb][h]) <= 3.402823466e38f && fabsf(vzero[kb][h]) <= 3.402823466e38f;
          // (and a scale that nobody sees must not set the unit)
          if (!finite || j >= j_hi || j < j_lo) vscale[kb][h] = vzero[kb][h] = 0.f;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const bool hidden = j > pos[nt][i] || (p.window > 0 && j <= pos[nt][i] - p.window);
              if (hidden) sc[kb][nt][2 * h + i] = -INFINITY;
              else if (!finite) sc[kb][nt][2 * h + i] = __int_as_float(0x7fc00000);
            }
        }
    }
    // (every key's score against the largest scale of the four: seldom more than a step's own, and the step that moves looks closely)
    const float widest = lg2(fmaxf(fmaxf(fabsf(vscale[0][0]), fabsf(vscale[0][1])), fmaxf(fabsf(vscale[1][0]), fabsf(vscale[1][1]))));
    bool moved = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        top[nt][i] = fmaxf(fmaxf(sc[0][nt][i], sc[0][nt][2 + i]), fmaxf(sc[1][nt][i], sc[1][nt][2 + i]));
        const float above = top[nt][i] - m[nt][i];
        moved |= above > SLACK || above + widest > top_v[nt][i] + SLACK;
      }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float f[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) top[nt][i] = fmaxf(top[nt][i], __shfl_xor_sync(0xffffffffu, top[nt][i], d));
          const float above = fmaxf(top[nt][i], m[nt][i]), shift = m[nt][i] - above;
          float wide = LOWEST;
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int h = 0; h < 2; ++h) wide = fmaxf(wide, sc[kb][nt][2 * h + i] - above + lg2(fabsf(vscale[kb][h])));
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) wide = fmaxf(wide, __shfl_xor_sync(0xffffffffu, wide, d));
          wide = fmaxf(wide, top_v[nt][i] + shift);
          // (where there was no scale but 0, o is 0)
          const float was = fminf(UNIT - top_v[nt][i], MAX_UNIT), is = fminf(UNIT - wide, MAX_UNIT);
          const float f_v = ex2(shift + (is - was));
          f[i] = ex2(shift);
          m[nt][i] = above;
          top_v[nt][i] = wide;
          unit[nt][i] = ex2(is);
          ps[nt][i] *= f_v;
          ps[nt][2 + i] *= f_v;
#pragma unroll
          for (int mt = 0; mt < D / 16; ++mt) { o[mt][nt][i] *= f_v; o[mt][nt][2 + i] *= f_v; }
        }
        l[nt] = f2_mul(l[nt], f2(f[0], f[1]));
        z[nt] = f2_mul(z[nt], f2(f[0], f[1]));
      }
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      uint32_t pb[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const F2 at = f2_add(f2(sc[kb][nt][2 * h], sc[kb][nt][2 * h + 1]), f2(-m[nt][0], -m[nt][1]));
          float x0, x1;
          f2_out(at, x0, x1);
          const F2 pr = f2(ex2(x0), ex2(x1));
          l[nt] = f2_add(l[nt], pr);
          z[nt] = f2_fma(pr, f2(vzero[kb][h], vzero[kb][h]), z[nt]);
          f2_out(f2_mul(f2_mul(pr, f2(unit[nt][0], unit[nt][1])), f2(vscale[kb][h], vscale[kb][h])), x0, x1);
          const __half2 two = __floats2half2_rn(x0, x1);
          const uint32_t bits = *reinterpret_cast<const uint32_t*>(&two);
          pb[nt][h] = transposed(bits);
        }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma_half(ps[nt], ONES, ONES, ONES, ONES, pb[nt][0], pb[nt][1]);
      // values: 16-bit units g UNITS .. of keys t, t + 4, t + 8, t + 12 of the group
      uint32_t u[4][(UNITS + 1) / 2];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const char* at = vs + (kb * 16 + t + 4 * q) * ROW_BYTES;
        if constexpr (UNITS % 8 == 0) {
          const uint4 x = reinterpret_cast<const uint4*>(at)[g];
          u[q][0] = x.x; u[q][1] = x.y; u[q][2] = x.z; u[q][3] = x.w;
        } else if constexpr (UNITS % 4 == 0) {
          const uint2 x = reinterpret_cast<const uint2*>(at)[g];
          u[q][0] = x.x; u[q][1] = x.y;
        } else if constexpr (UNITS % 2 == 0) {
#pragma unroll
          for (int i = 0; i < UNITS / 2; ++i) u[q][i] = reinterpret_cast<const uint32_t*>(at)[g * (UNITS / 2) + i];
        } else {
#pragma unroll
          for (int i = 0; i < UNITS; ++i) {
            const uint32_t x = reinterpret_cast<const uint16_t*>(at)[g * UNITS + i];
            u[q][i / 2] = i % 2 ? u[q][i / 2] | x << 16 : x;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < UNITS; ++i) {
        const uint32_t x0 = __byte_perm(u[0][i / 2], u[1][i / 2], i % 2 ? 0x7632 : 0x5410), x1 = __byte_perm(u[2][i / 2], u[3][i / 2], i % 2 ? 0x7632 : 0x5410);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_half(o[2 * i][nt], codes2<0>(x0), codes2<1>(x0), codes2<0>(x1), codes2<1>(x1), pb[nt][0], pb[nt][1]);
          mma_half(o[2 * i + 1][nt], codes2<2>(x0), codes2<3>(x0), codes2<2>(x1), codes2<3>(x1), pb[nt][0], pb[nt][1]);
        }
      }
    }
  }
  if (!ok) {
    // a wait ran out: the copies that may still be in flight land before their memory is used again or given up
    for (int i = 0; i < RING; ++i)
      for (int parity = 0; parity < 2; ++parity)
        for (uint32_t w = 0; w < WAIT_LIMIT && !mbar_try_wait(smem_u32(&full[warp][i]), parity); ++w) {}
  }

  // the warps' results meet in shared memory
  if (clustered) cluster_wait();                                   // (all peers run)
  __syncthreads();
  float* sm_o = reinterpret_cast<float*>(work);                    // [warp][column][MERGE_ROW]: output column d of lane group g at place (d's number there) * 8 + g
  float* sm_ml = sm_o + WARPS * C::NC * MERGE_ROW;             // [warp][column][3]
  float* box = reinterpret_cast<float*>(work + C::WORK_BYTES);     // (its own memory: a peer may send while this block still reads its ring)
  const int per_rank = (C::NC + p.splits - 1) / p.splits;
  auto send = [](uint32_t at, uint32_t rank, float v) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(rank));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote), "f"(v) : "memory");
  };
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float ls[2], zs[2];
    f2_out(l[nt], ls[0], ls[1]);
    f2_out(z[nt], zs[0], zs[1]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        ls[i] += __shfl_xor_sync(0xffffffffu, ls[i], d);
        zs[i] += __shfl_xor_sync(0xffffffffu, zs[i], d);
      }
      const int c = nt * 8 + 2 * t + i;
      const float back = 1.f / unit[nt][i];
      if (g == 0) {
        sm_ml[(warp * C::NC + c) * 3] = m[nt][i];
        sm_ml[(warp * C::NC + c) * 3 + 1] = ls[i];
        sm_ml[(warp * C::NC + c) * 3 + 2] = fmaf(-ABOVE * back, ps[nt][i], zs[i]);
      }
      float* dst = sm_o + (warp * C::NC + c) * MERGE_ROW + g;
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt) {
        dst[16 * mt] = o[mt][nt][i] * back;
        dst[16 * mt + 8] = o[mt][nt][2 + i] * back;
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nc * D; i += WARPS * 32) {
    const int c = i / D, place = i % D, r = c0 + c, head = kvh * G + r % G;
    // place 8 n + g: nibble n % 4 of unit g UNITS + n / 4
    const int unit = (place & 7) * UNITS + (place >> 5), d = 8 * (unit >> 1) + (unit & 1) + 2 * (place >> 3 & 3);
    const size_t row = (size_t)(q_begin + r / G) * p.H + head;
    const bool sink = p.splits == 1 && p.sinks != nullptr;
    const float sink2 = sink ? p.sinks[head] * LOG2E : LOWEST;
    float top = fmaxf(LOWEST, sink2);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, sm_ml[(w * C::NC + c) * 3]);
    float sum = 0.f, total = sink ? ex2(sink2 - top) : 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float* ml = sm_ml + (w * C::NC + c) * 3;
      const float f = ex2(ml[0] - top);
      total += f * ml[1];
      sum += f * (sm_o[(w * C::NC + c) * MERGE_ROW + place] + ml[2]);
    }
    if (p.splits == 1) {
      static_cast<bf16*>(p.out)[row * D + d] = __float2bfloat16_rn(total == 0.f ? 0.f : sum / total);
    } else if (p.part_o != nullptr) {
      p.part_o[(row * p.splits + split) * D + d] = sum;
      if (place == 0) {
        p.part_ml[(row * p.splits + split) * 2] = top;
        p.part_ml[(row * p.splits + split) * 2 + 1] = total;
      }
    } else {
      // to the block that owns the column (rank c % splits)
      const int at = split * per_rank + c / p.splits;
      send(smem_u32(box + at * MERGE_ROW + place), c % p.splits, sum);
      if (place < 2) send(smem_u32(box + at * MERGE_ROW + D + place), c % p.splits, place == 0 ? top : total);
    }
  }
  if (!clustered) return;
  cluster_arrive();
  cluster_wait();
  for (int i = threadIdx.x; i < per_rank * D; i += WARPS * 32) {
    const int c = i / D * p.splits + split, place = i % D, r = c0 + c, head = kvh * G + r % G;
    if (c >= nc) break;
    const int unit = (place & 7) * UNITS + (place >> 5), d = 8 * (unit >> 1) + (unit & 1) + 2 * (place >> 3 & 3);
    const float sink2 = p.sinks != nullptr ? p.sinks[head] * LOG2E : LOWEST;
    float top = fmaxf(LOWEST, sink2);
#pragma unroll
    for (int s = 0; s < C::MAX_CLUSTER; ++s)
      if (s < p.splits) top = fmaxf(top, box[(s * per_rank + i / D) * MERGE_ROW + D]);
    float sum = 0.f, total = p.sinks != nullptr ? ex2(sink2 - top) : 0.f;
#pragma unroll
    for (int s = 0; s < C::MAX_CLUSTER; ++s)
      if (s < p.splits) {
        const float* from = box + (s * per_rank + i / D) * MERGE_ROW;
        const float f = ex2(from[D] - top);
        sum += f * from[place];
        total += f * from[D + 1];
      }
    static_cast<bf16*>(p.out)[((size_t)(q_begin + r / G) * p.H + head) * D + d] = __float2bfloat16_rn(total == 0.f ? 0.f : sum / total);
  }
}

template <int NT, int WARPS>
int attend_mma(Int4Params p, int max_q_len, int sms, cudaStream_t stream) {
  using C = MmaCfg<NT, WARPS>;
  static SmemSet set;
  const cudaError_t sized = set.to(int4_mma_kernel<NT, WARPS>, C::SMEM);
  if (sized != cudaSuccess) return ts_fail("int4_attention: %s", cudaGetErrorString(sized));
  const int G = p.H / p.Hkv;
  const long long tiles = ((long long)max_q_len * G + C::NC - 1) / C::NC * p.Hkv;
  TS_REQUIRE(tiles <= 65535 && p.B <= 65535, "int4_attention: grid out of range");
  const dim3 grid(p.splits, (unsigned)tiles, p.B), block(WARPS * 32);
  // (when everything runs at once, order is no use)
  p.ordered = p.B > 1 && p.B <= MAX_ORDERED && tiles * p.splits * p.B > (long long)C::BLOCKS * sms;
  if (p.splits > 1 && p.part_o == nullptr) {
    // the key ranges of a tile are a cluster and merge in it
    const cudaError_t e = ts_launch_cluster(int4_mma_kernel<NT, WARPS>, grid, block, C::SMEM, stream, dim3(p.splits, 1, 1), p);
    if (e != cudaSuccess) return ts_fail("int4_attention (clusters of %d): %s", p.splits, cudaGetErrorString(e));
    return 0;
  }
  TS_LAUNCH("int4_attention", int4_mma_kernel<NT, WARPS>, grid, block, C::SMEM, stream, p);
  if (p.splits > 1)
    TS_LAUNCH("int4_attention (combine)", int4_combine_kernel<bf16>, dim3((unsigned)(p.T * p.H)), dim3(D < 128 ? D : 128), 0, stream, p);
  return 0;
}
#endif

int shift_of_page(int page_size) {
  for (int s = 0; s < 20; ++s)
    if (page_size == 1 << s) return s;
  return -1;
}

template <typename T>
int attend_simt(const Int4Params& p, cudaStream_t stream) {
  const int G = p.H / p.Hkv, head_tiles = (G + SIMT_HEADS - 1) / SIMT_HEADS;
  TS_REQUIRE(p.Hkv * head_tiles <= 65535 && p.splits <= 65535, "int4_attention: grid out of range");
  TS_LAUNCH("int4_attention", int4_attend_kernel<T>, dim3(p.T, p.Hkv * head_tiles, p.splits), dim3(SIMT_THREADS), 0, stream, p);
  if (p.splits > 1)
    TS_LAUNCH("int4_attention (combine)", int4_combine_kernel<T>, dim3((unsigned)(p.T * p.H)), dim3(D < 128 ? D : 128), 0, stream, p);
  return 0;
}

}  // namespace

#ifdef TS_INT4_MMA
// 1 if a block ever gave up on a wait since the library was loaded (reads device memory: syncs)
TS_EXPORT int ts_int4_attention_error() {
  int flag = 0;
  if (cudaMemcpyFromSymbol(&flag, g_error_flag, sizeof(int)) != cudaSuccess) return -1;
  return flag;
}
#endif

// k, v [T, Hkv, D] (strides in elements, columns contiguous) to the slots of slot_mapping [T] (< 0: skipped; slots are distinct)
static int int4_kvwrite(int dtype, const void* k, const void* v, long long k_row, long long k_head, long long v_row, long long v_head,
                        int T, int Hkv, void* k_codes, void* k_pairs, void* v_codes, void* v_pairs, const int* slot_mapping,
                        int page_size, int num_pages, cudaStream_t stream) {
  const int shift = shift_of_page(page_size);
  TS_REQUIRE(dtype == TS_F32 || dtype == TS_BF16, "int4_kvwrite: unknown dtype %d", dtype);
  TS_REQUIRE(T > 0 && Hkv > 0 && shift >= 0 && num_pages > 0, "int4_kvwrite: %d tokens, %d heads, pages of %d", T, Hkv, page_size);
  TS_REQUIRE((((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_pairs | (uintptr_t)v_pairs) & 3) == 0, "int4_kvwrite: the cache is not aligned to words");
  const int e = dtype == TS_F32 ? 4 : 2;
  const bool vec = ((((uintptr_t)k | (uintptr_t)v) | (uintptr_t)((k_row | k_head | v_row | v_head) * e)) & 15) == 0;
  WriteParams p = {k, v, k_row, k_head, v_row, v_head, (uint32_t*)k_codes, (uint32_t*)v_codes, (uint32_t*)k_pairs, (uint32_t*)v_pairs,
                   slot_mapping, T, Hkv, shift, (long long)num_pages << shift};
  if (dtype == TS_F32) return T < MANY_TOKENS ? launch_write<float, FEW_LANES>(p, vec, stream) : launch_write<float, MANY_LANES>(p, vec, stream);
  return T < MANY_TOKENS ? launch_write<bf16, FEW_LANES>(p, vec, stream) : launch_write<bf16, MANY_LANES>(p, vec, stream);
}
TS_ENTRY(int4_kvwrite)

// qkv [T, (H + 2 Hkv) D] contiguous -> q [T, H, D] and, with a slot_mapping, the cache; see RopeParams.  rot 0: no rotation, q_weight null: no norm.
static int int4_rope_kvwrite(int dtype, const void* qkv, void* q, const int* positions, const float* cos, const float* sin, int rot,
                             int interleaved, const void* q_weight, const void* k_weight, int weight_f32, float eps, int T, int H, int Hkv,
                             void* k_codes, void* k_pairs, void* v_codes, void* v_pairs, const int* slot_mapping, int page_size,
                             int num_pages, cudaStream_t stream) {
  const int shift = shift_of_page(page_size);
  TS_REQUIRE(dtype == TS_F32 || dtype == TS_BF16, "int4_rope_kvwrite: unknown dtype %d", dtype);
  TS_REQUIRE(T > 0 && H > 0 && Hkv > 0 && shift >= 0 && num_pages > 0, "int4_rope_kvwrite: %d tokens, %d and %d heads, pages of %d", T, H, Hkv, page_size);
  TS_REQUIRE(rot >= 0 && rot <= D && rot % 2 == 0 && (rot == 0 || (cos && sin && positions)), "int4_rope_kvwrite: a rotation over %d of %d columns", rot, D);
  TS_REQUIRE((q_weight == nullptr) == (k_weight == nullptr), "int4_rope_kvwrite: q and k norm weights come together");
  TS_REQUIRE((((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_pairs | (uintptr_t)v_pairs) & 3) == 0 && ((uintptr_t)q & 15) == 0, "int4_rope_kvwrite: the cache or q is not aligned");
  WriteParams p = {};
  p.kc = (uint32_t*)k_codes; p.vc = (uint32_t*)v_codes; p.kp = (uint32_t*)k_pairs; p.vp = (uint32_t*)v_pairs;
  p.slot_mapping = slot_mapping; p.T = T; p.Hkv = Hkv; p.page_shift = shift; p.slots = (long long)num_pages << shift;
  const RopeParams rp = {qkv, q, positions, rot ? cos : nullptr, sin, rot, interleaved, VecParam{q_weight, weight_f32}, VecParam{k_weight, weight_f32},
                         q_weight != nullptr, eps, H, ((uintptr_t)qkv & 15) == 0, (((uintptr_t)q_weight | (uintptr_t)k_weight) & 15) == 0,
                         !interleaved && rot % 16 == 0 && (((uintptr_t)cos | (uintptr_t)sin) & 15) == 0};
  if (dtype == TS_F32) return T < MANY_TOKENS ? launch_rope_write<float, FEW_LANES>(p, rp, stream) : launch_rope_write<float, MANY_LANES>(p, rp, stream);
  return T < MANY_TOKENS ? launch_rope_write<bf16, FEW_LANES>(p, rp, stream) : launch_rope_write<bf16, MANY_LANES>(p, rp, stream);
}
TS_ENTRY(int4_rope_kvwrite)

// q, out [T, H, D]; see Int4Params.  splits > 1 needs part_o and part_ml, or (with columns, up to 8) merges in clusters.  columns 8 or 16: the tensor-core kernel (bfloat16, heads in
// steps of 32 up to 256; 16 columns up to 128) with 8 warps a block, or 4 (8 columns, one key range, heads up to 128), whose grid covers max_q_len queries a request; 0: the 32-bit kernel.  most > 0 (with columns, for a step
// whose longer requests ts_int4_attention_tcgen05 has taken): requests with more queries than that are left alone.  sms: multiprocessors
// of the device.
static int int4_attention(int dtype, const void* q, long long q_row, long long q_head, void* out, const void* k_codes, const void* k_pairs,
                          const void* v_codes, const void* v_pairs, const int* block_table, const int* cu_q, const int* kv_lens,
                          int T, int B, int H, int Hkv, int page_size, int max_blocks, int table_stride, int num_pages, float scale,
                          int window, float softcap, const float* sinks, int splits, float* part_o, float* part_ml, int max_q_len,
                          int columns, int warps, int most, int sms, cudaStream_t stream) {
  const int shift = shift_of_page(page_size);
  TS_REQUIRE(dtype == TS_F32 || dtype == TS_BF16, "int4_attention: unknown dtype %d", dtype);
  TS_REQUIRE(T > 0 && B > 0 && Hkv > 0 && H > 0 && H % Hkv == 0 && shift >= 0 && num_pages > 0 && max_blocks > 0, "int4_attention: %d tokens of %d requests, %d heads on %d, pages of %d",
             T, B, H, Hkv, page_size);
  TS_REQUIRE((long long)T * H < (1LL << 31), "int4_attention: too many rows");
  TS_REQUIRE(splits >= 1 && (splits == 1 || (part_o && part_ml) || (columns > 0 && splits <= 8 && !part_o)), "int4_attention: key ranges need their scratch");
  Int4Params p = {q, q_row, q_head, out, (const uint32_t*)k_codes, (const uint32_t*)v_codes, (const uint32_t*)k_pairs, (const uint32_t*)v_pairs,
                  block_table, cu_q, kv_lens, T, B, H, Hkv, shift, max_blocks, table_stride, num_pages, scale, window, softcap, sinks,
                  splits, columns > 0 ? 1.f : LOG2E, most, 0, part_o, part_ml};
  if (columns > 0) {
#ifdef TS_INT4_MMA
    TS_REQUIRE(dtype == TS_BF16 && max_q_len > 0 && page_size >= 4, "int4_attention: the tensor-core kernel takes bfloat16 queries and pages of 4 and more");
    TS_REQUIRE(((long long)num_pages * Hkv << shift) < (1LL << 31), "int4_attention: the tensor-core kernel takes pools of fewer than 2^31 rows");
    TS_REQUIRE((((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_pairs | (uintptr_t)v_pairs) & 15) == 0, "int4_attention: the tensor-core kernel copies runs that begin on 16 bytes");
    if (columns == 8 && warps == 8) return attend_mma<1, 8>(p, max_q_len, sms, stream);
#if TS_HEAD_DIM <= 128
    if (columns == 8 && warps == 4 && splits == 1) return attend_mma<1, 4>(p, max_q_len, sms, stream);
    if (columns == 16 && warps == 8) return attend_mma<2, 8>(p, max_q_len, sms, stream);
#endif
#endif
    return ts_fail("int4_attention: no tensor-core kernel for heads of %d, %d columns and %d warps", D, columns, warps);
  }
  return dtype == TS_F32 ? attend_simt<float>(p, stream) : attend_simt<bf16>(p, stream);
}
TS_ENTRY(int4_attention)
