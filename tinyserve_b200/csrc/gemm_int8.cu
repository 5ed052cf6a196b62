// Matrix products in 8-bit integers: y[m, n] = (sum_k cx[m, k] cw[n, k]) sx[m] sw[n] (+ bias[n]).
//
// Rows of x (tokens) and of W (output channels) are held as codes of 8 bits and one 32-bit scale each:
//   scale = max |row| / 127, code = round(row / scale), halves to even; both operations in 32 bits.
// A row of zeros has scale 0 and codes 0; a row that holds an infinity or a NaN has scale NaN, and its products are NaN.
// The sums are exact: the tensor core adds products of 8-bit numbers in 32-bit integers (K up to 131,072: 127 * 127 * K < 2^31),
// so cutting K never changes a result, and the scales are applied once, in 32 bits.
//
// The product has the roles of gemm_tcgen05.cu: 128 rows of W are the M side of tcgen05.mma (kind::i8), TILE_T tokens its N side; a
// slice of K of 128 codes is 128 bytes, one swizzle row, so that shared memory, the TMA boxes and the four MMAs of a slice (32 bytes of
// K each) are those of 64 bfloat16.  K is cut over the blocks of a cluster, which add their integer sums through distributed shared
// memory: no scratch, no counters, nothing that two launches could share.
//
// For few tokens the bytes of W bound it: 8 tokens x 4,096 on 24,576 rows take 18.9 us with the rows' codes (101 MB, 5.3 TB/s), 64 x 12,288 on 4,096 rows
// 15.9 (50 MB, cut by eight); the smallest calls are launches (1 x 1,024 on 4,096 rows 5.4 us, both kernels).  A single launch that makes the
// rows' codes in every block's loader was slower (1 x 1,024: 7.4 us): every block waits for the whole row before its first MMA.
#include "entry.cuh"
#include "rounding.cuh"
#include "tcgen05.cuh"

TS_DEFINE_LAST_ERROR()

namespace {

using bf16 = __nv_bfloat16;

// ------------------------------------------------------------------------------------------ rows to 8 bits
// A row's block has up to 512 threads of eight neighbouring elements a step; up to four steps stay in registers between the search
// for the largest magnitude and the codes (longer rows are read twice, the second time from the caches).
constexpr int QUANT_THREADS = 512, QUANT_KEPT = 4;

struct QuantParams {
  const void* x;        // [M, K], leading dimension ldx
  signed char* codes;   // [M, K], leading dimension ldq (a multiple of 16)
  float* scales;        // [M]
  long long ldx, ldq;
  int K;
};

// Eight neighbouring elements of a row as they lie in memory; `top` keeps the largest magnitude as bits, where an infinity or a NaN is larger than
// every number.
template <typename T> struct Eight;
template <> struct Eight<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) { a = reinterpret_cast<const float4*>(p)[0]; b = reinterpret_cast<const float4*>(p)[1]; }
  __device__ __forceinline__ static uint32_t largest(uint32_t top, float x) { return max(top, __float_as_uint(x) & 0x7fffffffu); }
  __device__ __forceinline__ void look(uint32_t& top) const {
    top = largest(largest(largest(largest(top, a.x), a.y), a.z), a.w);
    top = largest(largest(largest(largest(top, b.x), b.y), b.z), b.w);
  }
  __device__ __forceinline__ void get(float (&x)[8]) const { x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w; }
  __device__ __forceinline__ static uint32_t bits(uint32_t top) { return top; }
};
template <> struct Eight<bf16> {
  uint4 raw;
  __device__ __forceinline__ void load(const bf16* p) { raw = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void look(uint32_t& top) const {          // (two magnitudes of 16 bits)
    top = __vmaxu2(__vmaxu2(top, raw.x & 0x7fff7fffu), raw.y & 0x7fff7fffu);
    top = __vmaxu2(__vmaxu2(top, raw.z & 0x7fff7fffu), raw.w & 0x7fff7fffu);
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
  __device__ __forceinline__ static uint32_t bits(uint32_t top) { return max(top << 16, top & 0xffff0000u); }
};

// round(x / scale) of the quotient rounded to 32 bits, as a byte; a division is only made where the reciprocal could overflow.  Adding
// 1.5 2^23 rounds to a whole number, halves to even, and leaves it in the low bits.
constexpr float ROUNDER = 12582912.f;
__device__ __noinline__ uint32_t divided_code(float x, float scale) {
  return (uint32_t)(int)fminf(fmaxf(rintf(__fdiv_rn(x, scale)), -127.f), 127.f) & 255u;
}
__device__ __forceinline__ uint32_t code_of(float x, float scale, float inverse) {
  if (!(scale > 1e-30f)) return divided_code(x, scale);
  float t, unused;
  f2_out(f2_quotient(f2(x, 0.f), f2(-scale, -scale), f2(inverse, inverse)), t, unused);
  return __float_as_uint(t + ROUNDER) & 255u;
}
__device__ __forceinline__ uint2 codes_of(const float (&x)[8], float scale, float inverse) {
  uint32_t c[8];
  if (scale > 1e-30f) {
    const F2 inv = f2(inverse, inverse), minus = f2(-scale, -scale), up = f2(ROUNDER, ROUNDER);
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      float t0, t1;
      f2_out(f2_add(f2_quotient(f2(x[e], x[e + 1]), minus, inv), up), t0, t1);
      c[e] = __float_as_uint(t0);
      c[e + 1] = __float_as_uint(t1);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = divided_code(x[e], scale);
  }
  // (the low bytes of four words side by side)
  return make_uint2(__byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410));
}

// a block a row; KEPT: steps that stay in registers (0: the row is read twice)
template <typename T, int KEPT>
__global__ void __launch_bounds__(QUANT_THREADS) quantize_rows_kernel(QuantParams p, bool vec) {
  __shared__ uint32_t tops[QUANT_THREADS / 32];
  const int threads = blockDim.x, warps = threads / 32;
  pdl_wait();
  pdl_trigger();
  const size_t m = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + m * p.ldx;
  signed char* out = p.codes + m * p.ldq;
  const int n8 = vec ? p.K / 8 : 0;
  uint32_t top = 0;
  Eight<T> kept[KEPT > 0 ? KEPT : 1];
  if constexpr (KEPT > 0) {
#pragma unroll
    for (int k = 0; k < KEPT; ++k)
      if (threadIdx.x + k * threads < n8) kept[k].load(x + (threadIdx.x + k * threads) * 8);
#pragma unroll
    for (int k = 0; k < KEPT; ++k)
      if (threadIdx.x + k * threads < n8) kept[k].look(top);
  } else {
    for (int i = threadIdx.x; i < n8; i += threads) {
      kept[0].load(x + i * 8);
      kept[0].look(top);
    }
  }
  top = Eight<T>::bits(top);
  for (int i = n8 * 8 + threadIdx.x; i < p.K; i += threads) top = Eight<float>::largest(top, to_f32<T>(x[i]));
  top = __reduce_max_sync(0xffffffffu, top);
  if (warps > 1) {
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, tops[(threadIdx.x & 31) % warps]);
  }
  const bool bad = top >= 0x7f800000u;
  const float scale = __fdiv_rn(__uint_as_float(top), 127.f);
  const bool zero = bad || !(scale > 0.f);
  if (threadIdx.x == 0) p.scales[m] = bad ? __int_as_float(0x7fc00000) : scale;
  const float inverse = 1.f / scale;
  auto write = [&](const Eight<T>& at, int i) {
    float v[8];
    at.get(v);
    *reinterpret_cast<uint2*>(out + i * 8) = zero ? make_uint2(0u, 0u) : codes_of(v, scale, inverse);
  };
  if constexpr (KEPT > 0) {
#pragma unroll
    for (int k = 0; k < KEPT; ++k)
      if (threadIdx.x + k * threads < n8) write(kept[k], threadIdx.x + k * threads);
  } else {
    for (int i = threadIdx.x; i < n8; i += threads) {
      kept[0].load(x + i * 8);
      write(kept[0], i);
    }
  }
  for (int i = n8 * 8 + threadIdx.x; i < p.K; i += threads) out[i] = zero ? 0 : (signed char)code_of(to_f32<T>(x[i]), scale, inverse);
}

// ------------------------------------------------------------------------------------------ the product
constexpr int TILE_N = 128;          // weight rows of a block (MMA M)
constexpr int BK = 128;              // codes of a stage: 128 bytes, one swizzle row
constexpr int K_STEPS = BK / 32;     // MMAs of a stage
constexpr int THREADS = 128;         // warp 0 loads, warp 1 issues, all four do the epilogue
constexpr int W_STAGE_BYTES = TILE_N * BK;
constexpr int MAX_SPLITS = 8;

struct I8Params {
  void* out;            // [M, ldc] bfloat16 or float
  const float* sx;      // [M]
  const float* sw;      // [N]
  VecParam bias;        // [N]; ptr null: none
  long long ldc;
  int M, N, K, splits, out_f32;
  int w_ready;          // nobody that may still run writes the codes of W: they are fetched before the dependency wait
};

// instruction descriptor: signed 8-bit x signed 8-bit -> 32-bit integers, both operands K-major, M = 128, N = tile_t
__host__ __device__ constexpr uint32_t instr_desc(int tile_t) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(tile_t >> 3) << 17) | (static_cast<uint32_t>(TILE_N >> 4) << 24);
}
__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
// four words of a peer's shared memory, at the place that `own_shared` names in this block's
__device__ __forceinline__ void cluster_store4(uint32_t own_shared, uint32_t rank, int a, int b, int c, int d) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(own_shared), "r"(rank));
  asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(remote), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

template <int TILE_T> struct Cfg {
  static constexpr int STAGE_BYTES = W_STAGE_BYTES + TILE_T * BK;
  static constexpr int RING = 110 * 1024;                     // two blocks share an SM
  static constexpr int STAGES = RING / STAGE_BYTES > 6 ? 6 : RING / STAGE_BYTES;
  static constexpr int TMEM_COLS = TILE_T < 32 ? 32 : TILE_T;
  static constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE_BYTES + 256;
  static_assert(STAGES >= 3 && STAGES * STAGE_BYTES >= (TILE_T + 4 * MAX_SPLITS) * TILE_N * 4, "the ring holds what the cluster sends");
};

template <int TILE_T>
__global__ void __launch_bounds__(THREADS, 2)
gemm_i8_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ I8Params p) {
  using C = Cfg<TILE_T>;
  extern __shared__ char smem_raw[];
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  char* ctrl = smem + (size_t)C::STAGES * C::STAGE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(ctrl);            // [STAGES]
  uint64_t* empty = full + C::STAGES;                            // [STAGES]
  uint64_t* accum = empty + C::STAGES;                           // [1]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(accum + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int t_tile = blockIdx.x, n_tile = blockIdx.y, split = blockIdx.z;          // the blocks that share a weight tile run together
  const int warp = threadIdx.x >> 5;
  const int kb_total = (p.K + BK - 1) / BK, per = (kb_total + p.splits - 1) / p.splits;
  const int kb0 = split * per, nkb = max(0, min(kb_total, kb0 + per) - kb0);

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    mbar_init(smem_u32(accum), 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n"
                 ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)C::TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  pdl_trigger();
  const uint32_t tmem_base = *tmem_slot;
  __shared__ float sx[TILE_T];          // (from global memory, a row's scale was waited for at every store: 5 us of 130 tokens x 1,024 on 4,096 rows)

  if (threadIdx.x == 0) {
    // loader: one slice of K per stage
    if (!p.w_ready) pdl_wait();
    const int pre = min(nkb, C::STAGES);
    for (int i = 0; i < pre; ++i) {
      const uint32_t bar = smem_u32(&full[i]);
      mbar_expect_tx(bar, C::STAGE_BYTES);
      tma_load_2d(smem_u32(smem + (size_t)i * C::STAGE_BYTES), &map_w, bar, (kb0 + i) * BK, n_tile * TILE_N);
    }
    pdl_wait();
    for (int i = 0; i < pre; ++i)
      tma_load_2d(smem_u32(smem + (size_t)i * C::STAGE_BYTES + W_STAGE_BYTES), &map_x, smem_u32(&full[i]), (kb0 + i) * BK, t_tile * TILE_T);
    int armed = pre;
    for (int i = pre; i < nkb; ++i) {
      const int s = i % C::STAGES;
      if (!mbar_wait(smem_u32(&empty[s]), ((i / C::STAGES) & 1) ^ 1, abort_flag)) break;
      const uint32_t bar = smem_u32(&full[s]);
      mbar_expect_tx(bar, C::STAGE_BYTES);
      char* stage = smem + (size_t)s * C::STAGE_BYTES;
      tma_load_2d(smem_u32(stage), &map_w, bar, (kb0 + i) * BK, n_tile * TILE_N);
      tma_load_2d(smem_u32(stage + W_STAGE_BYTES), &map_x, bar, (kb0 + i) * BK, t_tile * TILE_T);
      armed = i + 1;
    }
    if (*abort_flag) {
      // let the copies that are still in flight land before the block goes away
      for (int i = max(0, armed - C::STAGES); i < armed; ++i) {
        const uint32_t bar = smem_u32(&full[i % C::STAGES]);
        for (uint32_t w = 0; w < WAIT_LIMIT && !mbar_try_wait(bar, (i / C::STAGES) & 1); ++w) {}
      }
    }
  } else if (warp == 1 && elect_one()) {
    pdl_wait();
    const uint32_t idesc = instr_desc(TILE_T);
    const uint64_t desc0 = smem_desc(smem_u32(smem));
    bool ok = true;
    for (int i = 0; i < nkb && ok; ++i) {
      const int s = i % C::STAGES;
      ok = mbar_spin_wait(smem_u32(&full[s]), (i / C::STAGES) & 1, abort_flag);
      if (!ok) break;
      tcgen05_fence_after();
      const uint64_t ad = desc0 + (uint64_t)s * (C::STAGE_BYTES >> 4), bd = ad + (W_STAGE_BYTES >> 4);
#pragma unroll
      for (int k = 0; k < K_STEPS; ++k) umma_i8(tmem_base, ad + 2 * k, bd + 2 * k, idesc, i > 0 || k > 0 ? 1u : 0u);
      tcgen05_commit(smem_u32(&empty[s]));
    }
    if (ok && nkb > 0) tcgen05_commit(smem_u32(accum));
  } else {
    pdl_wait();
    for (int j = (int)threadIdx.x - 64; j >= 0 && j < TILE_T; j += 64) sx[j] = t_tile * TILE_T + j < p.M ? p.sx[t_tile * TILE_T + j] : 0.f;
  }
  __syncthreads();

  // epilogue: lane = weight row, columns = tokens
  bool have = nkb > 0;
  if (have) have = mbar_spin_wait(smem_u32(accum), 0, abort_flag);
  have = __all_sync(0xffffffffu, have);      // tcgen05.ld is warp-wide: decide per warp
  tcgen05_fence_after();
  const int n = n_tile * TILE_N + threadIdx.x, t0 = t_tile * TILE_T;
  const uint32_t taddr = tmem_base + (static_cast<uint32_t>(warp * 32) << 16);
  const float sw = n < p.N ? p.sw[n] : 0.f;
  const float bn = p.bias.ptr != nullptr && n < p.N ? p.bias[n] : 0.f;
  auto put = [&](int j, int sum) {          // token j of the tile
    const float y = (float)sum * (sx[j] * sw) + bn;
    if (p.out_f32) static_cast<float*>(p.out)[(t0 + j) * p.ldc + n] = y;
    else static_cast<bf16*>(p.out)[(t0 + j) * p.ldc + n] = __float2bfloat16_rn(y);
  };
  constexpr int COLS = TILE_T < 32 ? TILE_T : 32;           // tokens taken from tensor memory at a time
  auto take = [&](int c, int (&v)[COLS]) {
    if (!have) {
#pragma unroll
      for (int i = 0; i < COLS; ++i) v[i] = 0;
    } else if constexpr (COLS == 32) {
      float f[32];
      tmem_load32(taddr + c, f);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = __float_as_int(f[i]);
    } else {
#pragma unroll
      for (int h = 0; h < COLS; h += 8) {
        float f[8];
        tmem_load8(taddr + c + h, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[h + i] = __float_as_int(f[i]);
      }
    }
  };
  const int live = min(TILE_T, p.M - t0);
  if (p.splits == 1) {
#pragma unroll 1
    for (int c = 0; c < live; c += COLS) {
      int v[COLS];
      take(c, v);
      if (n < p.N) {
#pragma unroll
        for (int i = 0; i < COLS; ++i)
          if (c + i < live) put(c + i, v[i]);
      }
    }
  } else {
    // Once no block of the cluster reads its ring any more, every block sends its sums to the block that owns the token (rank r: `own` tokens
    // in a row from r own on, a multiple of four), which adds them up from its own shared memory.  (Loads from the peers instead, eight
    // in flight a thread, take a trip through the cluster for every token: 256 tokens x 4,096 on 4,096 rows 21 us.)
    const int own = ((live + p.splits - 1) / p.splits + 3) & ~3;
    const uint32_t box = smem_u32(smem);                    // [sender][four tokens of mine][weight row][token]: a warp's stores are one run
    // (by weight row first, 64 x 12,288 on 4,096 rows took 17.7 us instead of 13.9)
    cluster_arrive();
    cluster_wait();
#pragma unroll 1
    for (int c = 0; c < live; c += COLS) {
      int v[COLS];
      take(c, v);
#pragma unroll
      for (int i = 0; i < COLS; i += 4) {
        const int j = c + i, owner = j / own;
        if (j < live) cluster_store4(box + ((split * own + j - owner * own) * (TILE_N / 4) + threadIdx.x) * 16, owner, v[i], v[i + 1], v[i + 2], v[i + 3]);
      }
    }
    cluster_arrive();
    cluster_wait();
    const int4* sums = reinterpret_cast<const int4*>(smem);
    for (int j = 0; j < own && split * own + j < live; j += 4) {
      int4 sum = make_int4(0, 0, 0, 0);
#pragma unroll
      for (int s = 0; s < MAX_SPLITS; ++s)
        if (s < p.splits) {
          const int4 x = sums[(s * own + j) * (TILE_N / 4) + threadIdx.x];
          sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
        }
      if (n < p.N) {
        const int at = split * own + j, v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (at + i < live) put(at + i, v[i]);
      }
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 0) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"((uint32_t)C::TMEM_COLS) : "memory");
  }
}

// ---------------------------------------------------------------------------- host side
// rows x K codes with leading dimension ld; boxes of box_rows x 128
bool make_map(CUtensorMap* map, const void* base, long long rows, long long K, long long ld, int box_rows) {
  EncodeTiledFn fn = encode_tiled();
  if (!fn) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {BK, (cuuint32_t)box_rows};
  const cuuint32_t elem[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int TILE_T>
int launch(const CUtensorMap& map_w, const CUtensorMap& map_x, const I8Params& p, cudaStream_t stream) {
  static SmemSet set;
  const cudaError_t sized = set.to(gemm_i8_kernel<TILE_T>, (int)Cfg<TILE_T>::SMEM);
  if (sized != cudaSuccess) return ts_fail("gemm_int8: %s", cudaGetErrorString(sized));
  const dim3 grid((p.M + TILE_T - 1) / TILE_T, (p.N + TILE_N - 1) / TILE_N, p.splits);
  const cudaError_t e = ts_launch_cluster(gemm_i8_kernel<TILE_T>, grid, dim3(THREADS), Cfg<TILE_T>::SMEM, stream, dim3(1, 1, p.splits), map_w, map_x, p);
  if (e != cudaSuccess) return ts_fail("gemm_int8 (clusters of %d): %s", p.splits, cudaGetErrorString(e));
  return 0;
}

template <typename T>
int launch_quantize(const QuantParams& p, bool vec, int M, cudaStream_t stream) {
  // many rows: fewer threads with more of a row each (a block is short, and there are enough of them); few rows: as many as there are
  const int n8 = (p.K + 7) / 8, share = M >= 512 ? (n8 + QUANT_KEPT - 1) / QUANT_KEPT : n8;
  const int threads = share >= QUANT_THREADS ? QUANT_THREADS : (share + 31) / 32 * 32;
  if (!vec || n8 > QUANT_KEPT * threads) TS_LAUNCH("quantize_rows", (quantize_rows_kernel<T, 0>), dim3(M), dim3(vec ? threads : QUANT_THREADS), 0, stream, p, vec);
  else if (n8 <= threads) TS_LAUNCH("quantize_rows", (quantize_rows_kernel<T, 1>), dim3(M), dim3(threads), 0, stream, p, vec);
  else TS_LAUNCH("quantize_rows", (quantize_rows_kernel<T, QUANT_KEPT>), dim3(M), dim3(threads), 0, stream, p, vec);
  return 0;
}

int quantize(int dtype, const void* x, long long ldx, void* codes, long long ldq, float* scales, int M, int K, cudaStream_t stream) {
  const int e = dtype == TS_F32 ? 4 : 2;
  const bool vec = (((uintptr_t)x | (uintptr_t)(ldx * e)) & 15) == 0 && (((uintptr_t)codes | (uintptr_t)ldq) & 7) == 0;
  const QuantParams p = {x, static_cast<signed char*>(codes), scales, ldx, ldq, K};
  return dtype == TS_F32 ? launch_quantize<float>(p, vec, M, stream) : launch_quantize<bf16>(p, vec, M, stream);
}

}  // namespace

// 1 if a block ever gave up on a wait since the library was loaded (reads device memory: syncs)
TS_EXPORT int ts_gemm_int8_error() {
  int flag = 0;
  if (cudaMemcpyFromSymbol(&flag, g_error_flag, sizeof(int)) != cudaSuccess) return -1;
  return flag;
}

// codes [M, K] (leading dimension ldq) and scales [M] of the rows of x [M, K] (ldx)
static int quantize_rows(int dtype, const void* x, long long ldx, void* codes, long long ldq, float* scales, int M, int K, cudaStream_t stream) {
  TS_REQUIRE(dtype == TS_F32 || dtype == TS_BF16, "quantize_rows: unknown dtype %d", dtype);
  TS_REQUIRE(M > 0 && K > 0, "quantize_rows: empty operand");
  return quantize(dtype, x, ldx, codes, ldq, scales, M, K, stream);
}
TS_ENTRY(quantize_rows)

// out [M, N] (ldc; float where out_f32, else bfloat16) from codes and scales of x and w (leading dimensions multiples of 16).
// x_dtype >= 0: x is a tensor of that type (leading dimension ldx) whose rows are brought to cx, sx first; -1: cx and sx are given.
// tile_t: tokens of a tile (16, 32, 64 or 128); splits: cuts along K (a cluster of up to 8 blocks).  w_constant: nobody that may still run writes w, whose first
// codes are then fetched before the product's dependency wait.
static int gemm_int8(int x_dtype, const void* x, long long ldx, void* cx, long long ldcx, float* sx, const void* cw, long long ldw,
                     const float* sw, const void* bias, int bias_f32, void* out, long long ldc, int out_f32, int M, int N, int K,
                     int tile_t, int splits, int w_constant, cudaStream_t stream) {
  TS_REQUIRE(M > 0 && N > 0 && K > 0 && K <= 131072, "gemm_int8: M=%d N=%d K=%d (K up to 131072: the sums are 32-bit integers)", M, N, K);
  TS_REQUIRE((ldcx | ldw) % 16 == 0 && (((uintptr_t)cx | (uintptr_t)cw) & 15) == 0, "gemm_int8: rows of codes begin on 16 bytes");
  TS_REQUIRE(splits >= 1 && splits <= MAX_SPLITS, "gemm_int8: splits out of range");
  TS_REQUIRE(tile_t == 16 || tile_t == 32 || tile_t == 64 || tile_t == 128, "gemm_int8: tiles of %d tokens", tile_t);
  TS_REQUIRE((N + TILE_N - 1) / TILE_N <= 65535, "gemm_int8: too many outputs");
  if (x_dtype >= 0) {
    TS_REQUIRE(x_dtype == TS_F32 || x_dtype == TS_BF16, "gemm_int8: unknown dtype %d", x_dtype);
    const int rc = quantize(x_dtype, x, ldx, cx, ldcx, sx, M, K, stream);
    if (rc != 0) return rc;
  }
  CUtensorMap map_w, map_x;
  TS_REQUIRE(make_map(&map_w, cw, N, K, ldw, TILE_N) && make_map(&map_x, cx, M, K, ldcx, tile_t), "gemm_int8: cuTensorMapEncodeTiled failed");
  const I8Params p = {out, sx, sw, VecParam{bias, bias_f32}, ldc, M, N, K, splits, out_f32, w_constant};
  switch (tile_t) {
    case 16: return launch<16>(map_w, map_x, p, stream);
    case 32: return launch<32>(map_w, map_x, p, stream);
    case 64: return launch<64>(map_w, map_x, p, stream);
    default: return launch<128>(map_w, map_x, p, stream);
  }
}
TS_ENTRY(gemm_int8)
