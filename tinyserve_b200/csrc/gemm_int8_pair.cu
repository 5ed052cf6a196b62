// The 8-bit product y[m, n] = (sum_k cx[m, k] cw[n, k]) sx[m] sw[n] (+ bias[n]) of many tokens (see gemm_int8.cu for the codes), on pairs of SMs:
// tcgen05.mma.cta_group::2, kind::i8, sums in 32-bit integers.
//
// The arrangement is that of gemm_pair_tcgen05.cu, whose stages, boxes and swizzle carry over byte for byte (a slice of K of 128 codes is the
// 128 bytes of 64 bfloat16): two blocks of a cluster share a tile of 256 tokens x 256 weight rows, each loads its 128 token rows
// and half of the weight rows by TMA, one thread of the first block issues and commits to both, two accumulators take turns so that a
// tile's epilogue runs beside the next one's MMAs, the grid is persistent.  2,048 tokens x 4,096 on 24,576 rows: 131 us, 3.1 POPS;
// with tiles of 512 weight rows (half again as many MMAs for a byte loaded, but one accumulator) 157 us, with blocks on their own (tiles of
// 128 x 128, gemm_int8.cu) 284; the library's bfloat16 product takes 273.  What bounds it: a slice's MMAs take 512 cycles for 32 KB that
// each SM loads.
//
// The epilogue scales a row's sums by sx[m] sw[n] in 32 bits and reaches global memory through tiles of 128 rows x 128 bytes in shared memory, so that
// stores cover whole lines.  Every wait is bounded; a block that gives up tells its partner.
#include "entry.cuh"
#include "tcgen05.cuh"

TS_DEFINE_LAST_ERROR()

namespace {

using bf16 = __nv_bfloat16;
constexpr int BM = 128;              // token rows of a block (256 of the pair)
constexpr int HALF_N = 256;          // weight rows of one MMA over the pair (128 in each block's shared memory)
constexpr int BK = 128;              // codes of a stage: 128 bytes, one swizzle row
constexpr int A_BYTES = BM * BK, B_BYTES = HALF_N / 2 * BK;
constexpr int K_STEPS = BK / 32;
constexpr int LOAD_WARP = 4, ISSUE_WARP0 = 5;        // warps 0-3: epilogue; 4: loads; 5: issues
constexpr int TMEM_COLS = 512;
constexpr int CHUNK = 32;

constexpr int STAGE_BYTES = A_BYTES + B_BYTES, STAGES = 5, THREADS = 32 * (ISSUE_WARP0 + 1);
constexpr int UNITS = 8;             // 16-byte units of a row of the epilogue's tile
constexpr int TILE_BYTES = BM * UNITS * 16;
constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE_BYTES + TILE_BYTES + 2 * HALF_N * 4 + 256;

struct PairParams {
  void* out;              // [M, ldc] bfloat16 or float
  const float* sx;        // [M]
  const float* sw;        // [N]
  VecParam bias;          // [N]; ptr null: none
  long long ldc;
  int out_f32, M, N, K;
  int tiles_m, tiles, pairs, slices;
};

__device__ __forceinline__ uint32_t map_to_rank(uint32_t local, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  return remote;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(cluster_addr) : "memory");
}
// a TMA load of this block's shared memory whose bytes are counted on an mbarrier of either block
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar_cluster, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void umma_pair_i8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
// arrives on the mbarrier at this shared-memory offset in both blocks once this thread's MMAs are done
__device__ __forceinline__ void commit_pair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n"
      ::"r"(bar), "h"((uint16_t)3) : "memory");
}
// the four warps of the epilogue meet
__device__ __forceinline__ void epi_barrier() { asm volatile("bar.sync 1, 128;\n" ::: "memory"); }
// true if `ok` holds for every thread of them
__device__ __forceinline__ bool epi_all(bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "bar.red.and.pred p, 1, 128, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(r) : "r"((uint32_t)ok) : "memory");
  return r != 0;
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
// unit u (16 bytes) of row r of an epilogue tile: rows that are written together use different banks
__device__ __forceinline__ uint4* tile_unit(char* tile, int r, int u) {
  return reinterpret_cast<uint4*>(tile + r * UNITS * 16 + ((u ^ (r & 7)) << 4));
}

// The epilogue of a pair's i-th tile, by four warps of each block.  A thread owns a token row of the tensor memory; global memory is reached
// with eight threads on the 128 bytes of a row.  Returns false if a wait ran out.
__device__ __forceinline__ bool epilogue(const PairParams& p, int tile, int i, int quarter, int lane, uint32_t rank,
                                              uint32_t tmem_base, uint64_t* acc_full, uint32_t acc_empty0, char* stage, float* scales,
                                              volatile int* abort_flag) {
  const int buf = i & 1;
  const uint32_t parity = (uint32_t)(i >> 1) & 1u;
  const int r_in = quarter * 32 + lane;                        // the row this thread owns in tensor memory
  const int tm = tile % p.tiles_m, tn = tile / p.tiles_m;
  const int row0 = tm * 2 * BM + (int)rank * BM;               // first row of this block's half of the tile
  const int col0 = tn * HALF_N;
  const uint32_t acc = tmem_base + ((uint32_t)(quarter * 32) << 16) + buf * HALF_N;
  const int u = r_in % UNITS, rb = r_in / UNITS;               // the other arrangement: unit u of rows rb + 16 j
  // (scales and bias do not depend on the MMAs: they are read during the wait)
  float* bias = scales + HALF_N;
  for (int c = r_in; c < HALF_N; c += 128) {
    const int n = col0 + c;
    scales[c] = n < p.N ? p.sw[n] : 0.f;
    bias[c] = p.bias.ptr != nullptr && n < p.N ? p.bias[n] : 0.f;
  }
  const float sx = row0 + r_in < p.M ? p.sx[row0 + r_in] : 0.f;
  // (all four warps go on or none does: they meet at barriers below)
  if (!epi_all(mbar_wait(smem_u32(&acc_full[buf]), parity, abort_flag))) return false;
  tcgen05_fence_after();
  // 128 bytes of output a row at a time: 32 columns of float or 64 of bfloat16
  const int cols = p.out_f32 ? 32 : 64, esize = p.out_f32 ? 4 : 2;
  for (int c0 = 0; c0 < HALF_N && col0 + c0 < p.N; c0 += cols) {
    for (int sub = 0; sub < cols; sub += CHUNK) {
      float v[CHUNK];
      tmem_load32(acc + c0 + sub, v);
#pragma unroll
      for (int e = 0; e < CHUNK; e += 4) {
        const float4 s = *reinterpret_cast<const float4*>(scales + c0 + sub + e), b = *reinterpret_cast<const float4*>(bias + c0 + sub + e);
        v[e] = (float)__float_as_int(v[e]) * (sx * s.x) + b.x;
        v[e + 1] = (float)__float_as_int(v[e + 1]) * (sx * s.y) + b.y;
        v[e + 2] = (float)__float_as_int(v[e + 2]) * (sx * s.z) + b.z;
        v[e + 3] = (float)__float_as_int(v[e + 3]) * (sx * s.w) + b.w;
      }
      if (p.out_f32) {
#pragma unroll
        for (int q = 0; q < 8; ++q)
          *tile_unit(stage, r_in, q) = make_uint4(__float_as_uint(v[4 * q]), __float_as_uint(v[4 * q + 1]), __float_as_uint(v[4 * q + 2]), __float_as_uint(v[4 * q + 3]));
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *tile_unit(stage, r_in, sub / 8 + q) = make_uint4(pack2(v[8 * q], v[8 * q + 1]), pack2(v[8 * q + 2], v[8 * q + 3]),
                                                            pack2(v[8 * q + 4], v[8 * q + 5]), pack2(v[8 * q + 6], v[8 * q + 7]));
      }
    }
    epi_barrier();
    if ((col0 + c0) * esize + u * 16 < p.N * esize) {
      char* out = static_cast<char*>(p.out) + ((size_t)row0 * p.ldc + col0 + c0) * esize;
#pragma unroll
      for (int j = 0; j < BM / 16; ++j) {
        const int r = rb + 16 * j;
        if (row0 + r < p.M) *reinterpret_cast<uint4*>(out + (size_t)r * p.ldc * esize + u * 16) = *tile_unit(stage, r, u);
      }
    }
    epi_barrier();          // the tile is written again
  }
  tcgen05_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive_cluster(acc_empty0 + buf * 8);
  return true;
}

__global__ void __launch_bounds__(THREADS, 1)
gemm_i8_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, PairParams p) {
  extern __shared__ char smem_raw[];
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  char* tiles = smem + (size_t)STAGES * STAGE_BYTES;       // the epilogue's
  float* scales = reinterpret_cast<float*>(tiles + TILE_BYTES);      // [2][256]
  char* ctrl = reinterpret_cast<char*>(scales + 2 * HALF_N);
  uint64_t* full = reinterpret_cast<uint64_t*>(ctrl);            // [STAGES], used in the first block
  uint64_t* empty = full + STAGES;                            // [STAGES], in both blocks
  uint64_t* acc_full = empty + STAGES;                        // [2], in both blocks
  uint64_t* acc_empty = acc_full + 2;                            // [2], used in the first block
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();                          // 0: the block that issues the MMAs
  const int pair = blockIdx.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&acc_full[b]), 1);
      mbar_init(smem_u32(&acc_empty[b]), 2 * 4);     // every epilogue warp of both blocks
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == LOAD_WARP) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n"
                 ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  // both blocks' barriers exist before either block's loads or commits may reach them
  cluster_arrive();
  cluster_wait();
  tcgen05_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_trigger();
  pdl_wait();

  auto tell_partner = [&]() {
    const uint32_t remote = map_to_rank(smem_u32(const_cast<int*>(abort_flag)), rank ^ 1u);
    asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(remote), "r"(1u) : "memory");
  };
  const uint32_t acc_empty0 = map_to_rank(smem_u32(acc_empty), 0);
  if (warp == LOAD_WARP) {
    if (lane == 0) {
      const uint32_t full0 = map_to_rank(smem_u32(full), 0);     // the first block's barriers
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < p.tiles; tile += p.pairs) {
        const int row_x = (tile % p.tiles_m) * 2 * BM + (int)rank * BM;
        const int row_w = (tile / p.tiles_m) * HALF_N + (int)rank * (HALF_N / 2);
        for (int s = 0; s < p.slices; ++s) {
          ok = mbar_wait(smem_u32(&empty[stage]), phase ^ 1u, abort_flag);
          if (!ok) break;
          if (rank == 0) mbar_expect_tx(smem_u32(&full[stage]), 2 * STAGE_BYTES);
          const uint32_t dst = smem_u32(smem + (size_t)stage * STAGE_BYTES);
          tma_load_2d_pair(dst, &map_x, full0 + stage * 8, s * BK, row_x);
          tma_load_2d_pair(dst + A_BYTES, &map_w, full0 + stage * 8, s * BK, row_w);
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
      }
      if (!ok) tell_partner();
    }
  } else if (warp >= ISSUE_WARP0) {
    // signed 8-bit x signed 8-bit -> 32-bit integers, both operands K-major, M = 256 over the pair, N = 256
    const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(HALF_N >> 3) << 17) | ((uint32_t)((2 * BM) >> 4) << 24);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    int i = 0;
    for (int tile = pair; ok && tile < p.tiles; tile += p.pairs, ++i) {
      if (rank == 0 && elect_one()) {
        const int buf = i & 1;
        const uint32_t parity = (uint32_t)(i >> 1) & 1u;
        // (a buffer is free at the start: the wait on the phase before the first returns at once)
        ok = mbar_spin_wait(smem_u32(&acc_empty[buf]), parity ^ 1u, abort_flag);
        tcgen05_fence_after();
        const uint32_t d = tmem_base + buf * HALF_N;
        for (int s = 0; ok && s < p.slices; ++s) {
          ok = mbar_spin_wait(smem_u32(&full[stage]), phase, abort_flag);
          if (!ok) break;
          tcgen05_fence_after();
          const uint64_t a = smem_desc(smem_u32(smem + (size_t)stage * STAGE_BYTES));
#pragma unroll
          for (int k = 0; k < K_STEPS; ++k) umma_pair_i8(d, a + k * 2, a + (A_BYTES >> 4) + k * 2, idesc, s > 0 || k > 0 ? 1u : 0u);
          commit_pair(smem_u32(&empty[stage]));
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
        if (ok) commit_pair(smem_u32(&acc_full[buf]));
        if (!ok) tell_partner();
      }
      // the issuing thread's outcome is its warp's (which meets again here before the next election)
      ok = __all_sync(0xffffffffu, ok) != 0;
    }
  } else {
    bool ok = true;
    int i = 0;
    for (int tile = pair; ok && tile < p.tiles; tile += p.pairs, ++i)
      ok = epilogue(p, tile, i, warp, lane, rank, tmem_base, acc_full, acc_empty0, tiles, scales, abort_flag);
    if (!ok && lane == 0) tell_partner();
  }
  // neither block leaves (or frees its tensor memory) while the other may still reach its barriers
  tcgen05_fence_before();
  __syncthreads();
  cluster_arrive();
  cluster_wait();
  if (warp == LOAD_WARP) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"((uint32_t)TMEM_COLS) : "memory");
  }
}

bool make_map(CUtensorMap* map, const void* base, int rows, int K, long long ld) {
  EncodeTiledFn fn = encode_tiled();
  if (!fn) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {BK, 128};
  const cuuint32_t elem[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int launch(const CUtensorMap& mx, const CUtensorMap& mw, PairParams p, int pairs, cudaStream_t stream) {
  static SmemSet set;
  const cudaError_t sized = set.to(gemm_i8_pair_kernel, (int)SMEM);
  if (sized != cudaSuccess) return ts_fail("gemm_int8_pair: %s", cudaGetErrorString(sized));
  p.tiles = p.tiles_m * ((p.N + HALF_N - 1) / HALF_N);
  p.pairs = pairs < p.tiles ? pairs : p.tiles;
  const cudaError_t e = ts_launch_cluster(gemm_i8_pair_kernel, dim3(2 * p.pairs), dim3(THREADS), SMEM, stream, dim3(2, 1, 1), mx, mw, p);
  if (e != cudaSuccess) return ts_fail("gemm_int8_pair: %s", cudaGetErrorString(e));
  return 0;
}

}  // namespace

TS_EXPORT int ts_gemm_int8_pair_error() {
  int flag = 0;
  if (cudaMemcpyFromSymbol(&flag, g_error_flag, sizeof(int)) != cudaSuccess) return -1;
  return flag;
}

// out [M, N] (ldc; float where out_f32, else bfloat16; rows of whole 16 bytes) from codes and scales of x and w (leading dimensions multiples of 16).
// pairs: SM pairs of the device.
static int gemm_int8_pair(const void* cx, long long ldcx, const float* sx, const void* cw, long long ldw, const float* sw, const void* bias,
                          int bias_f32, void* out, long long ldc, int out_f32, int M, int N, int K, int pairs, cudaStream_t stream) {
  TS_REQUIRE(M > 0 && N > 0 && K > 0 && K <= 131072 && pairs > 0, "gemm_int8_pair: M=%d N=%d K=%d (K up to 131072: the sums are 32-bit integers)", M, N, K);
  TS_REQUIRE((ldcx | ldw) % 16 == 0 && (((uintptr_t)cx | (uintptr_t)cw) & 15) == 0, "gemm_int8_pair: rows of codes begin on 16 bytes");
  const int e = out_f32 ? 4 : 2;
  TS_REQUIRE(ldc * e % 16 == 0 && N * e % 16 == 0 && ((uintptr_t)out & 15) == 0, "gemm_int8_pair: rows of the output are whole 16 bytes");
  CUtensorMap mx, mw;
  TS_REQUIRE(make_map(&mx, cx, M, K, ldcx) && make_map(&mw, cw, N, K, ldw), "gemm_int8_pair: cuTensorMapEncodeTiled failed");
  PairParams p = {};
  p.out = out; p.sx = sx; p.sw = sw; p.bias = VecParam{bias, bias_f32}; p.ldc = ldc; p.out_f32 = out_f32; p.M = M; p.N = N; p.K = K;
  p.tiles_m = (M + 2 * BM - 1) / (2 * BM);
  p.slices = (K + BK - 1) / BK;
  return launch(mx, mw, p, pairs, stream);
}
TS_ENTRY(gemm_int8_pair)
