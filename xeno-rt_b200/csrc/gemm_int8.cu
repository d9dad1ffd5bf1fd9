// out[M, N] = (codes[M, K] . W[N, K]^T) * scales[m] * w_scales[n] (+ bias[n]) of signed 8-bit integers, on the
// fifth-generation tensor cores (tcgen05.mma kind::i8): the sums over K are 32-bit integers and exact, whatever their
// order, and are rounded to 32-bit floating point once, before the scales.  K is bounded by the caller's check, so that
// 128 * 128 * K stays below 2^31.
//
// Many rows: a persistent block, or a pair of blocks as one (cta_group::2, Int8Shape), one block a multiprocessor, walks output
// tiles of 128 (a pair: 256) rows and BN columns.  Seven warps a block:
//   warps 0, 1  producers, one of the block's 128 rows of codes, one of its rows of W (in a pair half of the tile's): for each
//               128-wide slab of K a TMA load into the next free stage of a ring; what a tile has beyond M, N or K
//               arrives as zeros.
//   warp 2      owns TMEM (two accumulators of 128 lanes x BN columns) and issues the MMAs (in a pair the first block's does,
//               for both): four a stage, each 32 bytes of K.
//   warps 3-6   epilogue: each warp reads its 32 TMEM lanes (rows), 32 columns at a time, applies the scales and writes
//               patches of 32 rows x 128 bytes to shared memory, which a TMA store takes (or a TMA reduction adds into the
//               output), while the MMA warp fills the other accumulator.  Outputs whose rows do not begin and end
//               every 16 bytes are stored by the warp, a row of 32 columns at a time.
// What bounds it: the tensor pipe, 93 percent of whose cycles are taken while a block runs (2,048 rows of 28,672 outputs, 4,096
// inputs 145-153 us; 8,192 546, 3,527 TOP/s, until the power limit lowers the clock: 655 in a loop of seconds).  Products of one
// wave of tiles are their walk over K and the ends: 512 rows of 4,096, 4,096 11.2 us, 333 of 5,003, 1,999 7.7 (of 5,008, 2,048,
// whose output rows begin every 16 bytes, 7.2).  Few rows: see there.
//
// Every wait on an mbarrier is bounded.  A wait that runs out raises the error flag and an abort flag in shared memory; all
// roles leave their loops, the block waits for its copies in flight (bounded too), frees its TMEM and returns.
#include <stddef.h>

#include <type_traits>

#include "tcgen05.cuh"

namespace xrt {

using namespace sm100;

constexpr int I8_BM = 128, I8_BK = 128, I8_UMMA_K = 32;
constexpr int I8_THREADS = 32 * 7;
template <bool PAIR, int BN> struct Int8Shape {
  static constexpr int A_BYTES = I8_BM * I8_BK;
  static constexpr int B_ROWS = PAIR ? BN / 2 : BN;  // of the W tile, in one block
  static constexpr int STAGE_BYTES = A_BYTES + B_ROWS * I8_BK;
  static constexpr int STAGES = 196608 / STAGE_BYTES;
  static constexpr int PATCH_BYTES = 5120;             // an epilogue warp's: 32 x 128 bytes, or 32 rows of 33 floats
  static constexpr int STAGING_BYTES = 4 * PATCH_BYTES;
  static constexpr int FACTOR_BYTES = 2 * 2 * BN * 4;  // scales and biases of a tile's columns, one set an accumulator
  static constexpr int SMEM = STAGES * STAGE_BYTES + STAGING_BYTES + FACTOR_BYTES + 512 + 1024;
};

// What the sums are multiplied by and what is added.
struct Int8Scales {
  const float* rows;     // [M]
  const float* columns;  // [N]
  const float* bias;     // [N] or null
};

// Where a tile lies.  Tiles that run at the same time should share operands in the L2: the walk goes down 4,096 rows of codes,
// then to the next column of tiles, and only after the last column to the next such group of rows.
template <int TILE_ROWS>
__device__ __forceinline__ void int8_tile_place(int tile, int tiles_m, int tiles_n, int& m_blk, int& n_blk) {
  constexpr int GROUP = 4096 / TILE_ROWS;
  const int per_group = GROUP * tiles_n;
  const int group = tile / per_group, in_group = tile - group * per_group;
  const int rows = min(GROUP, tiles_m - group * GROUP);
  n_blk = in_group / rows;
  m_blk = group * GROUP + (in_group - n_blk * rows);
}

// 16 bytes of a patch's row: four float32 or eight bfloat16 from value `at` on.
template <typename TO>
__device__ __forceinline__ uint4 int8_unit(const float (&v)[32], int at);
template <>
__device__ __forceinline__ uint4 int8_unit<float>(const float (&v)[32], int at) {
  return make_uint4(__float_as_uint(v[at]), __float_as_uint(v[at + 1]), __float_as_uint(v[at + 2]), __float_as_uint(v[at + 3]));
}
template <>
__device__ __forceinline__ uint4 int8_unit<__nv_bfloat16>(const float (&v)[32], int at) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 two = __floats2bfloat162_rn(v[at + 2 * i], v[at + 2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&two);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// MODE 0: store, 1: add into float out.
template <int MODE, bool PAIR, int BN, typename TO>
__global__ void __launch_bounds__(I8_THREADS, 1)
gemm_int8_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                 const __grid_constant__ CUtensorMap map_out, TO* out, int by_tma, int M, int N, int K, int ldo,
                 const Int8Scales scales, int* error_flag) {
  using Shape = Int8Shape<PAIR, BN>;
  constexpr int STAGES = Shape::STAGES, TILE_ROWS = (PAIR ? 2 : 1) * I8_BM;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
  unsigned char* a_stages = smem;
  unsigned char* b_stages = smem + STAGES * Shape::A_BYTES;
  unsigned char* staging = smem + STAGES * Shape::STAGE_BYTES;
  float* factors = reinterpret_cast<float*>(staging + Shape::STAGING_BYTES);  // [accumulator][scales, biases][column]
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + Shape::STAGING_BYTES + Shape::FACTOR_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles_m = (M + TILE_ROWS - 1) / TILE_ROWS, tiles_n = (N + BN - 1) / BN;
  const int n_tiles = tiles_m * tiles_n;
  const int k_iters = (K + I8_BK - 1) / I8_BK;
  const int rank = PAIR ? (int)(blockIdx.x & 1) : 0;  // the block's place in its pair
  const int unit = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x, units = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;

  if (threadIdx.x == 0) {
    // a stage is full when both operands' bytes have been announced (each by its producer, in a pair by the first block's for both
    // blocks) and are there
    for (int s = 0; s < STAGES; ++s) { mbar_init(smem_u32(&full[s]), 2); mbar_init(smem_u32(&empty[s]), 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(smem_u32(&acc_full[a]), 1); mbar_init(smem_u32(&acc_empty[a]), PAIR ? 256 : 128); }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(2 * BN));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(2 * BN));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    pdl_trigger();  // not before: see common.cuh
  }
  fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();  // the other block's barriers stand before anything arrives on them
  fence_after();
  const uint32_t tmem_base = *tmem_slot;

  bool ok = true;
  auto give_up = [&]() {  // a wait ran out: every role leaves
    *abort_flag = 1;
    if (error_flag != nullptr) atomicExch(error_flag, 6);
  };
  if (warp < 2) {
    if (elect_one()) {
      const bool codes = warp == 0;
      const CUtensorMap* map = codes ? &map_x : &map_w;
      asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
      if (!codes) {  // the first of W on its way to the L2 while the kernel before finishes
        int m_blk, n_blk;
        int8_tile_place<TILE_ROWS>(unit, tiles_m, tiles_n, m_blk, n_blk);
        for (int kb = 0; kb < min(STAGES, k_iters); ++kb) tma_prefetch_2d(map, kb * I8_BK, n_blk * BN + rank * Shape::B_ROWS);
      }
      pdl_wait();
      const uint32_t stages = smem_u32(codes ? a_stages : b_stages), bytes = codes ? Shape::A_BYTES : Shape::B_ROWS * I8_BK;
      int s = 0;
      uint32_t turn = 1;
      for (int tile = unit; tile < n_tiles && ok; tile += units) {
        int m_blk, n_blk;
        int8_tile_place<TILE_ROWS>(tile, tiles_m, tiles_n, m_blk, n_blk);
        const int row0 = codes ? m_blk * TILE_ROWS + rank * I8_BM : n_blk * BN + rank * Shape::B_ROWS;
        for (int kb = 0; kb < k_iters; ++kb) {
          ok = mbar_wait(smem_u32(&empty[s]), turn, abort_flag);
          if (!ok) break;
          if (PAIR) {
            // both blocks' copies complete on the first block's barrier, which alone the MMAs wait for; the bytes of both are
            // announced there (a copy of the second block may complete before that: the phase cannot end without the
            // arrivals, and the second block reuses a stage only after the MMAs have released it)
            if (rank == 0) mbar_arrive_expect_tx(smem_u32(&full[s]), 2 * bytes);
            tma_load_2d_pair(stages + s * bytes, map, kb * I8_BK, row0, first_block_address(smem_u32(&full[s])));
          } else {
            mbar_arrive_expect_tx(smem_u32(&full[s]), bytes);
            tma_load_2d(stages + s * bytes, map, kb * I8_BK, row0, smem_u32(&full[s]));
          }
          if (++s == STAGES) { s = 0; turn ^= 1; }
        }
      }
      // a block of a pair leaves only when the other's MMAs have let go of its last stages
      for (int j = 0; PAIR && ok && j < STAGES; ++j) {
        ok = mbar_wait(smem_u32(&empty[s]), turn, abort_flag);
        if (++s == STAGES) { s = 0; turn ^= 1; }
      }
      if (!ok) give_up();
    }
  } else if (warp == 2) {
    if (rank == 0 && elect_one()) {
      constexpr uint32_t idesc = instr_desc_i8(TILE_ROWS, BN);
      auto slab = [&](uint32_t d, int s, auto adds) {  // `adds`: whether to the sums so far
        const uint64_t desc_a = desc_k_major(smem_u32(a_stages + s * Shape::A_BYTES));
        const uint64_t desc_b = desc_k_major(smem_u32(b_stages + s * Shape::B_ROWS * I8_BK));
#pragma unroll
        for (int k = 0; k < I8_BK / I8_UMMA_K; ++k) {  // 32 bytes further along K inside the swizzle atom
          if (PAIR) mma_i8_pair(d, desc_a + 2 * k, desc_b + 2 * k, idesc, decltype(adds)::value || k > 0);
          else mma_i8(d, desc_a + 2 * k, desc_b + 2 * k, idesc, decltype(adds)::value || k > 0);
        }
        if (PAIR) commit_pair(smem_u32(&empty[s]));
        else commit(smem_u32(&empty[s]));
      };
      int s = 0, a = 0;
      uint32_t turn = 0, acc_turn = 1;
      for (int tile = unit; tile < n_tiles && ok; tile += units) {
        ok = mbar_wait(smem_u32(&acc_empty[a]), acc_turn, abort_flag);
        if (!ok) break;
        fence_after();
        for (int kb = 0; kb < k_iters; ++kb) {
          ok = mbar_wait(smem_u32(&full[s]), turn, abort_flag);
          if (!ok) break;
          fence_after();
          if (kb == 0) slab(tmem_base + a * BN, s, std::false_type());
          else slab(tmem_base + a * BN, s, std::true_type());
          if (++s == STAGES) { s = 0; turn ^= 1; }
        }
        if (!ok) break;
        if (PAIR) commit_pair(smem_u32(&acc_full[a]));
        else commit(smem_u32(&acc_full[a]));
        if (++a == 2) { a = 0; acc_turn ^= 1; }
      }
      if (!ok) give_up();
    }
  } else {
    constexpr int CHUNK = 128 / sizeof(TO);  // columns of a patch
    const int quarter = warp & 3;            // the TMEM lanes this warp may read
    unsigned char* patch = staging + quarter * Shape::PATCH_BYTES;
    pdl_wait();
    int a = 0;
    uint32_t acc_turn = 0;
    for (int tile = unit; tile < n_tiles; tile += units) {
      int m_blk, n_blk;
      int8_tile_place<TILE_ROWS>(tile, tiles_m, tiles_n, m_blk, n_blk);
      const int row0 = m_blk * TILE_ROWS + rank * I8_BM + quarter * 32, col0 = n_blk * BN;
      const float row_scale = row0 + lane < M ? scales.rows[row0 + lane] : 0.f;
      float* by_column = factors + a * 2 * BN;
      for (int i = (int)threadIdx.x - 96; i < BN; i += 128) {
        const int n = min(col0 + i, N - 1);
        by_column[i] = scales.columns[n];
        by_column[BN + i] = scales.bias != nullptr ? scales.bias[n] : 0.f;
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");  // (the set of the tile before last is not read any more)
      // A warp whose wait ran out says so at once, and from then on only meets the others at this barrier, which they may
      // still come to.
      if (!ok) continue;
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&acc_full[a]), acc_turn, abort_flag));
      if (!ok) {
        if (lane == 0) give_up();
        continue;
      }
      fence_after();
      const uint32_t tmem_row = tmem_base + ((uint32_t)(quarter * 32) << 16) + a * BN;
#pragma unroll 1
      for (int c = 0; c < BN; c += 32) {
        uint32_t v[32];
        tmem_ld32(v, tmem_row + c);
        tmem_wait_ld();
        float value[32];
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const float4 f = *reinterpret_cast<const float4*>(by_column + c + j), b = *reinterpret_cast<const float4*>(by_column + BN + c + j);
          value[j] = fmaf(__int2float_rn((int)v[j]) * row_scale, f.x, b.x);
          value[j + 1] = fmaf(__int2float_rn((int)v[j + 1]) * row_scale, f.y, b.y);
          value[j + 2] = fmaf(__int2float_rn((int)v[j + 2]) * row_scale, f.z, b.z);
          value[j + 3] = fmaf(__int2float_rn((int)v[j + 3]) * row_scale, f.w, b.w);
        }
        if (by_tma) {
          const int part = c % CHUNK;  // where in the patch
          if (part == 0) {
            tma_stores_read();
            __syncwarp();
          }
#pragma unroll
          for (int j = 0; j < 32; j += 16 / sizeof(TO)) {
            const int u = (part + j) * (int)sizeof(TO) / 16;
            *reinterpret_cast<uint4*>(patch + lane * 128 + ((u ^ (lane & 7)) << 4)) = int8_unit<TO>(value, j);
          }
          if (part + 32 == CHUNK) {
            fence_to_async();
            __syncwarp();
            if (elect_one() && row0 < M && col0 + c - part < N) tma_store_2d(&map_out, col0 + c - part, row0, smem_u32(patch), MODE == 1);
          }
        } else {
          float* square = reinterpret_cast<float*>(patch);  // 32 rows, 33 floats apart
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 32; ++j) square[lane * 33 + j] = value[j];
          __syncwarp();
          const int col = col0 + c + lane, rows = min(32, M - row0);
          TO* dst = out + (size_t)row0 * ldo + col;
          if (col < N) {
            if (MODE == 0 && rows == 32) {
#pragma unroll
              for (int r = 0; r < 32; ++r, dst += ldo) *dst = from_float<TO>(square[r * 33 + lane]);
            } else {
#pragma unroll 1
              for (int r0 = 0; r0 < rows; r0 += 8) {
                // what is added into is asked for before the first store, which might be to the same memory
                float old[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) old[r] = MODE == 1 && r0 + r < rows ? to_float(dst[(size_t)(r0 + r) * ldo]) : 0.f;
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                  const float sum = square[min(r0 + r, 31) * 33 + lane];
                  if (r0 + r < rows) dst[(size_t)(r0 + r) * ldo] = from_float<TO>(MODE == 1 ? old[r] + sum : sum);
                }
              }
            }
          }
        }
      }
      fence_before();
      if (PAIR) mbar_arrive_remote(first_block_address(smem_u32(&acc_empty[a])));
      else mbar_arrive(smem_u32(&acc_empty[a]));
      if (++a == 2) { a = 0; acc_turn ^= 1; }
    }
    tma_stores_done();
  }

  fence_before();
  __syncthreads();
  if (*abort_flag && rank == 0 && threadIdx.x == 0) mbar_wait_copies(full, STAGES);  // (a pair's copies: all of them)
  if (PAIR) cluster_sync();  // neither block leaves while the other may still arrive on its barriers or read its shared memory
  if (warp == 2) {
    fence_after();
    if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2 * BN));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2 * BN));
  }
}

// A product's operands as the launchers pass them on.
struct Int8Product {
  void* out;
  const void* codes;
  const void* w;
  int M, N, K, ldx, ldw, ldo;
  Int8Scales scales;
  int sm_count;
  int* error_flag;
};

template <int MODE, bool PAIR, int BN, typename TO>
int launch_gemm_int8_tiled(const Int8Product& p, cudaStream_t stream) {
  using Shape = Int8Shape<PAIR, BN>;
  constexpr auto kernel = gemm_int8_kernel<MODE, PAIR, BN, TO>;
  const cudaError_t err = allow_shared_memory_once<kernel>(Shape::SMEM);
  if (err != cudaSuccess) return (int)err;
  CUtensorMap map_x, map_w, map_out = {};
  if (!make_map_int8_2d(&map_x, p.codes, p.M, p.K, p.ldx, I8_BM) || !make_map_int8_2d(&map_w, p.w, p.N, p.K, p.ldw, Shape::B_ROWS))
    return XRT_ERR_UNSUPPORTED;
  // A TMA store writes whole pieces of 16 bytes: what a row's last one has beyond N would be overwritten with zeros.
  const int by_tma = (((uintptr_t)p.out | (size_t)p.ldo * sizeof(TO) | (size_t)p.N * sizeof(TO)) & 15) == 0;
  if (by_tma && !make_map_result_2d(&map_out, p.out, p.M, p.N, p.ldo, sizeof(TO))) return XRT_ERR_UNSUPPORTED;
  constexpr int tile_rows = (PAIR ? 2 : 1) * I8_BM;
  const long long tiles = (long long)((p.M + tile_rows - 1) / tile_rows) * ((p.N + BN - 1) / BN);
  const int units = PAIR ? p.sm_count / 2 : p.sm_count;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)(tiles < units ? tiles : units) * (PAIR ? 2 : 1));
  config.blockDim = dim3(I8_THREADS);
  config.dynamicSmemBytes = Shape::SMEM;
  config.stream = stream;
  cudaLaunchAttribute attrs[2];
  int n_attrs = 0;
  if (pdl_enabled()) {  // (a block fills its multiprocessor's shared memory: placed early, none shares one)
    attrs[n_attrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[n_attrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (PAIR) {
    attrs[n_attrs].id = cudaLaunchAttributeClusterDimension;
    attrs[n_attrs].val.clusterDim.x = 2; attrs[n_attrs].val.clusterDim.y = 1; attrs[n_attrs++].val.clusterDim.z = 1;
  }
  config.attrs = attrs;
  config.numAttrs = n_attrs;
  cudaLaunchKernelEx(&config, kernel, map_x, map_w, map_out, (TO*)p.out, by_tma, p.M, p.N, p.K, p.ldo, p.scales, p.error_flag);
  return launch_status();
}

// The tile: 0 pairs of 256 x 256, 1 pairs of 256 x 128, 2 single blocks of 128 x 256, 3 of 128 x 128: the least of what it takes
// to begin and end, the longer of the rounds of tiles (microseconds a 128-wide slab of K) and the operands from memory, and a fifth of
// the shorter; fitted to the times of 104 products of 136 to 8,192 rows with all four on a B200, the operands in memory (the
// choice is on average 0.1 percent above the best of them).  Microseconds (0 / 1 / 2 / 3): 256 rows of 6,144 outputs, 4,096 inputs
// 15.1 / 11.6 / 16.6 / 11.4; 256 of 28,672, 4,096 31.6 / 33.8 / 34.9 / 36.9; 512 of 4,096, 14,336 39.0 / 26.0 / 44.6 / 28.7; 333 of
// 10,240, 5,120 29.7 / 26.9 / 21.3 / 22.5; 8,192 of 28,672, 4,096 565 / 703 / 626 / 839 (546 at best, 3,527 TOP/s).
struct Int8Form {
  int form;
  double us;
};
static Int8Form int8_form(const Int8Product& p) {
  constexpr int rows[4] = {256, 256, 128, 128}, columns[4] = {256, 128, 256, 128};
  constexpr double slab_us[4] = {0.26, 0.154, 0.302, 0.204}, ends_us[4] = {6.6, 8.1, 8.2, 4.0};
  const double memory_us = ((double)p.M + p.N) * p.K / 6.3e6;
  const long long slabs = (p.K + I8_BK - 1) / I8_BK;
  Int8Form best = {0, 0};
  for (int form = 0; form < 4; ++form) {
    const long long tiles = (long long)((p.M + rows[form] - 1) / rows[form]) * ((p.N + columns[form] - 1) / columns[form]);
    const int units = rows[form] == 256 ? p.sm_count / 2 : p.sm_count;
    const double walk_us = (double)((tiles + units - 1) / units * slabs) * slab_us[form];
    const double longer = walk_us > memory_us ? walk_us : memory_us;
    const double us = ends_us[form] + longer + 0.2 * (walk_us + memory_us - longer);
    if (form == 0 || us < best.us) best = {form, us};
  }
  return best;
}

template <int MODE, typename TO>
int launch_gemm_int8(const Int8Product& p, int form, cudaStream_t stream) {
  if (form == 0) return launch_gemm_int8_tiled<MODE, true, 256, TO>(p, stream);
  if (form == 1) return launch_gemm_int8_tiled<MODE, true, 128, TO>(p, stream);
  if (form == 2) return launch_gemm_int8_tiled<MODE, false, 256, TO>(p, stream);
  return launch_gemm_int8_tiled<MODE, false, 128, TO>(p, stream);
}

// ---------------------------------------------------------------- few rows
// Up to 128 rows the operands are swapped: WEIGHT rows are the MMA's lanes and the rows of codes its N (16 .. 128), and the
// time is the time to stream W from memory and through every multiprocessor's port to the L2.  A block takes a tile of
// any number of weight rows up to 256 (one or two MMAs; lanes beyond the tile's rows hold whatever lies behind them in shared
// memory and are never read) and one of `splits` parts of K, so that every multiprocessor gets the same share of W.  The
// parts of a tile are the blocks of a cluster: every block sends its sums for a share of the tile's rows to the block
// that finishes them (remote stores into shared memory that no ring uses), the cluster meets once, and every block adds its
// rows' sums: whole numbers, so their order does not matter.
//
// Nine warps: warps 0-3 issue the copies, every fourth slab of K each, because the copies of one warp run few at a
// time (measured with boxes of 128 rows x 128 bytes from memory, GB/s into one multiprocessor: one warp 55, two 98, four 127);
// warp 4 owns the TMEM and issues the MMAs; warps 5-8 bring the accumulators to shared memory, where all warps finish them.  A
// kernel this short also pays for every instruction that it meets for the first time (its code comes from the L2): the
// finish is one short loop, and while warps 5-8 wait they walk it once into a place that nobody reads.
//
// Measured on a B200, operands from memory, microseconds, the weight constant (its bytes and the codes' at the copy rate of 6.55 TB/s,
// which reads alone may pass): 1 row of 6,144 outputs, 4,096 inputs 7.3 (3.9), 8 of 4,096, 14,336 12.3 (9.0), of 28,672,
// 4,096 20.0 (18.1), of 51,200, 5,120 40.4 (40.3), 64 of 28,672, 4,096 21.9 (18.5).  With a weight that may have just been written 0.2
// to 1.2 more.
constexpr int FEW_MAX_ROWS = 128, FEW_MAX_SPLITS = 4, FEW_MAX_STAGES = 24;
constexpr int FEW_PRODUCERS = 4;  // (the walk below counts on four)
constexpr int FEW_THREADS = 32 * (FEW_PRODUCERS + 1 + 4);
constexpr int FEW_TAIL_BYTES = 512 + 4 * (FEW_MAX_ROWS + 2 * 256);  // barriers, flags, a place that nobody reads; scales, biases

struct FewShape {
  int M, N, ldo;
  int nb;        // rows of codes, padded to a multiple of 16
  int rows;      // weight rows of a tile
  int splits;
  int slabs;     // of 128 of K in a stage: 1, 2 or 4
  int stages;
  int k_iters;   // stages' worth of K: the first `k_more` parts have k_each + 1, the others k_each
  int k_each, k_more;
  int early;     // the weight may be read before the kernel before this one is done
};

__host__ __device__ inline int few_columns(const FewShape& s) {  // of tensor memory
  int columns = 32;
  while (columns < (s.rows > 128 ? 2 : 1) * s.nb) columns *= 2;
  return columns;
}
__host__ __device__ inline int few_w_bytes(const FewShape& s) { return (s.rows * I8_BK + 1023) & ~1023; }  // of a slab
__host__ __device__ inline int few_stage_bytes(const FewShape& s) { return s.slabs * (few_w_bytes(s) + s.nb * I8_BK); }
// Weight rows that one block of a cluster finishes; the last has the remainder.
__host__ __device__ inline int few_rows_per_block(const FewShape& s) { return (s.rows + s.splits - 1) / s.splits; }
__host__ __device__ inline int few_recv_row(const FewShape& s) { return s.nb + 4; }  // ints; quads of neighbouring rows in other banks
__host__ __device__ inline int few_recv_bytes(const FewShape& s) { return s.splits * few_rows_per_block(s) * few_recv_row(s) * 4; }
// The ring, and what the MMAs of its last slab read beyond the tile's rows; the sums, where they take the ring's place.
__host__ __device__ inline int few_ring_bytes(const FewShape& s) {
  const int lanes = s.rows > 128 ? 256 : 128;
  int bytes = s.stages * few_stage_bytes(s);
  const int reach = (s.stages - 1) * few_stage_bytes(s) + (s.slabs - 1) * few_w_bytes(s) + lanes * I8_BK;
  if (reach > bytes) bytes = reach;
  if (s.splits == 1 && few_recv_bytes(s) > bytes) bytes = (few_recv_bytes(s) + 1023) & ~1023;
  return bytes;
}

template <int MODE, typename TO>
__global__ void __launch_bounds__(FEW_THREADS)
gemm_int8_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, TO* out,
                     const FewShape shape, const Int8Scales scales, int* error_flag) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
  const int stages = shape.stages, nb = shape.nb, splits = shape.splits, slabs = shape.slabs;
  const int w_bytes = few_w_bytes(shape), x_bytes = nb * I8_BK, stage_bytes = few_stage_bytes(shape);
  unsigned char* tail = smem + few_ring_bytes(shape);
  uint64_t* full = reinterpret_cast<uint64_t*>(tail);
  uint64_t* empty = full + FEW_MAX_STAGES;
  uint64_t* acc_full = empty + FEW_MAX_STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* row_scales = reinterpret_cast<float*>(tail + 512);  // [M]
  float* column_scales = row_scales + FEW_MAX_ROWS;          // [weight row of the tile]
  float* biases = column_scales + 256;
  unsigned char* nowhere = tail + 448;  // 16 bytes
  // [split][weight row][row of codes]; where K is not split, the ring is free when the sums come
  int* recv = reinterpret_cast<int*>(splits > 1 ? tail + FEW_TAIL_BYTES : smem);

  if (splits > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // (nothing here divides: what a block does before its first copies is a tenth of a short product)
  const int tile = (int)blockIdx.y, split = (int)blockIdx.x;
  const int kb0 = shape.k_each * split + min(split, shape.k_more), kb1 = kb0 + shape.k_each + (split < shape.k_more ? 1 : 0);
  const int groups = shape.rows > 128 ? 2 : 1, tmem_cols = few_columns(shape);
  const int per = few_rows_per_block(shape), recv_row = few_recv_row(shape);

  if (warp == 0) {
    if (lane < stages) { mbar_init(smem_u32(&full[lane]), slabs); mbar_init(smem_u32(&empty[lane]), 1); }
    if (lane == 0) { mbar_init(smem_u32(acc_full), 1); *abort_flag = 0; }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();

  bool ok = true;
  auto give_up = [&]() {  // a wait ran out: every role leaves
    *abort_flag = 1;
    if (error_flag != nullptr) atomicExch(error_flag, 6);
  };
  uint32_t tmem_base = 0;
  if (warp < FEW_PRODUCERS) {
    if (elect_one()) {
      // Slabs are counted from the start of the block's walk: slab u lies in stage u / slabs and is copied by warp u % 4, with the
      // rows of codes that belong to it.  Neighbouring tiles start their walk over K at different places: blocks that run at the
      // same time would else ask for the same lines of the codes, and for addresses a whole weight row apart, at the same moment.
      const uint64_t once = policy_evict_first();
      const int count = kb1 - kb0, first = (tile * 5 & 15) * count >> 4;
      const int units = count * slabs, ahead = min(stages, count) * slabs;
      const int w_load = shape.rows * I8_BK;
      struct Walk {
        int s, i, k;  // stage, slab in the stage, and the stage's place in K
      };
      auto begin = [&]() {
        Walk at;
        at.s = slabs == 1 ? warp : slabs == 2 ? warp >> 1 : 0;
        at.i = warp & (slabs - 1);
        at.k = first + at.s;
        while (at.s >= stages) at.s -= stages;
        while (at.k >= count) at.k -= count;
        return at;
      };
      auto step = [&](Walk& at) {  // four slabs further
        const int on = slabs == 1 ? 4 : slabs == 2 ? 2 : 1;
        at.s += on;
        while (at.s >= stages) at.s -= stages;
        at.k += on;
        while (at.k >= count) at.k -= count;
      };
      auto load_w = [&](const Walk& at) {
        tma_load_2d(smem_u32(smem) + at.s * stage_bytes + at.i * w_bytes, &map_w, ((kb0 + at.k) * slabs + at.i) * I8_BK,
                    tile * shape.rows, smem_u32(&full[at.s]), once);
      };
      auto load_x = [&](const Walk& at) {
        tma_load_2d(smem_u32(smem) + at.s * stage_bytes + slabs * w_bytes + at.i * x_bytes, &map_x,
                    ((kb0 + at.k) * slabs + at.i) * I8_BK, 0, smem_u32(&full[at.s]));
      };
      Walk at = begin();
      if (!shape.early) {  // into the L2 at least (more than the ring was slower: 8 rows of 4,096, 14,336 12.7 -> 13.5 us)
        for (int u = warp; u < ahead; u += FEW_PRODUCERS, step(at))
          tma_prefetch_2d(&map_w, ((kb0 + at.k) * slabs + at.i) * I8_BK, tile * shape.rows);
        at = begin();
        pdl_wait();
      }
      for (int u = warp; u < ahead; u += FEW_PRODUCERS, step(at)) {
        mbar_expect_tx(smem_u32(&full[at.s]), w_load);
        load_w(at);
      }
      if (shape.early) pdl_wait();
      at = begin();
      int u = warp;
      for (; u < ahead; u += FEW_PRODUCERS, step(at)) {
        mbar_arrive_expect_tx(smem_u32(&full[at.s]), x_bytes);
        load_x(at);
      }
      uint32_t turn = 0;
      int turn_end = 2 * ahead;  // the slab with which the ring's next turn begins
      for (; u < units; u += FEW_PRODUCERS, step(at)) {
        while (u >= turn_end) { turn ^= 1; turn_end += ahead; }
        ok = mbar_wait(smem_u32(&empty[at.s]), turn, abort_flag);
        if (!ok) break;
        mbar_arrive_expect_tx(smem_u32(&full[at.s]), w_load + x_bytes);
        load_w(at);
        load_x(at);
      }
      if (!ok) give_up();
    }
  } else {
    if (warp == FEW_PRODUCERS) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(tmem_cols));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
      pdl_trigger();  // not before: see common.cuh
    }
    fence_before();
    asm volatile("bar.sync 2, 160;" ::: "memory");  // the MMA warp and the finishing warps
    fence_after();
    tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  }
  if (warp == FEW_PRODUCERS && elect_one()) {
    const uint32_t idesc = instr_desc_i8(128, nb);
    int s = 0;
    uint32_t turn = 0;
    auto slab = [&](uint64_t desc_w, uint64_t desc_x, auto adds) {  // `adds`: whether to the sums so far
#pragma unroll
      for (int k = 0; k < I8_BK / I8_UMMA_K; ++k) {  // 32 bytes further along K inside the swizzle atom
        mma_i8(tmem_base, desc_w + 2 * k, desc_x + 2 * k, idesc, decltype(adds)::value || k > 0);
        if (groups == 2) mma_i8(tmem_base + nb, desc_w + 2 * k + (128 * I8_BK >> 4), desc_x + 2 * k, idesc, decltype(adds)::value || k > 0);
      }
    };
    for (int kb = kb0; kb < kb1; ++kb) {  // in the order in which the producers walk
      ok = mbar_wait(smem_u32(&full[s]), turn, abort_flag);
      if (!ok) break;
      fence_after();
      const uint64_t desc_w = desc_k_major(smem_u32(smem) + s * stage_bytes);
      const uint64_t desc_x = desc_k_major(smem_u32(smem) + s * stage_bytes + slabs * w_bytes);
      if (kb == kb0) slab(desc_w, desc_x, std::false_type());
      else slab(desc_w, desc_x, std::true_type());
      for (int i = 1; i < slabs; ++i) slab(desc_w + (i * w_bytes >> 4), desc_x + (i * x_bytes >> 4), std::true_type());
      commit(smem_u32(&empty[s]));
      if (++s == stages) { s = 0; turn ^= 1; }
    }
    if (ok) commit(smem_u32(acc_full));
    else give_up();
  }
  if (warp > FEW_PRODUCERS) {
    const int tid = (int)threadIdx.x - 32 * (FEW_PRODUCERS + 1);
    pdl_wait();  // the scales, and the output, belong to the step
    for (int i = tid; i < nb; i += 128) row_scales[i] = i < shape.M ? scales.rows[i] : 0.f;
    for (int i = tid; i < shape.rows; i += 128) {
      const int n = min(tile * shape.rows + i, shape.N - 1);
      column_scales[i] = scales.columns[n];
      biases[i] = scales.bias != nullptr ? scales.bias[n] : 0.f;
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");
  }
  const int row_lo = split * per, n_lo = tile * shape.rows + row_lo;
  const int here = max(1, min(min(per, shape.rows - row_lo), shape.N - n_lo));
  const int eights = n_lo < shape.N && row_lo < shape.rows ? (shape.M + 7) / 8 : 0;
  // this thread's first sums, and from some to the next: eight rows of codes, weight rows inside
  const int eight0 = (int)threadIdx.x / here, local0 = (int)threadIdx.x - eight0 * here;
  const int eight_step = FEW_THREADS / here, local_step = FEW_THREADS - eight_step * here;
#pragma unroll 1
  for (int pass = warp > FEW_PRODUCERS ? 0 : 1; pass < 2; ++pass) {
    if (pass == 1) {
      if (splits > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");  // every block of the cluster runs
      if (warp > FEW_PRODUCERS) {
        const int quarter = warp & 3;
        ok = mbar_wait(smem_u32(acc_full), 0, abort_flag);
        if (!ok && lane == 0) give_up();
        fence_after();
        for (int g = 0; ok && g < groups; ++g) {
          const int r = g * 128 + quarter * 32 + lane, owner = min(r, shape.rows - 1) / per;
          uint32_t to;
          asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(recv)), "r"(owner));
          to += (uint32_t)((split * per + r - owner * per) * recv_row * 4);
#pragma unroll 1
          for (int c = 0; c < shape.M; c += 16) {
            uint32_t v[16];
            tmem_ld16(v, tmem_base + ((uint32_t)(quarter * 32) << 16) + g * nb + c);
            tmem_wait_ld();
            if (r < shape.rows) {
#pragma unroll
              for (int j = 0; j < 16; j += 4)
                asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to + (uint32_t)((c + j) * 4)), "r"(v[j]),
                             "r"(v[j + 1]), "r"(v[j + 2]), "r"(v[j + 3]) : "memory");
            }
          }
        }
        fence_before();
      }
      // Every thread of the cluster comes here, also after a wait that ran out.  After this meeting nothing touches another
      // block's memory, so a block may leave when it is done.
      if (splits > 1) asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;" ::: "memory");
      else __syncthreads();
      if (*abort_flag) break;
    }
    int eight = pass == 1 ? eight0 : 0, local = pass == 1 ? local0 : 0;
#pragma unroll 1
    while (eight < (pass == 1 ? eights : 1)) {
      int sums[8] = {};
#pragma unroll 1
      for (int sp = 0; sp < splits; ++sp) {
        const int4* part = reinterpret_cast<const int4*>(recv + (sp * per + local) * recv_row + eight * 8);
        const int4 lo = part[0], hi = part[1];
        sums[0] += lo.x; sums[1] += lo.y; sums[2] += lo.z; sums[3] += lo.w;
        sums[4] += hi.x; sums[5] += hi.y; sums[6] += hi.z; sums[7] += hi.w;
      }
      const float4 s_lo = *reinterpret_cast<const float4*>(row_scales + eight * 8);
      const float4 s_hi = *reinterpret_cast<const float4*>(row_scales + eight * 8 + 4);
      const float by_column = column_scales[row_lo + local], bias = biases[row_lo + local];
      const float factors[8] = {s_lo.x, s_lo.y, s_lo.z, s_lo.w, s_hi.x, s_hi.y, s_hi.z, s_hi.w};
      // rows beyond M, and all rows of the first walk, go nowhere; what is added into is asked for before the first store,
      // which might be to the same memory
      TO* dst[8];
      float old[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int m = eight * 8 + e;
        dst[e] = pass == 1 && m < shape.M ? out + (size_t)m * shape.ldo + n_lo + local : reinterpret_cast<TO*>(nowhere);
        old[e] = MODE == 1 ? to_float(*dst[e]) : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float value = fmaf(__int2float_rn(sums[e]) * factors[e], by_column, bias);
        *dst[e] = from_float<TO>(MODE == 1 ? old[e] + value : value);
      }
      if (pass == 0) break;
      eight += eight_step;
      local += local_step;
      if (local >= here) { local -= here; ++eight; }
    }
  }
  __syncthreads();
  if (*abort_flag && threadIdx.x == 0) mbar_wait_copies(full, stages);
  if (warp == FEW_PRODUCERS) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(tmem_cols));
  }
}

static int few_shared_bytes(const FewShape& s) {
  const int bytes = few_ring_bytes(s) + FEW_TAIL_BYTES + (s.splits > 1 ? few_recv_bytes(s) : 0) + 1024;
  const int least = shared_bytes_of_columns(few_columns(s));  // (two blocks a multiprocessor at most take half of it each)
  return bytes > least ? bytes : least;
}

// The tile, the parts of K and the ring of a product, from what was measured on a B200 (148 multiprocessors).
//
// Up to 128 weight rows a multiprocessor, one block each, the cheapest of some tiles and numbers of parts by this sum of
// microseconds (fitted to the times of 65 products of 1 to 128 rows with every one of them: on average 1.7 percent above the
// best): the longer of W from memory (6.3 TB/s in all, 0.11 TB/s into one multiprocessor, less with copies of fewer than 64
// rows) and a block's walk over its slabs (0.15 each, or their bytes at 0.11 TB/s), half of the shorter, 0.01 a block, 0.2 for
// each 1,000 sums that a block finishes, 0.3 where the parts of a tile meet and 0.3 for tiles of two MMAs.  The device does not
// hold clusters of 3 and 4 on all multiprocessors.  Chosen against other numbers of parts: 8 rows of 4,096 outputs, 14,336
// inputs 12.5 (4 parts; 3: 12.8, 1: 21); 6,144, 4,096 7.5 (2; 4: 7.4, 1: 8.5); 64 of 2,048, 2,048 4.8 (2; 4: 5.2).
//
// More weight rows than that: K is not split.  Two blocks a multiprocessor with a ring of four slabs each, if their
// tiles make one round of it or even tiles of 256 rows do not (8 rows of 28,672 outputs, 4,096 inputs 19.1 against 19.8 with one
// block, 64 rows 22.5 against 24.8); else one block with tiles of up to 256 rows (128 rows 30.7).
constexpr int FEW_SHARED_ONE = 227 * 1024, FEW_SHARED_TWO = 113 * 1024;

static void plan_few(FewShape& s, int K, int sm_count) {
  const int slabs = (K + I8_BK - 1) / I8_BK;
  auto even_rows = [&](int blocks) { return ((s.N + blocks - 1) / blocks + 7) / 8 * 8; };
  int limit = FEW_SHARED_ONE;
  if (even_rows(sm_count) <= 128) {
    double best = 0;
    s.splits = 0;
    for (int splits = 1; splits <= FEW_MAX_SPLITS && (splits == 1 || slabs >= 2 * splits); ++splits) {
      const int blocks = splits <= 2 ? sm_count : sm_count * 22 / 25;
      if (blocks < splits) break;
      const int even = even_rows(blocks / splits);
      for (int rows : {32, 64, 96, 128, even}) {
        if (rows > 256 || rows < even) continue;
        const int used = (s.N + rows - 1) / rows * splits;
        const double into = used * 0.11e6 * (rows < 64 ? rows / 64.0 : 1.0), slab_us = (rows + s.M) * 128 / 0.11e6;
        const double memory_us = (double)s.N * K / (into < 6.3e6 ? into : 6.3e6);
        const double walk_us = (slabs + splits - 1) / splits * (slab_us > 0.15 ? slab_us : 0.15);
        const double cost = (memory_us > walk_us ? memory_us + 0.5 * walk_us : walk_us + 0.5 * memory_us) + 0.01 * used +
                            0.2e-3 * rows * s.M + (splits > 1 ? 0.3 : 0.0) + (rows > 128 ? 0.3 : 0.0);
        if (s.splits == 0 || cost < best) { best = cost; s.splits = splits; s.rows = rows; }
      }
    }
  } else {
    const int two_most = 212 - s.nb;  // weight rows that leave room for four slabs
    const int two_rounds = (s.N + 2 * sm_count * two_most - 1) / (2 * sm_count * two_most);
    const int one_rounds = (s.N + sm_count * 256 - 1) / (sm_count * 256);
    const bool two = two_rounds == 1 || one_rounds > 1;
    s.splits = 1;
    s.rows = even_rows(two ? 2 * sm_count * two_rounds : sm_count);
    if (two) limit = FEW_SHARED_TWO;
  }
  // The ring: slabs a stage as many as leave three stages (or all that a block walks).  The producers, which take
  // every fourth slab each, need a ring of four slabs if it turns: two blocks a multiprocessor or parts of K that leave no
  // room for that are given up.
  for (;;) {
    for (s.slabs = 4; s.slabs > 1; s.slabs /= 2) {
      const int walked = ((slabs + s.slabs - 1) / s.slabs + s.splits - 1) / s.splits;
      s.stages = walked < 3 ? walked : 3;
      if (few_shared_bytes(s) <= limit && slabs >= s.slabs * s.splits) break;
    }
    s.k_iters = (slabs + s.slabs - 1) / s.slabs;
    const int share = (s.k_iters + s.splits - 1) / s.splits;
    s.stages = FEW_MAX_STAGES;
    while (s.stages > 1 && few_shared_bytes(s) > limit) --s.stages;
    if (s.stages > share) s.stages = share;
    if ((s.stages * s.slabs >= FEW_PRODUCERS || s.stages == share) && few_shared_bytes(s) <= limit) break;
    // (this ends: all of K with one block a multiprocessor has room for four slabs of 256 weight rows and 128 rows of codes)
    if (limit == FEW_SHARED_TWO) limit = FEW_SHARED_ONE;
    else --s.splits;
  }
}

static FewShape few_shape(const Int8Product& p) {
  FewShape shape = {};
  shape.M = p.M; shape.N = p.N; shape.ldo = p.ldo;
  shape.nb = (p.M + 15) / 16 * 16;
  plan_few(shape, p.K, p.sm_count);
  shape.k_each = shape.k_iters / shape.splits;
  shape.k_more = shape.k_iters - shape.k_each * shape.splits;
  return shape;
}

// Microseconds of a product by this kernel, for the choice between it and tiles: to begin and end, the longer of W from memory and
// of what a multiprocessor's blocks copy (the codes again for every tile), some of the shorter, and the sums that a block
// finishes; fitted, together with int8_form's, to the times of 188 products of 1 to 128 rows by both, in bfloat16.  The choice is
// on average 0.2 percent above the better one, and 8 at most; this kernel for all of them 5, and 50 at most.  Microseconds, this
// kernel / tiles: 48 rows of 10,240 outputs, 5,120 inputs 13.1 / 14.4, 96 16.4 / 14.6; 128 of 4,096, 14,336 18.4 / 24.5, of
// 6,400, 512 6.4 / 4.3, of 51,200, 5,120 72 / 47; 64 of 102,400, 1,024 29 / 24.  Up to 16 rows, and up to 48 where every block
// has a multiprocessor of its own, it was never behind, and is not compared.
static double few_us(const FewShape& s, int K, int sm_count) {
  const int blocks = (s.N + s.rows - 1) / s.rows * s.splits, each = (blocks + sm_count - 1) / sm_count;
  const int slabs = ((K + I8_BK - 1) / I8_BK + s.splits - 1) / s.splits;
  const double into = blocks * 0.11e6, slab_us = (s.rows + s.M) * 128 / 93e3;
  const double memory_us = (double)s.N * K / (into < 6.3e6 ? into : 6.3e6);
  const double walk_us = each * slabs * (slab_us > 0.15 ? slab_us : 0.15);
  const double longer = memory_us > walk_us ? memory_us : walk_us, shorter = memory_us + walk_us - longer;
  if (each > 1) return 0.4 + longer + 0.13 * shorter + 0.2e-3 * s.rows * s.M * each;  // (blocks begin and end beside others)
  return 3.8 + longer + 0.14 * shorter + 0.16e-3 * s.rows * s.M;
}

template <int MODE, typename TO>
int launch_gemm_int8_few(const Int8Product& p, FewShape shape, int constant_weight, cudaStream_t stream) {
  constexpr auto kernel = gemm_int8_few_kernel<MODE, TO>;
  const cudaError_t err = allow_shared_memory_once<kernel>(FEW_SHARED_ONE);
  if (err != cudaSuccess) return (int)err;
  shape.early = constant_weight;
  CUtensorMap map_w, map_x;
  if (!make_map_int8_2d(&map_x, p.codes, p.M, p.K, p.ldx, shape.nb) || !make_map_int8_2d(&map_w, p.w, p.N, p.K, p.ldw, shape.rows))
    return XRT_ERR_UNSUPPORTED;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)shape.splits, (unsigned)((shape.N + shape.rows - 1) / shape.rows));
  config.blockDim = dim3(FEW_THREADS);
  config.dynamicSmemBytes = few_shared_bytes(shape);
  config.stream = stream;
  cudaLaunchAttribute attrs[2];
  int n_attrs = 0;
  if (pdl_enabled()) {
    attrs[n_attrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[n_attrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  attrs[n_attrs].id = cudaLaunchAttributeClusterDimension;
  attrs[n_attrs].val.clusterDim.x = shape.splits; attrs[n_attrs].val.clusterDim.y = 1; attrs[n_attrs++].val.clusterDim.z = 1;
  config.attrs = attrs;
  config.numAttrs = n_attrs;
  cudaLaunchKernelEx(&config, kernel, map_w, map_x, (TO*)p.out, shape, p.scales, p.error_flag);
  return launch_status();
}

}  // namespace xrt

// A call as the caller packs it.  codes: int8 [M, K] with rows ldx bytes apart; w: int8 [N, K] with rows ldw bytes apart; both
// strides multiples of 16 and both bases 16-byte aligned; scales float32 [M], w_scales float32 [N], bias float32 [N] or null.
// out: [M, N] with row stride ldo; mode 0 stores, 1 adds into a float32 out.  constant_weight: none of the kernels that may
// still run wrote w, which is then read ahead of the wait for them.  error_flag (may be null) is set to 6 if a bounded wait
// ran out.
struct XrtInt8Call {
  void* out;
  const void* codes;
  const float* scales;
  const void* w;
  const float* w_scales;
  const float* bias;
  int* error_flag;
  int M, N, K, ldx, ldw, ldo, out_dtype, mode, constant_weight;
};
static_assert(offsetof(XrtInt8Call, M) == 56 && offsetof(XrtInt8Call, constant_weight) == 88, "seven pointers, then nine ints");

namespace xrt {

// The kernel that takes a product: the few rows' with `shape`, or tiles of `tiles.form`.
struct Int8Choice {
  bool few;
  FewShape shape;
  Int8Form tiles;
};
static Int8Choice int8_choice(const Int8Product& p) {
  // (The few rows' kernel: its tiles, of 64 weight rows at least, are a grid's second dimension.)
  Int8Choice c = {p.M <= FEW_MAX_ROWS && p.N <= 65535 * 64, {}, {0, 0}};
  if (c.few) c.shape = few_shape(p);
  const bool either = c.few && p.M > ((p.N + c.shape.rows - 1) / c.shape.rows * c.shape.splits > p.sm_count ? 16 : 48);
  if (!c.few || either) c.tiles = int8_form(p);
  if (either) c.few = few_us(c.shape, p.K, p.sm_count) <= c.tiles.us;
  return c;
}

}  // namespace xrt

// What the launcher would do with a product on a device of `sm_count` multiprocessors (host arithmetic): plan[0] = 0 to 3 the tile
// (int8_form), 4 the few rows' kernel; and of that one plan[1] = weight rows of a tile, plan[2] = parts of K, plan[3] = blocks,
// plan[4] = bytes of shared memory a block, plan[5] = columns of tensor memory a block (zeros for tiles).
XRT_EXPORT int xrt_gemm_int8_plan(int M, int N, int K, int sm_count, int* plan) {
  if (M <= 0 || M > XRT_INT8_MAX_SIZE || N <= 0 || N > XRT_INT8_MAX_SIZE || K <= 0 || K > 131071 || sm_count <= 1 || plan == nullptr)
    return XRT_ERR_ARGUMENT;
  xrt::Int8Product p = {};
  p.M = M; p.N = N; p.K = K; p.sm_count = sm_count;
  const xrt::Int8Choice c = xrt::int8_choice(p);
  for (int i = 0; i < 6; ++i) plan[i] = 0;
  plan[0] = c.few ? 4 : c.tiles.form;
  if (c.few) {
    plan[1] = c.shape.rows;
    plan[2] = c.shape.splits;
    plan[3] = (N + c.shape.rows - 1) / c.shape.rows * c.shape.splits;
    plan[4] = xrt::few_shared_bytes(c.shape);
    plan[5] = xrt::few_columns(c.shape);
  }
  return XRT_OK;
}

XRT_EXPORT int xrt_gemm_int8(const XrtInt8Call* call, cudaStream_t stream) {
  const XrtInt8Call& c = *call;
  if (c.M < 0 || c.N <= 0 || c.K <= 0 || c.K > 131071 || c.ldx < c.K || c.ldw < c.K || c.ldo < c.N || c.mode < 0 || c.mode > 1)
    return XRT_ERR_ARGUMENT;
  if (c.M > XRT_INT8_MAX_SIZE || c.N > XRT_INT8_MAX_SIZE) return XRT_ERR_ARGUMENT;
  if (c.mode == 1 && c.out_dtype != XRT_F32) return XRT_ERR_ARGUMENT;
  if (c.ldx % 16 != 0 || c.ldw % 16 != 0 || ((uintptr_t)c.codes & 15) || ((uintptr_t)c.w & 15)) return XRT_ERR_UNSUPPORTED;
  if (c.M == 0) return XRT_OK;
  const xrt::Int8Product p{c.out, c.codes, c.w, c.M, c.N, c.K, c.ldx, c.ldw, c.ldo, {c.scales, c.w_scales, c.bias},
                           xrt::multiprocessors(), c.error_flag};
  if (p.sm_count <= 1) return XRT_ERR_UNSUPPORTED;
  const xrt::Int8Choice choice = xrt::int8_choice(p);
  if (c.mode == 1)
    return choice.few ? xrt::launch_gemm_int8_few<1, float>(p, choice.shape, c.constant_weight, stream)
                      : xrt::launch_gemm_int8<1, float>(p, choice.tiles.form, stream);
  XRT_DISPATCH_DTYPE(c.out_dtype, TO, {
    return choice.few ? xrt::launch_gemm_int8_few<0, TO>(p, choice.shape, c.constant_weight, stream)
                      : xrt::launch_gemm_int8<0, TO>(p, choice.tiles.form, stream);
  });
}
