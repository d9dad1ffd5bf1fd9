// out[M, N] = (codes[M, K] . W[N, K]^T) * scales[m] * w_scales[n] (+ bias[n]) of signed 8-bit integers, on the
// fifth-generation tensor cores (tcgen05.mma kind::i8): the sums over K are 32-bit integers and exact, whatever their
// order, and are rounded to 32-bit floating point once, before the scales.  K is bounded by the caller's check, so that
// 128 * 128 * K stays below 2^31.
//
// A persistent block, one a multiprocessor, walks output tiles of 128 x 256.  Six warps a block:
//   warp 0     producer: for each 128-wide slab of K, TMA loads of the block's 128 rows of codes and 256 rows of W into the next
//              free stage of a ring; what a tile has beyond M, N or K arrives as zeros.
//   warp 1     allocates TMEM (two accumulators of 128 lanes x 256 columns) and issues the MMAs: four a stage, each 32 bytes
//              of K.
//   warps 2-5  epilogue: each warp reads its 32 TMEM lanes (rows), 32 columns at a time, applies the scales, turns the
//              patch around in shared memory and stores 16 bytes a lane, while the MMA warp fills the other accumulator.
// Every wait on an mbarrier is bounded.  A wait that runs out raises the error flag and an abort flag in shared memory; all
// roles leave their loops, the block frees its TMEM and returns.
#include "tcgen05.cuh"

namespace xrt {

using namespace sm100;

constexpr int I8_BM = 128, I8_BN = 256, I8_BK = 128, I8_UMMA_K = 32;
constexpr int I8_A_BYTES = I8_BM * I8_BK, I8_B_BYTES = I8_BN * I8_BK;
constexpr int I8_STAGES = 4, I8_STAGE_BYTES = I8_A_BYTES + I8_B_BYTES;
constexpr int I8_THREADS = 192;
constexpr int I8_STAGING_BYTES = 4 * 32 * 33 * 4;
constexpr int I8_SMEM = I8_STAGES * I8_STAGE_BYTES + I8_STAGING_BYTES + 256 + 1024;

// What the sums are multiplied by and what is added.
struct Int8Scales {
  const float* rows;     // [M]
  const float* columns;  // [N]
  const float* bias;     // [N] or null
};

// MODE 0: store, 1: add into float out.
template <int MODE, typename TO>
__global__ void __launch_bounds__(I8_THREADS, 1)
gemm_int8_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, TO* __restrict__ out,
                 int M, int N, int K, int ldo, const Int8Scales scales, int* __restrict__ error_flag) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  unsigned char* a_stages = smem;
  unsigned char* b_stages = smem + I8_STAGES * I8_A_BYTES;
  float* staging = reinterpret_cast<float*>(smem + I8_STAGES * I8_STAGE_BYTES);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + I8_STAGES * I8_STAGE_BYTES + I8_STAGING_BYTES);
  uint64_t* empty = full + I8_STAGES;
  uint64_t* acc_full = empty + I8_STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles_m = (M + I8_BM - 1) / I8_BM, tiles_n = (N + I8_BN - 1) / I8_BN;
  const int n_tiles = tiles_m * tiles_n;
  const int k_iters = (K + I8_BK - 1) / I8_BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < I8_STAGES; ++s) { mbar_init(smem_u32(&full[s]), 1); mbar_init(smem_u32(&empty[s]), 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(smem_u32(&acc_full[a]), 1); mbar_init(smem_u32(&acc_empty[a]), 128); }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem_base = *tmem_slot;

  bool ok = true;
  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      for (int tile = blockIdx.x; tile < n_tiles && ok; tile += gridDim.x) {
        const int m0 = tile % tiles_m * I8_BM, n0 = tile / tiles_m * I8_BN;
        for (int kb = 0; kb < k_iters; ++kb, ++it) {
          const int s = it % I8_STAGES;
          ok = mbar_wait(smem_u32(&empty[s]), ((it / I8_STAGES) & 1) ^ 1, abort_flag);
          if (!ok) break;
          const uint32_t bar = smem_u32(&full[s]), b_dst = smem_u32(b_stages + s * I8_B_BYTES);
          mbar_arrive_expect_tx(bar, I8_STAGE_BYTES);
          tma_load_2d(smem_u32(a_stages + s * I8_A_BYTES), &map_x, kb * I8_BK, m0, bar);
          tma_load_2d(b_dst, &map_w, kb * I8_BK, n0, bar);
          tma_load_2d(b_dst + I8_B_BYTES / 2, &map_w, kb * I8_BK, n0 + 128, bar);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = instr_desc_i8(I8_BM, I8_BN);
      int it = 0, tile_i = 0;
      for (int tile = blockIdx.x; tile < n_tiles && ok; tile += gridDim.x, ++tile_i) {
        const int a = tile_i & 1;
        ok = mbar_wait(smem_u32(&acc_empty[a]), ((tile_i >> 1) & 1) ^ 1, abort_flag);
        if (!ok) break;
        fence_after();
        for (int kb = 0; kb < k_iters; ++kb, ++it) {
          const int s = it % I8_STAGES;
          ok = mbar_wait(smem_u32(&full[s]), (it / I8_STAGES) & 1, abort_flag);
          if (!ok) break;
          fence_after();
          const uint64_t desc_a = desc_k_major(smem_u32(a_stages + s * I8_A_BYTES));
          const uint64_t desc_b = desc_k_major(smem_u32(b_stages + s * I8_B_BYTES));
#pragma unroll
          for (int k = 0; k < I8_BK / I8_UMMA_K; ++k)  // 32 bytes further along K inside the swizzle atom
            mma_i8(tmem_base + a * I8_BN, desc_a + 2 * k, desc_b + 2 * k, idesc, (kb | k) != 0);
          commit(smem_u32(&empty[s]));
        }
        if (ok) commit(smem_u32(&acc_full[a]));
      }
    }
  } else {
    const int quarter = warp & 3;  // the TMEM lanes this warp may read
    float* patch = staging + (warp - 2) * 32 * 33;
    const int sub_row = lane >> 3, sub_col = (lane & 7) * 4;
    int tile_i = 0;
    for (int tile = blockIdx.x; tile < n_tiles && ok; tile += gridDim.x, ++tile_i) {
      const int a = tile_i & 1;
      const int row0 = tile % tiles_m * I8_BM + quarter * 32, col0 = tile / tiles_m * I8_BN;
      const float row_scale = row0 + lane < M ? __ldg(scales.rows + row0 + lane) : 0.f;
      ok = mbar_wait(smem_u32(&acc_full[a]), (tile_i >> 1) & 1, abort_flag);
      if (!ok) break;
      fence_after();
      const uint32_t tmem_row = tmem_base + ((uint32_t)(quarter * 32) << 16) + a * I8_BN;
#pragma unroll 1
      for (int c = 0; c < I8_BN; c += 32) {
        const int col = col0 + c + sub_col;
        float factor[4], bias[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          factor[e] = col + e < N ? __ldg(scales.columns + col + e) : 0.f;
          bias[e] = scales.bias != nullptr && col + e < N ? __ldg(scales.bias + col + e) : 0.f;
        }
        uint32_t v[32];
        tmem_ld32(v, tmem_row + c);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; ++j) patch[lane * 33 + j] = __int2float_rn((int)v[j]) * row_scale;
        __syncwarp();
#pragma unroll
        for (int it = 0; it < 8; ++it) {
          const int row = row0 + it * 4 + sub_row;
          const float* src = patch + (it * 4 + sub_row) * 33 + sub_col;
          if (row < M) {
            TO* dst = out + (size_t)row * ldo + col;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (col + e < N) {
                const float value = fmaf(src[e], factor[e], bias[e]);
                dst[e] = from_float<TO>(MODE == 1 ? to_float(dst[e]) + value : value);
              }
          }
        }
        __syncwarp();
      }
      fence_before();
      mbar_arrive(smem_u32(&acc_empty[a]));
    }
  }
  if (!ok && lane == 0) { *abort_flag = 1; if (error_flag != nullptr) atomicExch(error_flag, 6); }

  fence_before();
  __syncthreads();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512));
  }
}

template <int MODE, typename TO>
int launch_gemm_int8(void* out, const CUtensorMap& map_x, const CUtensorMap& map_w, int M, int N, int K, int ldo,
                     const Int8Scales& scales, int sm_count, int* error_flag, cudaStream_t stream) {
  constexpr auto kernel = gemm_int8_kernel<MODE, TO>;
  const cudaError_t err = allow_shared_memory_once<kernel>(I8_SMEM);
  if (err != cudaSuccess) return (int)err;
  const long long tiles = (long long)((M + I8_BM - 1) / I8_BM) * ((N + I8_BN - 1) / I8_BN);
  launch_kernel_alone(kernel, dim3((unsigned)(tiles < sm_count ? tiles : sm_count)), dim3(I8_THREADS), (size_t)I8_SMEM, stream, map_x,
                      map_w, (TO*)out, M, N, K, ldo, scales, error_flag);
  return launch_status();
}

// ---------------------------------------------------------------- few rows
// Up to 128 rows the operands are swapped: 128 WEIGHT rows are the MMA's lanes and the rows of codes its N (16 .. 128), and the
// time is the time to stream W from memory.  A block takes one tile of 128 weight rows and one of `splits` parts of K; the
// parts of a tile are the blocks of a cluster.  Two blocks a multiprocessor are resident (their rings are cut to fit), so
// that the copies of one run while the other starts or finishes, and all of a product's blocks together hold many
// times the bytes in flight that the memory needs.  Every block sends its sums for a share of the tile's rows to the block
// that finishes them (remote stores into shared memory that no ring uses), the cluster meets once, and every block adds its
// rows' sums: whole numbers, so their order does not matter.
constexpr int FEW_MAX_ROWS = 128, FEW_MAX_SPLITS = 8;
constexpr int FEW_W_BYTES = 128 * I8_BK;
constexpr int FEW_THREADS = 192;
constexpr int FEW_TAIL_BYTES = 512;  // barriers and flags

struct FewShape {
  int M, N, ldo;
  int nb;       // rows of codes, padded to a multiple of 16
  int splits, stages;
  int k_iters;  // slabs of 128 of K
  int early;    // the weight may be read before the kernel before this one is done
};

__host__ __device__ inline int few_stage_bytes(int nb) { return FEW_W_BYTES + nb * I8_BK; }
// Weight rows that one block of a cluster finishes; the last has the remainder.
__host__ __device__ inline int few_rows_per_block(int splits) { return ((128 + splits - 1) / splits + 3) & ~3; }

template <int MODE, typename TO>
__device__ __forceinline__ void few_store(TO* dst, int sum, float row_scale, float column_scale, float bias) {
  const float value = fmaf(__int2float_rn(sum) * row_scale, column_scale, bias);
  *dst = from_float<TO>(MODE == 1 ? to_float(*dst) + value : value);
}

template <int MODE, typename TO>
__global__ void __launch_bounds__(FEW_THREADS)
gemm_int8_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, TO* out,
                     const FewShape shape, const Int8Scales scales, int* error_flag) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int stages = shape.stages, nb = shape.nb, splits = shape.splits;
  const int stage_bytes = few_stage_bytes(nb);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + stages * stage_bytes);
  uint64_t* empty = full + stages;
  uint64_t* acc_full = empty + stages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* recv = reinterpret_cast<int*>(smem + stages * stage_bytes + FEW_TAIL_BYTES);  // [split][row of codes][weight row]

  pdl_trigger();
  if (splits > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = (int)blockIdx.x / splits, split = (int)blockIdx.x - tile * splits;
  const int kb0 = shape.k_iters * split / splits, kb1 = shape.k_iters * (split + 1) / splits;
  int tmem_cols = 32;
  while (tmem_cols < nb) tmem_cols *= 2;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) { mbar_init(smem_u32(&full[s]), 1); mbar_init(smem_u32(&empty[s]), 1); }
    mbar_init(smem_u32(acc_full), 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(tmem_cols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem_base = *tmem_slot;

  bool ok = true;
  if (warp == 0) {
    if (lane == 0) {
      // Neighbouring tiles start their walk over K at different slabs: blocks that run at the same time would else ask for the
      // same lines of the codes, and for addresses a whole weight row apart, at the same moment.
      const uint64_t once = policy_evict_first();
      const uint32_t full0 = smem_u32(full), empty0 = smem_u32(empty), stage0 = smem_u32(smem);
      const int count = kb1 - kb0, first = kb0 + tile * 5 % count;
      auto slab = [&](int i) { const int kb = first + i; return (kb < kb1 ? kb : kb - count) * I8_BK; };
      const int ahead = min(stages, count);
      if (!shape.early) pdl_wait();
      for (int i = 0; i < ahead; ++i) {
        mbar_expect_tx(full0 + i * 8, FEW_W_BYTES);
        tma_load_2d(stage0 + i * stage_bytes, &map_w, slab(i), tile * 128, full0 + i * 8, once);
      }
      if (shape.early) pdl_wait();
      for (int i = 0; i < ahead; ++i) {
        mbar_arrive_expect_tx(full0 + i * 8, nb * I8_BK);
        tma_load_2d(stage0 + i * stage_bytes + FEW_W_BYTES, &map_x, slab(i), 0, full0 + i * 8);
      }
      int s = 0;
      uint32_t turn = 0;
      for (int i = ahead; i < count; ++i) {
        ok = mbar_wait(empty0 + s * 8, turn, abort_flag);
        if (!ok) break;
        mbar_arrive_expect_tx(full0 + s * 8, stage_bytes);
        tma_load_2d(stage0 + s * stage_bytes, &map_w, slab(i), tile * 128, full0 + s * 8, once);
        tma_load_2d(stage0 + s * stage_bytes + FEW_W_BYTES, &map_x, slab(i), 0, full0 + s * 8);
        if (++s == stages) { s = 0; turn ^= 1; }
      }
    }
    if (splits > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = instr_desc_i8(128, nb);
      int s = 0;
      uint32_t turn = 0;
      for (int kb = kb0; kb < kb1; ++kb) {  // in the order in which the producer walks
        ok = mbar_wait(smem_u32(&full[s]), turn, abort_flag);
        if (!ok) break;
        fence_after();
        const uint64_t desc_w = desc_k_major(smem_u32(smem + s * stage_bytes));
        const uint64_t desc_x = desc_k_major(smem_u32(smem + s * stage_bytes + FEW_W_BYTES));
#pragma unroll
        for (int k = 0; k < I8_BK / I8_UMMA_K; ++k)
          mma_i8(tmem_base, desc_w + 2 * k, desc_x + 2 * k, idesc, (kb > kb0 || k > 0) ? 1u : 0u);
        commit(smem_u32(&empty[s]));
        if (++s == stages) { s = 0; turn ^= 1; }
      }
      if (ok) commit(smem_u32(acc_full));
    }
    if (splits > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  } else {
    if (splits > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");  // every block of the cluster runs
    pdl_wait();  // the scales, and the output, belong to the step
    const int quarter = warp & 3, r = quarter * 32 + lane, n = tile * 128 + r;
    const bool inside = n < shape.N;
    const float column_scale = inside ? scales.columns[n] : 0.f;
    const float bias = inside && scales.bias != nullptr ? scales.bias[n] : 0.f;
    const uint32_t tmem_row = tmem_base + ((uint32_t)(quarter * 32) << 16);
    ok = mbar_wait(smem_u32(acc_full), 0, abort_flag);
    if (ok) {
      fence_after();
      const int per = few_rows_per_block(splits), owner = r / per;
      uint32_t remote = 0;
      if (splits > 1) {
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(recv)), "r"(owner));
        remote += (uint32_t)((split * nb * per + r - owner * per) * 4);
      }
      for (int c = 0; c < shape.M; c += 16) {
        uint32_t v[16];
        tmem_ld16(v, tmem_row + c);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if (c + j >= shape.M) break;
          if (splits > 1)
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote + (uint32_t)((c + j) * per * 4)), "r"(v[j]) : "memory");
          else if (inside)
            few_store<MODE>(out + (size_t)(c + j) * shape.ldo + n, (int)v[j], scales.rows[c + j], column_scale, bias);
        }
      }
      fence_before();
    }
  }
  if (!ok && lane == 0) { *abort_flag = 1; if (error_flag != nullptr) atomicExch(error_flag, 6); }

  if (splits > 1) {
    // Every thread of every block of the cluster comes here, also after a wait that ran out.  After the meeting nothing
    // touches another block's memory, so a block may leave when it is done.
    asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;" ::: "memory");
    if (warp >= 2 && !*abort_flag) {
      const int per = few_rows_per_block(splits), row_lo = split * per;
      const int n_lo = tile * 128 + row_lo, here = max(0, min(min(per, 128 - row_lo), shape.N - n_lo));
      for (int idx = (int)threadIdx.x - 64; idx < here * shape.M; idx += 128) {
        const int m = idx / here, local = idx - m * here, n = n_lo + local;
        int sum = 0;
        for (int sp = 0; sp < splits; ++sp) sum += recv[(sp * nb + m) * per + local];
        few_store<MODE>(out + (size_t)m * shape.ldo + n, sum, scales.rows[m], scales.columns[n],
                        scales.bias != nullptr ? scales.bias[n] : 0.f);
      }
    }
  }
  __syncthreads();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(tmem_cols));
  }
}

static int few_shared_bytes(int nb, int splits, int stages) {
  const int recv = splits > 1 ? splits * nb * few_rows_per_block(splits) * 4 : 0;
  return stages * few_stage_bytes(nb) + FEW_TAIL_BYTES + recv + 1024;
}

static int plan_few(FewShape& shape, int tiles, int sm_count) {
  const int two = 113 * 1024, most = 227 * 1024;
  int splits = 1;
  while (splits < FEW_MAX_SPLITS && tiles * (splits + 1) <= 2 * sm_count && shape.k_iters >= 4 * (splits + 1)) ++splits;
  shape.splits = splits;
  const int share = (shape.k_iters + splits - 1) / splits;
  for (int limit : {two, most}) {
    shape.stages = 12;
    while (shape.stages > 1 && few_shared_bytes(shape.nb, splits, shape.stages) > limit) --shape.stages;
    if (shape.stages >= 3) break;
  }
  if (shape.stages > share) shape.stages = share;
  return few_shared_bytes(shape.nb, splits, shape.stages);
}

template <int MODE, typename TO>
int launch_gemm_int8_few(void* out, const CUtensorMap& map_w, const CUtensorMap& map_x, FewShape shape, const Int8Scales& scales,
                         int sm_count, int* error_flag, cudaStream_t stream) {
  constexpr auto kernel = gemm_int8_few_kernel<MODE, TO>;
  const cudaError_t err = allow_shared_memory_once<kernel>(227 * 1024);
  if (err != cudaSuccess) return (int)err;
  const int tiles = (shape.N + 127) / 128;
  const int smem = plan_few(shape, tiles, sm_count);
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)tiles * shape.splits);
  config.blockDim = dim3(FEW_THREADS);
  config.dynamicSmemBytes = smem;
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
  cudaLaunchKernelEx(&config, kernel, map_w, map_x, (TO*)out, shape, scales, error_flag);
  return launch_status();
}

}  // namespace xrt

// codes: int8 [M, K] with rows ldx bytes apart; w: int8 [N, K] with rows ldw bytes apart; both strides multiples of 16 and both
// bases 16-byte aligned; scales float32 [M], w_scales float32 [N], bias float32 [N] or null.  out: [M, N] with row
// stride ldo; mode 0 stores, 1 adds into a float32 out.  constant_weight: none of the kernels that may still run wrote w, which
// is then read ahead of the wait for them.  error_flag (may be null) is set to 6 if a bounded wait ran out.
XRT_EXPORT int xrt_gemm_int8(void* out, const void* codes, const float* scales, const void* w, const float* w_scales,
                             const float* bias, int M, int N, int K, int ldx, int ldw, int ldo, int out_dtype, int mode,
                             int constant_weight, int* error_flag, cudaStream_t stream) {
  if (M < 0 || N <= 0 || K <= 0 || K > 131071 || ldx < K || ldw < K || ldo < N || mode < 0 || mode > 1) return XRT_ERR_ARGUMENT;
  if (mode == 1 && out_dtype != XRT_F32) return XRT_ERR_ARGUMENT;
  if (ldx % 16 != 0 || ldw % 16 != 0 || ((uintptr_t)codes & 15) || ((uintptr_t)w & 15)) return XRT_ERR_UNSUPPORTED;
  if (M == 0) return XRT_OK;
  const int sm_count = xrt::multiprocessors();
  if (sm_count <= 0) return XRT_ERR_UNSUPPORTED;
  CUtensorMap map_x, map_w;
  const xrt::Int8Scales factors{scales, w_scales, bias};
  if (M <= xrt::FEW_MAX_ROWS) {
    const xrt::FewShape shape{M, N, ldo, (M + 15) / 16 * 16, 1, 1, (K + xrt::I8_BK - 1) / xrt::I8_BK, constant_weight};
    if (!xrt::sm100::make_map_int8_2d(&map_x, codes, M, K, ldx, shape.nb) || !xrt::sm100::make_map_int8_2d(&map_w, w, N, K, ldw, 128))
      return XRT_ERR_UNSUPPORTED;
    if (mode == 1) return xrt::launch_gemm_int8_few<1, float>(out, map_w, map_x, shape, factors, sm_count, error_flag, stream);
    XRT_DISPATCH_DTYPE(out_dtype, TO, {
      return xrt::launch_gemm_int8_few<0, TO>(out, map_w, map_x, shape, factors, sm_count, error_flag, stream);
    });
  }
  if (!xrt::sm100::make_map_int8_2d(&map_x, codes, M, K, ldx, 128) || !xrt::sm100::make_map_int8_2d(&map_w, w, N, K, ldw, 128))
    return XRT_ERR_UNSUPPORTED;
  if (mode == 1)
    return xrt::launch_gemm_int8<1, float>(out, map_x, map_w, M, N, K, ldo, factors, sm_count, error_flag, stream);
  XRT_DISPATCH_DTYPE(out_dtype, TO, {
    return xrt::launch_gemm_int8<0, TO>(out, map_x, map_w, M, N, K, ldo, factors, sm_count, error_flag, stream);
  });
}
