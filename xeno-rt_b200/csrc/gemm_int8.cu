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
#include <type_traits>

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
    if (elect_one()) {
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
    if (elect_one()) {
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
  if (!ok) { *abort_flag = 1; if (error_flag != nullptr) atomicExch(error_flag, 6); }

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
constexpr int FEW_MAX_ROWS = 128, FEW_MAX_SPLITS = 8, FEW_MAX_STAGES = 24;
constexpr int FEW_PRODUCERS = 4;
constexpr int FEW_THREADS = 32 * (FEW_PRODUCERS + 1 + 4);
constexpr int FEW_TAIL_BYTES = 512 + 4 * (FEW_MAX_ROWS + 2 * 256);  // barriers, flags, a place that nobody reads; scales, biases

struct FewShape {
  int M, N, ldo;
  int nb;        // rows of codes, padded to a multiple of 16
  int rows;      // weight rows of a tile
  int splits;
  int slabs;     // of 128 of K in a stage: 1, 2 or 4
  int stages;
  int k_iters;   // stages' worth of K
  int early;     // the weight may be read before the kernel before this one is done
};

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
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
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

  pdl_trigger();
  if (splits > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = (int)blockIdx.x / splits, split = (int)blockIdx.x - tile * splits;
  const int kb0 = shape.k_iters * split / splits, kb1 = shape.k_iters * (split + 1) / splits;
  const int groups = shape.rows > 128 ? 2 : 1;
  int tmem_cols = 32;
  while (tmem_cols < groups * nb) tmem_cols *= 2;
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
      const int count = kb1 - kb0, first = tile * 5 % count;
      const int units = count * slabs, ahead = min(stages, count) * slabs;
      const int w_load = shape.rows * I8_BK;
      struct Walk {
        int s, i, k;  // stage, slab in the stage, and the stage's place in K
      };
      auto begin = [&]() {
        Walk at;
        at.s = warp / slabs;
        at.i = warp % slabs;
        at.k = first + at.s;
        while (at.s >= stages) at.s -= stages;
        while (at.k >= count) at.k -= count;
        return at;
      };
      auto step = [&](Walk& at) {  // four slabs further
        const int on = FEW_PRODUCERS / slabs;
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
      if (!shape.early) pdl_wait();
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
  const int here = max(0, min(min(per, shape.rows - row_lo), shape.N - n_lo)), quads = (shape.M + 3) / 4;
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
    const int begin = pass == 1 ? (int)threadIdx.x : 0, end = pass == 1 ? here * quads : 1, wide = max(here, 1);
#pragma unroll 1
    for (int idx = begin; idx < end; idx += FEW_THREADS) {
      const int quad = idx / wide, local = idx - quad * wide;
      int sums[4] = {0, 0, 0, 0};
#pragma unroll 1
      for (int sp = 0; sp < splits; ++sp) {
        const int4 part = *reinterpret_cast<const int4*>(recv + (sp * per + local) * recv_row + quad * 4);
        sums[0] += part.x; sums[1] += part.y; sums[2] += part.z; sums[3] += part.w;
      }
      const float4 by_row = *reinterpret_cast<const float4*>(row_scales + quad * 4);
      const float by_column = column_scales[row_lo + local], bias = biases[row_lo + local];
      const float factors[4] = {by_row.x, by_row.y, by_row.z, by_row.w};
      // rows beyond M, and all rows of the first walk, go nowhere; what is added into is asked for before the first store,
      // which might be to the same memory
      TO* dst[4];
      float old[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int m = quad * 4 + e;
        dst[e] = pass == 1 && m < shape.M ? out + (size_t)m * shape.ldo + n_lo + local : reinterpret_cast<TO*>(nowhere);
        old[e] = MODE == 1 ? to_float(*dst[e]) : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float value = fmaf(__int2float_rn(sums[e]) * factors[e], by_column, bias);
        *dst[e] = from_float<TO>(MODE == 1 ? old[e] + value : value);
      }
    }
  }
  __syncthreads();
  if (warp == FEW_PRODUCERS) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(tmem_cols));
  }
}

static int few_shared_bytes(const FewShape& s) {
  return few_ring_bytes(s) + FEW_TAIL_BYTES + (s.splits > 1 ? few_recv_bytes(s) : 0) + 1024;
}

// The tile, the parts of K and the ring of a product, from what was measured on a B200 (148 multiprocessors).
//
// Up to 128 weight rows a multiprocessor, one block each: the time is the longer of W from memory (6.3 TB/s in all, 110 GB/s
// into one multiprocessor) and a block's walk over its slabs (0.15 us each, or their bytes at 110 GB/s), a third of the
// shorter, and what it takes to begin and end: 2 us, and where the parts of a tile meet 0.8 us more and 0.4 us for each
// 1,000 sums that a block sends.  Clusters of 3 and 4 do not fill the device (45 and 33 are held; many fewer of 3 at once in
// practice).  Microseconds, chosen against the next best number of parts: 8 rows of 4,096 outputs, 4,096 inputs 5.9 (4 parts; 2: 6.0,
// 1: 7.8); 6,144, 4,096 7.1 (2; 4: 7.5); 4,096, 14,336 12.4 (4; 3: 12.8); 64 of 2,048, 2,048 4.8 (2; 4: 5.2).
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
    for (int splits = 1; splits <= 4 && (splits == 1 || slabs >= 4 * splits); ++splits) {
      const int blocks = splits <= 2 ? sm_count : splits == 3 ? sm_count * 4 / 5 : sm_count * 8 / 9;
      if (blocks < splits) break;
      const int even = even_rows(blocks / splits);
      for (int rows : {32, 64, 96, 128, even}) {
        if (rows > 256 || rows < even) continue;
        const int used = (s.N + rows - 1) / rows * splits;
        const double rate = used * 0.11e6 < 6.3e6 ? used * 0.11e6 : 6.3e6, slab_us = (rows + s.M) * 128 / 110e3;
        const double memory_us = (double)s.N * K / rate;
        const double walk_us = (slabs + splits - 1) / splits * (slab_us > 0.15 ? slab_us : 0.15);
        const double longer = memory_us > walk_us ? memory_us : walk_us;
        const double cost = longer + 0.3 * (memory_us + walk_us - longer) + (splits > 1 ? 0.8 + 0.4e-3 * rows * s.M : 0.0);
        if (s.splits == 0 || cost < best) { best = cost; s.splits = splits; s.rows = rows; }
      }
    }
  } else {
    const int two_most = 220 - s.nb;  // weight rows that leave room for four slabs
    const int two_rounds = (s.N + 2 * sm_count * two_most - 1) / (2 * sm_count * two_most);
    const int one_rounds = (s.N + sm_count * 256 - 1) / (sm_count * 256);
    const bool two = two_rounds == 1 || one_rounds > 1;
    s.splits = 1;
    s.rows = two ? even_rows(2 * sm_count * two_rounds) : even_rows(sm_count);
    if (two) limit = FEW_SHARED_TWO;
  }
  // slabs a stage: as many as leave a ring of three stages
  for (s.slabs = 4; s.slabs > 1; s.slabs /= 2) {
    s.stages = 3;
    if (few_shared_bytes(s) <= limit) break;
  }
  s.k_iters = (slabs + s.slabs - 1) / s.slabs;
  const int share = (s.k_iters + s.splits - 1) / s.splits;
  for (;;) {
    s.stages = FEW_MAX_STAGES;
    while (s.stages > 1 && few_shared_bytes(s) > limit) --s.stages;
    // the producers, which take every fourth slab each, need a ring of four slabs if it turns
    if (s.stages * s.slabs >= FEW_PRODUCERS || s.stages >= share || limit == FEW_SHARED_ONE) break;
    limit = FEW_SHARED_ONE;
  }
  if (s.stages > share) s.stages = share;
}

template <int MODE, typename TO>
int launch_gemm_int8_few(void* out, const CUtensorMap& map_w, const CUtensorMap& map_x, const FewShape& shape, const Int8Scales& scales,
                         int* error_flag, cudaStream_t stream) {
  constexpr auto kernel = gemm_int8_few_kernel<MODE, TO>;
  const cudaError_t err = allow_shared_memory_once<kernel>(FEW_SHARED_ONE);
  if (err != cudaSuccess) return (int)err;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)((shape.N + shape.rows - 1) / shape.rows) * shape.splits);
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
    xrt::FewShape shape = {};
    shape.M = M; shape.N = N; shape.ldo = ldo;
    shape.nb = (M + 15) / 16 * 16;
    shape.early = constant_weight;
    xrt::plan_few(shape, K, sm_count);
    if (!xrt::sm100::make_map_int8_2d(&map_x, codes, M, K, ldx, shape.nb) ||
        !xrt::sm100::make_map_int8_2d(&map_w, w, N, K, ldw, shape.rows))
      return XRT_ERR_UNSUPPORTED;
    if (mode == 1) return xrt::launch_gemm_int8_few<1, float>(out, map_w, map_x, shape, factors, error_flag, stream);
    XRT_DISPATCH_DTYPE(out_dtype, TO, {
      return xrt::launch_gemm_int8_few<0, TO>(out, map_w, map_x, shape, factors, error_flag, stream);
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
