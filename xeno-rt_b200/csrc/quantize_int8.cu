// Rows as 8-bit integers with one 32-bit scale a row, for the products of gemm_int8.cu:
//     scale = max(max_c |y[c]| / 127, 2^-126),   code[c] = y[c] / scale rounded to the nearest whole number, ties to even,
// where y is a row as it is, the hidden units of a gated feed-forward (activation.cu's formula), or the RMSNorm
// (norm.cu's formula) of the residual stream after something was added to it:
//     s = x + add,   y = s / sqrt(mean(s^2) + eps) * w.
// A row of zeros has codes 0 and the smallest scale.  A row with a NaN or an infinity has codes 0 and the scale NaN, so that
// every product with it is NaN.  Sums, statistics and y are 32-bit; the codes are the only rounding to fewer bits.
//
// One block a row, the row in registers: read once, one meeting of the block (the norm's sum of squares and the largest |s w|
// are found in the same pass, since the factor 1 / rms is the same for the whole row), codes written once.  The largest absolute
// value is found on the bits: for numbers without a sign their order is that of the integers, and every NaN lies above infinity.
//
// Few rows (steps): a block a row, its loads all in flight together.  More rows than blocks: blocks take every so many-th
// row from a ring in shared memory that bulk copies fill ahead (quantize_int8_ring_kernel), so that the memory is asked for the
// next rows while a block meets.  Rows beyond what 1,024 threads hold are walked twice.
//
// What bounds it: many long rows the memory, and beside it the instructions that a multiprocessor issues (hence Two, largest_of
// and four_sigmoid below: gates 64 -> 51 us, 4,096 plain rows of 8,192 22.6 -> 20.6); few rows the time of one load, one meeting and
// one store.  Measured on a B200, operands from memory, microseconds (bytes that it cannot do without at the copy rate of 6.55
// TB/s): norm after an addition of 1 row of 4,096 2.2, of 2,048 16.2 (14.1), of 8,191 of 5,120, float32 79-87 (83), without one of
// 2,048 of 4,096 10.4 (6.4); gate of 8 rows of 14,336 units 2.75, of 2,048 29.8 (22.4), of 2,000 of 25,600 52 (39); plain rows, 64
// of 4,096 1.5, 2,000 6.9 (3.8), 4,096 of 8,192 20.8 (15.4).  Rows of a width or an address that allows single values only take
// longer: norm of 2,047 of 4,095 35 (16.6), gates of 2,000 of 25,599 75 (39).
#include <stddef.h>

#include <type_traits>

#include "tcgen05.cuh"

namespace xrt {

constexpr float CODE_MAX = 127.0f, SMALLEST_SCALE = 1.17549435e-38f;
constexpr float ROUNDER = 12582912.0f;  // 1.5 * 2^23: v + ROUNDER has v, rounded to a whole number, in its low bits

// Two 32-bit numbers in one instruction: a row's arithmetic is bound by the instructions that a multiprocessor can issue.
struct Two {
  uint64_t bits;
  Two() = default;
  __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(bits) : "f"(a), "f"(b)); }
  __device__ __forceinline__ explicit Two(float a) : Two(a, a) {}
  __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(bits)); }
};
__device__ __forceinline__ Two operator*(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
  return r;
}
__device__ __forceinline__ Two operator+(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
  return r;
}
__device__ __forceinline__ Two fma_two(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits), "l"(c.bits));
  return r;
}

// The largest absolute value of a row's pieces; a NaN once any is one.
template <int VEC>
__device__ __forceinline__ float largest_of(float most, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(most) : "f"(most), "f"(fabsf(v[0])));
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 2)
      asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(most) : "f"(most), "f"(fabsf(v[i])), "f"(fabsf(v[i + 1])));
  }
  return most;
}

template <int VEC>
__device__ __forceinline__ void load_some(const float* p, float (&v)[VEC]) {
  if constexpr (VEC % 4 == 0) {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const float4 t = *reinterpret_cast<const float4*>(p + i);
      v[i] = t.x; v[i + 1] = t.y; v[i + 2] = t.z; v[i + 3] = t.w;
    }
  } else {
    v[0] = *p;
  }
}
template <int VEC>
__device__ __forceinline__ void load_some(const __nv_bfloat16* p, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = __bfloat162float(*p);
  } else {
    uint32_t raw[VEC / 2];
    if constexpr (VEC == 8) {
      const uint4 t = *reinterpret_cast<const uint4*>(p);
      raw[0] = t.x; raw[1] = t.y; raw[2] = t.z; raw[3] = t.w;
    } else {
      const uint2 t = *reinterpret_cast<const uint2*>(p);
      raw[0] = t.x; raw[1] = t.y;
    }
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      v[2 * i] = __uint_as_float(raw[i] << 16);
      v[2 * i + 1] = __uint_as_float(raw[i] & 0xffff0000u);
    }
  }
}
template <int VEC>
__device__ __forceinline__ void store_some(float* p, const float (&v)[VEC]) {
  if constexpr (VEC % 4 == 0) {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  } else {
    *p = v[0];
  }
}

// The codes of VEC values y / scale, `inverse` being 1 / scale; all zero with `broken`.  EXACT: of the quotient as a 32-bit division
// rounds it: the product with the inverse, corrected once by its remainder (Markstein's correction: IBM J. Res. Dev. 34, 1990; of
// bfloat16 values every such quotient is tested).  A row that is coded as it is needs that: its values
// have few bits, and quotients in the middle between two codes, which go to the even one, are many.  What was computed on
// the way here is not exact in its last bit.
template <int VEC, bool EXACT>
__device__ __forceinline__ void store_codes(int8_t* p, const float (&y)[VEC], float scale, float inverse, bool broken) {
  uint32_t bits[VEC];
  if constexpr (VEC == 1) {
    float q = y[0] * inverse;
    if constexpr (EXACT) q = fmaf(fmaf(-q, scale, y[0]), inverse, q) + ROUNDER;
    else q = fmaf(y[0], inverse, ROUNDER);
    bits[0] = __float_as_uint(q);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const Two both(y[i], y[i + 1]);
      Two code;
      if constexpr (EXACT) {
        const Two q = both * Two(inverse);
        code = fma_two(fma_two(q, Two(-scale), both), Two(inverse), q) + Two(ROUNDER);
      } else {
        code = fma_two(both, Two(inverse), Two(ROUNDER));
      }
      float first, second;
      code.get(first, second);
      bits[i] = __float_as_uint(first);
      bits[i + 1] = __float_as_uint(second);
    }
  }
  if constexpr (VEC == 1) {
    *p = broken ? 0 : (int8_t)(bits[0] & 0xff);
  } else {
    uint32_t word[VEC / 4];
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      const uint32_t lo = __byte_perm(bits[4 * i], bits[4 * i + 1], 0x0040), hi = __byte_perm(bits[4 * i + 2], bits[4 * i + 3], 0x0040);
      word[i] = broken ? 0u : __byte_perm(lo, hi, 0x5410);
    }
    if constexpr (VEC == 8) *reinterpret_cast<uint2*>(p) = make_uint2(word[0], word[1]);
    else *reinterpret_cast<uint32_t*>(p) = word[0];
  }
}

// What a row's values are made of: VEC of them from column c on, after `load` and `settle` (all loads of a thread come
// before its first store, which might be to the same memory).  NORMED: the sum of squares is wanted, and the values have
// to be multiplied by 1 / rms.
template <typename T>
struct PlainRows {
  static constexpr bool NORMED = false;
  static constexpr bool GATED = false, EXACT = true;
  static constexpr int STREAMS = 1;  // what a row consists of in memory: pieces of `length` elements of From<i>
  template <int I> using From = T;
  const T* x;
  template <int I> __host__ __device__ __forceinline__ const T* from() const { return x; }
  __host__ __device__ __forceinline__ static int length(int width) { return width; }
  static constexpr int early = 0;
  __device__ __forceinline__ void wait() { pdl_wait(x); }
  // the values from a row's streams where those lie in shared memory
  template <int VEC, class READ> __device__ __forceinline__ void read(int c, int, const READ& get, float (&v)[VEC]) const {
    get.template operator()<0, VEC>(c, v);
  }
  template <int VEC, bool LOOSE = false> __device__ __forceinline__ void ahead(int, int, float (&)[VEC]) const {}
  template <int VEC, bool AGAIN> __device__ __forceinline__ void load(int row, int c, int width, float (&v)[VEC]) const {
    load_some<VEC>(x + (size_t)row * width + c, v);
  }
  template <int VEC, bool AGAIN>
  __device__ __forceinline__ void settle(int, int, int, const float (&)[VEC], float (&)[VEC], float&) const {}
};

template <typename T>
struct GatedRows {
  static constexpr bool NORMED = false;
  static constexpr bool GATED = true, EXACT = false;
  static constexpr float GELU = 1.5957691216057308f;  // 2 sqrt(2 / pi)
  static constexpr int STREAMS = 1;
  template <int I> using From = T;
  const T* gate_up;  // [rows, 2 * width]
  RowScale gate;
  template <int I> __host__ __device__ __forceinline__ const T* from() const { return gate_up; }
  __host__ __device__ __forceinline__ static int length(int width) { return 2 * width; }
  static constexpr int early = 0;
  __device__ __forceinline__ void wait() { pdl_wait(gate_up); }
  // g sigmoid(a g) u as g / (1 + 2^(-a log2(e) g)) u: the exponential and the reciprocal as the multiprocessor has them (2 ulp and 1;
  // 8 bits are kept).  They give 0 for results below 2^-126, but sigmoid goes on to 2^-128 before 1 + 2^x is no 32-bit number
  // (and a gate of -88 alone in its row, times a large u, is the scale): hence 4 sigmoid, 1 / (1 / 4 + 2^(x - 2)), from x - 2,
  // which the exponent's last addition gives.  Beyond, the result is 0, as the formula's is in 32 bits.
  __device__ __forceinline__ static float four_sigmoid(float exponent_less_2) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(exponent_less_2));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(0.25f + e));
    return r;
  }
  // a limit lets what is no number through, so that its row is broken
  __device__ __forceinline__ static float smaller(float a, float b) {
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(b));
    return a;
  }
  __device__ __forceinline__ static float larger(float a, float b) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(b));
    return a;
  }
  template <int VEC> __device__ __forceinline__ void gated(float (&g)[VEC], float (&u)[VEC], int c) const {
    constexpr float LOG2E = 1.4426950408889634f;
    add_gate_biases<VEC, true>(g, u, c, gate);
    if (gate.gate_act == 2) {
      const float limit = gate.gate_limit, exponent = -gate.gate_alpha * LOG2E;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float x = smaller(g[i], limit);
        g[i] = 0.25f * x * four_sigmoid(fmaf(x, exponent, -2.0f)) * (smaller(larger(u[i], -limit), limit) + 1.0f);
      }
      return;
    }
    // 0.5 g (1 + tanh(z)) = g sigmoid(2 z), which loses nothing where tanh(z) is near -1: alone in its row, such a
    // value is the scale
    const bool tanh_form = gate.gate_act == 1;
    if constexpr (VEC == 1) {
      const float by = tanh_form ? fmaf(-GELU * 0.044715f * LOG2E, g[0] * g[0], -GELU * LOG2E) : -LOG2E;
      g[0] = 0.25f * g[0] * four_sigmoid(fmaf(g[0], by, -2.0f)) * u[0];
    } else {
#pragma unroll
      for (int i = 0; i < VEC; i += 2) {
        const Two x(g[i], g[i + 1]);
        const Two by = tanh_form ? fma_two(x * x, Two(-GELU * 0.044715f * LOG2E), Two(-GELU * LOG2E)) : Two(-LOG2E);
        float first, second;
        fma_two(x, by, Two(-2.0f)).get(first, second);
        (Two(0.25f) * x * Two(four_sigmoid(first), four_sigmoid(second)) * Two(u[i], u[i + 1])).get(g[i], g[i + 1]);
      }
    }
  }
  template <int VEC, class READ> __device__ __forceinline__ void read(int c, int width, const READ& get, float (&v)[VEC]) const {
    float u[VEC];
    get.template operator()<0, VEC>(c, v);
    get.template operator()<0, VEC>(width + c, u);
    gated<VEC>(v, u, c);
  }
  template <int VEC, bool LOOSE = false> __device__ __forceinline__ void ahead(int, int, float (&)[VEC]) const {}
  template <int VEC, bool AGAIN> __device__ __forceinline__ void load(int row, int c, int width, float (&v)[VEC]) const {
    const T* p = gate_up + (size_t)row * 2 * width + c;
    float u[VEC];
    load_some<VEC>(p, v);
    load_some<VEC>(p + width, u);
    gated<VEC>(v, u, c);
  }
  template <int VEC, bool AGAIN>
  __device__ __forceinline__ void settle(int, int, int, const float (&)[VEC], float (&)[VEC], float&) const {}
};

struct Nothing {};

// TA: what is added (Nothing: nothing is, and no sum is written).
template <typename TA, typename TW>
struct NormedRows {
  static constexpr bool NORMED = true;
  static constexpr bool ADDS = !std::is_same<TA, Nothing>::value;
  static constexpr bool GATED = false, EXACT = false;
  static constexpr int STREAMS = ADDS ? 2 : 1;
  template <int I> using From = std::conditional_t<I == 0, float, TA>;
  template <int I> __host__ __device__ __forceinline__ const From<I>* from() const {
    if constexpr (I == 0) return x;
    else return add;
  }
  __host__ __device__ __forceinline__ static int length(int width) { return width; }
  template <int VEC, class READ> __device__ __forceinline__ void read(int c, int, const READ& get, float (&v)[VEC]) const {
    get.template operator()<0, VEC>(c, v);
    if constexpr (ADDS) {
      float a[VEC];
      get.template operator()<1, VEC>(c, a);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] += a[i];
    }
  }
  const float* x;
  const TA* add;
  float* sum;  // may be x
  const TW* weight;
  float eps;
  int early;  // the weight may be read before the kernel before this one is done
  __device__ __forceinline__ void wait() { pdl_wait(x, add); }
  // LOOSE: pieces begin at any element, the last one with the row's last VEC elements
  template <int VEC, bool LOOSE = false> __device__ __forceinline__ void ahead(int c, int width, float (&w)[VEC]) const {
    if (c >= width) return;
    if constexpr (LOOSE) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) w[i] = to_float(weight[min(c, width - VEC) + i]);
    } else {
      load_some<VEC>(weight + c, w);
    }
  }
  template <int VEC, bool AGAIN> __device__ __forceinline__ void load(int row, int c, int width, float (&v)[VEC]) const {
    const size_t at = (size_t)row * width + c;
    if constexpr (ADDS && AGAIN) {
      load_some<VEC>(const_cast<const float*>(sum) + at, v);  // this thread wrote it
    } else {
      load_some<VEC>(x + at, v);
      if constexpr (ADDS) {
        float a[VEC];
        load_some<VEC>(add + at, a);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] += a[i];
      }
    }
  }
  template <int VEC, bool AGAIN, bool LOOSE = false>
  __device__ __forceinline__ void settle(int row, int c, int width, const float (&w)[VEC], float (&v)[VEC], float& squares) const {
    static_assert(!LOOSE || !ADDS, "a sum's pieces would be written in parts of the memory's 32 bytes");
    if constexpr (ADDS && !AGAIN) store_some<VEC>(sum + (size_t)row * width + c, v);
    const int first = LOOSE ? min(c, width - VEC) : c;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if (!LOOSE || first + i >= c) squares = fmaf(v[i], v[i], squares);  // (what lies before belongs to another piece too)
      v[i] *= w[i];
    }
  }
};

// The block's largest `bits` and the sum of `squares` (in a fixed order), with one meeting.
template <bool NORMED>
__device__ __forceinline__ void meet(uint32_t& bits, float& squares, uint32_t (&most)[32], float (&sums)[32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (int)blockDim.x >> 5;
  bits = __reduce_max_sync(0xffffffffu, bits);
  if (NORMED) squares = warp_sum(squares);
  if (warps == 1) return;
  if (lane == 0) {
    most[warp] = bits;
    if (NORMED) sums[warp] = squares;
  }
  __syncthreads();
  bits = __reduce_max_sync(0xffffffffu, lane < warps ? most[lane] : 0u);
  if (NORMED) squares = warp_sum(lane < warps ? sums[lane] : 0.f);
}

// The scale of a row whose largest value times `factor` is `bits`, and its codes from the values that the threads hold.
struct RowScaleOf {
  float factor, scale, inverse;
  bool broken;
};
// The exact quotients of store_codes need remainders that are no smaller than what 32 bits hold: rows whose scale is below
// TINY_SCALE are divided as LIFT times themselves, which changes no quotient.
constexpr float TINY_SCALE = 8.2718061e-25f, LIFT = 18446744073709551616.0f;  // 2^-80, 2^64
template <class ROWS>
__device__ __forceinline__ RowScaleOf scale_of(const ROWS& rows, int width, uint32_t bits, float squares) {
  RowScaleOf s;
  s.factor = 1.f;
  if constexpr (ROWS::NORMED) s.factor = 1.0f / sqrtf(squares / (float)width + rows.eps);
  const float largest = __uint_as_float(bits) * s.factor;
  s.broken = !(largest <= 3.402823466e38f);
  s.scale = s.broken ? __uint_as_float(0x7fc00000u) : fmaxf(largest / CODE_MAX, SMALLEST_SCALE);
  s.inverse = 1.0f / s.scale;
  return s;
}
template <class ROWS, int VEC, int ITEMS, bool LOOSE = false>
__device__ __forceinline__ void finish_row(int8_t* codes, float* scales, const ROWS& rows, int row, int width, int ld_codes, int stride,
                                           uint32_t bits, float squares, float (&v)[ITEMS][VEC]) {
  RowScaleOf s = scale_of(rows, width, bits, squares);
  if (threadIdx.x == 0) scales[row] = s.scale;
  int8_t* dst = codes + (size_t)row * ld_codes;
  if (ROWS::EXACT && s.scale < TINY_SCALE) {
    s.scale *= LIFT;
    s.inverse = 1.0f / s.scale;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] *= LIFT;
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int c = (int)threadIdx.x * VEC + i * stride;
    if (c < width) {
      if constexpr (ROWS::NORMED) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] *= s.factor;
      }
      if (LOOSE && c + VEC > width) {  // the row's last elements, one by one
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float one[1] = {v[i][j]};
          store_codes<1, ROWS::EXACT>(dst + width - VEC + j, one, s.scale, s.inverse, s.broken);
        }
      } else {
        store_codes<VEC, ROWS::EXACT>(dst + c, v[i], s.scale, s.inverse, s.broken);
      }
    }
  }
}

// ITEMS pieces of VEC values a thread; 0: as many as the row takes, walked twice.
template <class ROWS, int VEC, int ITEMS>
__global__ void __launch_bounds__(1024)
quantize_int8_kernel(int8_t* __restrict__ codes, float* __restrict__ scales, ROWS rows, int width, int ld_codes) {
  __shared__ uint32_t most[32];
  __shared__ float sums[32];
  constexpr int KEPT = ITEMS > 0 ? ITEMS : 1;
  constexpr bool AHEAD = ITEMS > 0 && ITEMS * VEC <= 16;
  pdl_trigger();
  float w[KEPT][VEC], v[KEPT][VEC];
  const int stride = (int)blockDim.x * VEC;
  const bool waited = !rows.early;
  if (waited) rows.wait();
  if constexpr (AHEAD) {  // a model's weight is on its way before the wait for the kernel before
#pragma unroll
    for (int i = 0; i < KEPT; ++i) rows.template ahead<VEC>((int)threadIdx.x * VEC + i * stride, width, w[i]);
  }
  if (!waited) rows.wait();
  const int row = blockIdx.x;
  float squares = 0.f, most_here = 0.f;
  if constexpr (ITEMS > 0) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = (int)threadIdx.x * VEC + i * stride;
      if (c < width) {
        rows.template load<VEC, false>(row, c, width, v[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = (int)threadIdx.x * VEC + i * stride;
      if (c < width) {
        if constexpr (!AHEAD) rows.template ahead<VEC>(c, width, w[i]);
        rows.template settle<VEC, false>(row, c, width, w[i], v[i], squares);
        most_here = largest_of<VEC>(most_here, v[i]);
      }
    }
  } else {
    for (int c = (int)threadIdx.x * VEC; c < width; c += stride) {
      rows.template ahead<VEC>(c, width, w[0]);
      rows.template load<VEC, false>(row, c, width, v[0]);
      rows.template settle<VEC, false>(row, c, width, w[0], v[0], squares);
      most_here = largest_of<VEC>(most_here, v[0]);
    }
  }
  uint32_t bits = __float_as_uint(most_here);
  meet<ROWS::NORMED>(bits, squares, most, sums);
  if constexpr (ITEMS > 0) {
    finish_row<ROWS, VEC, KEPT>(codes, scales, rows, row, width, ld_codes, stride, bits, squares, v);
  } else {
    RowScaleOf s = scale_of(rows, width, bits, squares);
    if (threadIdx.x == 0) scales[row] = s.scale;
    const bool lifted = ROWS::EXACT && s.scale < TINY_SCALE;
    if (lifted) {
      s.scale *= LIFT;
      s.inverse = 1.0f / s.scale;
    }
    int8_t* dst = codes + (size_t)row * ld_codes;
    for (int c = (int)threadIdx.x * VEC; c < width; c += stride) {
      rows.template ahead<VEC>(c, width, w[0]);
      rows.template load<VEC, true>(row, c, width, v[0]);
      rows.template settle<VEC, true>(row, c, width, w[0], v[0], squares);
      if constexpr (ROWS::NORMED) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[0][j] *= s.factor;
      }
      if (lifted) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[0][j] *= LIFT;
      }
      store_codes<VEC, ROWS::EXACT>(dst + c, v[0], s.scale, s.inverse, s.broken);
    }
  }
}

// The ring.  A stage holds one row's streams, each at its own 16-byte phase: what lies between the first and the last
// 16-byte boundary of a stream comes by one bulk copy, the few elements outside are put beside it by the lanes of the warp that
// asks for the copy.
constexpr int RING_MOST = 8;

// Which launches take the ring: enough rows for every block to have several, and rows long enough (`stage` bytes) that few of
// them fill a multiprocessor; shorter ones are served as well by many small blocks.  Measured on a B200 (microseconds, ring /
// a block a row): bfloat16 rows of 1,000 (2 KB), 4,096 of them, 6.0 / 4.6; gates of 2 x 14,336, 2,048 of them, 29.5 / 47; norms
// without an addition, 600 of 4,096 (16 KB) 4.9 / 5.3, 2,048 10.6 / 11.7, 2,048 of 8,192 16.8 / 22.7, 8,191 of 14,336 90 / 136.
// With an addition the sum is written as well, and longer rows are asked for: 4,096 of 8,192 and bfloat16 (48 KB) 67 / 58, and
// float32 (64 KB) 74 / 82, 600 14.9 / 15.3, 1,200 of 14,336 and bfloat16 (84 KB) 34 / 40.
template <class ROWS, int VEC>
inline bool ring_pays(int n, int grid, int stage) {
  if (ROWS::STREAMS == 1 || VEC == 1) return n > grid && stage >= 6 * 1024;
  return n > 3 * grid && stage >= 60 * 1024;
}
// Threads of a block by the values a thread holds: 32 of them need more registers than 1,024 threads have.
constexpr int ring_threads(int per) { return per > 16 ? 832 : 1024; }
template <class ROWS, int I>
__host__ __device__ __forceinline__ int ring_room(int width) {  // of a stream in a stage
  return (ROWS::length(width) * (int)sizeof(typename ROWS::template From<I>) + 16 + 127) / 128 * 128;
}
template <class ROWS>
__host__ __device__ __forceinline__ int ring_stage(int width) {
  int bytes = ring_room<ROWS, 0>(width);
  if constexpr (ROWS::STREAMS == 2) bytes += ring_room<ROWS, 1>(width);
  return bytes;
}

template <class ROWS, int I>
__device__ __forceinline__ const typename ROWS::template From<I>* ring_source(const ROWS& rows, int row, int width) {
  return rows.template from<I>() + (size_t)row * ROWS::length(width);
}
// The bulk copy of a stream of a row to its place in a stage: where the row begins, and the copy's ends.  (Rows in a ring are
// thousands of bytes long, see ring_pays: none lies between two boundaries.)
struct RingCopy {
  uintptr_t begin, lo, hi;
  __device__ __forceinline__ uint32_t bytes() const { return (uint32_t)(hi - lo); }
  __device__ __forceinline__ void go(uint32_t place, uint32_t bar) const {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(place + (uint32_t)(lo - (begin & ~(uintptr_t)15))), "l"(lo), "r"(bytes()), "r"(bar) : "memory");
  }
};
template <class ROWS, int I>
__device__ __forceinline__ RingCopy ring_copy(const ROWS& rows, int row, int width) {
  RingCopy copy;
  copy.begin = (uintptr_t)ring_source<ROWS, I>(rows, row, width);
  const uintptr_t end = copy.begin + (size_t)ROWS::length(width) * sizeof(typename ROWS::template From<I>);
  copy.lo = (copy.begin + 15) & ~(uintptr_t)15;
  copy.hi = end & ~(uintptr_t)15;
  return copy;
}
// The elements outside that copy, by the lanes of a warp: at most 7 (of 2 bytes) before and 7 behind.
template <class ROWS, int I>
__device__ __forceinline__ void ring_edges(const ROWS& rows, int row, int width, unsigned char* place, int lane) {
  using T = typename ROWS::template From<I>;
  const RingCopy copy = ring_copy<ROWS, I>(rows, row, width);
  const uint32_t count = ROWS::length(width), size = sizeof(T);  // (unsigned: a signed division by 2 or 4 is not a shift)
  const int before = (uint32_t)(copy.lo - copy.begin) / size, behind = count - (uint32_t)(copy.hi - copy.begin) / size;
  const int i = lane < 16 ? lane : (int)count - behind + lane - 16;
  if (lane < 16 ? lane < before : lane - 16 < behind)
    reinterpret_cast<T*>(place + (copy.begin & 15))[i] = reinterpret_cast<const T*>(copy.begin)[i];
}

// A row's elements in its stage.  LOOSE: pieces begin at any element, and are read one by one.
template <class ROWS, bool LOOSE>
struct RingRow {
  const unsigned char* first;
  const unsigned char* second;  // of the streams: the places of element 0
  template <int I, int VEC>
  __device__ __forceinline__ void operator()(int c, float (&v)[VEC]) const {
    const auto* from = reinterpret_cast<const typename ROWS::template From<I>*>(I == 0 ? first : second) + c;
    if constexpr (LOOSE) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = to_float(from[j]);
    } else {
      load_some<VEC>(from, v);
    }
  }
};

// Rows blockIdx.x, blockIdx.x + gridDim.x, ..  LOOSE: rows whose width or address allows no pieces of VEC in memory, whose codes'
// addresses do: the last piece is the row's last VEC elements then, some of them for the second time.
template <class ROWS, int VEC, int ITEMS, bool LOOSE>
__global__ void __launch_bounds__(ring_threads(VEC * ITEMS))
quantize_int8_ring_kernel(int8_t* __restrict__ codes, float* __restrict__ scales, ROWS rows, int n, int width, int ld_codes, int stages,
                          int* error_flag) {
  using namespace sm100;
  extern __shared__ __align__(128) unsigned char ring[];
  __shared__ uint32_t most[2][32];
  __shared__ float sums[2][32];
  __shared__ uint64_t full[RING_MOST];
  __shared__ int abort_flag;
  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) mbar_init(smem_u32(&full[s]), 1);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  const int stride = (int)blockDim.x * VEC, stage_bytes = ring_stage<ROWS>(width), room0 = ring_room<ROWS, 0>(width);
  const int lane = threadIdx.x & 31;
  __syncthreads();
  // A thread has the same columns of every row: it keeps their weights, where they leave room for the values.  Microseconds, kept /
  // read again for every row: without an addition 2,048 rows of 8,192 16.8 / 18.9, 8,191 of 14,336 90 / 110; with one, 600 of
  // 8,192, float32 15.0 / 17.1, 2,048 39 / 41, 4,096 75 / 75.5, 8,191 153.6 / 147, and of 14,336, bfloat16 600 20.8 / 22.8, 4,096 115 /
  // 112.5, 8,191 226 / 215: thousands of long rows with an addition lose 2 to 5 percent by it, fewer gain 5 to 13.
  constexpr bool KEEPS = ROWS::NORMED && VEC * ITEMS <= 16;
  float kept[KEEPS ? ITEMS : 1][VEC];
  auto keep = [&]() {
    if constexpr (KEEPS) {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) rows.template ahead<VEC, LOOSE>((int)threadIdx.x * VEC + i * stride, width, kept[i]);
    }
  };
  if (rows.early) keep();
  rows.wait();
  auto fetch = [&](int row, int s) {  // the first warp
    unsigned char* place = ring + s * stage_bytes;
    const uint32_t bar = smem_u32(&full[s]);
    if constexpr (VEC < 8) {  // (else rows begin and end at 16-byte boundaries)
      ring_edges<ROWS, 0>(rows, row, width, place, lane);
      if constexpr (ROWS::STREAMS == 2) ring_edges<ROWS, 1>(rows, row, width, place + room0, lane);
      __syncwarp();
    }
    if (elect_one()) {
      const RingCopy copy = ring_copy<ROWS, 0>(rows, row, width);
      if constexpr (ROWS::STREAMS == 2) {
        const RingCopy second = ring_copy<ROWS, 1>(rows, row, width);
        mbar_arrive_expect_tx(bar, copy.bytes() + second.bytes());
        second.go(smem_u32(place) + room0, bar);
      } else {
        mbar_arrive_expect_tx(bar, copy.bytes());
      }
      copy.go(smem_u32(place), bar);
    }
  };
  if (threadIdx.x < 32)
    for (int s = 0, row = blockIdx.x; s < stages && row < n; ++s, row += gridDim.x) fetch(row, s);
  if (!rows.early) keep();
  int s = 0, turn = 0, side = 0;
  for (int row = blockIdx.x; row < n; row += gridDim.x) {
    if (!mbar_wait(smem_u32(&full[s]), turn, &abort_flag)) {
      abort_flag = 1;
      if (error_flag != nullptr) atomicExch(error_flag, 7);
    }
    const unsigned char* place = ring + s * stage_bytes;
    RingRow<ROWS, LOOSE> from{place, place + room0};
    if constexpr (VEC < 8) {
      from.first += (uintptr_t)ring_source<ROWS, 0>(rows, row, width) & 15;
      if constexpr (ROWS::STREAMS == 2) from.second += (uintptr_t)ring_source<ROWS, 1>(rows, row, width) & 15;
    }
    float v[ITEMS][VEC], squares = 0.f, most_here = 0.f;
    // Pieces beyond the row are its last piece again (which changes no largest value), so that no branch keeps the pieces from
    // being worked out side by side.
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      rows.template read<VEC>(min((int)threadIdx.x * VEC + i * stride, width - VEC), width, from, v[i]);
      if (ROWS::GATED && VEC * ITEMS > 16) asm volatile("" ::: "memory");  // 32 units and their gates would not fit the registers
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = (int)threadIdx.x * VEC + i * stride;
      if (!ROWS::NORMED || c < width) {
        if constexpr (KEEPS) {
          rows.template settle<VEC, false, LOOSE>(row, c, width, kept[i], v[i], squares);
        } else if constexpr (ROWS::NORMED) {
          float w[VEC];
          rows.template ahead<VEC, LOOSE>(c, width, w);
          rows.template settle<VEC, false, LOOSE>(row, c, width, w, v[i], squares);
        }
        most_here = largest_of<VEC>(most_here, v[i]);
      }
    }
    uint32_t bits = __float_as_uint(most_here);
    meet<ROWS::NORMED>(bits, squares, most[side], sums[side]);
    side ^= 1;
    const bool given_up = *reinterpret_cast<volatile int*>(&abort_flag) != 0;
    // every thread has its values: the stage is free for the row that comes so many turns later
    if (threadIdx.x < 32) {
      __syncwarp();
      if (row + (long long)stages * gridDim.x < n && !given_up) fetch(row + stages * gridDim.x, s);
    }
    finish_row<ROWS, VEC, ITEMS, LOOSE>(codes, scales, rows, row, width, ld_codes, stride, bits, squares, v);
    if (++s == stages) { s = 0; turn ^= 1; }
    if (given_up) {
      if (threadIdx.x == 0) mbar_wait_copies(full, stages);
      break;
    }
  }
}

// Whether pieces of VEC values of a T of every row may be read or written at once: rows of `width` T's begin at p.
template <typename T>
inline bool pieces_fit(const T* p, int width, int vec) {
  const uintptr_t bytes = (uintptr_t)(vec * sizeof(T) < 16 ? vec * sizeof(T) : 16);
  return p == nullptr || ((uintptr_t)p % bytes == 0 && (size_t)width * sizeof(T) % bytes == 0);
}
template <typename T> bool fits(const PlainRows<T>& r, int width, int vec) { return pieces_fit(r.x, width, vec); }
template <typename T> bool fits(const GatedRows<T>& r, int width, int vec) { return pieces_fit(r.gate_up, width, vec); }
template <typename TW> bool fits(const NormedRows<Nothing, TW>& r, int width, int vec) {
  return pieces_fit(r.x, width, vec) && pieces_fit(r.weight, width, vec);
}
template <typename TA, typename TW> bool fits(const NormedRows<TA, TW>& r, int width, int vec) {
  return pieces_fit(r.x, width, vec) && pieces_fit(r.weight, width, vec) && pieces_fit(r.add, width, vec) && pieces_fit(r.sum, width, vec);
}

template <class ROWS, int VEC, int PER, bool LOOSE = false>
int launch_quantize_ring(int8_t* codes, float* scales, const ROWS& rows, int n, int width, int ld_codes, int* error_flag,
                         cudaStream_t stream, bool& taken) {
  // Single values, but codes that allow pieces of four: four neighbours a thread, read one by one.  Microseconds, so / single
  // values: 2,000 gates of 25,599 units 75 / 208, 600 of 5,003 7.9 / 13.2; 4,000 plain rows of 4,001 17.2 / 26.4;
  // 2,047 norms of 4,095 16.5 / 18.6.  With an addition (whose sums would be written in parts of 32 bytes) 8,191 of 4,097 185 / 117, and
  // single values stay.
  if constexpr (VEC == 1 && ROWS::STREAMS == 1)
    if (((uintptr_t)codes | (uintptr_t)ld_codes) % 4 == 0)
      return launch_quantize_ring<ROWS, 4, PER, true>(codes, scales, rows, n, width, ld_codes, error_flag, stream, taken);
  constexpr auto kernel = quantize_int8_ring_kernel<ROWS, VEC, PER / VEC, LOOSE>;
  const int threads = ((width + PER - 1) / PER + 31) / 32 * 32, stage = ring_stage<ROWS>(width), room = 208 * 1024;
  if (threads > ring_threads(PER)) return XRT_OK;
  int blocks = ring_threads(PER) / threads < 8 ? ring_threads(PER) / threads : 8;
  while (blocks > 1 && 2 * stage * blocks > room) --blocks;
  int stages = room / blocks / stage;
  if (stages > RING_MOST) stages = RING_MOST;
  const int grid = blocks * multiprocessors();
  taken = stages >= 2 && ring_pays<ROWS, VEC>(n, grid, stage);
  if (!taken) return XRT_OK;
  const cudaError_t err = allow_shared_memory_once<kernel>(room);
  if (err != cudaSuccess) return (int)err;
  launch_kernel(kernel, dim3(grid), dim3(threads), (size_t)stages * stage, stream, codes, scales, rows, n, width, ld_codes, stages, error_flag);
  return launch_status();
}

template <class ROWS, int VEC>
int launch_quantize(int8_t* codes, float* scales, const ROWS& rows, int n, int width, int ld_codes, int* error_flag, cudaStream_t stream) {
  bool taken = false;
  int status = XRT_OK;
  // Microseconds with 16 / 32 values a thread: 2,048 gates of 14,336 units 29.8 / 34.8, 600 13.2 / 14.1; plain rows between
  // 20.5 / 19.2 (8,191 of 4,096) and 8.2 / 8.0 (600 of 14,336).
  if (width <= 16 * 1024)
    status = launch_quantize_ring<ROWS, VEC, 16>(codes, scales, rows, n, width, ld_codes, error_flag, stream, taken);
  else if (width <= 32 * 1024)
    status = launch_quantize_ring<ROWS, VEC, 32>(codes, scales, rows, n, width, ld_codes, error_flag, stream, taken);
  if (taken || status != XRT_OK) return status;
  auto launch = [&](auto kernel, int per) {
    const int threads = per > 0 ? ((width + per - 1) / per + 31) / 32 * 32 : 1024;
    launch_kernel(kernel, dim3(n), dim3(threads), 0, stream, codes, scales, rows, width, ld_codes);
    return launch_status();
  };
  // The fewest values a thread that 1,024 threads allow, which keeps the most loads in flight.  Microseconds with 8 / 16 a thread:
  // norm of 1 row of 4,096 2.0 / 2.25, of 2,048 16.4 / 18.5, gate of 600 of 8,192 8.1 / 9.2, 600 plain rows of 8,192 5.3 / 5.5.
  if (width <= 8 * 1024) return launch(quantize_int8_kernel<ROWS, VEC, 8 / VEC>, 8);
  if (width <= 16 * 1024) return launch(quantize_int8_kernel<ROWS, VEC, 16 / VEC>, 16);
  if (width <= 32 * 1024) return launch(quantize_int8_kernel<ROWS, VEC, 32 / VEC>, 32);
  return launch(quantize_int8_kernel<ROWS, VEC, 0>, 0);
}

// Pieces of eight, four or one value at a time: the most that rows of this width and these addresses allow.
template <class ROWS>
int quantize(int8_t* codes, float* scales, const ROWS& rows, int n, int width, int ld_codes, int* error_flag, cudaStream_t stream) {
  if (n < 0 || n > XRT_INT8_MAX_SIZE || width <= 0 || width > XRT_INT8_MAX_SIZE || ld_codes < width) return XRT_ERR_ARGUMENT;
  if (n == 0) return XRT_OK;
  auto whole = [&](int vec) {
    return width % vec == 0 && fits(rows, width, vec) && ((uintptr_t)codes | (uintptr_t)ld_codes) % vec == 0;
  };
  if (whole(8)) return launch_quantize<ROWS, 8>(codes, scales, rows, n, width, ld_codes, error_flag, stream);
  if (whole(4)) return launch_quantize<ROWS, 4>(codes, scales, rows, n, width, ld_codes, error_flag, stream);
  return launch_quantize<ROWS, 1>(codes, scales, rows, n, width, ld_codes, error_flag, stream);
}

}  // namespace xrt

// A call as the caller packs it.  codes: int8 [n, width] with rows ld_codes bytes apart; scales: float32 [n]; error_flag (may be
// null) is set to 7 if a bounded wait ran out.
struct XrtRowsCall {
  void* codes;
  float* scales;
  const void* x;
  const void* add;
  float* sum;
  const void* weight;
  const xrt::GateOptions* gate;
  int* error_flag;
  int n, width, ld_codes, x_dtype, add_dtype, w_dtype, act, constant_weight;
  float eps;
};
static_assert(offsetof(XrtRowsCall, n) == 64 && offsetof(XrtRowsCall, eps) == 96, "eight pointers, eight ints, a float");

template <class ROWS>
static int quantize_call(const XrtRowsCall& c, const ROWS& rows, cudaStream_t stream) {
  return xrt::quantize((int8_t*)c.codes, c.scales, rows, c.n, c.width, c.ld_codes, c.error_flag, stream);
}

// x [n, width], float32 or bfloat16.
XRT_EXPORT int xrt_quantize_rows(const XrtRowsCall* call, cudaStream_t stream) {
  const XrtRowsCall& c = *call;
  XRT_DISPATCH_DTYPE(c.x_dtype, T, { return quantize_call(c, xrt::PlainRows<T>{(const T*)c.x}, stream); });
}

// x: gate_up [n, 2 * width], float32 or bfloat16; act and gate as for xrt_swiglu.
XRT_EXPORT int xrt_swiglu_int8(const XrtRowsCall* call, cudaStream_t stream) {
  const XrtRowsCall& c = *call;
  if (c.act < 0 || c.act > 2) return XRT_ERR_ARGUMENT;
  xrt::RowScale gate;
  gate.gate_act = c.act;
  if (!xrt::take_gate_options(c.gate, 2, c.width, gate)) return XRT_ERR_ARGUMENT;
  XRT_DISPATCH_DTYPE(c.x_dtype, T, { return quantize_call(c, xrt::GatedRows<T>{(const T*)c.x, gate}, stream); });
}

// x float32 [n, width]; add (may be null) [n, width], float32 or bfloat16; with it sum [n, width] gets x + add (sum may be x).
// constant_weight: none of the kernels that may still run wrote the weight.
XRT_EXPORT int xrt_rmsnorm_int8(const XrtRowsCall* call, cudaStream_t stream) {
  const XrtRowsCall& c = *call;
  if (c.add != nullptr && c.sum == nullptr) return XRT_ERR_ARGUMENT;
  const float* x = (const float*)c.x;
  XRT_DISPATCH_DTYPE(c.w_dtype, TW, {
    const TW* weight = (const TW*)c.weight;
    if (c.add == nullptr)
      return quantize_call(c, xrt::NormedRows<xrt::Nothing, TW>{x, nullptr, nullptr, weight, c.eps, c.constant_weight}, stream);
    XRT_DISPATCH_DTYPE(c.add_dtype, TA, {
      return quantize_call(c, xrt::NormedRows<TA, TW>{x, (const TA*)c.add, c.sum, weight, c.eps, c.constant_weight}, stream);
    });
  });
}
