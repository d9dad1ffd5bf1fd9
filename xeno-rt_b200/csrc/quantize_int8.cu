// Rows as 8-bit integers with one 32-bit scale a row, for the products of gemm_int8.cu:
//     scale = max(max_c |y[c]| / 127, 2^-126),   code[c] = y[c] / scale rounded to the nearest whole number, ties to even,
// where y is a row as it is, the hidden units of a gated feed-forward (activation.cu's formula), or the RMSNorm
// (norm.cu's formula) of the residual stream after something was added to it:
//     s = x + add,   y = s / sqrt(mean(s^2) + eps) * w.
// A row of zeros has codes 0 and the smallest scale.  A row with a NaN or an infinity has codes 0 and the scale NaN, so that
// every product with it is NaN.  Sums, statistics and y are 32-bit; the codes are the only rounding to fewer bits.
//
// One block a row, the row in registers: read once with loads that are all in flight together, one meeting of the block
// (the norm's sum of squares and the largest |s w| are found in the same pass, since the factor 1 / rms is the
// same for the whole row), codes written once.  The largest absolute value is found on the bits: for numbers without
// a sign their order is that of the integers, and every NaN lies above infinity.
// Rows beyond what 1,024 threads hold are walked twice.
#include <type_traits>

#include "common.cuh"

namespace xrt {

constexpr float CODE_MAX = 127.0f, SMALLEST_SCALE = 1.17549435e-38f;
constexpr float ROUNDER = 12582912.0f;  // 1.5 * 2^23: v + ROUNDER has v, rounded to a whole number, in its low bits

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

// The codes of VEC values y * inverse; all zero with `broken`.
template <int VEC>
__device__ __forceinline__ void store_codes(int8_t* p, const float (&y)[VEC], float inverse, bool broken) {
  uint32_t bits[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) bits[i] = __float_as_uint(fmaf(y[i], inverse, ROUNDER));
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
  const T* x;
  __device__ __forceinline__ void wait() { pdl_wait(x); }
  template <int VEC> __device__ __forceinline__ void ahead(int, int, float (&)[VEC]) const {}
  template <int VEC, bool AGAIN> __device__ __forceinline__ void load(int row, int c, int width, float (&v)[VEC]) const {
    load_some<VEC>(x + (size_t)row * width + c, v);
  }
  template <int VEC, bool AGAIN>
  __device__ __forceinline__ void settle(int, int, int, const float (&)[VEC], float (&)[VEC], float&) const {}
};

template <typename T>
struct GatedRows {
  static constexpr bool NORMED = false;
  const T* gate_up;  // [rows, 2 * width]
  RowScale gate;
  __device__ __forceinline__ void wait() { pdl_wait(gate_up); }
  template <int VEC> __device__ __forceinline__ void ahead(int, int, float (&)[VEC]) const {}
  template <int VEC, bool AGAIN> __device__ __forceinline__ void load(int row, int c, int width, float (&v)[VEC]) const {
    const T* p = gate_up + (size_t)row * 2 * width + c;
    float u[VEC];
    load_some<VEC>(p, v);
    load_some<VEC>(p + width, u);
    // the fast exponential and division, as for a bfloat16 result: 8 bits are kept
    if (gate.gate_act == 1) {
      // 0.5 g (1 + tanh(z)) = g sigmoid(2 z), which loses nothing where tanh(z) is near -1: alone in its row, such a
      // value is the scale
      add_gate_biases<VEC, true>(v, u, c, gate);
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        v[i] = swish_for<__nv_bfloat16>(v[i], 1.5957691216057308f * fmaf(0.044715f * v[i], v[i], 1.0f)) * u[i];
    } else {
      gated_units<__nv_bfloat16, VEC, true>(v, u, c, gate);
    }
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
  const float* x;
  const TA* add;
  float* sum;  // may be x
  const TW* weight;
  float eps;
  __device__ __forceinline__ void wait() { pdl_wait(x, add); }
  // the weight does not depend on the step: it is on its way before the wait for the kernel before
  template <int VEC> __device__ __forceinline__ void ahead(int c, int width, float (&w)[VEC]) const {
    if (c < width) load_some<VEC>(weight + c, w);
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
  template <int VEC, bool AGAIN>
  __device__ __forceinline__ void settle(int row, int c, int width, const float (&w)[VEC], float (&v)[VEC], float& squares) const {
    if constexpr (ADDS && !AGAIN) store_some<VEC>(sum + (size_t)row * width + c, v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      squares = fmaf(v[i], v[i], squares);
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

// ITEMS pieces of VEC values a thread; 0: as many as the row takes, walked twice.
template <class ROWS, int VEC, int ITEMS>
__global__ void __launch_bounds__(1024)
quantize_int8_kernel(int8_t* __restrict__ codes, float* __restrict__ scales, ROWS rows, int width, int ld_codes) {
  __shared__ uint32_t most[32];
  __shared__ float sums[32];
  constexpr int KEPT = ITEMS > 0 ? ITEMS : 1;
  constexpr bool AHEAD = ITEMS > 0 && ITEMS * VEC <= 8;
  pdl_trigger();
  float w[KEPT][VEC], v[KEPT][VEC];
  const int stride = (int)blockDim.x * VEC;
  if constexpr (AHEAD) {
#pragma unroll
    for (int i = 0; i < KEPT; ++i) rows.template ahead<VEC>((int)threadIdx.x * VEC + i * stride, width, w[i]);
  }
  rows.wait();
  const int row = blockIdx.x;
  float squares = 0.f;
  uint32_t bits = 0;
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
#pragma unroll
        for (int j = 0; j < VEC; ++j) bits = max(bits, __float_as_uint(v[i][j]) & 0x7fffffffu);
      }
    }
  } else {
    for (int c = (int)threadIdx.x * VEC; c < width; c += stride) {
      rows.template ahead<VEC>(c, width, w[0]);
      rows.template load<VEC, false>(row, c, width, v[0]);
      rows.template settle<VEC, false>(row, c, width, w[0], v[0], squares);
#pragma unroll
      for (int j = 0; j < VEC; ++j) bits = max(bits, __float_as_uint(v[0][j]) & 0x7fffffffu);
    }
  }
  meet<ROWS::NORMED>(bits, squares, most, sums);
  float factor = 1.f;
  if constexpr (ROWS::NORMED) factor = 1.0f / sqrtf(squares / (float)width + rows.eps);
  const float largest = __uint_as_float(bits) * factor;
  const bool broken = !(largest <= 3.402823466e38f);
  const float scale = fmaxf(largest / CODE_MAX, SMALLEST_SCALE);
  const float inverse = 1.0f / scale;
  if (threadIdx.x == 0) scales[row] = broken ? __uint_as_float(0x7fc00000u) : scale;
  int8_t* dst = codes + (size_t)row * ld_codes;
  if constexpr (ITEMS > 0) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = (int)threadIdx.x * VEC + i * stride;
      if (c < width) {
        if constexpr (ROWS::NORMED) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) v[i][j] *= factor;
        }
        store_codes<VEC>(dst + c, v[i], inverse, broken);
      }
    }
  } else {
    for (int c = (int)threadIdx.x * VEC; c < width; c += stride) {
      rows.template ahead<VEC>(c, width, w[0]);
      rows.template load<VEC, true>(row, c, width, v[0]);
      rows.template settle<VEC, true>(row, c, width, w[0], v[0], squares);
      if constexpr (ROWS::NORMED) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[0][j] *= factor;
      }
      store_codes<VEC>(dst + c, v[0], inverse, broken);
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

template <class ROWS, int VEC>
int launch_quantize(int8_t* codes, float* scales, const ROWS& rows, int n, int width, int ld_codes, cudaStream_t stream) {
  auto launch = [&](auto kernel, int per) {
    const int threads = per > 0 ? ((width + per - 1) / per + 31) / 32 * 32 : 1024;
    launch_kernel(kernel, dim3(n), dim3(threads), 0, stream, codes, scales, rows, width, ld_codes);
    return launch_status();
  };
  if (width <= 8 * 1024) return launch(quantize_int8_kernel<ROWS, VEC, 8 / VEC>, 8);
  if (width <= 16 * 1024) return launch(quantize_int8_kernel<ROWS, VEC, 16 / VEC>, 16);
  if (width <= 32 * 1024) return launch(quantize_int8_kernel<ROWS, VEC, 32 / VEC>, 32);
  return launch(quantize_int8_kernel<ROWS, VEC, 0>, 0);
}

// Pieces of eight, four or one value at a time: the most that rows of this width and these addresses allow.
template <class ROWS>
int quantize(int8_t* codes, float* scales, const ROWS& rows, int n, int width, int ld_codes, cudaStream_t stream) {
  if (n < 0 || width <= 0 || ld_codes < width) return XRT_ERR_ARGUMENT;
  if (n == 0) return XRT_OK;
  auto whole = [&](int vec) {
    return width % vec == 0 && fits(rows, width, vec) && ((uintptr_t)codes | (uintptr_t)ld_codes) % vec == 0;
  };
  if (whole(8)) return launch_quantize<ROWS, 8>(codes, scales, rows, n, width, ld_codes, stream);
  if (whole(4)) return launch_quantize<ROWS, 4>(codes, scales, rows, n, width, ld_codes, stream);
  return launch_quantize<ROWS, 1>(codes, scales, rows, n, width, ld_codes, stream);
}

}  // namespace xrt

// codes: int8 [n, width] with rows ld_codes bytes apart; scales: float32 [n].

// x [n, width], float32 or bfloat16.
XRT_EXPORT int xrt_quantize_rows(void* codes, float* scales, const void* x, int n, int width, int ld_codes, int x_dtype,
                                 cudaStream_t stream) {
  XRT_DISPATCH_DTYPE(x_dtype, T, {
    return xrt::quantize((int8_t*)codes, scales, xrt::PlainRows<T>{(const T*)x}, n, width, ld_codes, stream);
  });
}

// gate_up [n, 2 * width], float32 or bfloat16; act and options as for xrt_swiglu.
XRT_EXPORT int xrt_swiglu_int8(void* codes, float* scales, const void* gate_up, int n, int width, int ld_codes, int in_dtype,
                               int act, const xrt::GateOptions* options, cudaStream_t stream) {
  if (act < 0 || act > 2) return XRT_ERR_ARGUMENT;
  xrt::RowScale gate;
  gate.gate_act = act;
  if (!xrt::take_gate_options(options, 2, width, gate)) return XRT_ERR_ARGUMENT;
  XRT_DISPATCH_DTYPE(in_dtype, T, {
    return xrt::quantize((int8_t*)codes, scales, xrt::GatedRows<T>{(const T*)gate_up, gate}, n, width, ld_codes, stream);
  });
}

// x float32 [n, width]; add (may be null) [n, width], float32 or bfloat16; with it sum [n, width] gets x + add (sum may be x).
XRT_EXPORT int xrt_rmsnorm_int8(void* codes, float* scales, const float* x, const void* add, float* sum, const void* weight,
                                int n, int width, int ld_codes, float eps, int add_dtype, int w_dtype, cudaStream_t stream) {
  if (add != nullptr && sum == nullptr) return XRT_ERR_ARGUMENT;
  XRT_DISPATCH_DTYPE(w_dtype, TW, {
    if (add == nullptr) {
      const xrt::NormedRows<xrt::Nothing, TW> rows{x, nullptr, nullptr, (const TW*)weight, eps};
      return xrt::quantize((int8_t*)codes, scales, rows, n, width, ld_codes, stream);
    }
    XRT_DISPATCH_DTYPE(add_dtype, TA, {
      const xrt::NormedRows<TA, TW> rows{x, (const TA*)add, sum, (const TW*)weight, eps};
      return xrt::quantize((int8_t*)codes, scales, rows, n, width, ld_codes, stream);
    });
  });
}
