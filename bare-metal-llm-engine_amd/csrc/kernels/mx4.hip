// mx4.hip -- microscaled 4-bit floating point (OCP Microscaling Formats v1.0,
// MXFP4): quantisation of rows, and the values back (mx4_linear.hip has the linear
// layers on such weights).
//
// Format: 32 values along a row share a scale byte s (E8M0: 2^(s - 127), 255 a
// NaN); each value is a 4-bit E2M1 code, sign and one of 0, 0.5, 1, 1.5, 2, 3,
// 4, 6. A row of `cols` values is ceil(cols / 32) blocks: 16 bytes of codes a
// block, the even element in the low nibble, and one scale byte; the last block
// is filled with zeros, so every row's codes begin on 16 bytes whatever cols is.
#include "launch.hpp"

#include <algorithm>

namespace eng {
namespace {

typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kBlock = 32;  // values that share a scale

// ------------------------------------------------------------- quantisation

// Eight values from p (n of them in the row; the others are zero).
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* __restrict__ p, long long n, float (&v)[8]) {
  if constexpr (VEC) {
    typedef T V __attribute__((ext_vector_type(16 / sizeof(T))));
    constexpr int W = 16 / sizeof(T);
    if (n >= 8) {
#pragma unroll
      for (int i = 0; i < 8; i += W) {
        const V x = __builtin_nontemporal_load(reinterpret_cast<const V*>(p + i));
#pragma unroll
        for (int e = 0; e < W; ++e) v[i + e] = static_cast<float>(x[e]);
      }
      return;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = e < n ? static_cast<float>(p[e]) : 0.0f;
}

// Four lanes share a block of 32, eight values each. The block's exponent is
// the exponent field of its largest magnitude less 2 (6 is the largest E2M1
// value, 4 <= amax / 2^e < 8), and v_cvt_scalef32_pk_fp4_f32 divides by the
// scale, rounds to nearest even and saturates at 6. A block with a NaN or an
// infinity gets the NaN scale and zero codes. Memory bound: each value is read
// once, in 16-byte loads where the rows allow (VEC): 11008 x 4096 fp16, 114 MB, 21.7 us,
// 5.3 TB/s (a copy of 1 GiB runs at 5.2); fp32, 204 MB, 38.1 us, 5.4 TB/s. Other rows go
// value by value: 11008 x 4095 fp16 54.5 us, fp32 80.0.
template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void mx4_quantize_kernel(
    const T* __restrict__ src, unsigned* __restrict__ codes, unsigned char* __restrict__ scales,
    unsigned long long items, unsigned per_row, long long cols) {
  // item = (row, eighth e of the row): values 8 e .. + 7, one word of codes
  const unsigned long long stride = static_cast<unsigned long long>(gridDim.x) * kThreads;
  for (unsigned long long i = static_cast<unsigned long long>(blockIdx.x) * kThreads + threadIdx.x;
       i < items; i += stride) {
    unsigned long long row;
    unsigned e;
    if (items <= 0xffffffffull) {
      row = static_cast<unsigned>(i) / per_row;
      e = static_cast<unsigned>(i) - static_cast<unsigned>(row) * per_row;
    } else {
      row = i / per_row;
      e = static_cast<unsigned>(i - row * per_row);
    }
    const long long c = 8ll * e;
    float v[8];
    load8<T, VEC>(src + row * cols + (c < cols ? c : 0), c < cols ? cols - c : 0, v);
    unsigned top = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(v[k]) & 0x7fffffffu);
    // the block's four lanes (items come in groups of four: per_row is a
    // multiple of 4, so a quad of lanes is in or out of the loop together)
    top = max(top, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(top), 0xB1, 0xF, 0xF, false)));
    top = max(top, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(top), 0x4E, 0xF, 0xF, false)));
    const unsigned ex = top >> 23;
    const unsigned s = ex == 255 ? 255u : ex > 2 ? ex - 2 : 0u;
    unsigned w = 0;
#if defined(__HIP_DEVICE_COMPILE__)
    if (s != 255) {
      const float scale = __uint_as_float(s << 23);  // only its exponent field is read
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
    }
#endif
    codes[i] = w;
    if ((e & 3) == 0) scales[i >> 2] = static_cast<unsigned char>(s);
  }
}

// The values back: one word of codes, eight values a thread. Memory bound: 11008 x 4096
// to fp16, 114 MB, 18.1 us over three sets of buffers (the codes partly from the 256 MB
// cache), 24.4 over five; to fp32, 204 MB, 48.9 us over five. Rows that are not whole 16
// bytes go value by value: 11008 x 4095 to fp16 65.3 us, to fp32 116.5.
template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void mx4_dequantize_kernel(
    const unsigned* __restrict__ codes, const unsigned char* __restrict__ scales,
    T* __restrict__ dst, unsigned long long items, unsigned per_row, long long cols) {
  const unsigned long long stride = static_cast<unsigned long long>(gridDim.x) * kThreads;
  for (unsigned long long i = static_cast<unsigned long long>(blockIdx.x) * kThreads + threadIdx.x;
       i < items; i += stride) {
    unsigned long long row;
    unsigned e;
    if (items <= 0xffffffffull) {
      row = static_cast<unsigned>(i) / per_row;
      e = static_cast<unsigned>(i) - static_cast<unsigned>(row) * per_row;
    } else {
      row = i / per_row;
      e = static_cast<unsigned>(i - row * per_row);
    }
    const long long c = 8ll * e;
    if (c >= cols) continue;
    [[maybe_unused]] const unsigned w = codes[i];
    T v[8];
#if defined(__HIP_DEVICE_COMPILE__)
    const float scale = __uint_as_float(static_cast<unsigned>(scales[i >> 2]) << 23);
    auto two = [&](auto sel) {
      constexpr int B = decltype(sel)::value;
      if constexpr (sizeof(T) == 2) {
        const halfx2 p = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, B);
        v[2 * B] = p[0];
        v[2 * B + 1] = p[1];
      } else {
        const floatx2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, B);
        v[2 * B] = p[0];
        v[2 * B + 1] = p[1];
      }
    };
    two(std::integral_constant<int, 0>{});
    two(std::integral_constant<int, 1>{});
    two(std::integral_constant<int, 2>{});
    two(std::integral_constant<int, 3>{});
#endif
    T* out = dst + row * cols + c;
    if (VEC && c + 8 <= cols) {
      typedef T V __attribute__((ext_vector_type(16 / sizeof(T))));
      constexpr int W = 16 / sizeof(T);
#pragma unroll
      for (int k = 0; k < 8; k += W) {
        V x;
#pragma unroll
        for (int q = 0; q < W; ++q) x[q] = v[k + q];
        *reinterpret_cast<V*>(out + k) = x;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (c + k < cols) out[k] = v[k];
    }
  }
}

void check_pack(const char* what, const void* a, const void* codes, const void* scales, int64_t rows,
                int64_t cols) {
  const std::string name(what);
  ENG_CHECK(rows >= 0 && cols >= 0, name + ": negative dimension");
  if (rows == 0 || cols == 0) return;
  ENG_CHECK(a != nullptr && codes != nullptr && scales != nullptr, name + ": null device pointer");
  ENG_CHECK(aligned_to(codes, 16), name + ": codes must be 16-byte aligned");
  ENG_CHECK(cols <= (1ll << 34) && rows <= (1ll << 60) / cols, name + ": dimensions too large");
}

unsigned pack_grid(unsigned long long items) {
  const unsigned long long most = 64ull * device_cu_count();
  return static_cast<unsigned>(std::max(1ull, std::min((items + kThreads - 1) / kThreads, most)));
}

template <typename T>
void quantize_any(const T* src, std::uint8_t* codes, std::uint8_t* scales, int64_t rows,
                  int64_t cols, eng_stream stream) {
  check_pack("mx4_quantize", src, codes, scales, rows, cols);
  if (rows == 0 || cols == 0) return;
  const unsigned per_row = static_cast<unsigned>((cols + kBlock - 1) / kBlock * 4);
  const unsigned long long items = static_cast<unsigned long long>(rows) * per_row;
  const bool vec = aligned_to(src, 16) && cols * sizeof(T) % 16 == 0;
  auto go = [&](auto kernel) {
    kernel<<<pack_grid(items), kThreads, 0, as_stream(stream)>>>(
        src, reinterpret_cast<unsigned*>(codes), scales, items, per_row, cols);
  };
  if (vec) go(mx4_quantize_kernel<T, true>);
  else go(mx4_quantize_kernel<T, false>);
  ENG_LAUNCH_CHECK();
}

template <typename T>
void dequantize_any(const std::uint8_t* codes, const std::uint8_t* scales, T* dst, int64_t rows,
                    int64_t cols, eng_stream stream) {
  check_pack("mx4_dequantize", dst, codes, scales, rows, cols);
  if (rows == 0 || cols == 0) return;
  const unsigned per_row = static_cast<unsigned>((cols + kBlock - 1) / kBlock * 4);
  const unsigned long long items = static_cast<unsigned long long>(rows) * per_row;
  const bool vec = aligned_to(dst, 16) && cols * sizeof(T) % 16 == 0;
  auto go = [&](auto kernel) {
    kernel<<<pack_grid(items), kThreads, 0, as_stream(stream)>>>(
        reinterpret_cast<const unsigned*>(codes), scales, dst, items, per_row, cols);
  };
  if (vec) go(mx4_dequantize_kernel<T, true>);
  else go(mx4_dequantize_kernel<T, false>);
  ENG_LAUNCH_CHECK();
}

}  // namespace
}  // namespace eng

extern "C" {

int eng_mx4_quantize_f32(const float* src, uint8_t* codes, uint8_t* scales, int64_t rows,
                         int64_t cols, eng_stream stream) {
  return eng::guarded([&] { eng::quantize_any(src, codes, scales, rows, cols, stream); });
}

int eng_mx4_quantize_f16(const eng_half* src, uint8_t* codes, uint8_t* scales, int64_t rows,
                         int64_t cols, eng_stream stream) {
  return eng::guarded([&] {
    eng::quantize_any(reinterpret_cast<const _Float16*>(src), codes, scales, rows, cols, stream);
  });
}

int eng_mx4_dequantize_f32(const uint8_t* codes, const uint8_t* scales, float* dst, int64_t rows,
                           int64_t cols, eng_stream stream) {
  return eng::guarded([&] { eng::dequantize_any(codes, scales, dst, rows, cols, stream); });
}

int eng_mx4_dequantize_f16(const uint8_t* codes, const uint8_t* scales, eng_half* dst,
                           int64_t rows, int64_t cols, eng_stream stream) {
  return eng::guarded([&] {
    eng::dequantize_any(codes, scales, reinterpret_cast<_Float16*>(dst), rows, cols, stream);
  });
}

}  // extern "C"
