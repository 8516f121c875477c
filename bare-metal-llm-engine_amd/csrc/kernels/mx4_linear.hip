// mx4_linear.hip -- linear layers on MXFP4 weights (the format of mx4.hip):
// Y[M x N] = s_m (X[m] * gamma) . W^T, W [N x K] as codes and scale bytes, fp32
// X and Y, s_m = 1 / sqrt(mean X[m]^2 + eps) or 1.
//
// Arithmetic. An E2M1 value times its power-of-two scale is exact in bf16 (two
// significant bits, bf16's exponent is fp32's), and an fp32 activation is the
// exact sum of three bf16 terms, each the truncation of what the earlier ones
// leave (bits below 2^-133 aside). Every product on v_mfma_f32_16x16x32_bf16 is
// then exact and the sums are fp32: the arithmetic of the fp16-weight layers.
// v_cvt_scalef32_pk_bf16_fp4 makes two weights, scale included, in one
// instruction; a NaN scale makes NaNs of the whole block.
//
// Operand layout. Lane (i, g) = (lane % 16, lane / 16) of the instruction holds
// row (column) i and 8 values of k, group g. K goes by chunks of 128: lane group
// g takes the 32-block g of the chunk, and step j = 0 .. 3 its values 8 j .. + 7,
// so a lane's part of the weights is one 16-byte load (word j feeds step j) and
// one scale byte, and nothing is moved between lanes.
//
//   M <= 4            mx4_decode_kernel: the three terms of row m are rows 4 m ..
//                     4 m + 2 of one A operand, split once per workgroup into LDS
//   5 <= M <= 32      mx4_rows_kernel: a workgroup's waves split K, X split in
//                     registers
//   M > 32            mx4_gemm_kernel on planes made by mx4_planes_kernel
#include "device_sync.hpp"
#include "gemv_kernels.hpp"
#include "launch.hpp"

#include <algorithm>
#include <type_traits>

namespace eng {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned uintx2 __attribute__((ext_vector_type(2)));
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));

[[maybe_unused]] constexpr int kRsrcWord3 = 0x00020000;  // buffer descriptor: raw, 32-bit elements
constexpr int kChunk = 128;  // k of a chunk: one 16-byte weight load per lane

struct Mx4Args {
  const float* x;
  const float* gamma;  // rms only, may be null
  const unsigned char* codes;
  const unsigned char* scales;
  float* y;
  long long M, N, K;
  bool rms;
  float eps;
};

// The top 16 bits of a and b as one word of two bf16 (b in the upper half).
__device__ __forceinline__ unsigned pack_hi(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

// v as three bf16 terms, left in the top halves of t[0..2]. An infinity is its
// own first term with zeros after it; a NaN stays a NaN.
__device__ __forceinline__ void split3(float v, float (&t)[3]) {
  const unsigned b = __float_as_uint(v);
  const bool fin = (b & 0x7f800000u) != 0x7f800000u;
  const float h = __uint_as_float(b & 0xffff0000u);
  const float r = fin ? v - h : 0.0f;
  const float m = __uint_as_float(__float_as_uint(r) & 0xffff0000u);
  t[0] = v != v ? __uint_as_float(b | 0x00400000u) : h;
  t[1] = m;
  t[2] = r - m;
}

// The eight bf16 weights of one code word.
__device__ __forceinline__ bf16x8 weights8(unsigned w, float scale) {
  bf16x8 r = {};
#if defined(__HIP_DEVICE_COMPILE__)
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
  r[0] = a[0], r[1] = a[1], r[2] = b[0], r[3] = b[1];
  r[4] = c[0], r[5] = c[1], r[6] = d[0], r[7] = d[1];
#endif
  return r;
}

__device__ __forceinline__ float scale_of(unsigned byte) { return __uint_as_float(byte << 23); }

__device__ __forceinline__ floatx4 mfma(bf16x8 a, bf16x8 b, floatx4 c) {
#if defined(__HIP_DEVICE_COMPILE__)
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
#endif
  return c;
}

// ---------------------------------------------------------------- 1 to 4 rows
//
// A workgroup of 8 waves owns 16 weight rows; the waves split K by chunks. X is
// split into LDS once per workgroup (MR rows x 3 terms, a segment of `seg` k at
// a time); the first four chunks of weights are already on their way while it
// is. Terms sit 16 bytes apart modulo the banks' 256, so the reads of a step
// (3 MR rows x 4 groups) spread over the banks.
constexpr int kDecodeWaves = 8;
constexpr int kDecodeRing = 4;  // chunks of weights in flight per wave
constexpr int kDecodeLds = 120 * 1024;

template <int MR, bool RMS, bool VEC>
__global__ __launch_bounds__(64 * kDecodeWaves) void mx4_decode_kernel(
    const float* __restrict__ x, const float* __restrict__ gamma,
    const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales,
    float* __restrict__ y, long long N, int K, int nb, int seg, float eps) {
  constexpr int THREADS = 64 * kDecodeWaves;
  extern __shared__ __attribute__((aligned(16))) unsigned short planes[];  // [MR][3][seg + 8]
  __shared__ float red[kDecodeWaves][MR][16];
  __shared__ float red_ss[kDecodeWaves][MR];
  const int pitch = seg + 8;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15;
  const int g = lane >> 4;
  const long long n0 = 16ll * blockIdx.x;
  const long long n = std::min(n0 + i, N - 1);
  const unsigned char* crow = codes + n * (16ll * nb);
  const unsigned char* srow = scales + n * nb;
  // A row 4 m + p: term p of x row m; p == 3 and m >= MR are zero
  const int am = i >> 2;
  const int ap = i & 3;
  const bool a_on = am < MR && ap < 3;
  const unsigned short* abase = planes + (a_on ? (am * 3 + ap) * pitch : 0) + 32 * g;

  floatx4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  float ss[MR];
#pragma unroll
  for (int m = 0; m < MR; ++m) ss[m] = 0.0f;

  for (int k0 = 0; k0 < K; k0 += seg) {
    const int klen = min(seg, K - k0);
    const int chunks = (klen + kChunk - 1) / kChunk;
    const int c0 = chunks * wave / kDecodeWaves;
    const int c1 = chunks * (wave + 1) / kDecodeWaves;
    const int b0 = k0 / 32 + g;
    uintx4 w[kDecodeRing];
    unsigned s[kDecodeRing];
    auto load = [&](int r, int c) {
      const int b = min(b0 + 4 * min(c, chunks - 1), nb - 1);
      w[r] = __builtin_nontemporal_load(reinterpret_cast<const uintx4*>(crow + 16ll * b));
      s[r] = srow[b];
    };
#pragma unroll
    for (int r = 0; r < kDecodeRing; ++r) load(r, c0 + r);

    if (k0 > 0) __syncthreads();  // the last segment's planes have been read
    // whole chunks are staged: zeros past K
    for (int q = 4 * tid; q < chunks * kChunk; q += 4 * THREADS) {
      const int k = k0 + q;
      float gm[4] = {1.0f, 1.0f, 1.0f, 1.0f};
      if constexpr (RMS) {
        if (gamma != nullptr) {
#pragma unroll
          for (int e = 0; e < 4; ++e) gm[e] = gamma[min(k + e, K - 1)];
        }
      }
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        float v[4];
        const float* xp = x + static_cast<long long>(m) * K + k;
        if constexpr (VEC) {
          floatx4 t = {0.0f, 0.0f, 0.0f, 0.0f};
          if (k < K) t = *reinterpret_cast<const floatx4*>(xp);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = t[e];
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = k + e < K ? xp[e] : 0.0f;
        }
        float t[4][3];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (RMS) {
            ss[m] = fmaf(v[e], v[e], ss[m]);
            v[e] = k + e < K ? v[e] * gm[e] : 0.0f;
          }
          split3(v[e], t[e]);
        }
#pragma unroll
        for (int p = 0; p < 3; ++p)
          *reinterpret_cast<uintx2*>(planes + (m * 3 + p) * pitch + q) =
              uintx2{pack_hi(t[0][p], t[1][p]), pack_hi(t[2][p], t[3][p])};
      }
    }
    __syncthreads();

    for (int c = c0; c < c1; c += kDecodeRing) {
#pragma unroll
      for (int r = 0; r < kDecodeRing; ++r) {
        if (c + r < c1) {
          const float sc = scale_of(s[r]);
          const unsigned short* ap0 = abase + (c + r) * kChunk;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            bf16x8 a = *reinterpret_cast<const bf16x8*>(ap0 + 8 * j);
            if (!a_on) a = bf16x8{};
            acc = mfma(a, weights8(w[r][j], sc), acc);
          }
          if (c + r + kDecodeRing < c1) load(r, c + r + kDecodeRing);
        }
      }
    }
  }

  // lane (i, g): element r of acc is A row 4 g + r, weight row i
  if (g < MR) red[wave][g][i] = (acc[0] + acc[1]) + acc[2];
  if constexpr (RMS) {
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      const float t = gemv::wave_sum(ss[m]);
      if (lane == 0) red_ss[wave][m] = t;
    }
  }
  __syncthreads();
  if (tid < 16 * MR) {
    const int m = tid >> 4;
    const int col = tid & 15;
    float v = red[0][m][col];
#pragma unroll
    for (int q = 1; q < kDecodeWaves; ++q) v += red[q][m][col];
    if constexpr (RMS) {
      float t = red_ss[0][m];
#pragma unroll
      for (int q = 1; q < kDecodeWaves; ++q) t += red_ss[q][m];
      v *= 1.0f / sqrtf(t / static_cast<float>(K) + eps);
    }
    if (n0 + col < N) y[m * N + n0 + col] = v;
  }
}

template <int MR>
void run_decode(const Mx4Args& a, hipStream_t stream) {
  const long long grid = (a.N + 15) / 16;
  ENG_CHECK(grid <= 0x7fffffffLL, "linear_mx4w: grid too large for one launch");
  const int K = static_cast<int>(a.K);
  const int nb = (K + 31) / 32;
  const bool vec = a.K % 4 == 0 && aligned_to(a.x, 16);
  const int cap = (kDecodeLds / (6 * MR) - 8) / kChunk * kChunk;
  const int seg = std::min((K + kChunk - 1) / kChunk * kChunk, cap);
  const std::size_t lds = static_cast<std::size_t>(6) * MR * (seg + 8);
  auto go = [&](auto rms, auto v) {
    constexpr bool R = decltype(rms)::value;
    constexpr bool V = decltype(v)::value;
    static std::atomic<bool> done[64];
    allow_staged_lds(reinterpret_cast<const void*>(mx4_decode_kernel<MR, R, V>), done, lds);
    mx4_decode_kernel<MR, R, V><<<static_cast<unsigned>(grid), 64 * kDecodeWaves, lds, stream>>>(
        a.x, a.gamma, a.codes, a.scales, a.y, a.N, K, nb, seg, a.eps);
  };
  using T = std::true_type;
  using F = std::false_type;
  if (a.rms) vec ? go(T{}, T{}) : go(T{}, F{});
  else vec ? go(F{}, T{}) : go(F{}, F{});
  ENG_LAUNCH_CHECK();
}

// --------------------------------------------------------------- 5 to 32 rows
//
// A workgroup of 8 waves owns 16 NT weight rows and all of K, which the waves
// split by chunks. Each wave loads its own part of X (as fp32, straight into the
// operand's lanes) and splits it in registers, MB blocks of 16 rows.
constexpr int kRowsWaves = 8;

template <int MB, int NT, bool RMS, bool VEC>
__global__ __launch_bounds__(64 * kRowsWaves) void mx4_rows_kernel(
    const float* __restrict__ x, const float* __restrict__ gamma,
    const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales,
    float* __restrict__ y, int M, long long N, int K, int nb, float eps) {
  __shared__ float red[kRowsWaves][MB * NT][256];
  __shared__ float red_ss[kRowsWaves][16 * MB];
  __shared__ float row_scale[16 * MB];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15;
  const int g = lane >> 4;
  const long long n0 = 16ll * NT * blockIdx.x;
  const unsigned char* crow[NT];
  const unsigned char* srow[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const long long n = std::min(n0 + 16 * t + i, N - 1);
    crow[t] = codes + n * (16ll * nb);
    srow[t] = scales + n * nb;
  }
  const float* xrow[MB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
    xrow[mb] = x + static_cast<long long>(min(16 * mb + i, M - 1)) * K;
  const int chunks = (K + kChunk - 1) / kChunk;
  const int c0 = chunks * wave / kRowsWaves;
  const int c1 = chunks * (wave + 1) / kRowsWaves;

  floatx4 acc[MB][NT];
  float ss[MB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    ss[mb] = 0.0f;
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[mb][t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  uintx4 w[2][NT];
  unsigned s[2][NT];
  auto load_w = [&](auto r, int c) {
    constexpr int R = decltype(r)::value;
    const int b = min(4 * c + g, nb - 1);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      w[R][t] = __builtin_nontemporal_load(reinterpret_cast<const uintx4*>(crow[t] + 16ll * b));
      s[R][t] = srow[t][b];
    }
  };
  auto load4 = [&](const float* p, int k) {
    floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (VEC) {
      if (k < K) v = *reinterpret_cast<const floatx4*>(p + k);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = k + e < K ? p[k + e] : 0.0f;
    }
    return v;
  };
  auto compute = [&](auto r, int c) {
    constexpr int R = decltype(r)::value;
    floatx4 xv[4][MB][2];
    floatx4 gv[RMS ? 4 : 1][2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = c * kChunk + 32 * g + 8 * j;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        xv[j][mb][0] = load4(xrow[mb], k);
        xv[j][mb][1] = load4(xrow[mb], k + 4);
      }
      if constexpr (RMS) {
        if (gamma != nullptr) {
          gv[j][0] = load4(gamma, k);
          gv[j][1] = load4(gamma, k + 4);
        } else {
          gv[j][0] = gv[j][1] = floatx4{1.0f, 1.0f, 1.0f, 1.0f};
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bf16x8 b[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) b[t] = weights8(w[R][t][j], scale_of(s[R][t]));
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        float t3[8][3];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float v = xv[j][mb][e >> 2][e & 3];
          if constexpr (RMS) {
            ss[mb] = fmaf(v, v, ss[mb]);
            v *= gv[j][e >> 2][e & 3];
          }
          split3(v, t3[e]);
        }
#pragma unroll
        for (int p = 2; p >= 0; --p) {
          const uintx4 u = {pack_hi(t3[0][p], t3[1][p]), pack_hi(t3[2][p], t3[3][p]),
                            pack_hi(t3[4][p], t3[5][p]), pack_hi(t3[6][p], t3[7][p])};
          const bf16x8 av = __builtin_bit_cast(bf16x8, u);
#pragma unroll
          for (int t = 0; t < NT; ++t) acc[mb][t] = mfma(av, b[t], acc[mb][t]);
        }
      }
    }
  };
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  if (c0 < c1) load_w(I0{}, c0);
  for (int c = c0; c < c1; c += 2) {
    if (c + 1 < c1) load_w(I1{}, c + 1);
    compute(I0{}, c);
    if (c + 1 < c1) {
      if (c + 2 < c1) load_w(I0{}, c + 2);
      compute(I1{}, c + 1);
    }
  }

#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) red[wave][mb * NT + t][(4 * g + r) * 16 + i] = acc[mb][t][r];
    if constexpr (RMS) {
      float v = ss[mb];
      v += __shfl_xor(v, 16);
      v += __shfl_xor(v, 32);
      if (g == 0) red_ss[wave][16 * mb + i] = v;
    }
  }
  __syncthreads();
  if (tid < 16 * MB) {
    float sc = 1.0f;
    if constexpr (RMS) {
      float t = red_ss[0][tid];
#pragma unroll
      for (int q = 1; q < kRowsWaves; ++q) t += red_ss[q][tid];
      sc = 1.0f / sqrtf(t / static_cast<float>(K) + eps);
    }
    row_scale[tid] = sc;
  }
  __syncthreads();
  for (int q = tid; q < MB * NT * 256; q += 64 * kRowsWaves) {
    const int blk = q >> 8;
    const int row = 16 * (blk / NT) + ((q & 255) >> 4);
    const long long col = n0 + 16 * (blk % NT) + (q & 15);
    float v = red[0][blk][q & 255];
#pragma unroll
    for (int u = 1; u < kRowsWaves; ++u) v += red[u][blk][q & 255];
    if (row < M && col < N) y[row * N + col] = v * row_scale[row];
  }
}

template <int MB, int NT>
void run_rows(const Mx4Args& a, hipStream_t stream) {
  const long long grid = (a.N + 16 * NT - 1) / (16 * NT);
  ENG_CHECK(grid <= 0x7fffffffLL, "linear_mx4w: grid too large for one launch");
  const int K = static_cast<int>(a.K);
  const int nb = (K + 31) / 32;
  const bool vec = a.K % 4 == 0 && aligned_to(a.x, 16) && aligned_to(a.gamma, 16);
  auto go = [&](auto rms, auto v) {
    mx4_rows_kernel<MB, NT, decltype(rms)::value, decltype(v)::value>
        <<<static_cast<unsigned>(grid), 64 * kRowsWaves, 0, stream>>>(
            a.x, a.gamma, a.codes, a.scales, a.y, static_cast<int>(a.M), a.N, K, nb, a.eps);
  };
  using T = std::true_type;
  using F = std::false_type;
  if (a.rms) vec ? go(T{}, T{}) : go(T{}, F{});
  else vec ? go(F{}, T{}) : go(F{}, F{});
  ENG_LAUNCH_CHECK();
}

// -------------------------------------------------------------- 33 rows and up
//
// X split into planes first: 16 rows x 32 k of one term is a fragment, 1 KiB in the
// order the matrix instruction's lanes take it (lane (i, g): row i, the eight k of
// step j in its group's 32-block), fragments [M / 16][chunk][step j][term]. A tile's
// planes are then runs of whole KiB for the direct loads, and a fragment is one
// conflict-free 16-byte LDS read per lane. Rows past M and k past K are zeros.
// Beside them the sums of squares of each row over kPlaneK columns at a time.
constexpr int kPlaneK = 512;  // columns of a workgroup: a chunk per wave

template <bool RMS, bool VEC>
__global__ __launch_bounds__(256) void mx4_planes_kernel(const float* __restrict__ x,
                                                         const float* __restrict__ gamma,
                                                         unsigned short* __restrict__ planes,
                                                         float* __restrict__ part, long long M,
                                                         int K, int chunks) {
  __shared__ float red[4][16];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15;
  const int g = lane >> 4;
  const long long row = 16ll * blockIdx.x + i;
  const int c = blockIdx.y * (kPlaneK / kChunk) + wave;
  float ss = 0.0f;
  if (c < chunks) {
    const float* xr = x + (row < M ? row : 0) * K;
    auto load4 = [&](const float* p, int k) {
      floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
      if constexpr (VEC) {
        if (k < K) v = *reinterpret_cast<const floatx4*>(p + k);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = k + e < K ? p[k + e] : 0.0f;
      }
      return v;
    };
    floatx4 v[4][2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = c * kChunk + 32 * g + 8 * j;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        v[j][h] = load4(xr, k + 4 * h);
        if (row >= M) v[j][h] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (RMS) {
#pragma unroll
          for (int e = 0; e < 4; ++e) ss = fmaf(v[j][h][e], v[j][h][e], ss);
          if (gamma != nullptr) {
            const floatx4 gm = load4(gamma, k + 4 * h);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j][h][e] *= gm[e];
          }
        }
      }
    }
    uintx4* dst = reinterpret_cast<uintx4*>(planes) +
                  ((static_cast<long long>(blockIdx.x) * chunks + c) * 12) * 64 + lane;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float t[8][3];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float f = v[j][e >> 2][e & 3];
        split3(f, t[e]);
      }
#pragma unroll
      for (int p = 0; p < 3; ++p)
        dst[(3 * j + p) * 64] = uintx4{pack_hi(t[0][p], t[1][p]), pack_hi(t[2][p], t[3][p]),
                                       pack_hi(t[4][p], t[5][p]), pack_hi(t[6][p], t[7][p])};
    }
  }
  if constexpr (RMS) {
    ss += __shfl_xor(ss, 16);
    ss += __shfl_xor(ss, 32);
    if (g == 0) red[wave][i] = ss;
    __syncthreads();
    if (tid < 16 && row < M)
      part[row * gridDim.y + blockIdx.y] = (red[0][i] + red[1][i]) + (red[2][i] + red[3][i]);
  }
}

// C tiles of 16 BMB x 64 NT on BMB waves: BMB / 4 of them along M, 4 along N, each 64
// rows x 16 NT columns. A step is one j of a chunk (32 k): its 3 BMB plane fragments
// sit in one of four LDS stages, loaded three steps ahead by direct loads (three a
// wave); the weights of a chunk, which only one row of waves uses, come straight
// into registers a chunk ahead (4-bit: 16 NT bytes a lane and chunk) and are
// converted as their step begins.
template <int BMB, int NT, bool RMS>
__global__ __launch_bounds__(64 * BMB, 2) void mx4_gemm_kernel(
    const unsigned short* __restrict__ planes, const float* __restrict__ part,
    const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales,
    float* __restrict__ y, long long M, long long N, int K, int nb, int tiles_m, int mblocks,
    int groups, float eps) {
  static_assert(BMB == 8 || BMB == 4, "64- or 128-row tiles");
  constexpr int STAGE = BMB * 3 * 512;  // bf16 of a stage
  __shared__ __attribute__((aligned(1024))) unsigned short st0[STAGE];
  __shared__ __attribute__((aligned(1024))) unsigned short st1[STAGE];
  __shared__ __attribute__((aligned(1024))) unsigned short st2[STAGE];
  __shared__ __attribute__((aligned(1024))) unsigned short st3[STAGE];
  __shared__ float row_scale[16 * BMB];
  auto stage = [&](auto j) -> unsigned short* {
    if constexpr (decltype(j)::value == 0) return st0;
    else if constexpr (decltype(j)::value == 1) return st1;
    else if constexpr (decltype(j)::value == 2) return st2;
    else return st3;
  };

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15;
  const int g = lane >> 4;
  const int wm = wave >> 2;
  const int wn = wave & 3;
  const long long logical = gemv::xcd_contiguous(blockIdx.x, gridDim.x);
  const int tm = static_cast<int>(logical % tiles_m);
  const long long n0 = (logical / tiles_m) * (64 * NT);
  const long long m0 = 16ll * BMB * tm;
  const int chunks = (K + kChunk - 1) / kChunk;

  if constexpr (RMS) {
    if (tid < 16 * BMB) {
      const long long row = std::min(m0 + tid, M - 1);
      float t = 0.0f;
      for (int q = 0; q < groups; ++q) t += part[row * groups + q];
      row_scale[tid] = 1.0f / sqrtf(t / static_cast<float>(K) + eps);
    }
  }

  // This wave stages the three planes of m-block `wave` (the last one again past
  // the matrix): 3 KiB a step, contiguous over all steps.
  const long long mb_src = std::min<long long>(static_cast<long long>(BMB) * tm + wave, mblocks - 1);
  [[maybe_unused]] const unsigned short* a_src = planes + mb_src * chunks * (12 * 512);
  // Weight rows of this wave; rows past N read as zeros.
  const long long nw = n0 + 16 * NT * wn;  // (uniform)
  [[maybe_unused]] const long long rows_left = std::max(std::min<long long>(N - nw, 16 * NT), 0ll);
#if defined(__HIP_DEVICE_COMPILE__)
  const auto ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned short*>(a_src), 0,
                                                    chunks * 12 * 1024, kRsrcWord3);
  const auto rc = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<unsigned char*>(codes + (rows_left > 0 ? nw : 0) * 16 * nb), 0,
      static_cast<int>(rows_left * 16 * nb), kRsrcWord3);
  const auto rs = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<unsigned char*>(scales + (rows_left > 0 ? nw : 0) * nb), 0,
      static_cast<int>(rows_left * nb), kRsrcWord3);
#endif
  [[maybe_unused]] const int steps = 4 * chunks;
  auto fetch_a = [&](unsigned short* dst, int step) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int so = min(step, steps - 1) * 3072;
    unsigned short* d = dst + wave * (3 * 512);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, d, 16, lane * 16, so, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, d + 512, 16, lane * 16, so + 1024, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, d + 1024, 16, lane * 16, so + 2048, 0, 0);
#endif
  };
  struct W {
    uintx4 w[NT];
    unsigned s[NT];
  };
  auto load_w = [&](W& x, int c) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int b = min(4 * min(c, chunks - 1) + g, nb - 1);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      x.w[t] = __builtin_amdgcn_raw_buffer_load_b128(rc, ((16 * t + i) * nb + b) * 16, 0, 0);
      x.s[t] = __builtin_amdgcn_raw_buffer_load_b8(rs, (16 * t + i) * nb + b, 0, 0);
    }
#endif
  };

  floatx4 acc[4][NT];
#pragma unroll
  for (int mb = 0; mb < 4; ++mb)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[mb][t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

  // Step (c, j): its planes have landed and every wave is past the step before;
  // the weights of the next chunk (at j == 0), then the planes three steps on go
  // out, into the stage read last. Younger loads that the wait leaves in flight:
  // two steps' planes (6), and the next chunk's weights where step 0 was one of
  // the two. LAST: the chunk after which nothing reads weights; it loads none (the
  // compiler would drop loads that nothing reads, and the count be too high).
  auto step = [&](auto jt, int c, const W& w, W& next, auto last) __attribute__((always_inline)) {
    constexpr int J = decltype(jt)::value;
    constexpr bool LAST = decltype(last)::value;
    using Prev = std::integral_constant<int, (J + 3) & 3>;
    [[maybe_unused]] constexpr int YOUNGER = 6 + (!LAST && (J == 1 || J == 2) ? 2 * NT : 0);
    __builtin_amdgcn_sched_barrier(0);
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_s_waitcnt(vmcnt_le(YOUNGER) & lgkmcnt_zero());
#endif
    barrier_no_fence();
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (J == 0 && !LAST) load_w(next, c + 1);
    __builtin_amdgcn_sched_barrier(0);
    fetch_a(stage(Prev{}), 4 * c + J + 3);
    __builtin_amdgcn_sched_barrier(0);
    const unsigned short* as = stage(jt) + (wm * 4) * (3 * 512) + 8 * lane;
    bf16x8 b[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) b[t] = weights8(w.w[t][J], scale_of(w.s[t]));
#pragma unroll
    for (int mb = 0; mb < 4; ++mb) {
#pragma unroll
      for (int p = 2; p >= 0; --p) {
        const bf16x8 a = *reinterpret_cast<const bf16x8*>(as + (mb * 3 + p) * 512);
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[mb][t] = mfma(a, b[t], acc[mb][t]);
      }
    }
  };
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I3 = std::integral_constant<int, 3>;
  W w0, w1;
  auto chunk = [&](int c, const W& w, W& next, auto last) __attribute__((always_inline)) {
    step(I0{}, c, w, next, last);
    step(I1{}, c, w, next, last);
    step(I2{}, c, w, next, last);
    step(I3{}, c, w, next, last);
  };
  load_w(w0, 0);
  __builtin_amdgcn_sched_barrier(0);
  fetch_a(st0, 0);
  __builtin_amdgcn_sched_barrier(0);
  fetch_a(st1, 1);
  __builtin_amdgcn_sched_barrier(0);
  fetch_a(st2, 2);
  int c = 0;
  for (; c + 1 < chunks; c += 2) {
    chunk(c, w0, w1, std::false_type{});
    chunk(c + 1, w1, w0, std::false_type{});
  }
  if (c < chunks) chunk(c, w0, w1, std::true_type{});
  // no direct load may be in flight when the workgroup gives its LDS back
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_s_waitcnt(0);
#endif

  // lane (i, g): element r of acc is row 4 g + r, column i
#pragma unroll
  for (int mb = 0; mb < 4; ++mb) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int rt = 16 * (4 * wm + mb) + 4 * g + r;
      const long long row = m0 + rt;
      const float sc = RMS ? row_scale[rt] : 1.0f;
      if (row < M) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const long long col = nw + 16 * t + i;
          if (col < N) y[row * N + col] = acc[mb][t][r] * sc;
        }
      }
    }
  }
}

struct Mx4Planes {
  unsigned short* planes;
  float* part;
};

template <int BMB, int NT>
void run_gemm(const Mx4Args& a, const Mx4Planes& p, hipStream_t stream) {
  const int K = static_cast<int>(a.K);
  const int nb = (K + 31) / 32;
  const int mblocks = static_cast<int>((a.M + 15) / 16);
  const int tiles_m = (mblocks + BMB - 1) / BMB;
  const long long tiles = tiles_m * ((a.N + 64 * NT - 1) / (64 * NT));
  ENG_CHECK(tiles <= 0x7fffffffLL, "linear_mx4w: too many tiles for one launch");
  const int groups = (K + kPlaneK - 1) / kPlaneK;
  auto go = [&](auto rms) {
    mx4_gemm_kernel<BMB, NT, decltype(rms)::value>
        <<<static_cast<unsigned>(tiles), 64 * BMB, 0, stream>>>(
            p.planes, p.part, a.codes, a.scales, a.y, a.M, a.N, K, nb, tiles_m, mblocks, groups,
            a.eps);
  };
  if (a.rms) go(std::true_type{});
  else go(std::false_type{});
  ENG_LAUNCH_CHECK();
}

// Buffer offsets are 32-bit: a tile's weight rows (256) and an m-block's planes
// stay below 2^31 bytes.
constexpr long long kGemmMaxK = 1ll << 23;

void launch_mx4_gemm(const Mx4Args& a, hipStream_t stream) {
  const int K = static_cast<int>(a.K);
  const int chunks = (K + kChunk - 1) / kChunk;
  const int groups = (K + kPlaneK - 1) / kPlaneK;
  const long long mblocks = (a.M + 15) / 16;
  const std::size_t plane_bytes = static_cast<std::size_t>(mblocks) * chunks * 12 * 1024;
  StreamScratch ws(stream, plane_bytes + static_cast<std::size_t>(a.M) * groups * sizeof(float));
  Mx4Planes p;
  p.planes = static_cast<unsigned short*>(ws.get());
  p.part = reinterpret_cast<float*>(static_cast<char*>(ws.get()) + plane_bytes);
  const bool vec = a.K % 4 == 0 && aligned_to(a.x, 16) && aligned_to(a.gamma, 16);
  auto split = [&](auto rms, auto v) {
    mx4_planes_kernel<decltype(rms)::value, decltype(v)::value>
        <<<dim3(static_cast<unsigned>(mblocks), static_cast<unsigned>(groups)), 256, 0, stream>>>(
            a.x, a.gamma, p.planes, p.part, a.M, K, chunks);
  };
  using T = std::true_type;
  using F = std::false_type;
  if (a.rms) vec ? split(T{}, T{}) : split(T{}, F{});
  else vec ? split(F{}, T{}) : split(F{}, F{});
  ENG_LAUNCH_CHECK();
  if (a.M <= 64) {
    run_gemm<4, 2>(a, p, stream);
    return;
  }
  // the width whose tiles take the least time in whole rounds of one per CU
  const long long cus = device_cu_count();
  long long best = 0;
  int nt = 0;
  for (int cand : {4, 3, 2}) {
    const long long tiles = (mblocks + 7) / 8 * ((a.N + 64 * cand - 1) / (64 * cand));
    const long long cost = (tiles + cus - 1) / cus * (16 * cand + 6);
    if (nt == 0 || cost < best) best = cost, nt = cand;
  }
  if (nt == 4) run_gemm<8, 4>(a, p, stream);
  else if (nt == 3) run_gemm<8, 3>(a, p, stream);
  else run_gemm<8, 2>(a, p, stream);
}

// Up to 32 rows at a.x, a.y.
void launch_few(const Mx4Args& a, hipStream_t stream) {
  switch (a.M) {
    case 1: run_decode<1>(a, stream); return;
    case 2: run_decode<2>(a, stream); return;
    case 3: run_decode<3>(a, stream); return;
    case 4: run_decode<4>(a, stream); return;
    default: break;
  }
  if (a.M <= 16) run_rows<1, 2>(a, stream);
  else run_rows<2, 2>(a, stream);
}

// Rows in passes whose planes take at most 256 MiB of the stream's arena.
void linear_mx4w(const Mx4Args& a, hipStream_t stream) {
  const bool gemm = a.M > 32 && a.K <= kGemmMaxK;
  const long long row_bytes = (a.K + kChunk - 1) / kChunk * kChunk * 6;
  const long long pass = gemm ? std::max(128ll, (256ll << 20) / row_bytes / 128 * 128) : 32;
  for (long long m = 0; m < a.M; m += pass) {
    Mx4Args p = a;
    p.M = std::min(pass, a.M - m);
    p.x = a.x + m * a.K;
    p.y = a.y + m * a.N;
    if (gemm && p.M > 32) launch_mx4_gemm(p, stream);
    else launch_few(p, stream);
  }
}

void check_linear(const std::string& name, const void* x, const void* codes, const void* scales,
                  const void* y, int64_t M, int64_t N, int64_t K) {
  ENG_CHECK(M >= 0 && N >= 0 && K >= 0, name + ": negative dimension");
  ENG_CHECK(x != nullptr && codes != nullptr && scales != nullptr && y != nullptr,
            name + ": null device pointer");
  ENG_CHECK(aligned_to(codes, 16), name + ": codes must be 16-byte aligned");
  ENG_CHECK(K <= 0x7fffff00LL, name + ": K too large");
}

}  // namespace
}  // namespace eng

extern "C" {

int eng_linear_mx4w_nk(const float* x, const uint8_t* codes, const uint8_t* scales, float* y,
                       int64_t M, int64_t N, int64_t K, eng_stream stream) {
  return eng::guarded([&] {
    eng::check_linear("linear_mx4w", x, codes, scales, y, M, N, K);
    if (M == 0 || N == 0) return;
    if (K == 0) {
      eng::fill_zero_async(y, static_cast<std::size_t>(M) * N * sizeof(float),
                           eng::as_stream(stream));
      return;
    }
    eng::linear_mx4w({x, nullptr, codes, scales, y, M, N, K, false, 0.0f}, eng::as_stream(stream));
  });
}

int eng_rmsnorm_linear_mx4w_nk(const float* in, const float* rms_weight, const uint8_t* codes,
                               const uint8_t* scales, float* out, int64_t M, int64_t N, int64_t K,
                               float eps, eng_stream stream) {
  return eng::guarded([&] {
    eng::check_linear("rmsnorm_linear_mx4w", in, codes, scales, out, M, N, K);
    ENG_CHECK(eps >= 0.0f, "rmsnorm_linear_mx4w: eps must be non-negative");
    if (M == 0 || N == 0 || K == 0) return;
    eng::linear_mx4w({in, rms_weight, codes, scales, out, M, N, K, true, eps},
                     eng::as_stream(stream));
  });
}

}  // extern "C"
