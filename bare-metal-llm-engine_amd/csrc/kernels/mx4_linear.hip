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
//   M <= 64           mx4_slice_kernel: workgroups split K, then a reduce
//   M > 64            mx4_planes_kernel, then mx4_gemm_kernel: tiles of C
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
// four floats at any float's address (the hardware's loads need no more)
typedef float floatx4u __attribute__((ext_vector_type(4), aligned(4)));
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

// v as three bf16 terms, left in the top halves of t[0..2]. An infinity is its own
// first term with zeros after it; a NaN's difference, and so the second term, is a
// NaN with its top bit set, which the first need not be (payloads in the low bits).
__device__ __forceinline__ void split3(float v, float (&t)[3]) {
  const float h = __uint_as_float(__float_as_uint(v) & 0xffff0000u);
  const float r = __builtin_isinf(v) ? 0.0f : v - h;
  const float m = __uint_as_float(__float_as_uint(r) & 0xffff0000u);
  t[0] = h;
  t[1] = m;
  t[2] = r - m;
}

// v, loaded at K - 4 where its own place lies past it, as the values at k = K - 4 + past
// on: zeros from K on.
__device__ __forceinline__ floatx4 aligned4(const floatx4& v, int past) {
  floatx4 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float t = past <= 0 ? v[e] : 0.0f;
#pragma unroll
    for (int d = 1; e + d < 4; ++d) t = past == d ? v[e + d] : t;
    r[e] = t;
  }
  return r;
}

// Four values of a row of K at k, zeros from K on.
__device__ __forceinline__ floatx4 load4(const float* __restrict__ row, int k, int K) {
  if (K < 4) {  // (uniform)
    floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (k + e < K) v[e] = row[k + e];
    return v;
  }
  const floatx4 v = *reinterpret_cast<const floatx4u*>(row + min(k, K - 4));
  return k <= K - 4 ? v : aligned4(v, k - (K - 4));
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

// A unit of weights: 256 k of NT tiles of 16 rows, two chunks, so that the pieces of a
// 128-byte line are asked for together (64-byte pieces asked for one by one made the
// caches fetch lines twice). Lane (i, g) holds blocks 8 u + g and 8 u + 4 + g of row
// i; their scale bytes come out of one 8-byte load where rows of scales are whole
// eights of bytes (SV), else as two bytes. Blocks past the row read its last one.
constexpr int kUnit = 2 * kChunk;

template <int NT, bool SV>
struct Unit {
  uintx4 w[2][NT];
  uintx2 s[NT];
  __device__ __forceinline__ void load(int t, const unsigned char* crow, const unsigned char* srow,
                                       int u, int g, int nb) {
    const int b0 = min(8 * u + g, nb - 1);
    const int b1 = min(8 * u + 4 + g, nb - 1);
    w[0][t] = *reinterpret_cast<const uintx4*>(crow + 16ll * b0);
    w[1][t] = *reinterpret_cast<const uintx4*>(crow + 16ll * b1);
    if constexpr (SV) s[t] = *reinterpret_cast<const uintx2*>(srow + 8 * u);
    else s[t] = uintx2{srow[b0], srow[b1]};
  }
  // the scale of half h
  __device__ __forceinline__ float scale(int t, int h, int g) const {
    const unsigned v = s[t][h];
    return scale_of(SV ? (v >> (8 * g)) & 255u : v);
  }
};

// ---------------------------------------------------------------- 1 to 4 rows
//
// One workgroup of 16 waves per CU. X is split into LDS once (MR rows x 3 terms x K);
// then the workgroup goes through its share of the weight rows, equal to within one row, in
// tiles of 16, the waves splitting K by units (whole tiles dealt out in turn left some CUs
// half a tile more: 1 x 11008 x 4096 7.7 us, 1 x 6144 x 4096 6.0 against 5.5). A wave's
// weights come P units ahead, across the tiles, so the stream does not stop where a tile ends: there the waves leave their
// sums in LDS (two buffers in turn, one barrier a tile that waits for no load) and
// one wave, another for each tile, adds and writes them. Rows 4 m + p of the A
// operand are term p of row m; rows that are no term's read some other term (no
// output comes from them). Terms sit 16 bytes apart modulo the banks' 256, so the
// reads of a step (3 MR rows x 4 groups) spread over the banks.
// Bound by the weights' bytes once they are many (1 x 152064 x 4096, 331 MB: 59 us,
// 5.6 TB/s; 1 x 11008 x 4096, 24 MB: 7.4 us), below that by the latencies of one pass
// (X, its split, one unit of weights, the sum: 4.0 us at 1 x 2051 x 1023). Two units in
// flight: with three or four the last ones, which nothing needs, cost more (1 x 4096 x
// 4096, 4.4 us, 0.6 and 1.0 us).
constexpr int kDecodeWaves = 16;
constexpr int kDecodeLds = 120 * 1024;
constexpr int kDecodeTiles = 48;  // most tiles of a workgroup

constexpr int decode_pitch(int K) { return (K + kUnit - 1) / kUnit * kUnit + 8; }
// Whether M rows of X fit the decode kernel's LDS.
bool decode_applies(long long M, long long K) {
  return M <= 4 && K <= kDecodeLds && 6 * M * decode_pitch(static_cast<int>(K)) <= kDecodeLds;
}

template <int MR, bool RMS, bool SV>
__global__ __launch_bounds__(64 * kDecodeWaves) void mx4_decode_kernel(
    const float* __restrict__ x, const float* __restrict__ gamma,
    const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales,
    float* __restrict__ y, long long N, int K, int nb, int rows_each, unsigned more, float eps) {
  constexpr int THREADS = 64 * kDecodeWaves;
  constexpr int PX = MR == 1 ? 3 : MR == 2 ? 2 : 1;  // X loads ahead of the weights'
  constexpr int P = 2;                               // units of weights in flight
  extern __shared__ __attribute__((aligned(16))) unsigned short planes[];  // [MR][3][pitch]
  __shared__ float red[2][kDecodeWaves][MR][16];
  __shared__ float red_ss[kDecodeWaves][MR];
  __shared__ float out[kDecodeTiles][MR][16];
  const int pitch = decode_pitch(K);

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15;
  const int g = lane >> 4;
  const int units = (K + kUnit - 1) / kUnit;
  const int staged = units * kUnit;  // whole units: zeros past K
  const int u0 = units * wave / kDecodeWaves;
  const int u1 = units * (wave + 1) / kDecodeWaves;
  // its rows of W: `rows_each`, and one more for the first `more` workgroups
  const int rows = rows_each + (blockIdx.x < more ? 1 : 0);
  const long long first = static_cast<long long>(blockIdx.x) * rows_each + std::min(blockIdx.x, more);
  const int mine = (rows + 15) / 16;

  struct X {
    floatx4 v[MR];
    floatx4 gm;
  };
  auto load_x = [&](X& r, int k) {
#pragma unroll
    for (int m = 0; m < MR; ++m) r.v[m] = load4(x + static_cast<long long>(m) * K, k, K);
    r.gm = floatx4{1.0f, 1.0f, 1.0f, 1.0f};
    if constexpr (RMS) {
      if (gamma != nullptr) r.gm = load4(gamma, k, K);
    }
  };
  float ss[MR];
#pragma unroll
  for (int m = 0; m < MR; ++m) ss[m] = 0.0f;
  auto put_x = [&](const X& r, int q) {
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      float t[4][3];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v = r.v[m][e];
        if constexpr (RMS) {
          ss[m] = fmaf(v, v, ss[m]);
          v *= r.gm[e];
        }
        split3(v, t[e]);
      }
#pragma unroll
      for (int p = 0; p < 3; ++p)
        *reinterpret_cast<uintx2*>(planes + (m * 3 + p) * pitch + q) =
            uintx2{pack_hi(t[0][p], t[1][p]), pack_hi(t[2][p], t[3][p])};
    }
  };

  X xr[PX];
#pragma unroll
  for (int u = 0; u < PX; ++u)
    if (4 * (tid + u * THREADS) < staged) load_x(xr[u], 4 * (tid + u * THREADS));
  __builtin_amdgcn_sched_barrier(0);

  // The next weights to ask for: unit fu of this workgroup's tile ft. Past the last
  // tile every lane asks for the same first bytes (the waits count loads, so some
  // have to go out; no one uses them).
  Unit<1, SV> w[P];
  int ft = 0, fu = u0;
  const unsigned char* crow;
  const unsigned char* srow;
  auto seek = [&] {
    const long long n = ft < mine ? first + min(16 * ft + i, rows - 1) : 0;
    crow = codes + n * (16ll * nb);
    srow = scales + n * nb;
  };
  auto load_w = [&](int r) {
    const bool live = ft < mine;
    w[r].load(0, crow, srow, live ? fu : 0, live ? g : 0, nb);
    if (++fu >= u1) {
      fu = u0;
      ++ft;
      seek();
    }
  };
  seek();
#pragma unroll
  for (int r = 0; r < P; ++r) load_w(r);
  __builtin_amdgcn_sched_barrier(0);

#pragma unroll
  for (int u = 0; u < PX; ++u)
    if (4 * (tid + u * THREADS) < staged) put_x(xr[u], 4 * (tid + u * THREADS));
  for (int q = 4 * (tid + PX * THREADS); q < staged; q += 4 * THREADS) {
    load_x(xr[0], q);
    put_x(xr[0], q);
  }
  if constexpr (RMS) {
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      const float t = gemv::wave_sum(ss[m]);
      if (lane == 0) red_ss[wave][m] = t;
    }
  }
  lds_barrier();
  [[maybe_unused]] float row_scale = 1.0f;  // of row lane / 16
  if constexpr (RMS) {
    float t = 0.0f;
#pragma unroll
    for (int q = 0; q < kDecodeWaves; ++q) t += red_ss[q][min(g, MR - 1)];
    row_scale = 1.0f / sqrtf(t / static_cast<float>(K) + eps);
  }

  const unsigned short* abase =
      planes + (min(i >> 2, MR - 1) * 3 + min(i & 3, 2)) * pitch + 32 * g;
  floatx4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  int tile = 0;
  // lane (i, g): element r of acc is A row 4 g + r, weight row i. The rows of y stay
  // in LDS until the end: a store among the loads would make every later wait one
  // for all of them.
  auto finish = [&] {
    float (*rb)[MR][16] = red[tile & 1];
    if (g < MR) rb[wave][g][i] = (acc[0] + acc[1]) + acc[2];
    acc = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    lds_barrier();
    if (wave == (tile & (kDecodeWaves - 1)) && g < MR) {
      float v = rb[0][g][i];
#pragma unroll
      for (int q = 1; q < kDecodeWaves; ++q) v += rb[q][g][i];
      out[tile][g][i] = v * row_scale;
    }
    ++tile;
  };
  int u = u0;
  auto compute = [&](const Unit<1, SV>& x) __attribute__((always_inline)) {
    const unsigned short* ap = abase + u * kUnit;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float sc = x.scale(0, h, g);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        acc = mfma(*reinterpret_cast<const bf16x8*>(ap + h * kChunk + 8 * j),
                   weights8(x.w[h][0][j], sc), acc);
    }
    if (++u == u1) {
      u = u0;
      finish();
    }
  };
  // (a wave without units, where K has fewer than waves, only joins the barriers)
  const int items = mine * (u1 - u0);
  int it = 0;
  for (; it + P < items; it += P) {
#pragma unroll
    for (int r = 0; r < P; ++r) {
      compute(w[r]);
      load_w(r);
    }
  }
#pragma unroll
  for (int r = 0; r < P; ++r)
    if (it + r < items) compute(w[r]);
  while (tile < mine) finish();
  lds_barrier();
  for (int q = tid; q < 16 * MR * mine; q += THREADS) {
    const int t = q / (16 * MR);
    const int m = q / 16 % MR;
    const int n = 16 * t + q % 16;
    if (n < rows) y[m * N + first + n] = out[t][m][q % 16];
  }
}

// f with both truth values as types.
template <class F>
void with_flags(bool a, bool b, F&& f) {
  using T = std::true_type;
  using N = std::false_type;
  if (a) b ? f(T{}, T{}) : f(T{}, N{});
  else b ? f(N{}, T{}) : f(N{}, N{});
}

// Whether every row's scale bytes are whole aligned eights (Unit's SV).
bool scales_by_8(const Mx4Args& a) {
  return (a.K + 31) / 32 % 8 == 0 && aligned_to(a.scales, 8);
}

template <int MR>
void run_decode(const Mx4Args& a, hipStream_t stream) {
  const int K = static_cast<int>(a.K);
  const int nb = (K + 31) / 32;
  const std::size_t lds = static_cast<std::size_t>(6) * MR * decode_pitch(K);
  const long long tiles = (a.N + 15) / 16;
  const long long least = (tiles + kDecodeTiles - 1) / kDecodeTiles;
  ENG_CHECK(threads_fit(least, 64 * kDecodeWaves), "linear_mx4w: N too large for one launch");
  const long long wgs = std::min<long long>(tiles, std::max<long long>(device_cu_count(), least));
  const unsigned grid = static_cast<unsigned>(wgs);
  auto go = [&](auto rms, auto sv) {
    constexpr bool R = decltype(rms)::value;
    constexpr bool SV = decltype(sv)::value;
    static std::atomic<bool> done[64];
    allow_staged_lds(reinterpret_cast<const void*>(mx4_decode_kernel<MR, R, SV>), done, lds);
    mx4_decode_kernel<MR, R, SV><<<grid, 64 * kDecodeWaves, lds, stream>>>(
        a.x, a.gamma, a.codes, a.scales, a.y, a.N, K, nb, static_cast<int>(a.N / wgs),
        static_cast<unsigned>(a.N % wgs), a.eps);
  };
  with_flags(a.rms, scales_by_8(a), go);
  ENG_LAUNCH_CHECK();
}

// ------------------------------------------------------------- planes of X
//
// For the GEMM X is split into planes first: 16 rows x 32 k of one term is a fragment,
// 1 KiB in the order the matrix instruction's lanes take it (lane (i, g): row i, the
// eight k of step j in its group's 32-block), fragments [M / 16][chunk][step j][term].
// A wave's load of a fragment is then 1 KiB in one piece, and one of X as it stands 64
// pieces of 16 bytes. Rows past M and k past K are zeros. Beside them the sums of
// squares of each row's chunks. Bound by its bytes and one round trip (512 x 4096, 21
// MB: 7.8 us).
template <bool RMS>
__global__ __launch_bounds__(256) void mx4_planes_kernel(const float* __restrict__ x,
                                                         const float* __restrict__ gamma,
                                                         unsigned short* __restrict__ planes,
                                                         float* __restrict__ part, long long M,
                                                         int K, int chunks) {
  // thread (row i of 16, eighth of 16 of the chunk): 8 values, one lane's of a step
  const int i = threadIdx.x >> 4;
  const int e8 = threadIdx.x & 15;
  const int c = blockIdx.x;
  const long long mb = blockIdx.y;
  const long long row = 16 * mb + i;
  const int k = c * kChunk + 8 * e8;
  const int kr = row < M ? k : K;  // rows past M count as past K
  float v[8];
  float ss = 0.0f;
  const float* xr = x + (row < M ? row : 0) * K;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const floatx4 f = load4(xr, kr + 4 * h, K);
    floatx4 gm = {1.0f, 1.0f, 1.0f, 1.0f};
    if (RMS && gamma != nullptr) gm = load4(gamma, kr + 4 * h, K);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[4 * h + e] = f[e];
      if constexpr (RMS) {
        ss = fmaf(f[e], f[e], ss);
        v[4 * h + e] = f[e] * gm[e];
      }
    }
  }
  float t[8][3];
#pragma unroll
  for (int e = 0; e < 8; ++e) split3(v[e], t[e]);
  uintx4* dst = reinterpret_cast<uintx4*>(planes) + ((mb * chunks + c) * 12 + 3 * (e8 & 3)) * 64 +
                (i + 16 * (e8 >> 2));
#pragma unroll
  for (int p = 0; p < 3; ++p)
    dst[p * 64] = uintx4{pack_hi(t[0][p], t[1][p]), pack_hi(t[2][p], t[3][p]),
                         pack_hi(t[4][p], t[5][p]), pack_hi(t[6][p], t[7][p])};
  if constexpr (RMS) {
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) ss += __shfl_xor(ss, off);
    if (e8 == 0 && row < M) part[row * chunks + c] = ss;
  }
}

struct Mx4Planes {
  unsigned short* planes;
  float* part;
};

std::size_t plane_bytes(long long M, long long K) {
  return static_cast<std::size_t>((M + 15) / 16) * ((K + kChunk - 1) / kChunk) * 12 * 1024;
}
std::size_t planes_scratch(const Mx4Args& a) {
  return plane_bytes(a.M, a.K) +
         static_cast<std::size_t>(a.M) * ((a.K + kChunk - 1) / kChunk) * sizeof(float);
}

Mx4Planes launch_planes(const Mx4Args& a, void* scratch, hipStream_t stream) {
  Mx4Planes p;
  p.planes = static_cast<unsigned short*>(scratch);
  p.part = reinterpret_cast<float*>(static_cast<char*>(scratch) + plane_bytes(a.M, a.K));
  const int K = static_cast<int>(a.K);
  const int chunks = (K + kChunk - 1) / kChunk;
  const dim3 grid(static_cast<unsigned>(chunks), static_cast<unsigned>((a.M + 15) / 16));
  auto go = [&](auto kernel) {
    kernel<<<grid, 256, 0, stream>>>(a.x, a.gamma, p.planes, p.part, a.M, K, chunks);
  };
  if (a.rms) go(mx4_planes_kernel<true>);
  else go(mx4_planes_kernel<false>);
  ENG_LAUNCH_CHECK();
  return p;
}

// s_m of rows m0 .. m0 + ROWS - 1 (row M - 1's past the matrix) into LDS, by all
// THREADS of the workgroup: THREADS / ROWS of them share a row's partial sums.
template <int ROWS, int THREADS>
__device__ __forceinline__ void row_scales(const float* __restrict__ part, long long m0, long long M,
                                           int K, int chunks, float eps, float* row_scale) {
  constexpr int S = THREADS / ROWS;
  static_assert(S >= 1 && S <= 64 && (S & (S - 1)) == 0, "a power of two of neighbouring lanes");
  const int r = threadIdx.x / S;
  const float* p = part + std::min(m0 + r, M - 1) * chunks;
  float t = 0.0f;
#pragma unroll 4
  for (int q = threadIdx.x % S; q < chunks; q += S) t += p[q];
#pragma unroll
  for (int off = 1; off < S; off <<= 1) t += __shfl_xor(t, off);
  if (threadIdx.x % S == 0) row_scale[r] = 1.0f / sqrtf(t / static_cast<float>(K) + eps);
}

// --------------------------------------------------------------- 5 to 64 rows
//
// A workgroup of 8 waves owns 128 NT weight rows (16 NT a wave) and a slice of K, which
// it takes a unit at a time: it splits its unit of X into LDS, as the fragments of
// the matrix instruction (16 rows x 32 k of one term, 1 KiB in the order the lanes
// take it), and every wave multiplies them by its own weights. The next unit of X is
// on its way meanwhile, the next weights from there to the end of its split. With
// several slices the sums go to scratch, and mx4_slice_reduce_kernel adds them in
// slice order and applies the rows' scales (from the sums of squares that the first
// column of workgroups leaves); with one the workgroup scales and writes its rows of
// y itself.
// Slices, because X outweighs the weights otherwise: 16 rows are 96 bytes per k
// in three terms against 8 of a 16-row tile of weights, and with all of K in every
// workgroup their way from L2 set the time (16 x 11008 x 4096: 114 MB, 15 us).
// What bounds it: with a few units to a workgroup, the latencies of one pass and the
// instructions' own way in (a third of the wave's time at 16 x 11008 x 4096, 13.8 us
// with the reduce); with many, the sum of a unit's parts, which barriers keep from
// overlapping within a workgroup (16 x 57344 x 8192 83 us; its weights alone 48 at a
// large copy's rate). Weights a unit ahead in a second set of registers cost more than
// they hide: 16 x 152064 x 4096 105 us, 115 so.
constexpr int kSliceWaves = 8;

// Where lane (i, g)'s 16 bytes of step j sit in their fragment. A read is served in
// passes of 16 lanes, half of a lane group and the other half of its neighbour, a store
// in passes of eight consecutive lanes (of a row: two lane groups, four steps); with
// these bits changed both hit every bank once (no conflicts by the counter).
__device__ __forceinline__ int frag_slot(int i, int g, int j) { return 16 * g + (i ^ j ^ (-g & 3) << 2); }

template <int MB, int NT, bool RMS, bool SV>
__global__ __launch_bounds__(64 * kSliceWaves, 2) void mx4_slice_kernel(
    const float* __restrict__ x, const float* __restrict__ gamma,
    const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales,
    float* __restrict__ y, float* __restrict__ sums, float* __restrict__ squares, int M, long long N,
    int K, int nb, float eps) {
  __shared__ __attribute__((aligned(1024))) unsigned short frag[MB * 24 * 512];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15;
  const int g = lane >> 4;
  const int units = (K + kUnit - 1) / kUnit;
  const int slices = gridDim.y;
  const int slice = blockIdx.y;
  const int u0 = units * slice / slices;  // (units <= 2^15, slices <= 32)
  const int u1 = units * (slice + 1) / slices;

  // X: a thread splits values 8 e8 .. + 7 of chunk tid / 256 of the unit, of rows
  // 16 mb + r.
  const int r = (tid >> 4) & 15;
  const int e8 = tid & 15;
  struct X {
    floatx4 v[MB][2];
    floatx4 gm[2];
  };
  // Rows past M repeat the last one: nothing comes of them.
  unsigned row_at[MB];  // the row's first byte (x is at most 2^31 of them)
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
    row_at[mb] = 4u * static_cast<unsigned>(min(16 * mb + r, M - 1)) * static_cast<unsigned>(K);
  // The weight rows of this wave; those past N read as zeros.
  const long long nw = (static_cast<long long>(blockIdx.x) * kSliceWaves + wave) * (16 * NT);
  [[maybe_unused]] const long long rows_left = std::max(std::min<long long>(N - nw, 16 * NT), 0ll);
#if defined(__HIP_DEVICE_COMPILE__)
  const auto rx = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(x), 0,
                                                    static_cast<int>(4u * static_cast<unsigned>(M) *
                                                                     static_cast<unsigned>(K)),
                                                    kRsrcWord3);
  const auto rg = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(gamma), 0,
                                                    gamma != nullptr ? 4 * K : 0, kRsrcWord3);
  const auto rc = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<unsigned char*>(codes + (rows_left > 0 ? nw : 0) * 16 * nb), 0,
      static_cast<int>(rows_left * 16 * nb), kRsrcWord3);
  const auto rs = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<unsigned char*>(scales + (rows_left > 0 ? nw : 0) * nb), 0,
      static_cast<int>(rows_left * nb), kRsrcWord3);
#endif
  // Unit u's loads, the same ones every time, so that the waits between them are exact;
  // without `live` all are out of their buffers' range, and move nothing. Values past K - 4
  // are loaded at K - 4 and moved by align_x.
  const int k_thread = (tid >> 8) * kChunk + 8 * e8;
  auto load_x = [&](X& f, int u, bool live) __attribute__((always_inline)) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int dead = live ? 0 : 1 << 29;  // (uniform) 2^31 bytes on
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned at = 4u * static_cast<unsigned>(max(min(u * kUnit + k_thread + 4 * h, K - 4), dead));
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
        f.v[mb][h] = __builtin_bit_cast(
            floatx4, __builtin_amdgcn_raw_buffer_load_b128(rx, static_cast<int>(row_at[mb] + at), 0, 0));
      if constexpr (RMS)
        f.gm[h] = __builtin_bit_cast(
            floatx4, __builtin_amdgcn_raw_buffer_load_b128(rg, static_cast<int>(at), 0, 0));
    }
#endif
  };
  // K below 4: value by value.
  auto load_x_short = [&](X& f, int u) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = u * kUnit + k_thread + 4 * h;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
        f.v[mb][h] = load4(x + static_cast<long long>(min(16 * mb + r, M - 1)) * K, k, K);
      if constexpr (RMS) {
        f.gm[h] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        if (gamma != nullptr) f.gm[h] = load4(gamma, k, K);
      }
    }
  };
  auto align_x = [&](X& f, int u) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int past = u * kUnit + k_thread + 4 * h - (K - 4);
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) f.v[mb][h] = aligned4(f.v[mb][h], past);
      if constexpr (RMS) f.gm[h] = aligned4(f.gm[h], past);
    }
  };
  float ss[MB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) ss[mb] = 0.0f;
  auto put_x = [&](const X& f) __attribute__((always_inline)) {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      float t[8][3];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float v = f.v[mb][e >> 2][e & 3];
        if constexpr (RMS) {
          ss[mb] = fmaf(v, v, ss[mb]);
          v *= gamma != nullptr ? f.gm[e >> 2][e & 3] : 1.0f;
        }
        split3(v, t[e]);
      }
      // fragments [chunk][step][m-block][term]; this thread's is lane (r, group e8 / 4)
      // of step e8 % 4.
      uintx4* dst = reinterpret_cast<uintx4*>(frag) +
                    ((((tid >> 8) * 4 + (e8 & 3)) * MB + mb) * 3) * 64 + frag_slot(r, e8 >> 2, e8 & 3);
#pragma unroll
      for (int p = 0; p < 3; ++p)
        dst[p * 64] = uintx4{pack_hi(t[0][p], t[1][p]), pack_hi(t[2][p], t[3][p]),
                             pack_hi(t[4][p], t[5][p]), pack_hi(t[6][p], t[7][p])};
    }
  };
  Unit<NT, SV> w;
  auto load_w = [&](int u, bool live) __attribute__((always_inline)) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int dead = live ? 0 : 1 << 27;  // (uniform) a block past any row's last
    const int b0 = max(min(8 * u + g, nb - 1), dead);
    const int b1 = max(min(8 * u + 4 + g, nb - 1), dead);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int row = (16 * t + i) * nb;
      w.w[0][t] = __builtin_amdgcn_raw_buffer_load_b128(rc, static_cast<int>(16u * (row + b0)), 0, 0);
      w.w[1][t] = __builtin_amdgcn_raw_buffer_load_b128(rc, static_cast<int>(16u * (row + b1)), 0, 0);
      if constexpr (SV) {
        w.s[t] = __builtin_amdgcn_raw_buffer_load_b64(rs, row + max(8 * u, dead), 0, 0);
      } else {
        w.s[t][0] = __builtin_amdgcn_raw_buffer_load_b8(rs, row + b0, 0, 0);
        w.s[t][1] = __builtin_amdgcn_raw_buffer_load_b8(rs, row + b1, 0, 0);
      }
    }
#endif
  };
  floatx4 acc[MB][NT];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[mb][t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  auto compute = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned short* f = frag + ((4 * h + j) * MB * 3) * 512 + 8 * frag_slot(i, g, j);
        bf16x8 b[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) b[t] = weights8(w.w[h][t][j], w.scale(t, h, g));
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
#pragma unroll
          for (int p = 2; p >= 0; --p) {
            const bf16x8 av = *reinterpret_cast<const bf16x8*>(f + (mb * 3 + p) * 512);
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[mb][t] = mfma(av, b[t], acc[mb][t]);
          }
        }
      }
    }
  };

  X xv;
  if (K >= 4) load_x(xv, u0, true);  // (uniform)
  else load_x_short(xv, u0);
  __builtin_amdgcn_sched_barrier(0);
  load_w(u0, true);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll 1
  for (int u = u0; u < u1; ++u) {
    if ((u + 1) * kUnit > K && K >= 4) align_x(xv, u);  // (uniform)
    put_x(xv);
    lds_barrier();
    load_x(xv, u + 1, u + 1 < u1);
    __builtin_amdgcn_sched_barrier(0);
    compute();
    __builtin_amdgcn_sched_barrier(0);
    load_w(u + 1, u + 1 < u1);
    __builtin_amdgcn_sched_barrier(0);
    lds_barrier();  // the fragments have been read
  }

  // The rows' sums of squares over the slice, in LDS (the fragments have been read).
  float* red = reinterpret_cast<float*>(frag);  // [2][16 MB]: the two halves of the threads
  if constexpr (RMS) {
    if (slices == 1 || blockIdx.x == 0) {  // (uniform)
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) ss[mb] += __shfl_xor(ss[mb], off);
        if (e8 == 0) red[(tid >> 8) * 16 * MB + 16 * mb + r] = ss[mb];
      }
      lds_barrier();
      if (slices > 1 && tid < 16 * MB && tid < M)
        squares[static_cast<long long>(tid) * slices + slice] = red[tid] + red[16 * MB + tid];
    }
  }
  // lane (i, g): element v of acc is row 4 g + v, column i
  float* out = slices == 1 ? y : sums + static_cast<long long>(slice) * M * N;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int row = 16 * mb + 4 * g + v;
      if (row < M) {
        float sc = 1.0f;
        if (RMS && slices == 1)
          sc = 1.0f / sqrtf((red[row] + red[16 * MB + row]) / static_cast<float>(K) + eps);
        float* dst = out + row * N;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const long long n = nw + 16 * t + i;
          if (n < N) dst[n] = acc[mb][t][v] * sc;
        }
      }
    }
  }
}

// y[m][n] = s_m times the sum over the slices, in their order, C of them loaded
// together (past the last one, the last one again) and the row's sums of squares, in
// `parts` parts, beside them. blockIdx.y: a row. The sums are in L2 mostly; what it
// costs is a launch and one round trip (16 x 11008, 8 slices, 6.3 MB: 3.9 us).
template <int C, bool RMS>
__global__ __launch_bounds__(256) void mx4_slice_reduce_kernel(const float* __restrict__ sums,
                                                               const float* __restrict__ squares,
                                                               float* __restrict__ y, long long M,
                                                               long long N, int K, int slices,
                                                               int parts, float eps) {
  const long long row = blockIdx.y;
  const long long stride = M * N;
  // four columns a thread; the last ones of a row whose N is no multiple of four overlap
  // their neighbour's, and both write the same bits
  const long long n4 = 4 * (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x);
  const bool whole = n4 < N && N >= 4;
  const long long n = whole ? std::min(n4, N - 4) : 0;
  const float* p = sums + row * N + n;
  float t = 0.0f;
  if constexpr (RMS)
    for (int q = threadIdx.x & 63; q < parts; q += 64) t += squares[row * parts + q];
  floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  if (whole) {
    for (int s0 = 0; s0 < slices; s0 += C) {
      floatx4 a[C];
#pragma unroll
      for (int s = 0; s < C; ++s)
        a[s] = *reinterpret_cast<const floatx4u*>(p + min(s0 + s, slices - 1) * stride);
#pragma unroll
      for (int s = 0; s < C; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = s0 + s < slices ? v[e] + a[s][e] : v[e];
    }
  }
  const float sc = RMS ? 1.0f / sqrtf(gemv::wave_sum(t) / static_cast<float>(K) + eps) : 1.0f;
  float* out = y + row * N;
  if (whole) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= sc;
    *reinterpret_cast<floatx4u*>(out + n) = v;
  } else if (n4 < N) {
    for (int c = 0; c < N; ++c) {
      float u = 0.0f;
      for (int s = 0; s < slices; ++s) u += p[s * stride + c];
      out[c] = u * sc;
    }
  }
}

void launch_reduce(const Mx4Args& a, const float* sums, const float* squares, int slices, int parts,
                   hipStream_t stream) {
  ENG_CHECK(a.M <= 65535, "linear_mx4w: too many rows in a pass");
  const dim3 grid(static_cast<unsigned>((a.N + 1023) / 1024), static_cast<unsigned>(a.M));
  auto go = [&](auto kernel) {
    kernel<<<grid, 256, 0, stream>>>(sums, squares, a.y, a.M, a.N, static_cast<int>(a.K), slices, parts,
                                     a.eps);
  };
  if (slices <= 4) {
    if (a.rms) go(mx4_slice_reduce_kernel<4, true>);
    else go(mx4_slice_reduce_kernel<4, false>);
  } else {
    if (a.rms) go(mx4_slice_reduce_kernel<8, true>);
    else go(mx4_slice_reduce_kernel<8, false>);
  }
  ENG_LAUNCH_CHECK();
}

// Width (128 nt columns) and slices of K: the least estimate, in microseconds or so, of
// whole rounds of one workgroup per CU (mb + 1.7 nt for a unit of K, 1.25 beside the
// units) and, past one slice, the reduce launch and the sums' way out and back.
// Fitted to every width and 1 to 32 slices at 5 to 64 rows of eighteen matrices, 1024 x
// 4096 to 128256 x 8192: what it picks takes 0.4 % (geometric mean) more than the
// fastest of them, 7 % at most. One width for all loses at one end: 16 x 4096 x 4096
// 9.9, 11.1 and 12.2 us at its best slices with nt = 1, 2 and 3 (X is split more often,
// CUs idle), 64 x 11008 x 4096 38, 34 and 30.
void slice_shape(const Mx4Args& a, int mb, int& nt, int& slices) {
  const long long cus = device_cu_count();
  const long long units = (a.K + kUnit - 1) / kUnit;
  double best = 0.0;
  nt = 0;
  for (int cand : {1, 2, 3}) {
    const long long groups = (a.N + 128 * cand - 1) / (128 * cand);
    if (!threads_fit(groups, 64 * kSliceWaves)) continue;
    for (long long s = 1; s <= std::min(units, 32ll); ++s) {
      double time = static_cast<double>((groups * s + cus - 1) / cus) *
                    (static_cast<double>((units + s - 1) / s) * (mb + 1.7 * cand) + 1.25);
      if (s > 1) time += 0.5 + 0.25 * static_cast<double>(s) + 1.7e-6 * static_cast<double>(s * a.M * a.N);
      if (nt == 0 || time < best) best = time, nt = cand, slices = static_cast<int>(s);
    }
  }
}

template <int MB, int NT>
void run_slices(const Mx4Args& a, int slices, hipStream_t stream) {
  const int K = static_cast<int>(a.K);
  const int M = static_cast<int>(a.M);
  const int nb = (K + 31) / 32;
  const long long groups = (a.N + 128 * NT - 1) / (128 * NT);
  const dim3 grid(static_cast<unsigned>(groups), static_cast<unsigned>(slices));
  auto launch = [&](float* sums, float* squares) {
    with_flags(a.rms, scales_by_8(a), [&](auto rms, auto sv) {
      mx4_slice_kernel<MB, NT, decltype(rms)::value, decltype(sv)::value>
          <<<grid, 64 * kSliceWaves, 0, stream>>>(a.x, a.gamma, a.codes, a.scales, a.y, sums, squares, M,
                                                  a.N, K, nb, a.eps);
    });
    ENG_LAUNCH_CHECK();
  };
  if (slices == 1) {
    launch(nullptr, nullptr);
    return;
  }
  const std::size_t sum_bytes = (static_cast<std::size_t>(slices) * M * a.N + 3) / 4 * 16;
  StreamScratch ws(stream, sum_bytes + static_cast<std::size_t>(M) * slices * sizeof(float));
  float* sums = static_cast<float*>(ws.get());
  float* squares = reinterpret_cast<float*>(static_cast<char*>(ws.get()) + sum_bytes);
  launch(sums, squares);
  launch_reduce(a, sums, squares, slices, slices, stream);
}

template <int MB>
void launch_slices(const Mx4Args& a, hipStream_t stream) {
  ENG_CHECK(threads_fit(a.N / 384 + 1, 64 * kSliceWaves), "linear_mx4w: N too large for one launch");
  int nt = 0, slices = 1;
  slice_shape(a, MB, nt, slices);
  if (nt == 1) run_slices<MB, 1>(a, slices, stream);
  else if (nt == 2) run_slices<MB, 2>(a, slices, stream);
  else run_slices<MB, 3>(a, slices, stream);
}

// -------------------------------------------------------------- 65 rows and up
//
// C tiles of 128 x 64 NT on 8 waves: 2 of them along M, 4 along N, each 64 rows x 16
// NT columns. A step is one j of a chunk (32 k): its 24 plane fragments sit in one of
// four LDS stages, loaded four steps ahead by direct loads (three a wave); the
// weights of a chunk come straight into registers a chunk ahead (4-bit: 16 NT bytes a
// lane and chunk) and are converted as their step begins. Tiles with K split among
// gridDim.y slices leave their sums for mx4_slice_reduce_kernel.
// 2048 x 4096 x 4096 takes 189 us with the planes' pass, 1090 TFLOP/s of bf16 products
// (three per weight); a plain bf16 product of 8192^3 through the library runs at 1198 on the
// same card. That is no bound of the hardware: the matrix cores are busy 52 % of the kernel
// (46 % at 512 x 11008 x 4096, 232 tiles on 256 CUs). A wave spends 58 % of its
// time waiting to issue (54 %), behind its SIMD's other wave and its own matrix
// instructions, 2 % of it for the LDS, and 25 % (28 %) at the steps' waits and barriers,
// which keep the two waves of a SIMD in step. Waves of 32 rows by 32 NT columns, with half the LDS
// reads and twice the conversions, take 226 us.
constexpr int kGemmBlocks = 8;  // m-blocks of a tile, and waves

template <int NT, bool RMS>
__global__ __launch_bounds__(64 * kGemmBlocks, 2) void mx4_gemm_kernel(
    const unsigned short* __restrict__ planes, const float* __restrict__ part,
    const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales,
    float* __restrict__ y, float* __restrict__ sums, long long M, long long N, int K, int nb,
    int tiles_m, int mblocks, float eps) {
  constexpr int BMB = kGemmBlocks;
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
  const unsigned logical = static_cast<unsigned>(gemv::xcd_contiguous(blockIdx.x, gridDim.x));
  const unsigned tn = logical / static_cast<unsigned>(tiles_m);
  const int tm = static_cast<int>(logical - tn * static_cast<unsigned>(tiles_m));
  const long long n0 = static_cast<long long>(tn) * (64 * NT);
  const long long m0 = 16ll * BMB * tm;
  const int chunks = (K + kChunk - 1) / kChunk;

  // This slice's chunks. One slice writes scaled rows of y, several their sums.
  const int slices = gridDim.y;
  const int cb = chunks * static_cast<int>(blockIdx.y) / slices;  // (chunks <= 2^16, slices <= 16)
  const int ce = chunks * (static_cast<int>(blockIdx.y) + 1) / slices;
  const bool scaled = RMS && slices == 1;  // (uniform)
  if (scaled) row_scales<16 * BMB, 64 * BMB>(part, m0, M, K, chunks, eps, row_scale);

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
  [[maybe_unused]] const int steps = 4 * ce;
  auto fetch_a = [&](unsigned short* dst, int step) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int so = min(step, steps - 1) * (3 * 1024);
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
    const int b = min(4 * min(c, ce - 1) + g, nb - 1);
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

  // Fragments of m-blocks 2 h and 2 h + 1 of the wave.
  struct A {
    bf16x8 a[2][3];
  };
  auto read_a = [&](A& f, const unsigned short* st, int h) __attribute__((always_inline)) {
    const unsigned short* as = st + (wm * 4 + 2 * h) * (3 * 512) + 8 * lane;
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int p = 0; p < 3; ++p)
        f.a[mb][p] = *reinterpret_cast<const bf16x8*>(as + (mb * 3 + p) * 512);
  };
  auto mma = [&](const A& f, int h, const bf16x8 (&b)[NT]) __attribute__((always_inline)) {
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int p = 2; p >= 0; --p)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[2 * h + mb][t] = mfma(f.a[mb][p], b[t], acc[2 * h + mb][t]);
  };
  // Step (c, j), x holding its first two m-blocks: the other two are read while those
  // are multiplied, then the hand-over (the next step's planes have landed, and every
  // wave has read all of this one's): the next chunk's weights (at j == 0) and the
  // planes four steps on go out, into the stage just read, and the next step's first
  // two m-blocks are read while the second two are multiplied. Younger loads that the
  // wait leaves in flight: two steps' planes (6), and the next chunk's weights where
  // step 0 was one of the two before. LAST: the chunk after which nothing reads
  // weights; it loads none (the compiler would drop loads that nothing reads, and the
  // count be too high).
  A x, z;
  auto step = [&](auto jt, int c, const W& w, W& next, auto last) __attribute__((always_inline)) {
    constexpr int J = decltype(jt)::value;
    constexpr bool LAST = decltype(last)::value;
    using Next = std::integral_constant<int, (J + 1) & 3>;
    [[maybe_unused]] constexpr int YOUNGER = 6 + (!LAST && (J == 1 || J == 2) ? 2 * NT : 0);
    bf16x8 b[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) b[t] = weights8(w.w[t][J], scale_of(w.s[t]));
    read_a(z, stage(jt), 1);
    mma(x, 0, b);
    __builtin_amdgcn_sched_barrier(0);
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_s_waitcnt(vmcnt_le(YOUNGER) & lgkmcnt_zero());
#endif
    barrier_no_fence();
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (J == 0 && !LAST) load_w(next, c + 1);
    __builtin_amdgcn_sched_barrier(0);
    fetch_a(stage(jt), 4 * c + J + 4);
    __builtin_amdgcn_sched_barrier(0);
    read_a(x, stage(Next{}), 0);
    mma(z, 1, b);
    __builtin_amdgcn_sched_barrier(0);
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
  load_w(w0, cb);
  __builtin_amdgcn_sched_barrier(0);
  fetch_a(st0, 4 * cb);
  __builtin_amdgcn_sched_barrier(0);
  fetch_a(st1, 4 * cb + 1);
  __builtin_amdgcn_sched_barrier(0);
  fetch_a(st2, 4 * cb + 2);
  __builtin_amdgcn_sched_barrier(0);
  fetch_a(st3, 4 * cb + 3);
  __builtin_amdgcn_sched_barrier(0);
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_s_waitcnt(vmcnt_le(9));  // the first step's have landed
#endif
  lds_barrier();
  read_a(x, st0, 0);
  __builtin_amdgcn_sched_barrier(0);
  int c = cb;
  for (; c + 1 < ce; c += 2) {
    chunk(c, w0, w1, std::false_type{});
    chunk(c + 1, w1, w0, std::false_type{});
  }
  if (c < ce) chunk(c, w0, w1, std::true_type{});
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
      const float sc = scaled ? row_scale[rt] : 1.0f;
      if (row < M) {
        float* dst = slices == 1 ? y + row * N : sums + (blockIdx.y * M + row) * N;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const long long col = nw + 16 * t + i;
          if (col < N) dst[col] = acc[mb][t][r] * sc;
        }
      }
    }
  }
}

template <int NT>
void run_gemm(const Mx4Args& a, const Mx4Planes& p, float* sums, int slices, hipStream_t stream) {
  constexpr int BMB = kGemmBlocks;
  const int K = static_cast<int>(a.K);
  const int nb = (K + 31) / 32;
  const int mblocks = static_cast<int>((a.M + 15) / 16);
  const int tiles_m = (mblocks + BMB - 1) / BMB;
  const long long tiles = tiles_m * ((a.N + 64 * NT - 1) / (64 * NT));
  ENG_CHECK(threads_fit(tiles, 64 * BMB), "linear_mx4w: too many tiles for one launch");
  const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(slices));
  auto go = [&](auto rms) {
    mx4_gemm_kernel<NT, decltype(rms)::value><<<grid, 64 * BMB, 0, stream>>>(
        p.planes, p.part, a.codes, a.scales, a.y, sums, a.M, a.N, K, nb, tiles_m, mblocks, a.eps);
  };
  if (a.rms) go(std::true_type{});
  else go(std::false_type{});
  ENG_LAUNCH_CHECK();
}

// Tile width and slices of K: the least estimate, in microseconds, of whole rounds of
// one workgroup per CU (a chunk of a 128 x 64 NT tile: its 192 NT matrix
// instructions on four SIMDs and about a quarter of a microsecond; the fill and the
// end of a tile about 2) and, past one slice, the sums' way out and back and the
// reduce launch. Held against every width and 1 to 16 slices (3, 6 and 12 too) at 65 to
// 2048 rows of five matrices, 2051 x 1023 to 28672 x 8192: what it picks takes 3 %
// (geometric mean) more than the fastest of them, 21 % at most (512 x 2051 x 1023 30.3 us,
// 25.1 in three slices, a count that it does not try; 256 x 11008 x 4096 92 against 79).
void gemm_shape(const Mx4Args& a, int& nt, int& slices) {
  const long long cus = device_cu_count();
  const long long chunks = (a.K + kChunk - 1) / kChunk;
  double best = 0.0;
  nt = 0;
  for (int cand : {4, 3, 2}) {
    const long long tiles = (a.M + 127) / 128 * ((a.N + 64 * cand - 1) / (64 * cand));
    for (int s : {1, 2, 4, 8, 16}) {
      if (s > 1 && (2 * s > chunks || tiles * s > 2 * cus)) break;
      const double rounds = static_cast<double>((tiles * s + cus - 1) / cus);
      double us = rounds * (static_cast<double>((chunks + s - 1) / s) * (0.64 * cand + 0.25) + 2.0);
      if (s > 1) us += 4.0 + 8.0e-6 * s * a.M * a.N / 4.0;
      if (nt == 0 || us < best) best = us, nt = cand, slices = s;
    }
  }
}

void launch_mx4_gemm(const Mx4Args& a, hipStream_t stream) {
  int nt = 0, slices = 1;
  gemm_shape(a, nt, slices);
  const std::size_t planes = (planes_scratch(a) + 15) / 16 * 16;
  const std::size_t sum_bytes =
      slices > 1 ? static_cast<std::size_t>(slices) * a.M * a.N * sizeof(float) : 0;
  StreamScratch ws(stream, planes + sum_bytes);
  float* sums = reinterpret_cast<float*>(static_cast<char*>(ws.get()) + planes);
  const Mx4Planes p = launch_planes(a, ws.get(), stream);
  if (nt == 4) run_gemm<4>(a, p, sums, slices, stream);
  else if (nt == 3) run_gemm<3>(a, p, sums, slices, stream);
  else run_gemm<2>(a, p, sums, slices, stream);
  if (slices > 1)
    launch_reduce(a, sums, p.part, slices, static_cast<int>((a.K + kChunk - 1) / kChunk), stream);
}

// One pass of rows at a.x, a.y. The least m-blocks that hold the rows, and the GEMM past
// four: 16 x 28672 x 8192 takes 41.6 us in one m-block and 60 in two, 17 rows 59.7 in two
// and 90 in four, 64 rows 91.7 in four and 176 in the GEMM (at 4096 x 4096 9.3 and 11.2,
// 11.5 and 14.5, 18.9 and 28.0). Past 64 rows the GEMM pays for 128: 65 rows take 27.5 us
// at 4096 x 4096 and 169 at 28672 x 8192.
void launch_pass(const Mx4Args& a, hipStream_t stream) {
  if (decode_applies(a.M, a.K)) {
    switch (a.M) {
      case 1: run_decode<1>(a, stream); break;
      case 2: run_decode<2>(a, stream); break;
      case 3: run_decode<3>(a, stream); break;
      default: run_decode<4>(a, stream); break;
    }
    return;
  }
  if (a.M <= 16) {
    launch_slices<1>(a, stream);
  } else if (a.M <= 32) {
    launch_slices<2>(a, stream);
  } else if (a.M <= 64) {
    launch_slices<4>(a, stream);
  } else {
    launch_mx4_gemm(a, stream);
  }
}

// Rows in passes whose planes take at most 256 MiB of the stream's arena, or of 128 rows,
// a tile of the GEMM, where these take more (K past 349000; 6.4 GB at K = 2^23): fewer rows
// a pass would read the weights more often.
void linear_mx4w(const Mx4Args& a, hipStream_t stream) {
  const long long row_bytes = (a.K + kChunk - 1) / kChunk * kChunk * 6;
  const long long pass = std::clamp((256ll << 20) / row_bytes / 128 * 128, 128ll, 32768ll);
  for (long long m = 0; m < a.M; m += pass) {
    Mx4Args p = a;
    p.M = std::min(pass, a.M - m);
    p.x = a.x + m * a.K;
    p.y = a.y + m * a.N;
    launch_pass(p, stream);
  }
}

void check_linear(const std::string& name, const void* x, const void* codes, const void* scales,
                  const void* y, int64_t M, int64_t N, int64_t K) {
  ENG_CHECK(M >= 0 && N >= 0 && K >= 0, name + ": negative dimension");
  ENG_CHECK(x != nullptr && codes != nullptr && scales != nullptr && y != nullptr,
            name + ": null device pointer");
  ENG_CHECK(aligned_to(codes, 16), name + ": codes must be 16-byte aligned");
  // buffer offsets are 32-bit: a GEMM tile's weight rows and an m-block's planes stay
  // below 2^31 bytes
  ENG_CHECK(K <= (1ll << 23), name + ": K too large (at most 2^23)");
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
