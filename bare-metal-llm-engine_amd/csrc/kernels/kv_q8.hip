// kv_q8.hip -- a KV cache held in 8 bits: the append and the decode attention
// that reads it (the fp16 cache's are in attention.hip).
//
// Format: values are e4m3 (OCP FP8: 4 exponent bits, 3 of mantissa, largest
// 448, no infinity), head-major like the fp16 caches, key j of KV head h of
// sequence b at ((b n_kv_heads + h) kv_max_seq_len + j) D; each block of 32
// tokens of a (sequence, KV head) has one fp32 scale for K and one for V, a
// power of two, at (b n_kv_heads + h) ceil(kv_max_seq_len / 32) + j / 32. A
// power of two keeps a code's value when a block's scale grows (only values that
// fall below e4m3's normal range are rounded again), so a block filled token by
// token is as exact as one written at once to within that rounding.
#include "gemv_kernels.hpp"
#include "launch.hpp"

#include <algorithm>
#include <cmath>

namespace eng {
namespace {

typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef unsigned short ushortx2 __attribute__((ext_vector_type(2)));
typedef unsigned uintx2 __attribute__((ext_vector_type(2)));
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));

constexpr int kKvBlock = 32;  // tokens that share a scale
constexpr float kNegInf = -__builtin_huge_valf();
// V scales below this one, zero among them, count as it: their values are below 448
// 2^-40 < 2^-31 either way, and an fp16 output's half step is 2^-25 at the least.
constexpr float kLeastVScale = 0x1p-40f;
constexpr float kLog2e = 1.4426950408889634f;
[[maybe_unused]] constexpr int kRsrcWord3 = 0x00020000;  // buffer descriptor: raw, 32-bit elements
[[maybe_unused]] constexpr int kNonTemporal = 2;  // a buffer load's cache policy

// ------------------------------------------------------------------- append

constexpr int kWriteThreads = 256;

// Four values as e4m3 bytes (nearest even; infinities and NaN become NaN).
__device__ __forceinline__ unsigned fp8x4(float a, float b, float c, float d) {
  int w = 0;
#if defined(__HIP_DEVICE_COMPILE__)
  w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
#endif
  return static_cast<unsigned>(w);
}

// p is the fp32 value nearest to an exact p + rest: p with its last bit set (of the value
// next towards zero) where rest is not zero. Rounded to e4m3, it gives the code nearest to
// the exact value, where p could have become the middle between two codes. (|p| outside
// the range in which codes differ is left alone: infinities, NaN, and what becomes zero.)
__device__ __forceinline__ float to_odd(float p, float rest) {
  const unsigned u = __float_as_uint(p);
  const unsigned below = ((__float_as_uint(rest) ^ u) >> 31);  // the exact value is nearer to zero
  const bool inexact = rest != 0.0f && fabsf(p) >= 0x1p-12f && fabsf(p) < 0x1p16f;
  return inexact ? __uint_as_float((u - below) | 1u) : p;
}

// Whether s (the same in every lane, positive or zero) is a power of two, or zero.
__device__ __forceinline__ bool power_of_two(float s) {
  return (__builtin_amdgcn_readfirstlane(__float_as_int(s)) & 0x7fffff) == 0;
}

// The largest of the wave's values, none negative, in every lane.
template <int CTRL>
__device__ __forceinline__ int dpp_max(int x) {
  return max(x, __builtin_amdgcn_update_dpp(0, x, CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ int wave_max(int x) {
  x = dpp_max<0xB1>(x);   // quad_perm [1, 0, 3, 2]
  x = dpp_max<0x4E>(x);   // quad_perm [2, 3, 0, 1]
  x = dpp_max<0x141>(x);  // row_half_mirror
  x = dpp_max<0x140>(x);  // row_mirror
  return max(max(__builtin_amdgcn_readlane(x, 0), __builtin_amdgcn_readlane(x, 16)),
             max(__builtin_amdgcn_readlane(x, 32), __builtin_amdgcn_readlane(x, 48)));
}

// One wave per (K or V, sequence, head, block of 32 tokens). A lane holds 8
// consecutive dims of a token (16 bytes of the new rows, 8 of the cache), so a
// wave load covers 64 / (D / 8) tokens and the block's new rows are in flight
// together. The block's scale is the least power of two in [2^-15, 2^8] that
// brings its largest finite new magnitude to 448 or less (2^-15 already holds
// fp16's smallest steps), and no less than the scale of earlier tokens kept in
// the block; if it grows, their codes are brought to it. (Both roundings are right for any
// scale kept from a cache written elsewhere: past powers of two, division and a sticky bit,
// in branches of their own.) Tokens at or past
// kv_max_seq_len are dropped. Blocks belong to one wave each: no atomics.
// Bound by the bytes of the new rows and their codes, and for a token each by the round
// trips of position, then new rows, old codes and scale together (4 prompts of up to 1000
// tokens, 8 heads of 128: 5.6 us; one token each of 32 sequences of 32 heads 4.0).
template <int D>
__global__ __launch_bounds__(kWriteThreads) void kv_write_q8_kernel(
    const _Float16* __restrict__ k_new, const _Float16* __restrict__ v_new,
    unsigned char* __restrict__ k_cache, unsigned char* __restrict__ v_cache,
    float* __restrict__ k_scale, float* __restrict__ v_scale, const int* __restrict__ pos,
    const int* __restrict__ n_new, unsigned units, long long s_new, long long n_kv_heads,
    long long kv_max, int reach) {
  constexpr int LPT = D / 8;         // lanes per token
  constexpr int TPL = 64 / LPT;      // tokens per wave load
  constexpr int LOADS = kKvBlock / TPL;
  const int lane = threadIdx.x & 63;
  const int sub = lane / LPT;
  const int d0 = (lane % LPT) * 8;
  // unit = ((b reach + block) heads + h) 2 + (K or V)
  const unsigned unit = blockIdx.x * (kWriteThreads / 64) +
                        __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (unit >= units) return;
  const bool is_v = (unit & 1) != 0;
  const unsigned heads = static_cast<unsigned>(n_kv_heads);
  const unsigned rest = (unit >> 1) / heads;
  const long long h = (unit >> 1) - rest * heads;
  const long long b = rest / static_cast<unsigned>(reach);
  const long long p = pos[b];
  const long long n = n_new != nullptr ? std::min<long long>(n_new[b], s_new) : s_new;
  if (p < 0 || n <= 0) return;
  const long long blk = p / kKvBlock + (rest - b * reach);  // (p >= 0)
  const long long first = blk * kKvBlock;
  const long long lo = std::max(p, first);
  const long long hi = std::min(std::min(p + n, kv_max), first + kKvBlock);
  if (lo >= hi) return;

  const _Float16* src = (is_v ? v_new : k_new) + ((b * s_new - p) * n_kv_heads + h) * D + d0;
  unsigned char* dst = (is_v ? v_cache : k_cache) + ((b * n_kv_heads + h) * kv_max + first) * D + d0;
  float* sp = (is_v ? v_scale : k_scale) + (b * n_kv_heads + h) * ((kv_max + kKvBlock - 1) / kKvBlock) + blk;

  // Lanes without a new token (or an old one) take the nearest: no branches between the
  // loads, and the maximum does not change.
  halfx8 x[LOADS];
#pragma unroll
  for (int r = 0; r < LOADS; ++r)
    x[r] = *reinterpret_cast<const halfx8*>(
        src + std::min(std::max(first + r * TPL + sub, lo), hi - 1) * n_kv_heads * D);
  const bool kept = lo > first;
  float s_old = 0.0f;
  uintx2 old[LOADS];
  if (kept) {  // (uniform)
    s_old = *sp;
#pragma unroll
    for (int r = 0; r < LOADS; ++r)
      old[r] = *reinterpret_cast<const uintx2*>(dst + std::min<long long>(r * TPL + sub, lo - first - 1) * D);
  }
  ushortx2 top2 = {0, 0};
#pragma unroll
  for (int r = 0; r < LOADS; ++r) {
    const uintx4 w = __builtin_bit_cast(uintx4, x[r]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const unsigned m = w[e] & 0x7fff7fffu;
      top2 = __builtin_elementwise_max(top2, __builtin_bit_cast(ushortx2, m));
    }
  }
  int top = wave_max(std::max<int>(top2[0], top2[1]));
  if (top >= 0x7c00) {  // (uniform) infinities or NaN among them: the finite ones' maximum
    top = 0;
#pragma unroll
    for (int r = 0; r < LOADS; ++r) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const _Float16 v = x[r][e];  // (bit-casting a vector's element in place reads element 0)
        const int m = __builtin_bit_cast(unsigned short, v) & 0x7fff;
        top = max(top, m < 0x7c00 ? m : 0);
      }
    }
    top = wave_max(top);
  }
  const float amax = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<unsigned short>(top)));
  // amax = 1.m 2^E: 448 = 1.75 2^8 holds it at 2^(E - 8) up to m = 0.75
  const int bits = __float_as_int(amax);
  int e = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  e = min(max(e, -15), 8);
  const float s = fmaxf(__int_as_float((e + 127) << 23), s_old);
  const float inv = 1.0f / s;
  if (power_of_two(s)) {
#pragma unroll
    for (int r = 0; r < LOADS; ++r) {
      const int t = r * TPL + sub;
      if (first + t >= lo && first + t < hi) {
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = static_cast<float>(x[r][q]) * inv;
        *reinterpret_cast<uintx2*>(dst + t * D) =
            uintx2{fp8x4(v[0], v[1], v[2], v[3]), fp8x4(v[4], v[5], v[6], v[7])};
      }
    }
  } else {  // a scale kept from elsewhere; its rows again, so that this stays a small loop
#pragma unroll 1
    for (int t = sub; t < kKvBlock; t += TPL) {
      if (first + t >= lo && first + t < hi) {
        const halfx8 w = *reinterpret_cast<const halfx8*>(src + (first + t) * n_kv_heads * D);
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const float f = static_cast<float>(w[q]);
          v[q] = f / s;
          v[q] = to_odd(v[q], fmaf(-v[q], s, f));
        }
        *reinterpret_cast<uintx2*>(dst + t * D) =
            uintx2{fp8x4(v[0], v[1], v[2], v[3]), fp8x4(v[4], v[5], v[6], v[7])};
      }
    }
  }
  if (kept && s > s_old) {  // (s is a power of two)
    [[maybe_unused]] const float ratio = s_old * inv;
    if (power_of_two(s_old)) {
#pragma unroll
      for (int r = 0; r < LOADS; ++r) {
        const int t = r * TPL + sub;
        if (first + t < lo) {
          [[maybe_unused]] const uintx2 c = old[r];
          uintx2 o = {0, 0};
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const floatx2 a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(c[q]), false);
            const floatx2 z = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(c[q]), true);
            o[q] = fp8x4(a[0] * ratio, a[1] * ratio, z[0] * ratio, z[1] * ratio);
          }
#endif
          *reinterpret_cast<uintx2*>(dst + t * D) = o;
        }
      }
    } else {
#pragma unroll 1
      for (int t = sub; first + t < lo; t += TPL) {
        uintx2 c = *reinterpret_cast<const uintx2*>(dst + t * D);
#if defined(__HIP_DEVICE_COMPILE__)
        auto scaled = [&](float f) { return to_odd(f * ratio, fmaf(f, ratio, -(f * ratio))); };
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const floatx2 a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(c[q]), false);
          const floatx2 z = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(c[q]), true);
          c[q] = fp8x4(scaled(a[0]), scaled(a[1]), scaled(z[0]), scaled(z[1]));
        }
#endif
        *reinterpret_cast<uintx2*>(dst + t * D) = c;
      }
    }
  }
  if (lane == 0 && s != s_old) *sp = s;
}

// ---------------------------------------------------------------- attention

// 2^(a - b), 0 for a == -inf whatever b is; NaN stays NaN.
__device__ __forceinline__ float weight2(float a, float b) {
  const float w = __builtin_amdgcn_exp2f(a - b);
  return a == kNegInf ? 0.0f : w;
}

struct AttnArgs {
  const _Float16* q;
  const unsigned char* k;
  const unsigned char* v;
  const float* ks;
  const float* vs;
  _Float16* out;
  const int* lens;
  long long n_heads, n_kv_heads, max_len, kv_max;
  int group, tiles;   // query heads per KV head; 16-head tiles of it
  int split_blocks;   // 32-token blocks per split
  int nsplit;
  float scale;
};

// One workgroup per (sequence, KV head, tile of up to 16 of its query heads,
// split of `split_blocks` 32-token blocks), NW waves, block t of the split to
// wave t % NW, P blocks in flight per wave (RING: more than P of them, the loads of
// one P blocks on following each compute). The matrix cores do both products:
// scores S^T = K . Q^T with K as the A operand (the e4m3 bytes converted to
// fp16, exact), O^T = V^T . P^T with the score accumulators, in place, as the B
// operand: A row i is key (i / 4) + 4 (i % 4) of its 16, so accumulator element
// r of lane group g is key g + 4 r, which is also the key that group loads of V.
// K is 16-byte pieces of a key's row, V D / 16 bytes of a key for each lane.
//
// A block's K scale multiplies its scores. Its V scale joins the weights: with
// s' = s + log2(v scale) the weight 2^(s' - m) multiplies the codes themselves
// and 2^(s' - m) / (v scale) adds to l, so O needs no second accumulator. m runs
// over s', is raised only when a score passes it by 8 or more, and the weights
// carry 2^7 so that their fp16 high and low terms hold 22 bits down to 2^-10 of
// the largest (as in the fp16 cache's kernel). Sums, m and l are fp32.
// With V scales from 2^-40 (smaller ones count as it) to 2^24, m passes the largest
// score s by 24 at the most, so l, in units of 2^-7, is 2^-17 or more. A weight below
// 2^-126, lost, would have added less than 2^-86 to it, 2^31 of them 2^-55; a split's l,
// 2^15 2^40 2^23 at the most, under a lost weight of the merge 2^-48. Neither shows.
//
// Bound by the cache's bytes: 131072 tokens of 32 / 8 heads, D = 128 (270 MB) in 46
// us with the merge, 5.9 TB/s. Workgroups of 4 waves, three to a CU, cover the
// latency of a split's start and end (16 unlike sequences of up to 8192 tokens: 29
// us, 35 on 8 waves). K's 64-byte pieces stay cacheable, since two loads share a
// line; V's whole rows are read past the caches (16 sequences 29 us, 32 with V
// cached, 33 with K uncached as well).
template <int D, int NW, int P, bool RING, bool PARTIAL>
__global__ __launch_bounds__(64 * NW, NW == 4 ? 3 : 1) void decode_q8_kernel(AttnArgs a, float* __restrict__ part_o,
                                                            float* __restrict__ part_ml) {
  static_assert(D == 64 || D == 128, "head_dim 64 or 128");
  constexpr int KS = D / 32;       // 32-dim steps of a score
  constexpr int KL = D / 64;       // 16-byte loads of a key per lane
  constexpr int VW = D / 16;       // dims of a value per lane: V words are VW / 4
  constexpr int VD = VW / 4;
  // One wave's state in LDS, for the heads that the tile has: o [heads][D], m, l.
  extern __shared__ __attribute__((aligned(16))) float s_state[];
  const int heads = min(a.group, 16);
  const int WS = heads * (D + 2);

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15;
  const int grp = lane >> 4;
  const unsigned n_kv = static_cast<unsigned>(a.n_kv_heads);  // 32-bit division: below 2^31
  const unsigned bh32 = blockIdx.x / static_cast<unsigned>(a.tiles);
  const int tile = static_cast<int>(blockIdx.x - bh32 * static_cast<unsigned>(a.tiles));
  const long long bh = bh32;  // sequence and KV head
  const long long b = bh32 / n_kv;
  const long long kvh = bh - b * a.n_kv_heads;
  const int split = static_cast<int>(blockIdx.y);
  const int gq = min(a.group - 16 * tile, 16);
  const long long h0 = b * a.n_heads + kvh * a.group + 16 * tile;  // first (sequence, head)
  const int len = static_cast<int>(std::min<long long>(max(a.lens[b], 0), a.max_len));
  const int blocks = (len + kKvBlock - 1) / kKvBlock;
  const long long t0 = static_cast<long long>(split) * a.split_blocks;
  if (t0 >= blocks) {
    // nothing here; a sequence without tokens gets zeros where no merge follows
    if (!PARTIAL && blocks == 0) {
      for (int i = tid; i < gq * D; i += 64 * NW) a.out[h0 * D + i] = static_cast<_Float16>(0.0f);
    }
    return;
  }
  const int nblocks = min(a.split_blocks, static_cast<int>(blocks - t0));
  const int nkeys = min(nblocks * kKvBlock, static_cast<int>(len - t0 * kKvBlock));
  const int nb = wave < nblocks ? (nblocks - wave + NW - 1) / NW : 0;  // this wave's blocks

  // q^T as the score B operand: dims 64 (s / 2) + 16 grp + 8 (s % 2) + j of head col
  halfx8 qb[KS];
  const _Float16* qh = a.q + (h0 + min(col, gq - 1)) * D + 16 * grp;
  if ((reinterpret_cast<std::uintptr_t>(a.q) & 15) == 0) {
#pragma unroll
    for (int s = 0; s < KS; ++s)
      qb[s] = *reinterpret_cast<const halfx8*>(qh + 64 * (s >> 1) + 8 * (s & 1));
  } else {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
#pragma unroll
      for (int j = 0; j < 8; ++j) qb[s][j] = qh[64 * (s >> 1) + 8 * (s & 1) + j];
    }
  }
  const float scale2 = a.scale * kLog2e;
  // The split's part of each cache through a buffer descriptor that ends with its
  // last token: rows past it read as zeros (weight 0, and no stale code can reach a
  // product), and a block's loads need one address each for K and V.
  [[maybe_unused]] const long long row0 = (bh * a.kv_max + t0 * kKvBlock) * D;
#if defined(__HIP_DEVICE_COMPILE__)
  const auto rk = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(a.k + row0), 0,
                                                    nkeys * D, kRsrcWord3);
  const auto rv = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(a.v + row0), 0,
                                                    nkeys * D, kRsrcWord3);
#endif
  [[maybe_unused]] const int koff = ((col >> 2) + 4 * (col & 3)) * D + 16 * grp;
  [[maybe_unused]] const int voff = grp * D + VW * col;
  const long long sb = bh * ((a.kv_max + kKvBlock - 1) / kKvBlock) + t0;

  typedef unsigned vword __attribute__((ext_vector_type(VD)));
  struct Block {
    uintx4 k[2][KL];
    vword v[8];
    float ks, vs;
  };
  // Every call issues the same loads, whether or not the wave has a block t (past
  // the last one they return zeros without a memory access), so that the waits
  // count exactly the blocks in flight behind the one a compute needs.
  auto load = [&](Block& x, int t) __attribute__((always_inline)) {
    const int blk = wave + NW * t;
#if defined(__HIP_DEVICE_COMPILE__)
    const int at = blk * (kKvBlock * D);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int s = 0; s < KL; ++s)
        x.k[h][s] = __builtin_amdgcn_raw_buffer_load_b128(rk, at + koff + 16 * h * D + 64 * s, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int o = at + voff + (16 * (e >> 2) + 4 * (e & 3)) * D;
      if constexpr (VD == 2) x.v[e] = __builtin_amdgcn_raw_buffer_load_b64(rv, o, 0, kNonTemporal);
      else x.v[e][0] = __builtin_amdgcn_raw_buffer_load_b32(rv, o, 0, kNonTemporal);
    }
#endif
    const int sblk = min(blk, nblocks - 1);
    x.ks = a.ks[sb + sblk];
    x.vs = a.vs[sb + sblk];
  };
  // Largest of x over the four lanes of a head (each swap leaves this lane's value
  // and its partner's in the two results, copied to scalars before they are cast).
  auto group_max = [](float x) __attribute__((always_inline)) {
#if defined(__HIP_DEVICE_COMPILE__)
    const unsigned u = __float_as_uint(x);
    const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const unsigned p0 = p[0], p1 = p[1];
    x = fmaxf(__uint_as_float(p0), __uint_as_float(p1));
    const unsigned w = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    const unsigned r0 = r[0], r1 = r[1];
    x = fmaxf(__uint_as_float(r0), __uint_as_float(r1));
#endif
    return x;
  };

  constexpr float kLazy = 8.0f;
  constexpr float kWeightShift = 7.0f;
  float m = kNegInf;
  float lsum = 0.0f;
  floatx4 o[VW];
#pragma unroll
  for (int mb = 0; mb < VW; ++mb) o[mb] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

  // two e4m3 bytes (half H of a word) as fp16
  auto two = [](unsigned w, auto half) __attribute__((always_inline)) {
    halfx2 r = {};
#if defined(__HIP_DEVICE_COMPILE__)
    r = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, decltype(half)::value);
#endif
    return r;
  };
  using Lo = std::false_type;
  using Hi = std::true_type;
  auto compute = [&](const Block& x, int t) __attribute__((always_inline)) {
    floatx4 sc[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sc[h] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const unsigned w0 = x.k[h][s >> 1][2 * (s & 1)];
        const unsigned w1 = x.k[h][s >> 1][2 * (s & 1) + 1];
        const halfx2 c0 = two(w0, Lo{}), c1 = two(w0, Hi{}), c2 = two(w1, Lo{}), c3 = two(w1, Hi{});
        [[maybe_unused]] const halfx8 ka = {c0[0], c0[1], c1[0], c1[1], c2[0], c2[1], c3[0], c3[1]};
#if defined(__HIP_DEVICE_COMPILE__)
        sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qb[s], sc[h], 0, 0, 0);
#endif
      }
    }
    const int left = nkeys - (wave + NW * t) * kKvBlock;  // keys from the block's first one on
    const float f = scale2 * x.ks;
    const float vs = fabsf(x.vs) < kLeastVScale ? kLeastVScale : x.vs;
    const float lv = __builtin_amdgcn_logf(vs);  // log2
    const float ivs = __builtin_amdgcn_rcpf(vs);
    float sv[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) sv[e] = fmaf(sc[e >> 2][e & 3], f, lv);
    if (left < kKvBlock) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (grp + 16 * (e >> 2) + 4 * (e & 3) >= left) sv[e] = kNegInf;
    }
    float mx = fmaxf(fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3])),
                     fmaxf(fmaxf(sv[4], sv[5]), fmaxf(sv[6], sv[7])));
    mx = group_max(mx);
    if (__any(mx > m + kLazy)) {
      const float mn = fmaxf(m, mx);
      const float alpha = weight2(m, mn);
      m = mn;
      lsum *= alpha;
#pragma unroll
      for (int mb = 0; mb < VW; ++mb) o[mb] *= alpha;
    }
    // (while every score so far is -inf, against 0: weights 0, not NaN)
    const float ref = m == kNegInf ? 0.0f : m - kWeightShift;
    [[maybe_unused]] halfx8 ph, pl;
    float ls = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float p0 = __builtin_amdgcn_exp2f(sv[e] - ref);
      const float p1 = __builtin_amdgcn_exp2f(sv[e + 1] - ref);
      ls += p0 + p1;
#if defined(__HIP_DEVICE_COMPILE__)
      const halfx2 hi = __builtin_bit_cast(halfx2, __builtin_amdgcn_cvt_pkrtz(p0, p1));
      const halfx2 lo = __builtin_bit_cast(
          halfx2, __builtin_amdgcn_cvt_pkrtz(p0 - static_cast<float>(hi[0]), p1 - static_cast<float>(hi[1])));
      ph[e] = hi[0], ph[e + 1] = hi[1];
      pl[e] = lo[0], pl[e + 1] = lo[1];
#endif
    }
    lsum = fmaf(ls, ivs, lsum);
#pragma unroll
    for (int d = 0; d < VD; ++d) {
      halfx8 av[4];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const halfx2 c0 = two(x.v[e][d], Lo{}), c1 = two(x.v[e][d], Hi{});
        av[0][e] = c0[0], av[1][e] = c0[1], av[2][e] = c1[0], av[3][e] = c1[1];
      }
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        o[4 * d + u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av[u], pl, o[4 * d + u], 0, 0, 0);
        o[4 * d + u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av[u], ph, o[4 * d + u], 0, 0, 0);
      }
#endif
    }
  };

  Block buf[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    load(buf[i], i);
    __builtin_amdgcn_sched_barrier(0);
  }
  if constexpr (!RING) {
#pragma unroll
    for (int i = 0; i < P; ++i)
      if (i < nb) compute(buf[i], i);
  } else {
    for (int t = 0; t < nb; t += P) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        if (t + i < nb) compute(buf[i], t + i);
        __builtin_amdgcn_sched_barrier(0);
        load(buf[i], t + i + P);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  // Lane (col, grp) holds dims VW (4 grp + r) + mb of head col in o[mb][r].
  float lt = lsum + __shfl_xor(lsum, 16);
  lt += __shfl_xor(lt, 32);
  if constexpr (NW == 1) {
    if (col < gq) {
      const long long h = h0 + col;
      const long long slot = h * a.nsplit + split;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
#pragma unroll
        for (int mb = 0; mb < VW; ++mb) {
          const int d = VW * (4 * grp + r) + mb;
          if constexpr (PARTIAL) part_o[slot * D + d] = o[mb][r];
          else a.out[h * D + d] = static_cast<_Float16>(o[mb][r] / lt);
        }
      }
      if (PARTIAL && grp == 0) {
        part_ml[2 * slot] = m;
        part_ml[2 * slot + 1] = lt;
      }
    }
    return;
  }
  float* const ws = s_state + wave * WS;
  if (col < gq) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
      for (int c = 0; c < VW; c += 2)  // (a state's start is 8-byte aligned)
        *reinterpret_cast<floatx2*>(ws + col * D + VW * (4 * grp + r) + c) =
            floatx2{o[c][r], o[c + 1][r]};
    }
    if (grp == 0) {
      ws[heads * D + col] = m;
      ws[heads * (D + 1) + col] = lt;
    }
  }
  __syncthreads();
  const int live = min(NW, nblocks);  // waves with a block
  for (int idx = tid; idx < gq * D; idx += 64 * NW) {
    const int gh = idx / D;
    const int d = idx - gh * D;
    float mb = kNegInf;
    for (int w = 0; w < live; ++w) mb = fmaxf(mb, s_state[w * WS + heads * D + gh]);
    float lb = 0.0f, ob = 0.0f;
    for (int w = 0; w < live; ++w) {
      const float wt = weight2(s_state[w * WS + heads * D + gh], mb);
      lb = fmaf(s_state[w * WS + heads * (D + 1) + gh], wt, lb);
      ob = fmaf(s_state[w * WS + gh * D + d], wt, ob);
    }
    const long long h = h0 + gh;
    if constexpr (PARTIAL) {
      const long long slot = h * a.nsplit + split;
      part_o[slot * D + d] = ob;
      if (d == 0) {
        part_ml[2 * slot] = mb;
        part_ml[2 * slot + 1] = lb;
      }
    } else {
      a.out[h * D + d] = static_cast<_Float16>(ob / lb);
    }
  }
}

// out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s over the splits that the
// sequence's length reaches: one wave per (sequence, head), in split order. Lane s
// holds state s's (m, l), every lane its D / 64 dims of all states, C states at a
// time and their loads issued together, so up to C splits cost one round trip;
// the weight of state s is read from lane s. Bound by the round trips of length and
// states: 2.9 us at 32 heads and 16 splits.
template <int D, int C>
__global__ __launch_bounds__(64) void merge_q8_kernel(const float* __restrict__ part_o,
                                                      const float* __restrict__ part_ml,
                                                      const int* __restrict__ lens,
                                                      _Float16* __restrict__ out, long long n_heads,
                                                      long long max_len, int split_blocks,
                                                      int nsplit) {
  static_assert(C <= 64, "a lane per state");
  constexpr int DPL = D / 64;
  const int lane = threadIdx.x;
  const long long h = blockIdx.x;
  const unsigned b = blockIdx.x / static_cast<unsigned>(n_heads);
  const int len = static_cast<int>(std::min<long long>(max(lens[b], 0), max_len));
  const int blocks = (len + kKvBlock - 1) / kKvBlock;
  const int ns = (blocks + split_blocks - 1) / split_blocks;
  const long long base = h * nsplit;
  float m = kNegInf, l = 0.0f;
  float o[DPL];
#pragma unroll
  for (int j = 0; j < DPL; ++j) o[j] = 0.0f;
  for (int s0 = 0; s0 < ns; s0 += C) {
    // states past the last one are read as the last one, with weight 0
    const long long sl = base + min(s0 + min(lane, C - 1), ns - 1);
    const float ms = part_ml[2 * sl];
    const float ls = part_ml[2 * sl + 1];
    float os[C][DPL];
#pragma unroll
    for (int s = 0; s < C; ++s) {
      const long long slot = base + min(s0 + s, ns - 1);
#pragma unroll
      for (int j = 0; j < DPL; ++j) os[s][j] = part_o[slot * D + lane + 64 * j];
    }
    const bool live = lane < C && s0 + lane < ns;
    float mx = live ? ms : kNegInf;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) mx = fmaxf(mx, __shfl_xor(mx, off));
    const float mn = fmaxf(m, mx);
    const float was = weight2(m, mn);
    m = mn;
    const float w = live ? weight2(ms, mn) : 0.0f;
    l = l * was + gemv::wave_sum(live ? w * ls : 0.0f);
#pragma unroll
    for (int j = 0; j < DPL; ++j) o[j] *= was;
#pragma unroll
    for (int s = 0; s < C; ++s) {
      const float ws = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), s));
#pragma unroll
      for (int j = 0; j < DPL; ++j) o[j] = s0 + s < ns ? fmaf(ws, os[s][j], o[j]) : o[j];
    }
  }
#pragma unroll
  for (int j = 0; j < DPL; ++j)
    out[h * D + lane + 64 * j] = static_cast<_Float16>(ns == 0 ? 0.0f : o[j] / l);
}

// Splits when the caller passes split_kv = 0: the largest power of two that keeps
// one workgroup per CU or fewer over all (sequence, KV head) units (splits of
// unlike lengths, as a division that does not come out even makes, were 5-25%
// slower), at least four blocks per split, one per wave, past 32 blocks, and one
// split, without the merge's launch, up to 12 blocks at D = 128 or 24 at D = 64
// (300 tokens, 32 / 4 heads of 64 5.3 us, 6.5 in 8 splits; 600 tokens, 32 / 8 heads
// of 128 7.8 us, 7.1 in 16). A sweep of 1 to 64 splits over 18 shapes put it at the best count or within 6%:
// 32 / 32 heads, D = 128, 8192 tokens 8 splits 15.4 us (16: 16.7, 4: 18.1); 32 / 8
// heads, 131072 tokens 32 splits 46 us (16: 59, 64: 49); 32 sequences of 32 / 8
// heads, 4096 tokens 1 split 43 us (2: 47.5, 8: 54.6); 1000 tokens, 32 / 8 heads 32
// splits 6.3 us (8: 7.3, 1: 9.5).
int auto_splits(long long blocks, long long units, long long head_dim) {
  if (blocks * head_dim <= 12 * 128) return 1;
  const long long cus = device_cu_count();
  const long long most = std::min(256ll, blocks <= 32 ? blocks : blocks / 4);
  long long s = 1;
  while (2 * s <= most && 2 * s * units <= cus) s *= 2;
  return static_cast<int>(s);
}

// A split's cache bytes stay below 2^31: buffer offsets are 32-bit.
constexpr long long kMaxSplitBlocks = (1ll << 30) / (128 * kKvBlock);

template <int D, bool PARTIAL>
void launch_decode(const AttnArgs& a, float* part_o, float* part_ml, dim3 grid, hipStream_t s) {
  auto go = [&](auto kernel, int waves) {
    const std::size_t lds =  // at most 33 KiB
        waves == 1 ? 0 : static_cast<std::size_t>(waves) * std::min(a.group, 16) * (D + 2) * 4;
    kernel<<<grid, 64 * waves, lds, s>>>(a, part_o, part_ml);
  };
  constexpr int W = 4;
  if (a.split_blocks <= 1) go(decode_q8_kernel<D, 1, 1, false, PARTIAL>, 1);
  else if (a.split_blocks <= 2) go(decode_q8_kernel<D, 2, 1, false, PARTIAL>, 2);
  else if (a.split_blocks <= W) go(decode_q8_kernel<D, W, 1, false, PARTIAL>, W);
  else if (a.split_blocks <= 2 * W) go(decode_q8_kernel<D, W, 2, false, PARTIAL>, W);
  else go(decode_q8_kernel<D, W, 2, true, PARTIAL>, W);
  ENG_LAUNCH_CHECK();
}

template <int D>
void run_decode(AttnArgs a, long long batch, hipStream_t s) {
  const long long units = batch * a.n_kv_heads * a.tiles;
  ENG_CHECK(threads_fit(units, 256) && (a.nsplit == 1 || threads_fit(batch * a.n_heads, 64)),
            "attention_decode_q8: too many (sequence, head) pairs for one launch");
  const dim3 grid(static_cast<unsigned>(units), static_cast<unsigned>(a.nsplit));
  if (a.nsplit == 1) {
    launch_decode<D, false>(a, nullptr, nullptr, grid, s);
    return;
  }
  const std::size_t slots = static_cast<std::size_t>(batch) * a.n_heads * a.nsplit;
  StreamScratch scratch(s, slots * (D + 2) * sizeof(float));
  float* part_o = static_cast<float*>(scratch.get());
  float* part_ml = part_o + slots * D;
  launch_decode<D, true>(a, part_o, part_ml, grid, s);
  auto merge = [&](auto kernel) {
    kernel<<<static_cast<unsigned>(batch * a.n_heads), 64, 0, s>>>(
        part_o, part_ml, a.lens, a.out, a.n_heads, a.max_len, a.split_blocks, a.nsplit);
  };
  if (a.nsplit <= 8) merge(merge_q8_kernel<D, 8>);
  else if (a.nsplit <= 16) merge(merge_q8_kernel<D, 16>);
  else merge(merge_q8_kernel<D, 32>);
  ENG_LAUNCH_CHECK();
}

constexpr long long kMaxLen = 0x7fffffffLL - kKvBlock;  // positions are 32-bit on the device

}  // namespace
}  // namespace eng

using eng::guarded;

extern "C" {

int eng_kv_cache_write_q8(const eng_half* k_new, const eng_half* v_new, uint8_t* k_cache,
                          uint8_t* v_cache, float* k_scale, float* v_scale, const int32_t* pos,
                          const int32_t* n_new, int64_t batch, int64_t s_new, int64_t n_kv_heads,
                          int64_t head_dim, int64_t kv_max_seq_len, eng_stream stream) {
  return guarded([&] {
    ENG_CHECK(batch >= 0, "kv_cache_write_q8: batch must be non-negative");
    ENG_CHECK(s_new >= 0, "kv_cache_write_q8: s_new must be non-negative");
    ENG_CHECK(n_kv_heads > 0, "kv_cache_write_q8: n_kv_heads must be positive");
    ENG_CHECK(head_dim == 64 || head_dim == 128, "kv_cache_write_q8: head_dim must be 64 or 128");
    ENG_CHECK(kv_max_seq_len >= 0 && kv_max_seq_len <= eng::kMaxLen,
              "kv_cache_write_q8: kv_max_seq_len must be non-negative and below 2^31 - 32");
    ENG_CHECK(s_new <= kv_max_seq_len, "kv_cache_write_q8: kv_max_seq_len < s_new");
    if (batch == 0 || s_new == 0) return;
    ENG_CHECK(k_new != nullptr && v_new != nullptr, "kv_cache_write_q8: k_new/v_new is null");
    ENG_CHECK(k_cache != nullptr && v_cache != nullptr, "kv_cache_write_q8: k_cache/v_cache is null");
    ENG_CHECK(k_scale != nullptr && v_scale != nullptr, "kv_cache_write_q8: k_scale/v_scale is null");
    ENG_CHECK(pos != nullptr, "kv_cache_write_q8: pos is null");
    ENG_CHECK(eng::aligned_to(k_new, 16) && eng::aligned_to(v_new, 16) &&
                  eng::aligned_to(k_cache, 16) && eng::aligned_to(v_cache, 16),
              "kv_cache_write_q8: k_new, v_new and the caches must be 16-byte aligned");
    const int reach = static_cast<int>((s_new + eng::kKvBlock - 2) / eng::kKvBlock + 1);
    ENG_CHECK(batch <= 0x7fffffffLL && n_kv_heads <= 0x7fffffffLL &&
                  batch * n_kv_heads <= 0x7fffffffLL / reach &&
                  eng::threads_fit((batch * n_kv_heads * reach + 1) / 2, eng::kWriteThreads),
              "kv_cache_write_q8: too many (sequence, head, block) units for one launch");
    const unsigned units = 2u * static_cast<unsigned>(batch * n_kv_heads * reach);
    const unsigned grid = (units + 3) / 4;
    auto go = [&](auto kernel) {
      kernel<<<grid, eng::kWriteThreads, 0, eng::as_stream(stream)>>>(
          reinterpret_cast<const _Float16*>(k_new), reinterpret_cast<const _Float16*>(v_new),
          k_cache, v_cache, k_scale, v_scale, pos, n_new, units, s_new, n_kv_heads, kv_max_seq_len,
          reach);
    };
    if (head_dim == 64) go(eng::kv_write_q8_kernel<64>);
    else go(eng::kv_write_q8_kernel<128>);
    ENG_LAUNCH_CHECK();
  });
}

int eng_attention_decode_q8(const eng_half* q, const uint8_t* k_cache, const uint8_t* v_cache,
                            const float* k_scale, const float* v_scale, eng_half* out,
                            const int32_t* kv_len, int64_t batch, int64_t n_heads,
                            int64_t n_kv_heads, int64_t head_dim, int64_t max_kv_len,
                            int64_t kv_max_seq_len, float scale, int split_kv, eng_stream stream) {
  return guarded([&] {
    ENG_CHECK(q != nullptr, "attention_decode_q8: q is null");
    ENG_CHECK(k_cache != nullptr, "attention_decode_q8: k_cache is null");
    ENG_CHECK(v_cache != nullptr, "attention_decode_q8: v_cache is null");
    ENG_CHECK(k_scale != nullptr && v_scale != nullptr, "attention_decode_q8: k_scale/v_scale is null");
    ENG_CHECK(out != nullptr, "attention_decode_q8: out is null");
    ENG_CHECK(kv_len != nullptr, "attention_decode_q8: kv_len is null");
    ENG_CHECK(batch >= 0, "attention_decode_q8: batch must be non-negative");
    ENG_CHECK(n_heads > 0, "attention_decode_q8: n_heads must be positive");
    ENG_CHECK(n_kv_heads > 0, "attention_decode_q8: n_kv_heads must be positive");
    ENG_CHECK(n_heads % n_kv_heads == 0,
              "attention_decode_q8: n_heads must be divisible by n_kv_heads");
    ENG_CHECK(head_dim == 64 || head_dim == 128, "attention_decode_q8: head_dim must be 64 or 128");
    ENG_CHECK(max_kv_len >= 0, "attention_decode_q8: max_kv_len must be non-negative");
    ENG_CHECK(kv_max_seq_len >= max_kv_len, "attention_decode_q8: kv_max_seq_len < max_kv_len");
    ENG_CHECK(kv_max_seq_len <= eng::kMaxLen,
              "attention_decode_q8: kv_max_seq_len must be below 2^31 - 32");
    ENG_CHECK(std::isfinite(scale), "attention_decode_q8: scale must be finite");
    ENG_CHECK(split_kv >= 0, "attention_decode_q8: split_kv must be non-negative");
    ENG_CHECK(eng::aligned_to(k_cache, 16) && eng::aligned_to(v_cache, 16),
              "attention_decode_q8: the caches must be 16-byte aligned");
    if (batch == 0) return;
    ENG_CHECK(batch <= 0x7fffffffLL && n_heads <= 0x7fffffffLL && batch * n_heads <= 0x7fffffffLL,
              "attention_decode_q8: too many (sequence, head) pairs for one launch");
    hipStream_t s = eng::as_stream(stream);
    if (max_kv_len == 0) {
      eng::fill_zero_async(out, static_cast<std::size_t>(batch * n_heads * head_dim) * sizeof(eng_half), s);
      return;
    }
    eng::AttnArgs a;
    a.q = reinterpret_cast<const _Float16*>(q);
    a.k = k_cache;
    a.v = v_cache;
    a.ks = k_scale;
    a.vs = v_scale;
    a.out = reinterpret_cast<_Float16*>(out);
    a.lens = kv_len;
    a.n_heads = n_heads;
    a.n_kv_heads = n_kv_heads;
    a.max_len = max_kv_len;
    a.kv_max = kv_max_seq_len;
    a.group = static_cast<int>(n_heads / n_kv_heads);
    a.tiles = (a.group + 15) / 16;
    a.scale = scale;
    const long long blocks = (max_kv_len + eng::kKvBlock - 1) / eng::kKvBlock;
    const long long want = split_kv == 0
                               ? eng::auto_splits(blocks, batch * n_kv_heads * a.tiles, head_dim)
                               : std::min<long long>({split_kv, blocks, 256});
    a.split_blocks =
        static_cast<int>(std::min((blocks + want - 1) / want, eng::kMaxSplitBlocks));
    a.nsplit = static_cast<int>((blocks + a.split_blocks - 1) / a.split_blocks);
    if (head_dim == 64) eng::run_decode<64>(a, batch, s);
    else eng::run_decode<128>(a, batch, s);
  });
}

}  // extern "C"
