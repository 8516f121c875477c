// attention_tiles.hpp -- attention of many query rows over a KV cache on the matrix
// cores: tiles of 128 rows by 64 keys, for prompts (causal, sliding window, sinks) and
// for the sequences of a batch that share a prefix (every row sees every key).
//
// Rows: the query heads of a KV head's group share its keys, so the rows of a unit (a
// sequence or a shared prefix, and a KV head) are its (token, head of the group) pairs,
// token-major. With k tokens of new queries (or k sequences over one prefix) the unit has
// k group rows: a KV head's keys are read once for all of them.
//
// Softmax in one pass: O = sum_j 2^(s_j - m) v_j and l = sum_j 2^(s_j - m) over the keys
// so far, s in units of log2, m the row's running maximum; both are rescaled when m rises.
#pragma once

#include "gemv_kernels.hpp"
#include "launch.hpp"

#include <algorithm>
#include <type_traits>

namespace eng {
namespace attn {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
typedef _Float16 halfx4 __attribute__((ext_vector_type(4)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef unsigned uintx2 __attribute__((ext_vector_type(2)));
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));

constexpr int kKvBlock = 32;  // tokens that share a scale in an 8-bit cache
constexpr float kNegInf = -__builtin_huge_valf();
constexpr float kLog2e = 1.4426950408889634f;
// V scales below this one count as it (their values vanish in an fp16 output either way).
constexpr float kLeastVScale = 0x1p-40f;
// The weights carry 2^kWeightShift and m rises only when a score passes it by kLazy, so
// that they reach 2^15 at the most and keep fp16's full precision down to 2^-21 of the
// largest; below, their step is 2^-31 of it.
constexpr float kLazy = 8.0f;
constexpr float kWeightShift = 7.0f;

// 2^(a - b), 0 for a == -inf whatever b is; NaN stays NaN.
__device__ __forceinline__ float weight2(float a, float b) {
  const float w = __builtin_amdgcn_exp2f(a - b);
  return a == kNegInf ? 0.0f : w;
}

// The largest of x over a lane and the lane 32 away.
__device__ __forceinline__ float pair_max(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
  const unsigned w = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  const unsigned r0 = r[0], r1 = r[1];
  x = fmaxf(__uint_as_float(r0), __uint_as_float(r1));
#endif
  return x;
}

// two e4m3 bytes (half H of a word) as fp16, exact
template <bool HI>
__device__ __forceinline__ halfx2 two_fp8([[maybe_unused]] unsigned w) {
  halfx2 r = {};
#if defined(__HIP_DEVICE_COMPILE__)
  r = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI);
#endif
  return r;
}
__device__ __forceinline__ halfx8 eight_fp8(unsigned w0, unsigned w1) {
  const halfx2 a = two_fp8<false>(w0), b = two_fp8<true>(w0);
  const halfx2 c = two_fp8<false>(w1), d = two_fp8<true>(w1);
  return halfx8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Four rows' worth of a column from LDS: lane i of 16 gets column i of the 4 x 16 fp16
// whose row r lanes 4 r .. 4 r + 3 point at, 8 bytes each.
__device__ __forceinline__ halfx4 read_transposed([[maybe_unused]] const _Float16* p) {
  halfx4 v = {};
#if defined(__HIP_DEVICE_COMPILE__)
  typedef short shortx4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) shortx4 lds_shortx4;
  v = __builtin_bit_cast(halfx4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_shortx4*)p));
#endif
  return v;
}

struct Args {
  const _Float16* q;
  _Float16* out;  // or, where part_o is set, states into part_o and part_ml
  const void* k;
  const void* v;
  const float* ks;
  const float* vs;
  // causal: token i of unit b stands at pos[b] + i, and the first n_new[b] (all where
  // null) of its s_new tokens are there; pos[b] < 0: none. Otherwise its s_new tokens
  // see the first pos[b] keys each.
  const int* pos;
  const int* n_new;
  long long kv_max;   // tokens that a cache has room for
  long long n_heads;
  int n_kv, group, s_new;
  int max_len;        // keys at or past it are not seen
  bool causal;
  long long window;   // 0: none
  int sinks;
  long long units;    // (sequence or prefix, KV head) pairs
  int row_tiles, nsplit;
  // State of row r's split s (r counts the rows of out): r part_stride + part0 + s.
  int part_stride, part0;
  float scale;
  float* part_o;
  float* part_ml;
};

// The tokens of a unit that are there, and the position of the first; none: n == 0.
struct Unit {
  long long p0;
  int n;
};
__device__ __forceinline__ Unit unit_of(const Args& a, long long b) {
  Unit u;
  u.p0 = a.pos[b];
  u.n = a.s_new;
  if (a.causal) {
    if (a.n_new != nullptr) u.n = min(u.n, a.n_new[b]);
    if (u.p0 < 0) u.n = 0;
  }
  return u;
}
// The keys that token t sees: [0, hi) without [sinks, lo).
struct Seen {
  int lo, hi;
};
__device__ __forceinline__ Seen seen_by(const Args& a, const Unit& u, int t) {
  const long long end = a.causal ? u.p0 + t + 1 : u.p0;
  Seen s;
  s.hi = static_cast<int>(std::min<long long>(std::max(end, 0ll), a.max_len));
  s.lo = a.window == 0 ? 0
                       : static_cast<int>(std::min<long long>(std::max(end - a.window, 0ll), a.max_len));
  return s;
}

constexpr int kTileRows = 128;
constexpr int kTileKeys = 64;
constexpr int kTileWaves = 4;

// One workgroup per (unit, 128 rows, split of their keys), 4 waves of 32 rows. K and V
// tiles of 64 keys pass through LDS in two buffers as fp16 (e4m3 codes are converted on
// the way, exact; a block's scale multiplies its scores, a V block's joins the weights as
// in decode_q8_kernel). Products on v_mfma_f32_32x32x16_f16: S^T = K . Q^T with K as the
// A operand leaves a row's scores in two lanes, O^T = V^T . P^T takes them in place as the
// B operand: element r of half-wave g is key 8 (r / 4) + 4 g + r % 4 of its 32, and V is
// read from LDS transposed (4 keys of a dim for each lane) in that order. A row of an LDS
// tile is D fp16; its 16-byte pieces are permuted by the row so that neither read has
// bank conflicts.
// Weights are rounded to fp16 (2^-11 of each at the most, as the output is); m, l, O are
// fp32 and l sums the weights before rounding.
template <int D, bool Q8>
__global__ __launch_bounds__(64 * kTileWaves, 2) void tile_kernel(Args a) {
  static_assert(D == 64 || D == 128, "head_dim 64 or 128");
  constexpr int CPR = D / 8;   // 16-byte pieces of an LDS row
  constexpr int KS = D / 16;   // k-steps of a score
  constexpr int DB = D / 32;   // 32-dim blocks of an output
  constexpr int TILE = kTileKeys * D;
  __shared__ __attribute__((aligned(16))) _Float16 s_k[2][TILE];
  __shared__ __attribute__((aligned(16))) _Float16 s_v[2][TILE];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31;
  const int half = lane >> 5;
  // the rows with the most keys first
  const unsigned units = static_cast<unsigned>(a.units);
  const unsigned rank = blockIdx.x / units;
  const unsigned unit = blockIdx.x - rank * units;
  const int rt = a.row_tiles - 1 - static_cast<int>(rank);
  const long long b = unit / static_cast<unsigned>(a.n_kv);
  const long long kvh = unit - b * a.n_kv;
  const int split = static_cast<int>(blockIdx.y);
  const Unit u = unit_of(a, b);
  const int rows = u.n * a.group;
  const int row0 = rt * kTileRows;
  if (row0 >= rows) return;

  // the workgroup's keys, as tiles: sinks first, then from the window's start on
  const unsigned group = static_cast<unsigned>(a.group);
  const int tok_first = static_cast<int>(static_cast<unsigned>(row0) / group);
  const int tok_last = static_cast<int>(static_cast<unsigned>(min(row0 + kTileRows, rows) - 1) / group);
  const int hi = seen_by(a, u, tok_last).hi;
  const int lo = seen_by(a, u, tok_first).lo;
  const int sink_end = min(min(a.sinks, lo), hi);
  const int sink_tiles = (sink_end + kTileKeys - 1) / kTileKeys;
  const int start = max(lo / kKvBlock * kKvBlock, sink_tiles * kTileKeys);
  const int tiles = sink_tiles + (hi > start ? (hi - start + kTileKeys - 1) / kTileKeys : 0);
  const int per = (tiles + a.nsplit - 1) / a.nsplit;
  const int t0 = min(split * per, tiles);
  const int t1 = min(t0 + per, tiles);
  auto base_of = [&](int t) { return t < sink_tiles ? t * kTileKeys : start + (t - sink_tiles) * kTileKeys; };

  // the wave's rows, and this lane's
  const int wrow = row0 + 32 * wave;
  const int r = min(wrow + col, rows - 1);
  const int tok = static_cast<int>(static_cast<unsigned>(r) / group);
  const Seen mine = seen_by(a, u, tok);
  const Seen first = seen_by(a, u, static_cast<int>(static_cast<unsigned>(min(wrow, rows - 1)) / group));
  const Seen last = seen_by(a, u, static_cast<int>(static_cast<unsigned>(min(wrow + 31, rows - 1)) / group));
  const long long orow = (b * a.s_new + tok) * a.n_heads + kvh * a.group + (r - tok * a.group);

  halfx8 qf[KS];
  {
    const _Float16* qp = a.q + orow * D + 8 * half;
    if ((reinterpret_cast<std::uintptr_t>(a.q) & 15) == 0) {
#pragma unroll
      for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const halfx8*>(qp + 16 * s);
    } else {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
#pragma unroll
        for (int j = 0; j < 8; ++j) qf[s][j] = qp[16 * s + j];
      }
    }
    if (a.scale < 0.0f) {
#pragma unroll
      for (int s = 0; s < KS; ++s) qf[s] = -qf[s];
    }
  }
  const float scale2 = fabsf(a.scale) * kLog2e;

  const long long bh = b * a.n_kv + kvh;
  using Elem = std::conditional_t<Q8, unsigned char, _Float16>;
  const Elem* kg = static_cast<const Elem*>(a.k) + bh * a.kv_max * D;
  const Elem* vg = static_cast<const Elem*>(a.v) + bh * a.kv_max * D;
  [[maybe_unused]] const long long sb = bh * ((a.kv_max + kKvBlock - 1) / kKvBlock);
  auto swz = [](int row) { return D == 128 ? (row & 7) << 1 : ((row >> 1) & 3) << 1; };

  // ---- global to LDS. Keys past the last one are taken as the last one: finite where it
  // is, and masked.
  constexpr int LOADS = Q8 ? TILE / 16 / 256 : 1;
  [[maybe_unused]] uintx4 rk[LOADS], rv[LOADS];
  float ks_at[2][2] = {}, vs_at[2][2] = {};  // scales of the tile in use and the next one's
  auto stage = [&]([[maybe_unused]] int t, [[maybe_unused]] int buf) __attribute__((always_inline)) {
    if constexpr (!Q8) {
      const int base = base_of(t);
      constexpr int RPI = 64 / CPR;  // rows of a wave load
#pragma unroll
      for (int i = 0; i < TILE / 512 / kTileWaves; ++i) {
        const int ins = i * kTileWaves + wave;
        const int row = ins * RPI + lane / CPR;
        const int piece = (lane % CPR) ^ swz(row);
        const long long at = static_cast<long long>(min(base + row, hi - 1)) * D + 8 * piece;
        dma16(kg + at, &s_k[buf][ins * 512]);
        dma16(vg + at, &s_v[buf][ins * 512]);
      }
    }
  };
  auto fetch = [&]([[maybe_unused]] int t) __attribute__((always_inline)) {
    if constexpr (Q8) {
      const int base = base_of(t);
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int n = i * 256 + tid;
        const int row = n / (D / 16);
        const long long at = static_cast<long long>(min(base + row, hi - 1)) * D + 16 * (n % (D / 16));
        rk[i] = *reinterpret_cast<const uintx4*>(kg + at);
        rv[i] = *reinterpret_cast<const uintx4*>(vg + at);
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int blk = min(base / kKvBlock + s, (hi - 1) / kKvBlock);
        ks_at[1][s] = a.ks[sb + blk];
        vs_at[1][s] = a.vs[sb + blk];
      }
    }
  };
  auto put = [&]([[maybe_unused]] int buf) __attribute__((always_inline)) {
    if constexpr (Q8) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int n = i * 256 + tid;
        const int row = n / (D / 16);
        const int at = row * D + 8 * ((2 * (n % (D / 16))) ^ swz(row));
        *reinterpret_cast<halfx8*>(&s_k[buf][at]) = eight_fp8(rk[i][0], rk[i][1]);
        *reinterpret_cast<halfx8*>(&s_k[buf][at + 8]) = eight_fp8(rk[i][2], rk[i][3]);
        *reinterpret_cast<halfx8*>(&s_v[buf][at]) = eight_fp8(rv[i][0], rv[i][1]);
        *reinterpret_cast<halfx8*>(&s_v[buf][at + 8]) = eight_fp8(rv[i][2], rv[i][3]);
      }
    }
  };

  // ---- LDS addresses of the fragments
  const int kswz = swz(col);
  const int vrow = 4 * half + ((lane & 15) >> 2);  // + 16 s + 8 j + 32 sub
  const int vswz = swz(vrow);
  int vat[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d)
    vat[d] = vrow * D + 8 * ((4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ vswz) + 4 * (lane & 1);

  // Sixteen keys of V from `key0` on (A operand): infinities and NaN taken out, and added
  // to acc for the rows that see them, their number found by a product with 0 and 1.
  auto apart = [&](halfx8 av, int key0, floatx16& acc) __attribute__((always_inline)) {
    bool any = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) any |= !(fabsf(static_cast<float>(av[j])) < __builtin_huge_valf());
    if (!__any(any)) return av;
    halfx8 sees, kind[3], clean;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int key = key0 + 8 * (j >> 2) + 4 * half + (j & 3);
      sees[j] = static_cast<_Float16>(key < mine.hi && (key >= mine.lo || key < a.sinks) ? 1.0f : 0.0f);
      const float x = static_cast<float>(av[j]);
      kind[0][j] = static_cast<_Float16>(x == __builtin_huge_valf() ? 1.0f : 0.0f);
      kind[1][j] = static_cast<_Float16>(x == kNegInf ? 1.0f : 0.0f);
      kind[2][j] = static_cast<_Float16>(x != x ? 1.0f : 0.0f);
      clean[j] = fabsf(x) < __builtin_huge_valf() ? av[j] : static_cast<_Float16>(0.0f);
    }
#pragma unroll
    for (int n = 0; n < 3; ++n) {
      floatx16 c = {};
#if defined(__HIP_DEVICE_COMPILE__)
      c = __builtin_amdgcn_mfma_f32_32x32x16_f16(kind[n], sees, c, 0, 0, 0);
#endif
      const float x = n == 0 ? __builtin_huge_valf() : n == 1 ? kNegInf : __builtin_nanf("");
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[e] += c[e] > 0.0f ? x : 0.0f;
    }
    return clean;
  };

  float m, l;
  floatx16 o[DB];
  bool careful = false;  // the second time: V's infinities and NaN kept from rows that do not see them
  for (;;) {
    m = kNegInf;
    l = 0.0f;
#pragma unroll
    for (int d = 0; d < DB; ++d) {
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;
    }
    if (t0 < t1) {
      if constexpr (Q8) {
        fetch(t0);
        put(0);
#pragma unroll
        for (int s = 0; s < 2; ++s) ks_at[0][s] = ks_at[1][s], vs_at[0][s] = vs_at[1][s];
        if (t0 + 1 < t1) fetch(t0 + 1);
      } else {
        stage(t0, 0);
      }
    }
    for (int t = t0; t < t1; ++t) {
      const int buf = (t - t0) & 1;
      float f[2], lv[2], ivs[2];
      if constexpr (Q8) {
        lds_barrier();  // the tile is written, the other buffer read
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          // (at least 1e-30, so that a mask's -inf stays -inf under a scale of zero)
          f[s] = fmaxf(scale2 * ks_at[0][s], 1e-30f);
          const float vs = fmaxf(vs_at[0][s], kLeastVScale);
          lv[s] = __builtin_amdgcn_logf(vs);
          ivs[s] = __builtin_amdgcn_rcpf(vs);
        }
        if (t + 1 < t1) {
          put(buf ^ 1);
#pragma unroll
          for (int s = 0; s < 2; ++s) ks_at[0][s] = ks_at[1][s], vs_at[0][s] = vs_at[1][s];
          if (t + 2 < t1) fetch(t + 2);
        }
      } else {
#if defined(__HIP_DEVICE_COMPILE__)
        __builtin_amdgcn_s_waitcnt(vmcnt_le(0));
#endif
        lds_barrier();
        if (t + 1 < t1) stage(t + 1, buf ^ 1);
        f[0] = f[1] = fmaxf(scale2, 1e-30f);
        lv[0] = lv[1] = 0.0f;
        ivs[0] = ivs[1] = 1.0f;
      }
      const int base = base_of(t);
      if (base >= last.hi || (base >= a.sinks && base + kTileKeys <= first.lo)) continue;  // (uniform) unseen

      floatx16 sc[2];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[s][e] = 0.0f;
#pragma unroll
        for (int st = 0; st < KS; ++st) {
          [[maybe_unused]] const halfx8 ka = *reinterpret_cast<const halfx8*>(
              &s_k[buf][(32 * s + col) * D + 8 * ((2 * st + half) ^ kswz)]);
#if defined(__HIP_DEVICE_COMPILE__)
          sc[s] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, qf[st], sc[s], 0, 0, 0);
#endif
        }
      }
      const bool whole = base + kTileKeys <= first.hi && (last.lo <= base || base + kTileKeys <= a.sinks);
      if (!whole) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int j = base + 32 * s + 8 * (e >> 2) + 4 * half + (e & 3);
            if (j >= mine.hi || (j < mine.lo && j >= a.sinks)) sc[s][e] = kNegInf;
          }
        }
      }
      float mx = kNegInf;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        float x = sc[s][0];
#pragma unroll
        for (int e = 1; e < 16; ++e) x = fmaxf(x, sc[s][e]);
        mx = fmaxf(mx, fmaf(x, f[s], lv[s]));
      }
      mx = pair_max(mx);
      if (__any(mx > m + kLazy)) {
        const float mn = fmaxf(m, mx);
        const float alpha = weight2(m, mn);
        m = mn;
        l *= alpha;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] *= alpha;
      }
      const float ref = m == kNegInf ? 0.0f : m - kWeightShift;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const float add = lv[s] - ref;
        float ls = 0.0f;
        halfx8 pb[2];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float p = __builtin_amdgcn_exp2f(fmaf(sc[s][e], f[s], add));
          ls += p;
          pb[e >> 3][e & 7] = static_cast<_Float16>(p);
        }
        l = fmaf(ls, ivs[s], l);
#pragma unroll
        for (int st = 0; st < 2; ++st) {
#pragma unroll
          for (int d = 0; d < DB; ++d) {
            halfx8 av = {};
#if defined(__HIP_DEVICE_COMPILE__)
            const _Float16* vp = &s_v[buf][vat[d] + (32 * s + 16 * st) * D];
            const halfx4 v0 = read_transposed(vp), v1 = read_transposed(vp + 8 * D);
            av = halfx8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
#endif
            if (careful && !whole) av = apart(av, base + 32 * s + 16 * st, o[d]);
#if defined(__HIP_DEVICE_COMPILE__)
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(av, pb[st], o[d], 0, 0, 0);
#endif
          }
        }
      }
    }
    if (careful) break;
    float sum = 0.0f;
#pragma unroll
    for (int d = 0; d < DB; ++d) {
#pragma unroll
      for (int e = 0; e < 16; ++e) sum = fmaf(o[d][e], 0.0f, sum);
    }
    if (!__syncthreads_or(sum != sum)) break;
    careful = true;
  }

  l += __shfl_xor(l, 32);
  if (wrow + col >= rows) return;
  if (a.part_o != nullptr) {
    const long long slot = orow * a.part_stride + a.part0 + split;
#pragma unroll
    for (int d = 0; d < DB; ++d) {
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<floatx4*>(a.part_o + slot * D + 32 * d + 2 * e + 4 * half) =
            floatx4{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
    }
    if (half == 0) *reinterpret_cast<floatx2*>(a.part_ml + 2 * slot) = floatx2{m, l};
    return;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (no key seen: zeros)
  _Float16* op = a.out + orow * D + 4 * half;
  const bool aligned = (reinterpret_cast<std::uintptr_t>(a.out) & 7) == 0;
#pragma unroll
  for (int d = 0; d < DB; ++d) {
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      halfx4 y;
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = static_cast<_Float16>(o[d][e + j] * inv);
      _Float16* at = op + 32 * d + 2 * e;
      if (aligned) {
        *reinterpret_cast<halfx4*>(at) = y;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) at[j] = y[j];
      }
    }
  }
}

}  // namespace attn
}  // namespace eng
