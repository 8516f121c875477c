// attention_tiles.hpp -- attention of many query rows over a KV cache on the matrix
// cores: tiles of 128 or 256 rows by 64 keys, for prompts (causal, sliding window, sinks)
// and for the sequences of a batch that share a prefix (every row sees every key).
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

// 2^(a - b), 0 for a == -inf whatever b is, else at least 2^-126, so that a state's
// infinity stays one; NaN stays NaN.
__device__ __forceinline__ float weight2(float a, float b) {
  const float w = __builtin_amdgcn_exp2f(a - b);
  return a == kNegInf ? 0.0f : w < 0x1p-126f ? 0x1p-126f : w;
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
    // (below zero none: times the group it could come out above it)
    if (a.n_new != nullptr) u.n = max(min(u.n, a.n_new[b]), 0);
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

constexpr int kTileKeys = 64;
// LDS buffers of a tile of NW waves.
constexpr int tile_buffers(int NW) { return NW == 8 ? 3 : 2; }

// One workgroup per (unit, tile of 32 NW rows, split of their keys), NW waves of 32 rows.
// K and V tiles of 64 keys pass through LDS as fp16, by way of registers, K and V in turn
// (8-bit codes are converted on the way, exact; a K block's scale multiplies its scores, a
// V block's joins the weights as in few_kernel). Products on v_mfma_f32_32x32x16_f16: S^T =
// K . Q^T with K as the A operand leaves a row's scores in two lanes, O^T = V^T . P^T takes
// them in place as the B operand: element r of half-wave g is key 8 (r / 4) + 4 g + r % 4
// of its 32, and V is read from LDS transposed (4 keys of a dim for each lane) in that
// order. A row of an LDS tile is D fp16; its 16-byte pieces are permuted by the row so that
// neither read has bank conflicts: 235 bytes a clock and CU for K, 148 for V, against 123
// and 122 for one permutation that suits V's rows only.
//
// A wave takes 32 keys at a time. The exponentials of 32 keys' scores (16 of 12 cycles, as
// many multiply-adds, additions and halves of maxima and conversions) are issued among the
// matrix products of the next 32 keys' scores, then come the products with V; two waves on
// a SIMD fill each other's gaps. K fragments are read one such step ahead. Eight waves share
// a tile where that leaves a workgroup for every CU; else four, two workgroups to a CU, and
// at D = 64, with three to a CU, always (prompts of 777 tokens, window 256: 36 us, 49 with
// eight waves). The four-wave forms at D = 128 fill their 256 registers and spill 16 (8-bit)
// and 40 bytes (fp16) a lane.
// Bound by the matrix cores and power together, and by the longest of one workgroup to a
// CU: 2048 tokens after 6144, 32 / 8 heads of 128: 277-282 us, 870 TFLOP/s, at 1.8 to 2.1
// GHz (a large fp16 product of the library's 1175).
// Slower: the two waves of a SIMD one phase apart, exponentials against products, by
// barriers (309; a phase then waits for its own latencies); 64 rows to a wave, half the LDS
// reads (376 to 442; the compiler moves values between the register files); direct loads
// to LDS (their wait covers the next tile's: 638 TFLOP/s).
// Weights are rounded to fp16 (2^-11 of each at the most, as the output is); m, l, O are
// fp32 and l sums the weights before rounding.
//
// A NaN or an infinity in a V row would reach, as 0 times it, rows that do not see its
// key. So where a workgroup's sums are not all finite it computes them again with such
// values taken out and added for the rows that see them (careful_pass, about six times the
// time).
template <int D, bool Q8, int NW>
__global__ __launch_bounds__(64 * NW, D == 64 ? 3 : 2) void tile_kernel(Args a) {
  constexpr int kRows = 32 * NW;
  constexpr int NB = tile_buffers(NW);
  static_assert(D == 64 || D == 128, "head_dim 64 or 128");
  constexpr int CPR = D / 8;   // 16-byte pieces of an LDS row
  constexpr int KS = D / 16;   // k-steps of a score
  constexpr int DB = D / 32;   // 32-dim blocks of an output
  constexpr int TILE = kTileKeys * D;
  extern __shared__ __attribute__((aligned(16))) _Float16 s_tiles[];  // K [NB][TILE], V [NB][TILE]
  __shared__ __attribute__((aligned(16))) float s_scale[NB][2][4];  // of 32 keys: f, lv, 1 / v scale
  _Float16* const s_k = s_tiles;
  _Float16* const s_v = s_tiles + NB * TILE;

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
  const int row0 = rt * kRows;
  if (row0 >= rows) return;

  // the workgroup's keys, as tiles: sinks first, then from the window's start on
  const unsigned group = static_cast<unsigned>(a.group);
  auto token_of = [&](int r) { return static_cast<int>(static_cast<unsigned>(r) / group); };
  const int hi = seen_by(a, u, token_of(min(row0 + kRows, rows) - 1)).hi;
  const int lo = seen_by(a, u, token_of(row0)).lo;
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
  const Seen first = seen_by(a, u, token_of(min(wrow, rows - 1)));
  const Seen last = seen_by(a, u, token_of(min(wrow + 31, rows - 1)));
  const int r = min(wrow + col, rows - 1);
  const int tok = token_of(r);
  const Seen mine = seen_by(a, u, tok);
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
  auto k_swz = [](int row) { return D == 128 ? row & 15 : (row >> 1) & 7; };
  auto v_swz = [](int row) { return D == 128 ? (row & 3) << 2 : (row & 3) << 1; };

  // ---- global to LDS, by way of registers. Keys past the last one are taken as the last
  // one, and masked.
  constexpr int PIECES = TILE * static_cast<int>(sizeof(Elem)) / 16;
  constexpr int LOADS = PIECES / (64 * NW);
  static_assert(LOADS * 64 * NW == PIECES, "whole loads");
  constexpr int LPR = D * static_cast<int>(sizeof(Elem)) / 16;  // loads of a row
  uintx4 raw[LOADS];  // of K or V
  [[maybe_unused]] float raw_ks = 0.0f, raw_vs = 0.0f;
  auto fetch = [&](int t, const Elem* g) __attribute__((always_inline)) {
    const int base = base_of(t);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int n = i * 64 * NW + tid;
      const long long at = static_cast<long long>(min(base + n / LPR, hi - 1)) * D + (n % LPR) * (D / LPR);
      raw[i] = *reinterpret_cast<const uintx4*>(g + at);
    }
  };
  auto put = [&](_Float16* tile, auto swz) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int n = i * 64 * NW + tid;
      const int row = n / LPR;
      const int piece = n % LPR;
      if constexpr (Q8) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
          *reinterpret_cast<halfx8*>(tile + row * D + 8 * ((2 * piece + j) ^ swz(row))) =
              eight_fp8(raw[i][2 * j], raw[i][2 * j + 1]);
      } else {
        *reinterpret_cast<uintx4*>(tile + row * D + 8 * (piece ^ swz(row))) = raw[i];
      }
    }
  };
  auto fetch_k = [&](int t) __attribute__((always_inline)) {  // and the scales of both
    fetch(t, kg);
    if constexpr (Q8) {
      const long long blk = sb + min(base_of(t) / kKvBlock + (tid & 1), (hi - 1) / kKvBlock);
      raw_ks = a.ks[blk];
      raw_vs = a.vs[blk];
    }
  };
  auto fetch_v = [&](int t) __attribute__((always_inline)) { fetch(t, vg); };
  auto put_k = [&](int buf) __attribute__((always_inline)) {
    put(s_k + buf * TILE, k_swz);
    if constexpr (Q8) {
      if (tid < 2) {
        // (at least 1e-30, so that a mask's -inf stays -inf under a scale of zero)
        const float vs = fmaxf(raw_vs, kLeastVScale);
        *reinterpret_cast<floatx4*>(s_scale[buf][tid]) =
            floatx4{fmaxf(scale2 * raw_ks, 1e-30f), __builtin_amdgcn_logf(vs), __builtin_amdgcn_rcpf(vs), 0.0f};
      }
    }
  };
  auto put_v = [&](int buf) __attribute__((always_inline)) { put(s_v + buf * TILE, v_swz); };
  // The factor of a 32-key block's scores, log2 and inverse of its V scale.
  struct Scale {
    float f, lv, ivs;
  };
  auto scale_of = [&](int buf, int sub) __attribute__((always_inline)) {
    if constexpr (Q8) {
      const floatx4 x = *reinterpret_cast<const floatx4*>(s_scale[buf][sub]);
      return Scale{x[0], x[1], x[2]};
    } else {
      return Scale{fmaxf(scale2, 1e-30f), 0.0f, 1.0f};
    }
  };

  // ---- LDS addresses of the fragments
  const int kswz = k_swz(col);
  const int vrow = 4 * half + ((lane & 15) >> 2);  // + 16 s + 8 j + 32 sub
  const int vswz = v_swz(vrow);
  int vat[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d)
    vat[d] = vrow * D + 8 * ((4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ vswz) + 4 * (lane & 1);

  float m, l;
  floatx16 o[DB];
  auto clear = [&]() __attribute__((always_inline)) {
    m = kNegInf;
    l = 0.0f;
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = floatx16{};
  };
  // What a phase of products takes: fragments of K and V, and the weights.
  halfx8 kf[KS], vf[2][DB], pb[2];
  struct Scores {
    floatx16 x;
  };
  Scores even, odd;  // of a tile's first and second 32 keys
  auto read_k = [&](int buf, int sub) __attribute__((always_inline)) {
#pragma unroll
    for (int st = 0; st < KS; ++st)
      kf[st] = *reinterpret_cast<const halfx8*>(s_k + buf * TILE + (32 * sub + col) * D +
                                                8 * ((2 * st + half) ^ kswz));
  };
  auto read_v = [&](int buf, int sub) __attribute__((always_inline)) {
#pragma unroll
    for (int st = 0; st < 2; ++st) {
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const _Float16* vp = s_v + buf * TILE + vat[d] + (32 * sub + 16 * st) * D;
        const halfx4 v0 = read_transposed(vp), v1 = read_transposed(vp + 8 * D);
        vf[st][d] = halfx8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
      }
    }
  };
  auto scores = [&](Scores& s) __attribute__((always_inline)) {
    floatx16 sc = {};
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
    for (int st = 0; st < KS; ++st) sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[st], qf[st], sc, 0, 0, 0);
#endif
    s.x = sc;
  };
  auto products = [&]() __attribute__((always_inline)) {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
    for (int st = 0; st < 2; ++st) {
#pragma unroll
      for (int d = 0; d < DB; ++d)
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[st][d], pb[st], o[d], 0, 0, 0);
    }
#endif
  };
  auto whole = [&](int key0) {  // 32 keys, seen by all rows of the wave
    return key0 + kKvBlock <= first.hi && (last.lo <= key0 || key0 + kKvBlock <= a.sinks);
  };
  auto seen = [&](int key0, int keys) {  // by any
    return key0 < last.hi && (key0 + keys > first.lo || key0 < a.sinks);
  };
  // 32 keys' scores: hidden ones to -inf. An element's key is a constant from the lane's
  // first one on, so either end costs a comparison with it and a select.
  auto mask = [&](Scores& s, int key0) __attribute__((always_inline)) {
    const int at = key0 + 4 * half;
    if (key0 < a.sinks) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int j = at + 8 * (e >> 2) + (e & 3);
        s.x[e] = (j < mine.lo) & (j >= a.sinks) ? kNegInf : s.x[e];
      }
    } else if (last.lo > key0) {
      const int lo = mine.lo - at;
#pragma unroll
      for (int e = 0; e < 16; ++e) s.x[e] = 8 * (e >> 2) + (e & 3) < lo ? kNegInf : s.x[e];
    }
    if (key0 + kKvBlock > first.hi) {
      const int hi = mine.hi - at;
#pragma unroll
      for (int e = 0; e < 16; ++e) s.x[e] = 8 * (e >> 2) + (e & 3) >= hi ? kNegInf : s.x[e];
    }
  };
  auto largest = [&](const Scores& s, const Scale& c) __attribute__((always_inline)) {
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = fmaxf(fmaxf(s.x[e], s.x[e + 4]), fmaxf(s.x[e + 8], s.x[e + 12]));
    return pair_max(fmaf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), c.f, c.lv));
  };
  auto raise = [&](float mx) __attribute__((always_inline)) {
    if (!__any(mx > m + kLazy)) return;
    const float mn = fmaxf(m, mx);
    const float alpha = weight2(m, mn);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] *= alpha;
  };
  auto weigh = [&](const Scores& s, const Scale& c) __attribute__((always_inline)) {
    const float add = c.lv - (m == kNegInf ? 0.0f : m - kWeightShift);
    float ls[4] = {};
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float p = __builtin_amdgcn_exp2f(fmaf(s.x[e], c.f, add));
      ls[e & 3] += p;
      pb[e >> 3][e & 7] = static_cast<_Float16>(p);
    }
    l = fmaf((ls[0] + ls[1]) + (ls[2] + ls[3]), c.ivs, l);
  };

  clear();
  if (t0 < t1) {
    // (tiles past the last one are taken as the last one, and not used)
    auto at_most = [&](int t) { return min(t, t1 - 1); };
    fetch_k(t0);
    put_k(0);
    fetch_v(t0);
    put_v(0);
    if constexpr (NB == 3) {
      fetch_k(at_most(t0 + 1));
      put_k(1);
      fetch_v(at_most(t0 + 1));
      put_v(1);
    }
    fetch_k(at_most(t0 + NB - 1));
    float mx = 0.0f;
    bool primed = false;  // `even` holds the tile's scores, mx their largest, kf the second keys
    int buf = 0;
    for (int t = t0; t < t1; ++t) {
      // NB == 3: all waves are done with the tile before this one, whose buffer the tile
      // after the next takes; this one and the next are in LDS. NB == 2: the next one takes
      // it, and is there for the second 32 keys.
      const int next = buf + 1 == NB ? 0 : buf + 1;
      const int free = (buf + NB - 1) % NB;
      lds_barrier();
      const int base = base_of(t);
      if (seen(base, kTileKeys)) {
        const bool one = seen(base, kKvBlock), two = seen(base + kKvBlock, kKvBlock);
        Scale c = scale_of(buf, 0);
        if (!primed) {
          read_k(buf, 0);
          scores(even);
          read_k(buf, 1);
          mx = largest(even, c);
        }
        if (!whole(base)) {
          mask(even, base);
          mx = largest(even, c);
        }
        raise(mx);
        if (one) {
          read_v(buf, 0);
          put_k(free);
          fetch_v(at_most(t + NB - 1));
          scores(odd);
          weigh(even, c);
          if constexpr (NB == 3) read_k(next, 0);
          products();
        } else {
          put_k(free);
          fetch_v(at_most(t + NB - 1));
          scores(odd);
          if constexpr (NB == 3) read_k(next, 0);
        }
        c = scale_of(buf, 1);
        mx = largest(odd, c);
        if (!whole(base + kKvBlock)) {
          mask(odd, base + kKvBlock);
          mx = largest(odd, c);
        }
        raise(mx);
        if constexpr (NB == 2) {
          lds_barrier();
          read_k(next, 0);
        }
        if (two) {
          read_v(buf, 1);
          put_v(free);
          fetch_k(at_most(t + NB));
          if constexpr (NB == 3) scores(even);
          weigh(odd, c);
          if constexpr (NB == 2) scores(even);
          read_k(next, 1);
          products();
        } else {
          put_v(free);
          fetch_k(at_most(t + NB));
          scores(even);
          read_k(next, 1);
        }
        mx = largest(even, scale_of(next, 0));
        primed = t + 1 < t1;
      } else {
        put_k(free);
        fetch_v(at_most(t + NB - 1));
        if constexpr (NB == 2) lds_barrier();
        put_v(free);
        fetch_k(at_most(t + NB));
        primed = false;
      }
      buf = next;
    }
  }

  // Tile by tile as above, one phase after the other, values that are not finite kept apart.
  auto careful_pass = [&]() {
    clear();
    for (int t = t0; t < t1; ++t) {
      __syncthreads();
      fetch_k(t);
      put_k(0);
      fetch_v(t);
      put_v(0);
      __syncthreads();
#pragma unroll 1
      for (int sub = 0; sub < 2; ++sub) {
        const int key0 = base_of(t) + kKvBlock * sub;
        if (!seen(key0, kKvBlock)) continue;
        read_k(0, sub);
        read_v(0, sub);
        scores(even);
        const Scale c = scale_of(0, sub);
        mask(even, key0);
        raise(largest(even, c));
        weigh(even, c);
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          halfx8 sees;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int key = key0 + 16 * st + 8 * (j >> 2) + 4 * half + (j & 3);
            sees[j] = static_cast<_Float16>(key < mine.hi && (key >= mine.lo || key < a.sinks) ? 1.0f : 0.0f);
          }
#pragma unroll
          for (int d = 0; d < DB; ++d) {
            halfx8 clean, kind[3];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float x = static_cast<float>(vf[st][d][j]);
              kind[0][j] = static_cast<_Float16>(x == __builtin_huge_valf() ? 1.0f : 0.0f);
              kind[1][j] = static_cast<_Float16>(x == kNegInf ? 1.0f : 0.0f);
              kind[2][j] = static_cast<_Float16>(x != x ? 1.0f : 0.0f);
              clean[j] = fabsf(x) < __builtin_huge_valf() ? vf[st][d][j] : static_cast<_Float16>(0.0f);
            }
            // how many infinities and NaN a row sees in a dim
#pragma unroll
            for (int n = 0; n < 3; ++n) {
              floatx16 count = {};
#if defined(__HIP_DEVICE_COMPILE__)
              count = __builtin_amdgcn_mfma_f32_32x32x16_f16(kind[n], sees, count, 0, 0, 0);
#endif
              const float x = n == 0 ? __builtin_huge_valf() : n == 1 ? kNegInf : __builtin_nanf("");
#pragma unroll
              for (int e = 0; e < 16; ++e) o[d][e] += count[e] > 0.0f ? x : 0.0f;
            }
#if defined(__HIP_DEVICE_COMPILE__)
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(clean, pb[st], o[d], 0, 0, 0);
#endif
          }
        }
      }
    }
    // (a row without a score above -inf: none of them)
    if (m == kNegInf && l + __shfl_xor(l, 32) == 0.0f) {
#pragma unroll
      for (int d = 0; d < DB; ++d) o[d] = floatx16{};
    }
  };
  float sum = 0.0f;
#pragma unroll
  for (int d = 0; d < DB; ++d) {
#pragma unroll
    for (int e = 0; e < 16; ++e) sum = fmaf(o[d][e], 0.0f, sum);
  }
  if (__syncthreads_or(sum != sum)) careful_pass();

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
