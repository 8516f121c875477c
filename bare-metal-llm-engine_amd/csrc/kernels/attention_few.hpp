// attention_few.hpp -- attention of a few query rows that see the same keys: one token of
// each sequence, or a few sequences over a shared prefix. Bound by the caches' bytes.
#pragma once

#include "attention_tiles.hpp"

namespace eng {
namespace attn {

constexpr int kFewRows = 16;   // rows of a tile

// One workgroup per (unit, tile of 16 rows, split of the unit's keys), NW waves; a wave
// takes every NW-th block of 32 keys straight from memory into registers, two blocks in
// flight. Both products are on v_mfma_f32_16x16x32_f16: S^T = K . Q^T with K as the A
// operand, whose row i is key (i / 4) + 4 (i % 4) of 16, so that accumulator element r of
// lane group g is key g + 4 r; O^T = V^T . P^T takes the scores in place as the B operand,
// the keys that a lane group loads of V. Weights enter as two fp16 terms (22 bits). 8-bit
// codes are converted to fp16, exact, K's scale multiplies the scores and V's joins the
// weights: with s' = s + log2(v scale), 2^(s' - m) multiplies the codes themselves and
// 2^(s' - m) / (v scale) adds to l.
//
// The keys are [0, hi) without [sinks, lo) and a block's loads go through a descriptor
// that ends with its last key, so rows past it read as zeros; values of hidden keys before
// the window are set to zero, so nothing of either reaches a sum. An infinity that is seen
// would meet weights' second terms of 0. So a wave whose sums are not all finite computes
// them again with V's infinities and NaN taken out, and adds these: its rows all see them.
// (Of 8-bit values only NaN is not finite, and stays it. The question costs 0.2 us.)
//
// Bound by the caches' bytes: one token of 16 sequences of up to 8192, window 4096, 32 / 8
// heads of 128, 8-bit: 135 MB in 25 us, 5.4 TB/s; eight groups of four beams over 4096
// tokens of 32 heads 252 MB in 51 us. (On tile_kernel, whose tiles a few rows leave empty, 77
// and 164.) Up to 128 rows over one prefix the L2 serves the tiles after the first: 32
// sequences, 8 heads of 128, 8192 tokens 31 us, 63 MB.
template <int D, bool Q8, int NW>
__global__ __launch_bounds__(64 * NW, 2) void few_kernel(Args a0, Args a1, unsigned wgs0) {
  static_assert(D == 64 || D == 128, "head_dim 64 or 128");
  constexpr int KS = D / 32;            // 32-dim steps of a score
  constexpr int ES = Q8 ? 1 : 2;        // bytes of a value
  constexpr int KL = D * ES / 64;       // 16-byte loads of a key per lane
  constexpr int VW = D / 16;            // dims of a value per lane
  constexpr int VD = VW * ES / 4;       // in 32-bit words
  constexpr int kBlockBytes = kKvBlock * D * ES;
  constexpr int WS = kFewRows * (D + 2);  // a wave's state in LDS: o, m, l
  __shared__ __attribute__((aligned(16))) float s_state[NW * WS];

  const bool second = blockIdx.x >= wgs0;
  const Args& a = second ? a1 : a0;
  const unsigned id = second ? blockIdx.x - wgs0 : blockIdx.x;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15;
  const int grp = lane >> 4;
  // id = (tile nsplit + split) units + unit: the tiles of a split share an XCD's L2 where
  // units nsplit is a multiple of 8
  const unsigned units = static_cast<unsigned>(a.units);
  const unsigned rest = id / units;
  const unsigned unit = id - rest * units;
  const int tile = static_cast<int>(rest / static_cast<unsigned>(a.nsplit));
  const int split = static_cast<int>(rest) - tile * a.nsplit;
  const long long b = unit / static_cast<unsigned>(a.n_kv);
  const long long kvh = unit - b * a.n_kv;
  const Unit u = unit_of(a, b);
  const unsigned group = static_cast<unsigned>(a.group);
  const int rows = u.n * a.group;
  if (kFewRows * tile >= rows) return;
  auto out_row = [&](int r) {
    const unsigned tok = static_cast<unsigned>(r) / group;
    return (b * a.s_new + tok) * a.n_heads + kvh * a.group + (r - static_cast<int>(tok * group));
  };

  const Seen see = seen_by(a, u, 0);
  const int sink_end = min(min(a.sinks, see.lo), see.hi);
  const int sink_blocks = (sink_end + kKvBlock - 1) / kKvBlock;
  const int start = max(see.lo / kKvBlock, sink_blocks);
  const int end = (see.hi + kKvBlock - 1) / kKvBlock;
  const int blocks = sink_blocks + max(end - start, 0);
  const int per = (blocks + a.nsplit - 1) / a.nsplit;
  const int t0 = min(split * per, blocks);
  const int n = min(per, blocks - t0);                                // of this split
  const int nb = wave < n ? (n - wave + NW - 1) / NW : 0;  // of this wave
  auto block_of = [&](int i) {  // the wave's i-th
    const int t = t0 + wave + NW * i;
    return t < sink_blocks ? t : start + (t - sink_blocks);
  };

  // q^T as the score B operand. Dims of step s, lane group g, element j: 32 s + 8 g + j
  // of an fp16 cache (16 bytes of a key), 64 (s / 2) + 16 g + 8 (s % 2) + j of 8 bits.
  halfx8 qb[KS];
  const _Float16* qh = a.q + out_row(min(kFewRows * tile + col, rows - 1)) * D;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const _Float16* p = qh + (Q8 ? 64 * (s >> 1) + 16 * grp + 8 * (s & 1) : 32 * s + 8 * grp);
    if ((reinterpret_cast<std::uintptr_t>(a.q) & 15) == 0) {
      qb[s] = *reinterpret_cast<const halfx8*>(p);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) qb[s][j] = p[j];
    }
  }
  const float scale2 = a.scale * kLog2e;
  const long long bh = b * a.n_kv + kvh;
  [[maybe_unused]] const char* kg = static_cast<const char*>(a.k) + bh * a.kv_max * (D * ES);
  [[maybe_unused]] const char* vg = static_cast<const char*>(a.v) + bh * a.kv_max * (D * ES);
  [[maybe_unused]] const long long sb = bh * ((a.kv_max + kKvBlock - 1) / kKvBlock);
  [[maybe_unused]] const int koff = ((col >> 2) + 4 * (col & 3)) * D * ES + 16 * grp;
  [[maybe_unused]] const int voff = (grp * D + VW * col) * ES;

  typedef unsigned vword __attribute__((ext_vector_type(VD)));
  struct Block {
    uintx4 k[2][KL];
    vword v[8];
    float ks, vs;
  };
  // Every call issues the same loads, past the wave's last block without a memory access,
  // so that the waits count exactly the blocks in flight behind the one in use.
  auto load = [&](Block& x, int i) __attribute__((always_inline)) {
    const int blk = block_of(i);
    const int keys = i < nb ? min(see.hi - blk * kKvBlock, kKvBlock) : 0;
    const long long at = i < nb ? static_cast<long long>(blk) * kBlockBytes : 0;
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int kRsrcWord3 = 0x00020000;  // raw, 32-bit elements
    const auto rk = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(kg + at), 0, keys * D * ES, kRsrcWord3);
    const auto rv = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(vg + at), 0, keys * D * ES, kRsrcWord3);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int s = 0; s < KL; ++s)
        x.k[h][s] = __builtin_amdgcn_raw_buffer_load_b128(rk, koff + 16 * h * D * ES + 64 * s, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int o = voff + (16 * (e >> 2) + 4 * (e & 3)) * D * ES;
      if constexpr (VD == 4) x.v[e] = __builtin_amdgcn_raw_buffer_load_b128(rv, o, 0, 0);
      else if constexpr (VD == 2) x.v[e] = __builtin_amdgcn_raw_buffer_load_b64(rv, o, 0, 0);
      else x.v[e][0] = __builtin_amdgcn_raw_buffer_load_b32(rv, o, 0, 0);
    }
    if constexpr (Q8) {
      const auto rks = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(a.ks + sb + (keys > 0 ? blk : 0)), 0,
                                                         keys > 0 ? 4 : 0, kRsrcWord3);
      const auto rvs = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(a.vs + sb + (keys > 0 ? blk : 0)), 0,
                                                         keys > 0 ? 4 : 0, kRsrcWord3);
      x.ks = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rks, 0, 0, 0));
      x.vs = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rvs, 0, 0, 0));
    }
#endif
  };
  // Largest of x over the four lanes of a row.
  auto row_max = [](float x) __attribute__((always_inline)) {
#if defined(__HIP_DEVICE_COMPILE__)
    const unsigned w = __float_as_uint(x);
    const auto p = __builtin_amdgcn_permlane16_swap(w, w, false, false);
    const unsigned p0 = p[0], p1 = p[1];
    x = fmaxf(__uint_as_float(p0), __uint_as_float(p1));
#endif
    return pair_max(x);
  };

  float m = kNegInf;
  float lsum = 0.0f;
  floatx4 o[VW];
#pragma unroll
  for (int d = 0; d < VW; ++d) o[d] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

  [[maybe_unused]] float apart[VW] = {};  // of dims VW col + c: what is not finite, taken out
  auto compute = [&](Block& x, int i, auto careful) __attribute__((always_inline)) {
    const int first = block_of(i) * kKvBlock;
    floatx4 sc[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sc[h] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        [[maybe_unused]] halfx8 ka;
        if constexpr (Q8) ka = eight_fp8(x.k[h][s >> 1][2 * (s & 1)], x.k[h][s >> 1][2 * (s & 1) + 1]);
        else ka = __builtin_bit_cast(halfx8, x.k[h][s]);
#if defined(__HIP_DEVICE_COMPILE__)
        sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qb[s], sc[h], 0, 0, 0);
#endif
      }
    }
    float f = scale2, lv = 0.0f, ivs = 1.0f;
    if constexpr (Q8) {
      f = scale2 * x.ks;
      const float vs = fmaxf(x.vs, kLeastVScale);
      lv = __builtin_amdgcn_logf(vs);  // log2
      ivs = __builtin_amdgcn_rcpf(vs);
    }
    float sv[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) sv[e] = fmaf(sc[e >> 2][e & 3], f, lv);
    if (first + kKvBlock > see.hi || (first < see.lo && first + kKvBlock > a.sinks)) {  // (uniform)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int j = first + grp + 16 * (e >> 2) + 4 * (e & 3);
        if (j >= see.hi || (j < see.lo && j >= a.sinks)) {
          sv[e] = kNegInf;
#pragma unroll
          for (int w = 0; w < VD; ++w) x.v[e][w] = 0;
        }
      }
    }
    if constexpr (decltype(careful)::value) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
#pragma unroll
        for (int c = 0; c < VW; ++c) {
          const unsigned word = x.v[e][c / 2];
          const float y = static_cast<float>(__builtin_bit_cast(halfx2, word)[c % 2]);
          if (fabsf(y) < __builtin_huge_valf()) continue;
          apart[c] += y;
          x.v[e][c / 2] = word & (c % 2 == 0 ? 0xffff0000u : 0x0000ffffu);
        }
      }
    }
    float mx = fmaxf(fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3])),
                     fmaxf(fmaxf(sv[4], sv[5]), fmaxf(sv[6], sv[7])));
    mx = row_max(mx);
    if (__any(mx > m + kLazy)) {
      const float mn = fmaxf(m, mx);
      const float alpha = weight2(m, mn);
      m = mn;
      lsum *= alpha;
#pragma unroll
      for (int d = 0; d < VW; ++d) o[d] *= alpha;
    }
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
    auto product = [&](int d, const halfx8& av) __attribute__((always_inline)) {
#if defined(__HIP_DEVICE_COMPILE__)
      o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, pl, o[d], 0, 0, 0);
      o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, ph, o[d], 0, 0, 0);
#endif
    };
#pragma unroll
    for (int w = 0; w < VD; ++w) {
      if constexpr (Q8) {
        halfx8 av[4];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const halfx2 c0 = two_fp8<false>(x.v[e][w]), c1 = two_fp8<true>(x.v[e][w]);
          av[0][e] = c0[0], av[1][e] = c0[1], av[2][e] = c1[0], av[3][e] = c1[1];
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) product(4 * w + c, av[c]);
      } else {
        halfx8 av[2];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const unsigned word = x.v[e][w];
          const halfx2 c = __builtin_bit_cast(halfx2, word);
          av[0][e] = c[0], av[1][e] = c[1];
        }
        product(2 * w, av[0]);
        product(2 * w + 1, av[1]);
      }
    }
  };

  constexpr int P = 2;
  Block buf[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    load(buf[i], i);
    __builtin_amdgcn_sched_barrier(0);
  }
  for (int t = 0; t < nb; t += P) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      if (t + i < nb) compute(buf[i], t + i, std::false_type{});
      __builtin_amdgcn_sched_barrier(0);
      load(buf[i], t + i + P);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // Lane (col, grp) holds dims VW (4 grp + r) + d of row col in o[d][r].
  if constexpr (!Q8) {
    float sum = 0.0f;
#pragma unroll
    for (int d = 0; d < VW; ++d) {
#pragma unroll
      for (int r = 0; r < 4; ++r) sum = fmaf(o[d][r], 0.0f, sum);
    }
    if (__any(sum != sum)) {
      m = kNegInf;
      lsum = 0.0f;
#pragma unroll
      for (int d = 0; d < VW; ++d) o[d] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
      for (int t = 0; t < nb; ++t) {
        load(buf[0], t);
        compute(buf[0], t, std::true_type{});
      }
#pragma unroll
      for (int d = 0; d < VW; ++d) {
        apart[d] += __shfl_xor(apart[d], 16);
        apart[d] += __shfl_xor(apart[d], 32);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float seen = __shfl(apart[d], 4 * grp + r);
          o[d][r] += m == kNegInf ? 0.0f : seen;  // (no score above -inf: none of them)
        }
      }
    }
  }
  float lt = lsum + __shfl_xor(lsum, 16);
  lt += __shfl_xor(lt, 32);
  const int gq = min(rows - kFewRows * tile, kFewRows);
  float* const ws = s_state + wave * WS;
  if (col < gq) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
      for (int c = 0; c < VW; c += 4)
        *reinterpret_cast<floatx4*>(ws + col * D + VW * (4 * grp + r) + c) =
            floatx4{o[c][r], o[c + 1][r], o[c + 2][r], o[c + 3][r]};
    }
    if (grp == 0) {
      ws[kFewRows * D + col] = m;
      ws[kFewRows * (D + 1) + col] = lt;
    }
  }
  __syncthreads();
  const int live = min(NW, n);  // waves with a block
  for (int idx = tid; idx < gq * D; idx += 64 * NW) {
    const int r = idx / D;
    const int d = idx - r * D;
    float mb = kNegInf;
    for (int w = 0; w < live; ++w) mb = fmaxf(mb, s_state[w * WS + kFewRows * D + r]);
    float lb = 0.0f, ob = 0.0f;
    for (int w = 0; w < live; ++w) {
      const float wt = weight2(s_state[w * WS + kFewRows * D + r], mb);
      lb = fmaf(s_state[w * WS + kFewRows * (D + 1) + r], wt, lb);
      ob = fmaf(s_state[w * WS + r * D + d], wt, ob);
    }
    const long long orow = out_row(kFewRows * tile + r);
    if (a.part_o != nullptr) {
      const long long slot = orow * a.part_stride + a.part0 + split;
      a.part_o[slot * D + d] = ob;
      if (d == 0) *reinterpret_cast<floatx2*>(a.part_ml + 2 * slot) = floatx2{mb, lb};
    } else {
      a.out[orow * D + d] = static_cast<_Float16>(lb == 0.0f ? 0.0f : ob / lb);
    }
  }
}

}  // namespace attn
}  // namespace eng
