// beam.hip -- beam search: the best continuations over the beams of a group and the
// vocabulary, and the reordering of the beams' caches that follows from them.
//
// Selection: candidate (beam b, token t) has the score s_b + x_bt - L_b, with L_b =
// log sum_t exp x_bt. Within a beam the order is the logits' own, so the logits are read
// once: a pass over a piece of a row keeps the piece's best candidates by (logit, lowest
// token) as 64-bit keys and its max and sum of exponentials; a second kernel joins the
// pieces and compares candidates of unlike beams by their scores in 64 bits, with sums of
// fp32 exponentials where these tell the candidates apart and 64-bit ones where not.
#include "gemv_kernels.hpp"
#include "launch.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace eng {
namespace beam {
namespace {

typedef unsigned uintx2 __attribute__((ext_vector_type(2)));
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
typedef unsigned long long u64;

constexpr float kNegInf = -__builtin_huge_valf();
constexpr int kMaxOut = 64;    // candidates that a call may ask for
constexpr int kMaxBeams = 32;
constexpr int kWaves = 4;
constexpr int kVpt = 16;       // values of a lane in one step of a wave
constexpr int kWaveList = 64 * kVpt + kMaxOut;

// A logit as a number that orders like it.
__device__ __forceinline__ unsigned order_of(float x) {
  const unsigned u = __float_as_uint(x + 0.0f);  // (-0 as 0)
  return u ^ ((u >> 31) != 0 ? 0xffffffffu : 0x80000000u);
}
// Key of a candidate: larger logits first, then lower tokens. 0 stands for none.
__device__ __forceinline__ u64 key_of(float x, unsigned token) {
  return (static_cast<u64>(order_of(x)) << 32) | (0xffffffffu - token);
}
__device__ __forceinline__ float value_of(unsigned v) {
  return __uint_as_float(v ^ ((v >> 31) != 0 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ float logit_of(u64 key) { return value_of(static_cast<unsigned>(key >> 32)); }
__device__ __forceinline__ unsigned token_of(u64 key) { return 0xffffffffu - static_cast<unsigned>(key); }

// e^d in 64 bits, d < 700 and no NaN, to 2e-14: 2^k 2^f, t = k + f, |f| <= 1/2, 2^f by the
// polynomial of degree 9 that meets it in Chebyshev's points. Less than e^-700 counts as it.
__device__ __forceinline__ double exp64(double d) {
  constexpr double kLog2e = 1.4426950408889634, kRound = 0x1.8p52;
  d = fmax(d, -700.0);
  const double t = fma(d, kLog2e, kRound);  // (k in the lowest bits)
  const double f = fma(d, kLog2e, kRound - t);
  double p = 0x1.b69b333333333p-24;
  p = fma(p, f, 0x1.63f1a66666666p-20);
  p = fma(p, f, 0x1.ffcb2e3333335p-17);
  p = fma(p, f, 0x1.43088c34ccccbp-13);
  p = fma(p, f, 0x1.5d87fea9ba666p-10);
  p = fma(p, f, 0x1.3b2ab72c33333p-7);
  p = fma(p, f, 0x1.c6b08d70374acp-5);
  p = fma(p, f, 0x1.ebfbdff813d86p-3);
  p = fma(p, f, 0x1.62e42fefa3a31p-1);
  p = fma(p, f, 0x1.000000000003fp+0);
  uintx2 w = __builtin_bit_cast(uintx2, p);
  w[1] += __builtin_bit_cast(uintx2, t)[0] << 20;
  return __builtin_bit_cast(double, w);
}
// Sums of exponentials are kept as sums of 2^(x log2 e - n), n the whole number that belongs
// to the largest x, so that sums of unlike n are joined by shifts of exponents: exact.
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = 0x1p22f;  // past it n is not to be had in fp32
__device__ __forceinline__ float exponent_of(float m) {
  return fminf(fmaxf(rintf(m * kLog2e), -2.0f * kFar), 2.0f * kFar);
}
// A sum against m as one against top >= m.
__device__ __forceinline__ double against(double sum, float m, float top) {
  return __builtin_ldexp(sum, static_cast<int>(exponent_of(m) - exponent_of(top)));
}
// The sum over the wave, in every lane.
template <int CTRL>
__device__ __forceinline__ double dpp_add(double x) {
  uintx2 w = __builtin_bit_cast(uintx2, x);
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(w[i]), CTRL, 0xF, 0xF, false));
  return x + __builtin_bit_cast(double, w);
}
__device__ __forceinline__ double wave_sum(double x) {
  x = dpp_add<0xB1>(x);   // quad_perm [1, 0, 3, 2]
  x = dpp_add<0x4E>(x);   // quad_perm [2, 3, 0, 1]
  x = dpp_add<0x141>(x);  // row_half_mirror
  x = dpp_add<0x140>(x);  // row_mirror
  const uintx2 w = __builtin_bit_cast(uintx2, x);
  double r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r[i] = __builtin_bit_cast(double, uintx2{static_cast<unsigned>(__builtin_amdgcn_readlane(w[0], 16 * i)),
                                             static_cast<unsigned>(__builtin_amdgcn_readlane(w[1], 16 * i))});
  return (r[0] + r[1]) + (r[2] + r[3]);
}

// The largest of the wave's values, in every lane.
template <int CTRL>
__device__ __forceinline__ unsigned dpp_max(unsigned x) {
  return max(x, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, 0xF, 0xF, false)));
}
__device__ __forceinline__ unsigned wave_max(unsigned x) {
  x = dpp_max<0xB1>(x);   // quad_perm [1, 0, 3, 2]
  x = dpp_max<0x4E>(x);   // quad_perm [2, 3, 0, 1]
  x = dpp_max<0x141>(x);  // row_half_mirror
  x = dpp_max<0x140>(x);  // row_mirror
  const unsigned a = __builtin_amdgcn_readlane(x, 0), b = __builtin_amdgcn_readlane(x, 16);
  const unsigned c = __builtin_amdgcn_readlane(x, 32), d = __builtin_amdgcn_readlane(x, 48);
  return max(max(a, b), max(c, d));
}
__device__ __forceinline__ u64 wave_max(u64 x) {
  const unsigned hi = static_cast<unsigned>(x >> 32);
  const unsigned top = wave_max(hi);
  const unsigned low = wave_max(hi == top ? static_cast<unsigned>(x) : 0u);
  return (static_cast<u64>(top) << 32) | low;
}

__device__ __forceinline__ u64 lane_value(u64 x, int lane) {
  const unsigned lo = __builtin_amdgcn_readlane(static_cast<unsigned>(x), lane);
  const unsigned hi = __builtin_amdgcn_readlane(static_cast<unsigned>(x >> 32), lane);
  return (static_cast<u64>(hi) << 32) | lo;
}

// One wave's candidates, of which it keeps the `k` best. CAP: room in its list, in LDS.
template <int CAP>
struct Best {
  static constexpr int kSteps = (CAP + 63) / 64;
  u64* list;
  int k;
  int n;

  // A value that at least k lanes' `top` reach, few more where halving the interval 24
  // times finds one.
  __device__ __forceinline__ unsigned reached(unsigned top) const {
    unsigned hi = wave_max(top), lo = ~wave_max(~top);  // (all reach lo)
    int c = 64;
    for (int i = 0; i < 24 && c > k + 8 && hi - lo > 1; ++i) {
      const unsigned mid = lo + (hi - lo) / 2;
      const int reach = __builtin_popcountll(__ballot(top >= mid));
      if (reach >= k) lo = mid, c = reach;
      else hi = mid;
    }
    return lo;
  }

  // Adds those of N items of each lane that reach(i) says, item i being key_at(i) (0: none).
  template <int N, class R, class K>
  __device__ __forceinline__ void add(R&& reach, K&& key_at, int lane) {
    static_assert(64 * N + kMaxOut <= CAP, "the list holds them all");
    if (n > kMaxOut) sort(lane);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (__ballot(reach(i)) == 0) continue;
      const u64 key = key_at(i);
      const u64 mask = __ballot(reach(i) && key != 0);
      const int at = n + __builtin_amdgcn_mbcnt_hi(static_cast<unsigned>(mask >> 32),
                                                   __builtin_amdgcn_mbcnt_lo(static_cast<unsigned>(mask), 0));
      if (reach(i) && key != 0) list[at] = key;
      n += __builtin_popcountll(mask);
    }
  }

  // Brings the k best of list[0 .. n) to its front, in order: an entry's place is the
  // number of larger ones.
  __device__ __forceinline__ void sort(int lane) {
    wave_sync();
    const int keep = min(n, k);
    if (n <= 64) {
      const u64 mine = lane < n ? list[lane] : 0;
      int place = 0;
      for (int j = 0; j < n; ++j) place += lane_value(mine, j) > mine;
      wave_sync();
      if (lane < n && place < keep) list[place] = mine;
    } else {
      // Many equal logits, or k past 32. The k best by rounds, each the largest left.
      u64 mine[kSteps];
#pragma unroll
      for (int s = 0; s < kSteps; ++s) mine[s] = 64 * s + lane < n ? list[64 * s + lane] : 0;
      wave_sync();
      for (int j = 0; j < keep; ++j) {
        u64 top = 0;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) top = max(top, mine[s]);
        top = wave_max(top);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) mine[s] = mine[s] == top ? 0 : mine[s];
        if (lane == 0) list[j] = top;
      }
    }
    wave_sync();
    n = keep;
  }

  // LDS accesses of this wave before it are done before those behind it.
  __device__ static __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
};

struct SelectArgs {
  const void* logits;
  long long ld;
  const float* scores;
  const unsigned char* finished;
  float* out_scores;
  int* out_parent;
  int* out_token;
  unsigned char* out_finished;
  int beams, n_out, vocab, eos;
  int pieces;      // of a row
  u64* keys;       // [rows][pieces][n_out], 0 behind the last one
  double* sums;    // [rows][pieces]: of 2^(x log2 e - n), n the largest logit's exponent_of
  float* maxes;    // [rows][pieces]
  double* lse;     // [rows][2]: L as the largest logit and what is to be added; NaN: none
  double near;     // scores of unlike beams this close may be in the wrong order
};

constexpr int kStep = 64 * kWaves * kVpt;  // values of a workgroup's step

// One workgroup per (row, piece of STEPS steps), the whole piece in registers, 16 STEPS
// values of a lane. The k-th largest of the lanes' largest values bounds the k best from
// below, so few values are looked at one by one. A NaN in a row makes its sum NaN.
// 64 rows of 152064 fp32 (39 MB) take 15.3 us: their loads, issued together, about 7, the
// exponentials and the search behind them the rest (19 with a list kept over the steps, 17
// in pieces of two steps). 4 rows of 32000: 6.6 us, latencies.
template <typename T, bool VECTOR, int STEPS>
__global__ __launch_bounds__(64 * kWaves) void piece_kernel(SelectArgs a) {
  constexpr int VEC = 16 / sizeof(T);
  constexpr int LOADS = kVpt / VEC;
  __shared__ u64 s_list[kWaves][kWaveList];
  __shared__ float s_max[kWaves];
  __shared__ double s_sum[kWaves];
  __shared__ int s_count[kWaves];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const unsigned row = blockIdx.x / static_cast<unsigned>(a.pieces);
  const int piece = static_cast<int>(blockIdx.x - row * static_cast<unsigned>(a.pieces));
  const T* x = static_cast<const T*>(a.logits) + row * a.ld;
  const int begin = piece * (STEPS * kStep);
  const int end = min(begin + STEPS * kStep, a.vocab);

  uintx4 raw[STEPS][LOADS];  // as in memory; -inf behind the row's end
#pragma unroll
  for (int c = 0; c < STEPS; ++c) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int t0 = begin + c * kStep + (i * 64 * kWaves + tid) * VEC;
      if (VECTOR && t0 + VEC <= end) {
        raw[c][i] = *reinterpret_cast<const uintx4*>(x + t0);
      } else {
        T some[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) some[e] = t0 + e < end ? x[t0 + e] : static_cast<T>(kNegInf);
        raw[c][i] = __builtin_bit_cast(uintx4, some);
      }
    }
  }
  auto value = [&](int c, int i) __attribute__((always_inline)) {
    const unsigned w = raw[c][i / VEC][i % VEC * sizeof(T) / 4];
    if constexpr (sizeof(T) == 4) return __uint_as_float(w);
    else return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<unsigned short>(w >> (16 * (i % 2)))));
  };
  float m = kNegInf;
#pragma unroll
  for (int c = 0; c < STEPS; ++c) {
#pragma unroll
    for (int i = 0; i < kVpt; ++i) m = fmaxf(m, value(c, i));
  }
  const float shift = exponent_of(m);
  float part[STEPS];
#pragma unroll
  for (int c = 0; c < STEPS; ++c) {
    float e[kVpt];
#pragma unroll
    for (int i = 0; i < kVpt; ++i) e[i] = __builtin_amdgcn_exp2f(fmaf(value(c, i), kLog2e, -shift));
#pragma unroll
    for (int w = kVpt / 2; w > 0; w /= 2) {
#pragma unroll
      for (int i = 0; i < w; ++i) e[i] += e[i + w];
    }
    part[c] = e[0];
  }
#pragma unroll
  for (int w = STEPS / 2; w > 0; w /= 2) {
#pragma unroll
    for (int c = 0; c < w; ++c) part[c] += part[c + w];
  }
  Best<kWaveList> best = {s_list[wave], a.n_out, 0};
  const float least = value_of(best.reached(order_of(m)));
#pragma unroll
  for (int c = 0; c < STEPS; ++c)
    best.add<kVpt>([&](int i) { return value(c, i) >= least; }, [&](int i) {
      const int t = begin + c * kStep + (i / VEC * 64 * kWaves + tid) * VEC + i % VEC;
      return t < end ? key_of(value(c, i), static_cast<unsigned>(t)) : 0;
    }, lane);
  best.sort(lane);
  // the wave's max and sum
  const float wm = value_of(wave_max(order_of(m)));
  const double ws = wave_sum(against(part[0], m, wm));
  if (lane == 0) {
    s_max[wave] = wm;
    s_sum[wave] = ws;
    s_count[wave] = best.n;
  }
  __syncthreads();
  if (wave != 0) return;
  // the other waves' keys behind its own
  for (int w = 1; w < kWaves; ++w) {
    const int c = s_count[w];
    if (lane < c) best.list[best.n + lane] = s_list[w][lane];
    best.n += c;
  }
  best.sort(lane);
  const long long out = static_cast<long long>(blockIdx.x);
  for (int i = lane; i < a.n_out; i += 64) a.keys[out * a.n_out + i] = i < best.n ? best.list[i] : 0;
  if (lane == 0) {
    float top = kNegInf;
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, s_max[w]);
    double s = 0.0;
    for (int w = 0; w < kWaves; ++w) s += against(s_sum[w], s_max[w], top);
    a.sums[out] = s;
    a.maxes[out] = top;
  }
}

constexpr int kJoinWaves = 16;  // at the most: one for each beam
constexpr int kJoinKeys = 4;    // of a lane in one go
constexpr int kJoinList = 64 * kJoinKeys + kMaxOut;

// One workgroup per group, a wave for each beam up to kJoinWaves: a wave joins its beam's
// pieces; then the beams' candidates are put in order by (score, beam, token). A candidate
// whose score is no number, or of a beam without a finite score, counts as -inf; such a
// beam's come in the order of the tokens, so its first n_out stand for it. Bound by a chain
// of round trips (pieces, logarithm, sort, ranks): 4 beams 5.6-7.5 us, 10 beams of 10
// candidates 10, 32 of 32 56 (compared each with each, by four waves, 18 and 560).
//
// The sum of fp32 exponentials leaves L off by up to `near` / 2 (select_entry has the bound).
// Where a chosen candidate and one of another beam are closer than `near`, both beams' sums
// are formed again, from the logits, in 64 bits, and the candidates put in order again: of
// groups with gaps of 0.1 in score about one in three thousand, 90-140 us for two beams
// of 152064 (a workgroup's CU is all it has). The question costs 0.3 us. (All exponentials in 64 bits: 16 x 4 beams of
// 152064 in 29 us in place of 22.)
template <typename T>
__global__ __launch_bounds__(64 * kJoinWaves) void join_kernel(SelectArgs a) {
  __shared__ u64 s_list[kJoinWaves][kJoinList];
  __shared__ double s_score[kMaxBeams * kMaxOut];
  __shared__ int s_token[kMaxBeams * kMaxOut];
  const int threads = static_cast<int>(blockDim.x);
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const long long group = blockIdx.x;
  const int k = a.n_out;
  const double ninf = -__builtin_huge_val();
  for (int b = wave; b < a.beams; b += threads / 64) {
    const long long row = group * a.beams + b;
    const float given = a.scores[row];
    const bool done = a.finished != nullptr && a.finished[row] != 0;
    const long long n = static_cast<long long>(a.pieces) * k;
    u64 key[kJoinKeys];
    auto load_keys = [&](long long i0) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < kJoinKeys; ++j) {
        const long long i = i0 + 64 * j + lane;
        key[j] = i < n ? a.keys[row * n + i] : 0;
      }
    };
    load_keys(0);
    // a lane's first piece is loaded with the keys
    const float* maxes = a.maxes + row * a.pieces;
    const double* sums = a.sums + row * a.pieces;
    const float max0 = lane < a.pieces ? maxes[lane] : kNegInf;
    const double sum0 = lane < a.pieces ? sums[lane] : 0.0;
    float m = max0;
    for (int i = lane + 64; i < a.pieces; i += 64) m = fmaxf(m, maxes[i]);
    m = value_of(wave_max(order_of(m)));
    double part = against(sum0, max0, m);
    for (int i = lane + 64; i < a.pieces; i += 64) part += against(sums[i], maxes[i], m);
    const double sum = wave_sum(part);
    const bool finite = given > kNegInf && given < -kNegInf;
    // L = peak + more, kept apart: rows far from zero lose nothing
    const double peak = m;
    double more = log(sum) - 0.6931471805599453 * (peak * kLog2e - exponent_of(m));
    if (!done && finite && fabsf(m) > kFar && fabsf(m) < -kNegInf && sum == sum) {
      const T* x = static_cast<const T*>(a.logits) + row * a.ld;
      double slow = 0.0;
      for (int t = lane; t < a.vocab; t += 64) slow += exp64(static_cast<double>(x[t]) - peak);
      more = log(wave_sum(slow));
    }
    const bool plain = !done && finite && (peak + more) - (peak + more) == 0.0;
    if (lane == 0) {
      a.lse[2 * row] = plain ? peak : __builtin_nan("");
      a.lse[2 * row + 1] = more;
    }
    Best<kJoinList> best = {s_list[wave], k, 0};
    if (plain) {
      for (long long i0 = 0;; i0 += 64 * kJoinKeys) {
        unsigned top = 0;
#pragma unroll
        for (int j = 0; j < kJoinKeys; ++j) top = max(top, static_cast<unsigned>(key[j] >> 32));
        const unsigned least = best.reached(top);
        best.add<kJoinKeys>([&](int j) { return static_cast<unsigned>(key[j] >> 32) >= least; },
                    [&](int j) { return key[j]; }, lane);
        if (i0 + 64 * kJoinKeys >= n) break;
        load_keys(i0 + 64 * kJoinKeys);
      }
      best.sort(lane);
    }
    for (int i = lane; i < k; i += 64) {
      double score = ninf;
      int token = i;
      if (plain) {
        // (fewer than k tokens in the vocabulary: none)
        token = -1;
        if (i < best.n) {
          const u64 key = best.list[i];
          token = static_cast<int>(token_of(key));
          score = static_cast<double>(given) + ((static_cast<double>(logit_of(key)) - peak) - more);
        }
      } else if (done && finite) {
        // its end token first, then the others
        token = i == 0 ? a.eos : i - 1 < a.eos ? i - 1 : i;
        if (i == 0) score = given;
      }
      if (token >= a.vocab) token = -1;
      s_score[b * k + i] = score == score ? score : ninf;
      s_token[b * k + i] = token;
    }
  }
  // beams whose order is open, in wave 0's list, which it is done with; a wave's sum in the next
  unsigned* const s_open = reinterpret_cast<unsigned*>(s_list[0]);
  double* const s_part = reinterpret_cast<double*>(s_list[1]);
  if (tid == 0) *s_open = 0;
  __syncthreads();
  const int n = a.beams * k;
  // Places of a thread's candidates, k and more for none; the beams whose order is open.
  constexpr int kMine = (kMaxBeams * kMaxOut + 64 * kJoinWaves - 1) / (64 * kJoinWaves);
  int place[kMine];
  auto rank = [&] {
    unsigned open = 0;
#pragma unroll
    for (int q = 0; q < kMine; ++q) {
      const int i = tid + q * threads;
      place[q] = k;
      if (i >= n || s_token[i] < 0) continue;
      const double score = s_score[i];
      const int b = i / k;
      // Each beam's own are in order, those without a token last: counted up to the first that
      // comes behind this one. A place past the k-th is none.
      int at = i - b * k;
      unsigned close = 0;
      for (int c = 0; c < a.beams && at < k; ++c) {
        if (c == b) continue;
        double behind = ninf;
        for (int j = c * k; j < c * k + k && at < k; ++j) {
          behind = s_token[j] < 0 ? ninf : s_score[j];
          if (s_token[j] < 0 || !(behind > score || (behind == score && c < b))) break;
          ++at;
        }
        if (score - behind <= a.near) close |= (1u << b) | (1u << c);
      }
      place[q] = at;
      if (at < k) open |= close;
    }
    return open;
  };
  const unsigned open = rank();
  if (open != 0) atomicOr(s_open, open);
  __syncthreads();
  // Open beams whose sums agree in every bit have equal rows, whose order is that of the
  // logits and scores (others' agree by chance only, with L closer than a term's last bit).
  // Where all do, the order stands; sums in 64 bits otherwise.
  const double* const first = a.lse + 2 * group * a.beams;
  bool alike = true;
  for (unsigned rest = *s_open; rest != 0; rest &= rest - 1) {
    const int b = __builtin_ctz(rest), c = __builtin_ctz(*s_open);
    alike = alike && first[2 * b] == first[2 * c] && first[2 * b + 1] == first[2 * c + 1];
  }
  const unsigned settle = alike ? 0 : *s_open;
  for (unsigned again = settle; again != 0; again &= again - 1) {
    const int b = __builtin_ctz(again);
    const long long row = group * a.beams + b;
    const double peak = first[2 * b], more = first[2 * b + 1];
    if (peak != peak) continue;
    const T* x = static_cast<const T*>(a.logits) + row * a.ld;
    double part[4] = {};
    for (int t0 = tid; t0 < a.vocab; t0 += 4 * threads) {
      T v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = x[min(t0 + j * threads, a.vocab - 1)];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double e = exp64((static_cast<double>(v[j]) - peak) - more);
        part[j] += t0 + j * threads < a.vocab ? e : 0.0;
      }
    }
    const double mine = wave_sum((part[0] + part[1]) + (part[2] + part[3]));
    __syncthreads();  // (s_part is read for the beam before)
    if (lane == 0) s_part[wave] = mine;
    __syncthreads();
    double sum = 0.0;
    for (int w = 0; w < threads / 64; ++w) sum += s_part[w];
    const double change = log(sum);  // of L: terms against the old one add up to e^change
    for (int i = b * k + tid; i < b * k + k; i += threads) s_score[i] -= change;
  }
  if (settle != 0) {
    __syncthreads();
    rank();
  }
#pragma unroll
  for (int q = 0; q < kMine; ++q) {
    if (place[q] >= k) continue;
    const int i = tid + q * threads;
    const int b = i / k;
    const int token = s_token[i];
    const long long out = group * k + place[q];
    a.out_scores[out] = static_cast<float>(s_score[i]);
    a.out_parent[out] = b;
    a.out_token[out] = token;
    if (a.out_finished != nullptr)
      a.out_finished[out] = (a.finished != nullptr && a.finished[group * a.beams + b] != 0) || token == a.eos;
  }
}

// ---------------------------------------------------------------------- reorder

struct ReorderArgs {
  const unsigned char* src[2];
  unsigned char* dst[2];
  const float* src_scale[2];
  float* dst_scale[2];
  const int* parent;
  const int* lens;
  int beams, heads;
  long long max_len;
  long long head_bytes;    // of a head's cache
  long long scale_blocks;  // of a head
  unsigned chunks;         // workgroups of a head
  int row_bytes;           // of a token
  bool in_place;
};

// One workgroup per (group, head, K or V, 256 16-byte columns of the head's cache): a
// thread loads its column of every beam's parent, then stores to the beams, so the beams
// of a group may change places in their own buffers. A parent that several beams share is
// read once from memory and then from the caches. The thread of a 32-token block's first
// column moves the block's scale. Bound by memory: 64 beams of 1000 tokens, 32 heads of 128,
// 8-bit, into other buffers 162 us, 5.5 TB/s; 14 beams in two groups of 1724 tokens, 40 heads
// of 128, fp16, 170 us, 5.2 TB/s (271 with a branch around each load, which a wave then
// waits for one by one).
template <int MB>
__global__ __launch_bounds__(256) void reorder_kernel(ReorderArgs a) {
  const unsigned chunk = blockIdx.x % a.chunks;
  const unsigned rest = blockIdx.x / a.chunks;
  const int side = static_cast<int>(rest & 1);
  const unsigned heads = static_cast<unsigned>(a.heads);
  const unsigned gh = rest >> 1;
  const long long group = gh / heads;
  const long long head = gh - static_cast<unsigned>(group) * heads;
  const long long at = (static_cast<long long>(chunk) * 256 + threadIdx.x) * 16;
  const long long token = at / a.row_bytes;
  const long long first = group * a.beams;
  const long long beam_bytes = a.head_bytes * heads;
  const long long base = (first * heads + head) * a.head_bytes;
  // What each beam takes, the same in all threads: its parent's tokens, 0 of them where it
  // stays as it is. Such a beam loads what another one takes and does not store it: no
  // branches between the loads.
  const long long chunk_token = static_cast<long long>(chunk) * 4096 / a.row_bytes;
  int p[MB];
  long long n[MB];
  int some = -1;
#pragma unroll
  for (int j = 0; j < MB; ++j) {
    p[j] = __builtin_amdgcn_readfirstlane(a.parent[first + std::min(j, a.beams - 1)]);
    if (j >= a.beams || p[j] < 0 || p[j] >= a.beams || (a.in_place && p[j] == j)) p[j] = -1;
  }
#pragma unroll
  for (int j = 0; j < MB; ++j) {
    const int len = __builtin_amdgcn_readfirstlane(a.lens[first + std::max(p[j], 0)]);
    n[j] = p[j] < 0 ? 0 : std::min<long long>(len, a.max_len);
    some = n[j] > chunk_token ? p[j] : some;
  }
  if (some < 0) return;
  // (a thread past the last token loads the last one)
  const unsigned char* from = a.src[side] + base + std::min(at, a.max_len * a.row_bytes - 16);
  uintx4 v[MB];
#pragma unroll
  for (int j = 0; j < MB; ++j)
    v[j] = *reinterpret_cast<const uintx4*>(from + (n[j] > chunk_token ? p[j] : some) * beam_bytes);
  const long long beam_blocks = a.scale_blocks * heads;
  const long long sbase = (first * heads + head) * a.scale_blocks + token / 32;
  float s[MB] = {};
  const bool scales = a.src_scale[side] != nullptr && at % (32ll * a.row_bytes) == 0 && token < a.max_len;
  if (scales) {
#pragma unroll
    for (int j = 0; j < MB; ++j) s[j] = a.src_scale[side][sbase + (n[j] > chunk_token ? p[j] : some) * beam_blocks];
  }
#pragma unroll
  for (int j = 0; j < MB; ++j) {
    if (token < n[j]) {
      *reinterpret_cast<uintx4*>(a.dst[side] + base + at + j * beam_bytes) = v[j];
      if (scales) a.dst_scale[side][sbase + j * beam_blocks] = s[j];
    }
  }
}

void select_entry(const void* logits, bool half, int64_t ld, const float* scores, const uint8_t* finished,
                  float* out_scores, int32_t* out_parent, int32_t* out_token, uint8_t* out_finished,
                  int64_t batch, int64_t beams, int64_t n_out, int64_t vocab, int64_t eos, hipStream_t s) {
  ENG_CHECK(batch >= 0, "beam_select: batch must be non-negative");
  ENG_CHECK(beams > 0 && beams <= kMaxBeams, "beam_select: beams must be 1 to 32");
  ENG_CHECK(n_out > 0 && n_out <= kMaxOut, "beam_select: n_out must be 1 to 64");
  ENG_CHECK(vocab > 0 && vocab < 0x80000000LL - 65536, "beam_select: vocab must be positive and below 2^31 - 65536");
  ENG_CHECK(n_out <= beams * vocab, "beam_select: n_out > beams * vocab");
  ENG_CHECK(ld >= vocab, "beam_select: ld < vocab");
  ENG_CHECK(eos < vocab, "beam_select: eos >= vocab");
  if (batch == 0) return;
  ENG_CHECK(logits != nullptr, "beam_select: logits is null");
  ENG_CHECK(scores != nullptr, "beam_select: scores is null");
  ENG_CHECK(out_scores != nullptr && out_parent != nullptr && out_token != nullptr,
            "beam_select: out_scores/out_parent/out_token is null");
  ENG_CHECK(finished == nullptr || eos >= 0, "beam_select: finished beams need eos");
  const long long elem = half ? 2 : 4;
  ENG_CHECK(aligned_to(logits, elem), "beam_select: logits must be aligned to their type");
  SelectArgs a = {};
  a.logits = logits;
  a.ld = ld;
  a.scores = scores;
  a.finished = finished;
  a.out_scores = out_scores;
  a.out_parent = out_parent;
  a.out_token = out_token;
  a.out_finished = out_finished;
  a.beams = static_cast<int>(beams);
  a.n_out = static_cast<int>(n_out);
  a.vocab = static_cast<int>(vocab);
  a.eos = eos < 0 ? -1 : static_cast<int>(eos);
  // Steps of a piece: as many as leave two workgroups to a CU, up to four; one to a CU, where
  // the join would load a beam's candidates in more than one go (16 rows of 152064, 8 of
  // them: 15.3 us with 304 workgroups, 17.0 with 608; 48 rows of 50257 18.7 and 16.9).
  const long long steps = (vocab + kStep - 1) / kStep;
  ENG_CHECK(batch <= 0xffffffffLL / (64 * kWaves) / (beams * steps),
            "beam_select: too many logits for one launch");
  const long long rows = batch * beams;
  int per = 4;
  auto pieces = [&](int n) { return (steps + n - 1) / n; };
  while (per > 1 && rows * pieces(per) < 2ll * device_cu_count()) per /= 2;
  while (per < 4 && pieces(per) * n_out > 64 * kJoinKeys && rows * pieces(2 * per) >= device_cu_count()) per *= 2;
  a.pieces = static_cast<int>(pieces(per));
  const std::size_t lists = static_cast<std::size_t>(rows) * a.pieces;
  StreamScratch scratch(s, lists * (n_out * sizeof(u64) + sizeof(double) + sizeof(float)) +
                               static_cast<std::size_t>(rows) * 2 * sizeof(double));
  a.keys = static_cast<u64*>(scratch.get());
  a.sums = reinterpret_cast<double*>(a.keys + lists * n_out);
  a.lse = a.sums + lists;
  a.maxes = reinterpret_cast<float*>(a.lse + 2 * rows);
  const bool vector = aligned_to(logits, 16) && (ld * elem) % 16 == 0;
  const unsigned grid = static_cast<unsigned>(lists);
  auto go = [&](auto elem, auto vec) {
    using T = decltype(elem);
    constexpr bool kVector = decltype(vec)::value;
    if (per == 4) piece_kernel<T, kVector, 4><<<grid, 64 * kWaves, 0, s>>>(a);
    else if (per == 2) piece_kernel<T, kVector, 2><<<grid, 64 * kWaves, 0, s>>>(a);
    else piece_kernel<T, kVector, 1><<<grid, 64 * kWaves, 0, s>>>(a);
  };
  if (half) vector ? go(_Float16{}, std::true_type{}) : go(_Float16{}, std::false_type{});
  else vector ? go(float{}, std::true_type{}) : go(float{}, std::false_type{});
  ENG_LAUNCH_CHECK();
  // How far L may be off, u = 2^-24: a term by 1.22 |x - max| u (its argument's rounding, log2 e
  // as an fp32 number; the part of it that all terms share is known), over a row in the mean
  // 1.22 u log vocab at the most (the mean of -log w_i under w_i / S is an entropy less log
  // S, and S >= 1), 2 u of the exponential, and a lane's additions 6 u; what follows is in 64
  // bits. Twice that, and one u, for two beams.
  a.near = 2.0 * 0x1p-24 * (1.22 * std::log(static_cast<double>(vocab)) + 10.0);
  // At least four waves, for the sums in 64 bits; a thread has up to two candidates.
  const int join_threads = 64 * std::max(4, std::min(a.beams, kJoinWaves));
  if (half) join_kernel<_Float16><<<static_cast<unsigned>(batch), join_threads, 0, s>>>(a);
  else join_kernel<float><<<static_cast<unsigned>(batch), join_threads, 0, s>>>(a);
  ENG_LAUNCH_CHECK();
}

void reorder_entry(const void* k_src, const void* v_src, const float* ks_src, const float* vs_src, void* k_dst,
                   void* v_dst, float* ks_dst, float* vs_dst, bool q8, const int32_t* parent,
                   const int32_t* kv_len, int64_t batch, int64_t beams, int64_t n_kv_heads, int64_t head_dim,
                   int64_t max_kv_len, int64_t kv_max_seq_len, hipStream_t s) {
  ENG_CHECK(batch >= 0, "kv_cache_reorder: batch must be non-negative");
  ENG_CHECK(beams > 0 && beams <= kMaxBeams, "kv_cache_reorder: beams must be 1 to 32");
  ENG_CHECK(n_kv_heads > 0, "kv_cache_reorder: n_kv_heads must be positive");
  ENG_CHECK(head_dim == 64 || head_dim == 128, "kv_cache_reorder: head_dim must be 64 or 128");
  ENG_CHECK(max_kv_len >= 0, "kv_cache_reorder: max_kv_len must be non-negative");
  ENG_CHECK(kv_max_seq_len >= max_kv_len, "kv_cache_reorder: kv_max_seq_len < max_kv_len");
  ENG_CHECK(kv_max_seq_len <= 0x7fffffffLL - 32, "kv_cache_reorder: kv_max_seq_len must be below 2^31 - 32");
  if (batch == 0 || max_kv_len == 0) return;
  ENG_CHECK(k_src != nullptr && v_src != nullptr, "kv_cache_reorder: k_src/v_src is null");
  ENG_CHECK(k_dst != nullptr && v_dst != nullptr, "kv_cache_reorder: k_dst/v_dst is null");
  ENG_CHECK(!q8 || (ks_src != nullptr && vs_src != nullptr && ks_dst != nullptr && vs_dst != nullptr),
            "kv_cache_reorder: a scale buffer is null");
  ENG_CHECK(parent != nullptr, "kv_cache_reorder: parent is null");
  ENG_CHECK(kv_len != nullptr, "kv_cache_reorder: kv_len is null");
  ENG_CHECK(aligned_to(k_src, 16) && aligned_to(v_src, 16) && aligned_to(k_dst, 16) && aligned_to(v_dst, 16),
            "kv_cache_reorder: the caches must be 16-byte aligned");
  const bool in_place = k_src == k_dst;
  ENG_CHECK(in_place == (v_src == v_dst) && (!q8 || (in_place == (ks_src == ks_dst) && in_place == (vs_src == vs_dst))),
            "kv_cache_reorder: all buffers in place, or none");
  ReorderArgs a = {};
  a.src[0] = static_cast<const unsigned char*>(k_src);
  a.src[1] = static_cast<const unsigned char*>(v_src);
  a.dst[0] = static_cast<unsigned char*>(k_dst);
  a.dst[1] = static_cast<unsigned char*>(v_dst);
  a.src_scale[0] = ks_src;
  a.src_scale[1] = vs_src;
  a.dst_scale[0] = ks_dst;
  a.dst_scale[1] = vs_dst;
  a.parent = parent;
  a.lens = kv_len;
  a.beams = static_cast<int>(beams);
  a.max_len = max_kv_len;
  a.row_bytes = static_cast<int>(head_dim * (q8 ? 1 : 2));
  a.head_bytes = kv_max_seq_len * a.row_bytes;
  a.scale_blocks = (kv_max_seq_len + 31) / 32;
  a.in_place = in_place;
  const long long chunks = (max_kv_len * a.row_bytes / 16 + 255) / 256;
  ENG_CHECK(n_kv_heads <= 0x7fffffffLL && batch <= 0xffffffffLL / 256 / 2 / chunks / n_kv_heads,
            "kv_cache_reorder: too many (group, head, token) units for one launch");
  a.heads = static_cast<int>(n_kv_heads);
  a.chunks = static_cast<unsigned>(chunks);
  const unsigned grid = static_cast<unsigned>(batch * n_kv_heads * 2 * chunks);
  auto go = [&](auto kernel) { kernel<<<grid, 256, 0, s>>>(a); };
  if (beams <= 4) go(reorder_kernel<4>);
  else if (beams <= 8) go(reorder_kernel<8>);
  else if (beams <= 16) go(reorder_kernel<16>);
  else go(reorder_kernel<32>);
  ENG_LAUNCH_CHECK();
}

}  // namespace
}  // namespace beam
}  // namespace eng

using eng::guarded;

extern "C" {

int eng_beam_select_f32(const float* logits, int64_t ld, const float* scores, const uint8_t* finished,
                        float* out_scores, int32_t* out_parent, int32_t* out_token,
                        uint8_t* out_finished, int64_t batch, int64_t beams, int64_t n_out,
                        int64_t vocab, int64_t eos, eng_stream stream) {
  return guarded([&] {
    eng::beam::select_entry(logits, false, ld, scores, finished, out_scores, out_parent, out_token, out_finished,
                            batch, beams, n_out, vocab, eos, eng::as_stream(stream));
  });
}

int eng_beam_select_f16(const eng_half* logits, int64_t ld, const float* scores, const uint8_t* finished,
                        float* out_scores, int32_t* out_parent, int32_t* out_token,
                        uint8_t* out_finished, int64_t batch, int64_t beams, int64_t n_out,
                        int64_t vocab, int64_t eos, eng_stream stream) {
  return guarded([&] {
    eng::beam::select_entry(logits, true, ld, scores, finished, out_scores, out_parent, out_token, out_finished,
                            batch, beams, n_out, vocab, eos, eng::as_stream(stream));
  });
}

int eng_kv_cache_reorder_f16(const eng_half* k_src, const eng_half* v_src, eng_half* k_dst, eng_half* v_dst,
                             const int32_t* parent, const int32_t* kv_len, int64_t batch, int64_t beams,
                             int64_t n_kv_heads, int64_t head_dim, int64_t max_kv_len,
                             int64_t kv_max_seq_len, eng_stream stream) {
  return guarded([&] {
    eng::beam::reorder_entry(k_src, v_src, nullptr, nullptr, k_dst, v_dst, nullptr, nullptr, false, parent, kv_len,
                             batch, beams, n_kv_heads, head_dim, max_kv_len, kv_max_seq_len, eng::as_stream(stream));
  });
}

int eng_kv_cache_reorder_q8(const uint8_t* k_src, const uint8_t* v_src, const float* k_scale_src,
                            const float* v_scale_src, uint8_t* k_dst, uint8_t* v_dst, float* k_scale_dst,
                            float* v_scale_dst, const int32_t* parent, const int32_t* kv_len,
                            int64_t batch, int64_t beams, int64_t n_kv_heads, int64_t head_dim,
                            int64_t max_kv_len, int64_t kv_max_seq_len, eng_stream stream) {
  return guarded([&] {
    eng::beam::reorder_entry(k_src, v_src, k_scale_src, v_scale_src, k_dst, v_dst, k_scale_dst, v_scale_dst, true,
                             parent, kv_len, batch, beams, n_kv_heads, head_dim, max_kv_len, kv_max_seq_len,
                             eng::as_stream(stream));
  });
}

}  // extern "C"
