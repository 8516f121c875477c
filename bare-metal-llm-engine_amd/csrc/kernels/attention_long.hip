// attention_long.hip -- attention over long contexts: new tokens of a batch, a prompt or
// one token each, with a sliding window and first tokens that stay visible, and single
// tokens over a prefix that several sequences share. Caches are fp16 or e4m3 (kv_q8.hip
// has the format).
#include "attention_few.hpp"

#include <cmath>

namespace eng {
namespace attn {
namespace {

constexpr int kMaxStates = 256;  // states of a row that a merge takes

// out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s over a row's states: one wave per
// row, four rows to a workgroup, C states' loads issued together. Rows of tokens that are
// not there are left alone. Bound by the round trip of a state's loads: 3.1 us at 32 rows,
// 4.8 at 512 to 1024.
template <int D, int C>
__global__ __launch_bounds__(256) void merge_kernel(Args a, unsigned rows, int states) {
  constexpr int DPL = D / 64;
  const int lane = threadIdx.x & 63;
  const unsigned row = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= rows) return;
  if (a.causal) {
    const unsigned t = row / static_cast<unsigned>(a.n_heads);
    const unsigned b = t / static_cast<unsigned>(a.s_new);
    if (static_cast<int>(t - b * static_cast<unsigned>(a.s_new)) >= unit_of(a, b).n) return;
  }
  const long long base = static_cast<long long>(row) * states;
  float m = kNegInf, l = 0.0f;
  float o[DPL];
#pragma unroll
  for (int j = 0; j < DPL; ++j) o[j] = 0.0f;
  for (int s0 = 0; s0 < states; s0 += C) {
    // states past the last one are read as the last one, with weight 0
    const long long mine = base + min(s0 + min(lane, C - 1), states - 1);
    const floatx2 ml = *reinterpret_cast<const floatx2*>(a.part_ml + 2 * mine);
    float os[C][DPL];
#pragma unroll
    for (int s = 0; s < C; ++s) {
      const float* p = a.part_o + (base + min(s0 + s, states - 1)) * D + lane;
#pragma unroll
      for (int j = 0; j < DPL; ++j) os[s][j] = p[64 * j];
    }
    const bool live = lane < C && s0 + lane < states;
    float mx = live ? ml[0] : kNegInf;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) mx = fmaxf(mx, __shfl_xor(mx, off));
    const float mn = fmaxf(m, mx);
    const float was = weight2(m, mn);
    m = mn;
    const float w = live ? weight2(ml[0], mn) : 0.0f;
    l = l * was + gemv::wave_sum(live ? w * ml[1] : 0.0f);
#pragma unroll
    for (int j = 0; j < DPL; ++j) o[j] *= was;
#pragma unroll
    for (int s = 0; s < C; ++s) {
      const float ws = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), s));
#pragma unroll
      for (int j = 0; j < DPL; ++j) o[j] = s0 + s < states ? fmaf(ws, os[s][j], o[j]) : o[j];
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int j = 0; j < DPL; ++j)
    a.out[static_cast<long long>(row) * D + lane + 64 * j] = static_cast<_Float16>(o[j] * inv);
}

template <int D>
void merge(const Args& a, long long rows, int states, hipStream_t s) {
  const unsigned grid = static_cast<unsigned>((rows + 3) / 4);
  if (states <= 8) merge_kernel<D, 8><<<grid, 256, 0, s>>>(a, static_cast<unsigned>(rows), states);
  else merge_kernel<D, 16><<<grid, 256, 0, s>>>(a, static_cast<unsigned>(rows), states);
  ENG_LAUNCH_CHECK();
}

// Launches of a part: tiles of many rows, or up to two parts of few rows together.
constexpr int tile_rows(int waves) { return 32 * waves; }
template <int D, bool Q8, int NW>
void tiles(const Args& a, hipStream_t s) {
  constexpr std::size_t kLds = 2 * tile_buffers(NW) * kTileKeys * D * sizeof(_Float16);
  static std::atomic<bool> done[64];
  allow_staged_lds(reinterpret_cast<const void*>(tile_kernel<D, Q8, NW>), done, kLds);
  const dim3 grid(static_cast<unsigned>(a.units * a.row_tiles), static_cast<unsigned>(a.nsplit));
  tile_kernel<D, Q8, NW><<<grid, 64 * NW, kLds, s>>>(a);
  ENG_LAUNCH_CHECK();
}
template <int D>
void tiles(const Args& a, bool q8, int waves, hipStream_t s) {
  if constexpr (D == 128) {
    if (waves == 8) {
      q8 ? tiles<D, true, 8>(a, s) : tiles<D, false, 8>(a, s);
      return;
    }
  }
  q8 ? tiles<D, true, 4>(a, s) : tiles<D, false, 4>(a, s);
}
template <int D, bool Q8>
void few(const Args& a, const Args& b, int waves, hipStream_t s) {
  const long long wgs0 = a.units * a.row_tiles * a.nsplit;
  const auto wgs = static_cast<unsigned>(wgs0 + b.units * b.row_tiles * b.nsplit);
  const auto first = static_cast<unsigned>(wgs0);
  if (waves == 1) few_kernel<D, Q8, 1><<<wgs, 64, 0, s>>>(a, b, first);
  else few_kernel<D, Q8, 4><<<wgs, 64 * 4, 0, s>>>(a, b, first);
  ENG_LAUNCH_CHECK();
}
template <int D>
void few(const Args& a, const Args& b, bool q8, int waves, hipStream_t s) {
  q8 ? few<D, true>(a, b, waves, s) : few<D, false>(a, b, waves, s);
}

// Waves of a tile: at D = 128 eight where that leaves a workgroup for every CU, else four.
int tile_waves(long long units, long long unit_rows, long long D) {
  if (D == 64) return 4;
  return units * ((unit_rows + tile_rows(8) - 1) / tile_rows(8)) >= device_cu_count() ? 8 : 4;
}

int tiles_of(long long rows, int tile) { return static_cast<int>((rows + tile - 1) / tile); }

// Splits of the keys, up to `keys`, of `wgs` workgroups of many rows: as many as fill the
// CUs, two workgroups of four waves to each, at least four tiles a split.
int tile_splits(long long wgs, long long keys, int waves) {
  const long long want = (8 / waves) * static_cast<long long>(device_cu_count()) / wgs;
  return static_cast<int>(std::max(1ll, std::min({want, (keys + kTileKeys - 1) / kTileKeys / 4,
                                                  static_cast<long long>(kMaxStates)})));
}
// And of few rows: one workgroup to a CU, at least two blocks a split, and one split up to
// 12 blocks at D = 128 or 24 at D = 64 (one token of 32 heads: 300 tokens 7.3 us, 8.2 in
// four splits; 8192 tokens of 32 / 8 heads 12.5-13.3 in 16 or 32 splits, 16.5 in 8 or 64; 16
// sequences of 2048 30 in 1 to 4, 34 in 8). Where one split needs no merge, up to more
// blocks the fewer the splits that it stands for: 128 units of 600 tokens 10.3 us in one
// and 13.0 in two, of 1500 22.2 and 21.5; 64 units of 400 8.5 and 9.1 in four, of 1000 13.3
// and 12.1.
int few_splits(long long wgs, long long keys, long long D, bool merged) {
  const long long blocks = (keys + kKvBlock - 1) / kKvBlock;
  const long long want = device_cu_count() / wgs;
  const long long single = merged ? 12 : std::max(12ll, 72 / std::max(want, 1ll));
  if (blocks * D <= single * 128) return 1;
  return static_cast<int>(std::max(1ll, std::min({want, blocks / 2, static_cast<long long>(kMaxStates)})));
}

// Waves of a workgroup of few rows. One, without three that find nothing to do, where a split
// is one block, and up to four blocks where four workgroups for each CU hide the chain of
// loads: one token of 64 sequences of 32 heads of 128, fp16, 20 tokens 8.2 us (18.2 with
// four waves), 100 tokens 19.7 (27.2), 200 34 (36); of 16 sequences of 8 KV heads, 100 tokens
// 7.4 (6.2).
int few_waves(long long wgs, long long blocks) {
  return blocks <= 1 || (blocks <= 4 && wgs >= 4 * static_cast<long long>(device_cu_count())) ? 1 : 4;
}

constexpr long long kMaxLen = 0x7fffffffLL - 2 * kTileKeys;  // 32-bit positions, up to a tile past the end

// State of a call in the stream's arena: o [rows][states][D], then (m, l) of each.
std::size_t state_bytes(long long rows, int states, long long D) {
  return static_cast<std::size_t>(rows) * states * (D + 2) * sizeof(float);
}

void run_window(Args a, long long batch, long long D, int split_kv, bool q8, hipStream_t s) {
  const long long rows = batch * a.s_new * a.n_heads;
  const long long unit_rows = static_cast<long long>(a.s_new) * a.group;
  const bool one = a.s_new == 1;  // a unit's rows see the same keys
  a.units = batch * a.n_kv;
  const int waves = tile_waves(a.units, unit_rows, D);
  const int tile = one ? kFewRows : tile_rows(waves);
  ENG_CHECK(unit_rows <= 0x3fffffffLL && rows <= 0xffffffffLL - 4 && threads_fit((rows + 3) / 4, 256) &&
                threads_fit(a.units, 256) && threads_fit(a.units * tiles_of(unit_rows, tile), 512),
            "attention_window: too many query rows for one launch");
  a.row_tiles = tiles_of(unit_rows, tile);
  long long keys = a.max_len;  // what a tile of rows can see
  if (a.window != 0)
    keys = std::min(keys, a.window + a.sinks + std::min<long long>(a.s_new, tile / a.group + 2) + kKvBlock);
  const long long step = one ? kKvBlock : kTileKeys;
  const long long most = std::max(1ll, (keys + step - 1) / step);
  a.nsplit = split_kv == 0 ? (one ? few_splits(a.units * a.row_tiles, keys, D, false)
                                  : tile_splits(a.units * a.row_tiles, keys, waves))
                           : static_cast<int>(std::min<long long>({split_kv, most, kMaxStates}));
  if (one)
    ENG_CHECK(threads_fit(a.units * a.row_tiles * a.nsplit, 256),
              "attention_window: too many query rows for one launch");
  a.part_stride = a.nsplit;
  auto go = [&](auto dim) {
    constexpr int kD = decltype(dim)::value;
    auto launch = [&] {
      const long long wgs = a.units * a.row_tiles * a.nsplit;
      if (one) few<kD>(a, Args{}, q8, few_waves(wgs, (most + a.nsplit - 1) / a.nsplit), s);
      else tiles<kD>(a, q8, waves, s);
    };
    if (a.nsplit == 1) {
      launch();
      return;
    }
    StreamScratch scratch(s, state_bytes(rows, a.nsplit, kD));
    a.part_o = static_cast<float*>(scratch.get());
    a.part_ml = a.part_o + rows * a.nsplit * kD;
    launch();
    merge<kD>(a, rows, a.nsplit, s);
  };
  if (D == 64) go(std::integral_constant<int, 64>{});
  else go(std::integral_constant<int, 128>{});
}

// Shared rows of a KV head up to which the prefix is read in tiles of 16 of them, all in the
// launch that reads the sequences' own tokens, though each tile reads it (the L2 holds it):
// 64 rows, 2000 tokens, 4 heads of 64: 10.4 us, 16.4 in one tile of 128 rows; 128 rows, 8192
// tokens, 8 heads of 128 27-33 (30-35); eight such groups of 2000 tokens 47-68 (48-62); 256
// rows 38 (38).
constexpr long long kFewShared = 128;

void run_prefix(Args shared, Args mine, long long n_prefix, long long batch, long long D, int split_kv,
                bool q8, hipStream_t s) {
  const long long rows = batch * mine.n_heads;
  const long long unit_rows = static_cast<long long>(shared.s_new) * shared.group;
  const bool few_shared = unit_rows <= kFewShared;
  shared.units = n_prefix * shared.n_kv;
  const int waves = tile_waves(shared.units, unit_rows, D);
  const int tile = few_shared ? kFewRows : tile_rows(waves);
  mine.units = batch * mine.n_kv;
  ENG_CHECK(unit_rows <= 0x3fffffffLL && rows <= 0xffffffffLL - 4 && threads_fit((rows + 3) / 4, 256) &&
                threads_fit(shared.units, 256) && threads_fit(mine.units, 256),
            "attention_prefix: too many query rows for one launch");
  shared.row_tiles = tiles_of(unit_rows, tile);
  mine.row_tiles = tiles_of(mine.group, kFewRows);
  auto splits = [&](const Args& a, bool of_few) {
    if (a.max_len == 0) return 0;
    const long long step = of_few ? kKvBlock : kTileKeys;
    const long long wgs = a.units * a.row_tiles;
    const int chosen = split_kv != 0 ? static_cast<int>(std::min<long long>(split_kv, (a.max_len + step - 1) / step))
                       : of_few      ? few_splits(wgs, a.max_len, D, true)
                                     : tile_splits(wgs, a.max_len, waves);
    return std::min(chosen, kMaxStates / 2);
  };
  shared.nsplit = splits(shared, few_shared);
  mine.nsplit = splits(mine, true);
  ENG_CHECK(threads_fit(shared.units * shared.row_tiles * std::max(1, few_shared ? shared.nsplit : 1) +
                            mine.units * mine.row_tiles * std::max(1, mine.nsplit), 512),
            "attention_prefix: too many query rows for one launch");
  // of the launch of few rows: workgroups, and the blocks of a split at the most
  auto blocks_of = [](const Args& a) {
    const long long blocks = (a.max_len + kKvBlock - 1) / kKvBlock;
    return a.nsplit > 0 ? (blocks + a.nsplit - 1) / a.nsplit : 0;
  };
  long long wgs = mine.units * mine.row_tiles * mine.nsplit;
  long long blocks = blocks_of(mine);
  if (few_shared) {
    wgs += shared.units * shared.row_tiles * shared.nsplit;
    blocks = std::max(blocks, blocks_of(shared));
  }
  const int states = shared.nsplit + mine.nsplit;
  shared.part_stride = mine.part_stride = states;
  mine.part0 = shared.nsplit;
  auto go = [&](auto dim) {
    constexpr int kD = decltype(dim)::value;
    StreamScratch scratch(s, state_bytes(rows, states, kD));
    shared.part_o = mine.part_o = static_cast<float*>(scratch.get());
    shared.part_ml = mine.part_ml = shared.part_o + rows * states * kD;
    if (!few_shared && shared.nsplit > 0) tiles<kD>(shared, q8, waves, s);
    if (few_shared) few<kD>(shared, mine, q8, few_waves(wgs, blocks), s);
    else if (mine.nsplit > 0) few<kD>(mine, Args{}, q8, few_waves(wgs, blocks), s);
    merge<kD>(mine, rows, states, s);
  };
  if (D == 64) go(std::integral_constant<int, 64>{});
  else go(std::integral_constant<int, 128>{});
}

void window_entry(const eng_half* q, const void* k, const void* v, const float* ks, const float* vs,
                  bool q8, eng_half* out, const int32_t* pos, const int32_t* n_new, int64_t batch,
                  int64_t s_new, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim, int64_t window,
                  int64_t sinks, int64_t max_kv_len, int64_t kv_max_seq_len, float scale, int split_kv,
                  hipStream_t s) {
  ENG_CHECK(q != nullptr, "attention_window: q is null");
  ENG_CHECK(k != nullptr, "attention_window: k_cache is null");
  ENG_CHECK(v != nullptr, "attention_window: v_cache is null");
  ENG_CHECK(!q8 || (ks != nullptr && vs != nullptr), "attention_window: k_scale/v_scale is null");
  ENG_CHECK(out != nullptr, "attention_window: out is null");
  ENG_CHECK(pos != nullptr, "attention_window: pos is null");
  ENG_CHECK(batch >= 0, "attention_window: batch must be non-negative");
  ENG_CHECK(s_new >= 0, "attention_window: s_new must be non-negative");
  ENG_CHECK(n_heads > 0, "attention_window: n_heads must be positive");
  ENG_CHECK(n_kv_heads > 0, "attention_window: n_kv_heads must be positive");
  ENG_CHECK(n_heads % n_kv_heads == 0, "attention_window: n_heads must be divisible by n_kv_heads");
  ENG_CHECK(head_dim == 64 || head_dim == 128, "attention_window: head_dim must be 64 or 128");
  ENG_CHECK(window >= 0, "attention_window: window must be non-negative");
  ENG_CHECK(sinks >= 0, "attention_window: sinks must be non-negative");
  ENG_CHECK(max_kv_len >= 0, "attention_window: max_kv_len must be non-negative");
  ENG_CHECK(kv_max_seq_len >= max_kv_len, "attention_window: kv_max_seq_len < max_kv_len");
  ENG_CHECK(kv_max_seq_len <= kMaxLen, "attention_window: kv_max_seq_len must be below 2^31 - 128");
  ENG_CHECK(std::isfinite(scale), "attention_window: scale must be finite");
  ENG_CHECK(split_kv >= 0, "attention_window: split_kv must be non-negative");
  ENG_CHECK(aligned_to(k, 16) && aligned_to(v, 16), "attention_window: the caches must be 16-byte aligned");
  if (batch == 0 || s_new == 0) return;
  constexpr long long kMost = 0x7fffffffLL;
  ENG_CHECK(batch <= kMost && s_new <= kMost && n_heads <= kMost && batch * n_heads <= kMost &&
                batch * n_heads <= (kMost << 1) / s_new,
            "attention_window: too many query rows for one launch");
  Args a = {};
  a.q = reinterpret_cast<const _Float16*>(q);
  a.out = reinterpret_cast<_Float16*>(out);
  a.k = k;
  a.v = v;
  a.ks = ks;
  a.vs = vs;
  a.pos = pos;
  a.n_new = n_new;
  a.kv_max = kv_max_seq_len;
  a.n_heads = n_heads;
  a.n_kv = static_cast<int>(n_kv_heads);
  a.group = static_cast<int>(n_heads / n_kv_heads);
  a.s_new = static_cast<int>(s_new);
  a.max_len = static_cast<int>(max_kv_len);
  a.causal = true;
  a.window = std::min<int64_t>(window, 1ll << 40);
  a.sinks = window == 0 ? 0 : static_cast<int>(std::min(sinks, max_kv_len));
  a.scale = scale;
  run_window(a, batch, head_dim, split_kv, q8, s);
}

void prefix_entry(const eng_half* q, const void* kp, const void* vp, const float* kps, const float* vps,
                  const int32_t* prefix_len, const void* k, const void* v, const float* ks,
                  const float* vs, const int32_t* kv_len, bool q8, eng_half* out, int64_t n_prefix,
                  int64_t batch, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim,
                  int64_t max_prefix_len, int64_t prefix_max_seq_len, int64_t max_kv_len,
                  int64_t kv_max_seq_len, float scale, int split_kv, hipStream_t s) {
  ENG_CHECK(q != nullptr, "attention_prefix: q is null");
  ENG_CHECK(kp != nullptr && vp != nullptr, "attention_prefix: k_prefix/v_prefix is null");
  ENG_CHECK(k != nullptr && v != nullptr, "attention_prefix: k_cache/v_cache is null");
  ENG_CHECK(!q8 || (kps != nullptr && vps != nullptr), "attention_prefix: k_prefix_scale/v_prefix_scale is null");
  ENG_CHECK(!q8 || (ks != nullptr && vs != nullptr), "attention_prefix: k_scale/v_scale is null");
  ENG_CHECK(prefix_len != nullptr, "attention_prefix: prefix_len is null");
  ENG_CHECK(kv_len != nullptr, "attention_prefix: kv_len is null");
  ENG_CHECK(out != nullptr, "attention_prefix: out is null");
  ENG_CHECK(batch >= 0, "attention_prefix: batch must be non-negative");
  ENG_CHECK(n_prefix > 0, "attention_prefix: n_prefix must be positive");
  ENG_CHECK(batch % n_prefix == 0, "attention_prefix: batch must be divisible by n_prefix");
  ENG_CHECK(n_heads > 0, "attention_prefix: n_heads must be positive");
  ENG_CHECK(n_kv_heads > 0, "attention_prefix: n_kv_heads must be positive");
  ENG_CHECK(n_heads % n_kv_heads == 0, "attention_prefix: n_heads must be divisible by n_kv_heads");
  ENG_CHECK(head_dim == 64 || head_dim == 128, "attention_prefix: head_dim must be 64 or 128");
  ENG_CHECK(max_prefix_len >= 0, "attention_prefix: max_prefix_len must be non-negative");
  ENG_CHECK(max_kv_len >= 0, "attention_prefix: max_kv_len must be non-negative");
  ENG_CHECK(prefix_max_seq_len >= max_prefix_len, "attention_prefix: prefix_max_seq_len < max_prefix_len");
  ENG_CHECK(kv_max_seq_len >= max_kv_len, "attention_prefix: kv_max_seq_len < max_kv_len");
  ENG_CHECK(prefix_max_seq_len <= kMaxLen && kv_max_seq_len <= kMaxLen,
            "attention_prefix: prefix_max_seq_len and kv_max_seq_len must be below 2^31 - 128");
  ENG_CHECK(std::isfinite(scale), "attention_prefix: scale must be finite");
  ENG_CHECK(split_kv >= 0, "attention_prefix: split_kv must be non-negative");
  ENG_CHECK(aligned_to(kp, 16) && aligned_to(vp, 16) && aligned_to(k, 16) && aligned_to(v, 16),
            "attention_prefix: the caches must be 16-byte aligned");
  if (batch == 0) return;
  constexpr long long kMost = 0x7fffffffLL;
  ENG_CHECK(batch <= kMost && n_heads <= kMost && batch * n_heads <= kMost,
            "attention_prefix: too many query rows for one launch");
  if (max_prefix_len == 0 && max_kv_len == 0) {
    fill_zero_async(out, static_cast<std::size_t>(batch * n_heads * head_dim) * sizeof(eng_half), s);
    return;
  }
  Args a = {};
  a.q = reinterpret_cast<const _Float16*>(q);
  a.out = reinterpret_cast<_Float16*>(out);
  a.n_heads = n_heads;
  a.n_kv = static_cast<int>(n_kv_heads);
  a.group = static_cast<int>(n_heads / n_kv_heads);
  a.causal = false;
  a.scale = scale;
  Args shared = a, mine = a;
  shared.k = kp;
  shared.v = vp;
  shared.ks = kps;
  shared.vs = vps;
  shared.pos = prefix_len;
  shared.kv_max = prefix_max_seq_len;
  shared.max_len = static_cast<int>(max_prefix_len);
  shared.s_new = static_cast<int>(batch / n_prefix);
  mine.k = k;
  mine.v = v;
  mine.ks = ks;
  mine.vs = vs;
  mine.pos = kv_len;
  mine.kv_max = kv_max_seq_len;
  mine.max_len = static_cast<int>(max_kv_len);
  mine.s_new = 1;
  run_prefix(shared, mine, n_prefix, batch, head_dim, split_kv, q8, s);
}

}  // namespace
}  // namespace attn
}  // namespace eng

using eng::guarded;

extern "C" {

int eng_attention_window_f16(const eng_half* q, const eng_half* k_cache, const eng_half* v_cache,
                             eng_half* out, const int32_t* pos, const int32_t* n_new, int64_t batch,
                             int64_t s_new, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim,
                             int64_t window, int64_t sinks, int64_t max_kv_len,
                             int64_t kv_max_seq_len, float scale, int split_kv, eng_stream stream) {
  return guarded([&] {
    eng::attn::window_entry(q, k_cache, v_cache, nullptr, nullptr, false, out, pos, n_new, batch, s_new,
                            n_heads, n_kv_heads, head_dim, window, sinks, max_kv_len, kv_max_seq_len,
                            scale, split_kv, eng::as_stream(stream));
  });
}

int eng_attention_window_q8(const eng_half* q, const uint8_t* k_cache, const uint8_t* v_cache,
                            const float* k_scale, const float* v_scale, eng_half* out,
                            const int32_t* pos, const int32_t* n_new, int64_t batch, int64_t s_new,
                            int64_t n_heads, int64_t n_kv_heads, int64_t head_dim, int64_t window,
                            int64_t sinks, int64_t max_kv_len, int64_t kv_max_seq_len, float scale,
                            int split_kv, eng_stream stream) {
  return guarded([&] {
    eng::attn::window_entry(q, k_cache, v_cache, k_scale, v_scale, true, out, pos, n_new, batch, s_new,
                            n_heads, n_kv_heads, head_dim, window, sinks, max_kv_len, kv_max_seq_len,
                            scale, split_kv, eng::as_stream(stream));
  });
}

int eng_attention_prefix_f16(const eng_half* q, const eng_half* k_prefix, const eng_half* v_prefix,
                             const int32_t* prefix_len, const eng_half* k_cache,
                             const eng_half* v_cache, const int32_t* kv_len, eng_half* out,
                             int64_t n_prefix, int64_t batch, int64_t n_heads, int64_t n_kv_heads,
                             int64_t head_dim, int64_t max_prefix_len, int64_t prefix_max_seq_len,
                             int64_t max_kv_len, int64_t kv_max_seq_len, float scale, int split_kv,
                             eng_stream stream) {
  return guarded([&] {
    eng::attn::prefix_entry(q, k_prefix, v_prefix, nullptr, nullptr, prefix_len, k_cache, v_cache,
                            nullptr, nullptr, kv_len, false, out, n_prefix, batch, n_heads, n_kv_heads,
                            head_dim, max_prefix_len, prefix_max_seq_len, max_kv_len, kv_max_seq_len,
                            scale, split_kv, eng::as_stream(stream));
  });
}

int eng_attention_prefix_q8(const eng_half* q, const uint8_t* k_prefix, const uint8_t* v_prefix,
                            const float* k_prefix_scale, const float* v_prefix_scale,
                            const int32_t* prefix_len, const uint8_t* k_cache, const uint8_t* v_cache,
                            const float* k_scale, const float* v_scale, const int32_t* kv_len,
                            eng_half* out, int64_t n_prefix, int64_t batch, int64_t n_heads,
                            int64_t n_kv_heads, int64_t head_dim, int64_t max_prefix_len,
                            int64_t prefix_max_seq_len, int64_t max_kv_len, int64_t kv_max_seq_len,
                            float scale, int split_kv, eng_stream stream) {
  return guarded([&] {
    eng::attn::prefix_entry(q, k_prefix, v_prefix, k_prefix_scale, v_prefix_scale, prefix_len, k_cache,
                            v_cache, k_scale, v_scale, kv_len, true, out, n_prefix, batch, n_heads,
                            n_kv_heads, head_dim, max_prefix_len, prefix_max_seq_len, max_kv_len,
                            kv_max_seq_len, scale, split_kv, eng::as_stream(stream));
  });
}

}  // extern "C"
