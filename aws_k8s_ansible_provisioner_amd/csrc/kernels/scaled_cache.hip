// Appending to the scaled 8-bit cache: q and k heads normed (optional) and rotated, q written as bf16 rows,
// keys and values as codes of their page's scale (scaled_cache.h).
//
// A page's scale depends on all the entries that a call brings, and where it grows its old codes are rounded
// anew, so a page and head belong to one wave: the one that holds the page's first row of the call.  Rows
// whose slots follow each other inside a page are a run, its first row the leader; a wave looks over 32 rows
// of the batch for leaders (over one row where rows are single tokens of their sequences) and takes each run,
// its keys or its values: magnitudes first, then the codes, from registers where the run fits them.  The
// caller keeps the rows of a page together, in rising slots.
#include "scaled_cache.h"
#include "kernels.h"

namespace akap {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
constexpr int D = 128;

// cos and sin of a row's dims 8 (li & 7) .. + 7
struct Angles {
  f32x4 c[2], s[2];
};
__device__ __forceinline__ Angles angles(const ScaledAppend& p, int t, int li) {
  const int64_t pos = p.rope ? p.positions[t] : 0;
  const f32x4* at = reinterpret_cast<const f32x4*>(
      p.cos_sin + (size_t)(pos < 0 ? 0 : pos < p.max_pos ? pos : p.max_pos - 1) * D + 8 * (li & 7));
  return Angles{{at[0], at[1]}, {at[16], at[17]}};
}

// q: 16 lanes per row and four of its heads
constexpr int kQHeads = 4;
__device__ __forceinline__ void append_q(const ScaledAppend& p, int block) {
  const int per = (p.Hq + kQHeads - 1) / kQHeads;
  const long item = (long)block * 16 + (threadIdx.x >> 4);
  const int li = threadIdx.x & 15;
  if (item >= (long)p.q_rows * per) return;      // the 16 lanes of a row leave together
  const int t = (int)(item / per), h0 = (int)(item % per) * kQHeads;
  const bf16* row = p.qkv + (size_t)t * p.qkv_stride + 8 * li;
  bf16x8 raw[kQHeads];
#pragma unroll
  for (int j = 0; j < kQHeads; ++j)
    raw[j] = *reinterpret_cast<const bf16x8*>(row + min(h0 + j, p.Hq - 1) * D);
  const Angles a = angles(p, t, li);
  const bf16x8 w = p.q_w != nullptr ? *reinterpret_cast<const bf16x8*>(p.q_w + 8 * li) : bf16x8{};
#pragma unroll
  for (int j = 0; j < kQHeads; ++j) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = bf2f(raw[j][e]);
    norm_rotate(x, p.q_w != nullptr, w, p.rope, a.c, a.s, li, p.eps);
    bf16x8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = f2bf(x[e]);
    if (h0 + j < p.Hq) *reinterpret_cast<bf16x8*>(p.q_out + ((size_t)t * p.Hq + h0 + j) * D + 8 * li) = o;
  }
}

// Keys of a run: rows t .. t + n - 1 into the page from token `off` on.  16 lanes per token, 4 J tokens at a
// time, from a token that is a multiple of 4 on: four such tokens are 128-byte lines of the layout.
template <int J>
__device__ __forceinline__ void append_keys(const ScaledAppend& p, int h, int t, int n, int64_t blk, int off) {
  const int lane = threadIdx.x & 63, li = lane & 15, sub = lane >> 4;
  uint8_t* codes = p.k_cache + ((size_t)blk * p.Hkv + h) * p.BS * D;
  const bf16* src = p.qkv + (size_t)(p.Hq + h) * D + 8 * li;
  const bf16x8 w = p.k_w != nullptr ? *reinterpret_cast<const bf16x8*>(p.k_w + 8 * li) : bf16x8{};
  const int o0 = off & ~3, pieces = (off - o0 + n + 4 * J - 1) / (4 * J);
  float x[J][8];
  auto load = [&](int piece) {
    bf16x8 raw[J];
    int row[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      row[j] = t + min(max(o0 + (piece * J + j) * 4 + sub - off, 0), n - 1);
      raw[j] = *reinterpret_cast<const bf16x8*>(src + (size_t)row[j] * p.qkv_stride);
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[j][e] = bf2f(raw[j][e]);
      const Angles a = angles(p, row[j], li);
      norm_rotate(x[j], p.k_w != nullptr, w, p.rope, a.c, a.s, li, p.eps);
    }
  };
  float most = 0.f;
  for (int piece = 0; piece < pieces; ++piece) {
    load(piece);
#pragma unroll
    for (int j = 0; j < J; ++j)     // (rows beyond the run's are its first or last one again)
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fmaxf(most, scale_mag(x[j][e]));
  }
  const float inv = exp_scale(-page_exp<64>(wave_max_dpp(most), p.k_scale + (size_t)blk * p.Hkv + h, codes, off, p.BS));
  for (int piece = 0; piece < pieces; ++piece) {
    if (pieces > 1) load(piece);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int o = o0 + (piece * J + j) * 4 + sub;
      const u32x2 c = {codes4(x[j][0], x[j][1], x[j][2], x[j][3], inv),
                       codes4(x[j][4], x[j][5], x[j][6], x[j][7], inv)};
      if (o >= off && o < off + n)
        *reinterpret_cast<u32x2*>(codes + k_swz_offset(o) + k_dim_offset(8 * li)) = c;
    }
  }
}

// Values of a run: a lane holds dims 2 lane and 2 lane + 1 of 8 Q tokens, whole groups of the layout.
template <int Q>
__device__ __forceinline__ void append_values(const ScaledAppend& p, int h, int t, int n, int64_t blk, int off) {
  const int lane = threadIdx.x & 63;
  uint8_t* codes = p.v_cache + ((size_t)blk * p.Hkv + h) * p.BS * D;
  const bf16* src = p.qkv + (size_t)(p.Hq + p.Hkv + h) * D + 2 * lane;
  const int o0 = off & ~7, pieces = (off - o0 + n + 8 * Q - 1) / (8 * Q);
  bf16x2 x[Q * 8];
  auto load = [&](int piece) {
#pragma unroll
    for (int j = 0; j < Q * 8; ++j) {
      const int row = t + min(max(o0 + piece * Q * 8 + j - off, 0), n - 1);
      x[j] = *reinterpret_cast<const bf16x2*>(src + (size_t)row * p.qkv_stride);
    }
  };
  float most = 0.f;
  for (int piece = 0; piece < pieces; ++piece) {
    load(piece);
#pragma unroll
    for (int j = 0; j < Q * 8; ++j) most = fmaxf(most, fmaxf(scale_mag(bf2f(x[j][0])), scale_mag(bf2f(x[j][1]))));
  }
  const float inv = exp_scale(-page_exp<64>(wave_max_dpp(most), p.v_scale + (size_t)blk * p.Hkv + h, codes, off, p.BS));
  for (int piece = 0; piece < pieces; ++piece) {
    if (pieces > 1) load(piece);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int o = o0 + (piece * Q + q) * 8;      // the group's first token
      u32x4 c;
#pragma unroll
      for (int d = 0; d < 2; ++d)
#pragma unroll
        for (int k = 0; k < 2; ++k)
          c[2 * d + k] = codes4(bf2f(x[8 * q + 4 * k][d]), bf2f(x[8 * q + 4 * k + 1][d]),
                                bf2f(x[8 * q + 4 * k + 2][d]), bf2f(x[8 * q + 4 * k + 3][d]), inv);
      uint8_t* at = codes + (size_t)(o >> 3) * D * 8 + 16 * lane;
      if (o >= off && o + 8 <= off + n) {
        *reinterpret_cast<u32x4*>(at) = c;
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (o + k >= off && o + k < off + n) {
            at[k] = (uint8_t)(c[k >> 2] >> (8 * (k & 3)));
            at[8 + k] = (uint8_t)(c[2 + (k >> 2)] >> (8 * (k & 3)));
          }
      }
    }
  }
}

// Rows [t0, t0 + rows) of the batch (rows <= 32), one head, keys or values: the runs that begin there.
template <int ROWS>
__device__ __forceinline__ void append_runs(const ScaledAppend& p, int t0, int h, bool values) {
  const int lane = threadIdx.x & 63;
  const int64_t cap = (int64_t)p.num_blocks * p.BS;
  auto slot_of = [&](int t) -> int64_t {
    const int64_t s = t >= 0 && t < p.T ? p.slots[t] : -1;
    return s < cap ? s : -1;        // (a slot outside the cache is no slot)
  };
  const int t = t0 + lane;
  const int64_t mine = lane < ROWS ? slot_of(t) : -1;
  const int64_t before = lane < ROWS ? slot_of(t - 1) : -1;
  uint64_t leaders = __ballot(mine >= 0 && (before != mine - 1 || before < 0 || mine % p.BS == 0));
  while (leaders != 0) {
    const int l = __builtin_ctzll(leaders);
    leaders &= leaders - 1;
    const int64_t s = ((int64_t)__builtin_amdgcn_readlane((int)(mine >> 32), l) << 32) |
                      (uint32_t)__builtin_amdgcn_readlane((int)mine, l);
    const int64_t blk = s / p.BS;
    const int off = (int)(s % p.BS), room = p.BS - off;
    int n = 1;                       // rows of the run: as far as the slots go on, inside the page
    while (n < room) {
      const int i = n + lane;
      const uint64_t on = __ballot(i < room && slot_of(t0 + l + i) == s + i);
      const int more = on == ~0ull ? 64 : __builtin_ctzll(~on);
      n += more;
      if (more < 64) break;
    }
    if (values) append_values<ROWS == 1 ? 1 : 4>(p, h, t0 + l, n, blk, off);
    else append_keys<ROWS == 1 ? 1 : 8>(p, h, t0 + l, n, blk, off);
  }
}

__global__ __launch_bounds__(256) void scaled_append_kernel(ScaledAppend p, int single_blocks, int run_blocks) {
  int b = blockIdx.x;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per = 2 * p.Hkv;
  if (b < single_blocks) {
    const int item = b * 4 + w;
    if (item < p.singles * per) append_runs<1>(p, item / per, (item % per) >> 1, item & 1);
    return;
  }
  b -= single_blocks;
  if (b < run_blocks) {
    const int item = b * 4 + w, t0 = p.singles + item / per * 32;
    if (t0 < p.T) append_runs<32>(p, t0, (item % per) >> 1, item & 1);
    return;
  }
  append_q(p, b - run_blocks);
}

}  // namespace

void launch_scaled_append(const ScaledAppend& p, hipStream_t s) {
  const long per = 2 * p.Hkv;
  const long single = (p.singles * per + 3) / 4;
  const long runs = ((long)(p.T - p.singles + 31) / 32 * per + 3) / 4;
  const long q = ((long)p.q_rows * ((p.Hq + kQHeads - 1) / kQHeads) + 15) / 16;
  if (single + runs + q == 0) return;
  scaled_append_kernel<<<dim3((unsigned)(single + runs + q)), 256, 0, s>>>(p, (int)single, (int)runs);
}

}  // namespace akap
