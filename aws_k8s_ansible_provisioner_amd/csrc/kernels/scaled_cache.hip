// Appending to the scaled 8-bit cache: q and k heads normed (optional) and rotated, q written as bf16 rows,
// keys and values as codes of their page's scale (scaled_cache.h).
//
// A page's scale depends on all the entries that a call brings, and where it grows its old codes are rounded
// anew, so a page and head belong to one workgroup, or a wave: the one that finds the page's first row of the call.
// Rows whose slots follow each other inside a page are a run, its first row the leader; a workgroup looks over a span
// of 8 to 32 rows of the batch for leaders (a wave over one, where rows are single tokens of their sequences) and
// takes each run: magnitudes first, then the codes.  The caller keeps the rows of a page together, in rising slots.
// Many rows are bound by their bytes (11881 of 32 / 8 heads 55.6 us, 4.9 TB/s), few by a chain of loads: slots, positions,
// angles (one row 3.9 us in a graph).
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
__device__ __forceinline__ int place_of(const ScaledAppend& p, int t) {      // a row's position, inside the table
  const int64_t pos = p.rope ? p.positions[t] : 0;
  return (int)(pos < 0 ? 0 : pos < p.max_pos ? pos : p.max_pos - 1);
}
__device__ __forceinline__ Angles angles(const ScaledAppend& p, int place, int li) {
  const f32x4* at = reinterpret_cast<const f32x4*>(p.cos_sin + (size_t)place * D + 8 * (li & 7));
  return Angles{{at[0], at[1]}, {at[16], at[17]}};
}
// Places of the 64 rows from `from` on, one to a lane: asked for beside their slots.  (Each row for itself, behind them:
// 11881 rows 58.2 us for 55.6, 24 sequences of ~210 12.0 for 11.6.)
struct Places {
  int from, mine;
  __device__ __forceinline__ int of(const ScaledAppend& p, int t) const {
    int v = __shfl(mine, (t - from) & 63, 64);
    if (t - from >= 64) v = place_of(p, t);
    return v;
  }
};

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
  const Angles a = angles(p, place_of(p, t), li);
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

// dims 8 li .. + 7 of a row's key, normed and rotated
__device__ __forceinline__ void key_row(float (&x)[8], const ScaledAppend& p, const Places& places, int h, int row, int li,
                                        const bf16x8& w) {
  const bf16x8 raw = *reinterpret_cast<const bf16x8*>(p.qkv + (size_t)row * p.qkv_stride + (p.Hq + h) * D + 8 * li);
  const Angles a = angles(p, places.of(p, row), li);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = bf2f(raw[e]);
  norm_rotate(x, p.k_w != nullptr, w, p.rope, a.c, a.s, li, p.eps);
}
// four tokens from a multiple of 4 on are 128-byte lines of the layout
__device__ __forceinline__ void put_key(uint8_t* codes, int o, int li, const float (&x)[8], float inv) {
  *reinterpret_cast<u32x2*>(codes + k_swz_offset(o) + k_dim_offset(8 * li)) =
      u32x2{codes4(x[0], x[1], x[2], x[3], inv), codes4(x[4], x[5], x[6], x[7], inv)};
}
// dims 2 lane and 2 lane + 1 of the 8 values from the run's first + `from` on (beyond the run: its first or last)
__device__ __forceinline__ void value_rows(bf16x2 (&x)[8], const ScaledAppend& p, int h, int t, int n, int from, int lane) {
  const bf16* src = p.qkv + (size_t)(p.Hq + p.Hkv + h) * D + 2 * lane;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    x[j] = *reinterpret_cast<const bf16x2*>(src + (size_t)(t + min(max(from + j, 0), n - 1)) * p.qkv_stride);
}
__device__ __forceinline__ float value_mag(const bf16x2 (&x)[8]) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, fmaxf(scale_mag(bf2f(x[j][0])), scale_mag(bf2f(x[j][1]))));
  return m;
}
// the group of 8 tokens from o on, of which [off, off + n) are the run's
__device__ __forceinline__ void put_values(uint8_t* codes, int o, int off, int n, int lane, const bf16x2 (&x)[8], float inv) {
  u32x4 c;
#pragma unroll
  for (int d = 0; d < 2; ++d)
#pragma unroll
    for (int k = 0; k < 2; ++k)
      c[2 * d + k] = codes4(bf2f(x[4 * k][d]), bf2f(x[4 * k + 1][d]), bf2f(x[4 * k + 2][d]), bf2f(x[4 * k + 3][d]), inv);
  uint8_t* at = codes + (size_t)(o >> 3) * D * 8 + 16 * lane;
  if (o >= off && o + 8 <= off + n) {
    *reinterpret_cast<u32x4*>(at) = c;
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (o + k >= off && o + k < off + n) {
      at[k] = (uint8_t)(c[k >> 2] >> (8 * (k & 3)));
      at[8 + k] = (uint8_t)(c[2 + (k >> 2)] >> (8 * (k & 3)));
    }
}

// A run of a wave of its own, keys or values: rows t .. t + n - 1 (single tokens: one, as a rule) into the page from
// token `off` on, 4 tokens of keys or 8 of values at a time.
__device__ __forceinline__ void append_keys(const ScaledAppend& p, const Places& places, int h, int t, int n, int64_t blk, int off) {
  const int lane = threadIdx.x & 63, li = lane & 15, sub = lane >> 4;
  uint8_t* codes = p.k_cache + ((size_t)blk * p.Hkv + h) * p.BS * D;
  const bf16x8 w = p.k_w != nullptr ? *reinterpret_cast<const bf16x8*>(p.k_w + 8 * li) : bf16x8{};
  const int o0 = off & ~3, pieces = (off - o0 + n + 3) / 4;
  float x[8];
  auto load = [&](int piece) {
    const int row = t + min(max(o0 + piece * 4 + sub - off, 0), n - 1);   // (beyond the run: its first or last again)
    key_row(x, p, places, h, row, li, w);
  };
  float most = 0.f;
  for (int piece = 0; piece < pieces; ++piece) {
    load(piece);
#pragma unroll
    for (int e = 0; e < 8; ++e) most = fmaxf(most, scale_mag(x[e]));
  }
  const float inv = exp_scale(-page_exp<64>(wave_max_dpp(most), p.k_scale + (size_t)blk * p.Hkv + h, codes, off, p.BS));
  for (int piece = 0; piece < pieces; ++piece) {
    if (pieces > 1) load(piece);
    const int o = o0 + piece * 4 + sub;
    if (o >= off && o < off + n) put_key(codes, o, li, x, inv);
  }
}
__device__ __forceinline__ void append_values(const ScaledAppend& p, int h, int t, int n, int64_t blk, int off) {
  const int lane = threadIdx.x & 63;
  uint8_t* codes = p.v_cache + ((size_t)blk * p.Hkv + h) * p.BS * D;
  const int o0 = off & ~7, pieces = (off - o0 + n + 7) / 8;
  bf16x2 x[8];
  float most = 0.f;
  for (int piece = 0; piece < pieces; ++piece) {
    value_rows(x, p, h, t, n, o0 + piece * 8 - off, lane);
    most = fmaxf(most, value_mag(x));
  }
  const float inv = exp_scale(-page_exp<64>(wave_max_dpp(most), p.v_scale + (size_t)blk * p.Hkv + h, codes, off, p.BS));
  for (int piece = 0; piece < pieces; ++piece) {
    if (pieces > 1) value_rows(x, p, h, t, n, o0 + piece * 8 - off, lane);
    put_values(codes, o0 + piece * 8, off, n, lane, x, inv);
  }
}

// A run of a workgroup: its keys and its values, a wave 8 tokens of every 32, both on their way at once; kept in
// registers where the run fits kHeld such pieces (blocks of 32 tokens: one, of 64: two), else read a second time.  With a wave to
// a run's keys or values, all of its tokens one after the other, a step of 1000 rows (8 kv heads) took 15 us, of 5000
// rows in blocks of 64 (4 kv heads) 30.
template <int kHeld>
__device__ __forceinline__ void append_run(const ScaledAppend& p, const Places& places, int h, int t, int n, int64_t blk, int off,
                                           float (*red)[4]) {
  const int lane = threadIdx.x & 63, li = lane & 15, sub = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const size_t at = (size_t)blk * p.Hkv + h;
  uint8_t *kcodes = p.k_cache + at * p.BS * D, *vcodes = p.v_cache + at * p.BS * D;
  const bf16x8 kw = p.k_w != nullptr ? *reinterpret_cast<const bf16x8*>(p.k_w + 8 * li) : bf16x8{};
  const int o0 = (off & ~7) + 8 * w, pieces = ((off & 7) + n + 31) / 32;
  const int kwas = off > 0 ? stored_exp(p.k_scale[at]) : -100, vwas = off > 0 ? stored_exp(p.v_scale[at]) : -100;
  float x[kHeld][2][8];
  bf16x2 v[kHeld][8];
  // a piece's tokens of this wave; of none: nothing
  auto some = [&](int piece) { return o0 + 32 * piece + 8 > off && o0 + 32 * piece < off + n; };
  auto load = [&](float (&k)[2][8], bf16x2 (&y)[8], int piece) {
    const int o = o0 + 32 * piece;
    value_rows(y, p, h, t, n, o - off, lane);
#pragma unroll
    for (int j = 0; j < 2; ++j) key_row(k[j], p, places, h, t + min(max(o + 4 * j + sub - off, 0), n - 1), li, kw);
  };
  auto put = [&](const float (&k)[2][8], const bf16x2 (&y)[8], int piece, float kinv, float vinv) {
    const int o = o0 + 32 * piece;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int at = o + 4 * j + sub;
      if (at >= off && at < off + n) put_key(kcodes, at, li, k[j], kinv);
    }
    put_values(vcodes, o, off, n, lane, y, vinv);
  };
  float kmost = 0.f, vmost = 0.f;
  auto count = [&](const float (&k)[2][8], const bf16x2 (&y)[8]) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) kmost = fmaxf(kmost, scale_mag(k[j][e]));
    vmost = fmaxf(vmost, value_mag(y));
  };
  const bool held = pieces <= kHeld;
  if (held) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (some(i)) load(x[i], v[i], i);
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (some(i)) count(x[i], v[i]);
  } else {
    for (int i = 0; i < pieces; ++i)
      if (some(i)) {
        load(x[0], v[0], i);
        count(x[0], v[0]);
      }
  }
  kmost = wave_max_dpp(kmost);
  vmost = wave_max_dpp(vmost);
  if (lane == 0) {
    red[0][w] = kmost;
    red[1][w] = vmost;
  }
  __syncthreads();
  kmost = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  vmost = fmaxf(fmaxf(red[1][0], red[1][1]), fmaxf(red[1][2], red[1][3]));
  const int ke = max(scale_exp(kmost), kwas), ve = max(scale_exp(vmost), vwas);

  if (off > 0 && ke > kwas) codes_grow<256>(kcodes, kwas - ke, p.BS);
  if (off > 0 && ve > vwas) codes_grow<256>(vcodes, vwas - ve, p.BS);
  __syncthreads();      // (the codes rounded anew, before new ones; and `red` read, before the next run)
  if (threadIdx.x == 0) {
    p.k_scale[at] = exp_scale(ke);
    p.v_scale[at] = exp_scale(ve);
  }
  const float kinv = exp_scale(-ke), vinv = exp_scale(-ve);
  if (held) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (some(i)) put(x[i], v[i], i, kinv, vinv);
  } else {
    for (int i = 0; i < pieces; ++i)
      if (some(i)) {
        load(x[0], v[0], i);
        put(x[0], v[0], i, kinv, vinv);
      }
  }
}

// Rows [t0, t0 + rows) of the batch (rows <= 32): `run` for each run that begins there, the i-th, with whether the
// runs are few and some of them long.  The slots of 64 rows, one to a lane, tell where runs begin and, as a rule, end.
template <typename F>
__device__ __forceinline__ void for_runs(const ScaledAppend& p, int t0, int rows, const F& run) {
  const int lane = threadIdx.x & 63;
  const int64_t cap = (int64_t)p.num_blocks * p.BS;
  const bool narrow = cap < (1ll << 31);
  auto slot_of = [&](int t) -> int64_t {
    const int64_t s = t >= 0 && t < p.T ? p.slots[t] : -1;
    return s < cap ? s : -1;        // (a slot outside the cache is no slot)
  };
  const Places places{t0, place_of(p, min(t0 + lane, p.T - 1))};
  const int64_t mine = slot_of(t0 + lane), before = slot_of(t0 + lane - 1);
  const int64_t page = mine < 0 ? 0 : narrow ? (int64_t)((uint32_t)mine / (uint32_t)p.BS) : mine / p.BS;
  const int off = (int)(mine - page * p.BS);
  const bool follows = mine >= 0 && before == mine - 1 && off != 0;
  const uint64_t on = __ballot(follows);
  uint64_t leaders = __ballot(lane < rows && mine >= 0 && !follows);
  const int count = __popcll(leaders);
  uint64_t longer = on & on >> 1;
  longer &= longer >> 2;
  longer &= longer >> 4;
  longer &= longer >> 8;            // 16 rows that each follow the one before
  const bool few = count <= 3 && longer != 0;
  for (int i = 0; i < count; ++i) {
    const int l = __builtin_ctzll(leaders);
    leaders &= leaders - 1;
    const int64_t blk = ((int64_t)__builtin_amdgcn_readlane((int)(page >> 32), l) << 32) |
                        (uint32_t)__builtin_amdgcn_readlane((int)page, l);
    const int o = __builtin_amdgcn_readlane(off, l);
    int n = 1 + __builtin_ctzll(~(on >> 1 >> l));     // rows of the run (at most 64 - l)
    while (l + n >= 64 && n < p.BS - o) {             // and of what follows the 64
      const int at = n + lane;
      const uint64_t more = __ballot(at < p.BS - o && slot_of(t0 + l + at) == blk * p.BS + o + at);
      n += more == ~0ull ? 64 : __builtin_ctzll(~more);
      if (more != ~0ull) break;
    }
    run(i, few, places, t0 + l, n, blk, o);
  }
}

template <int HELD>
__global__ __launch_bounds__(256) void scaled_append_kernel(ScaledAppend p, int single_blocks, int run_blocks,
                                                            int rows) {
  __shared__ float red[2][4];
  int b = blockIdx.x;
  if (b < single_blocks) {
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), per = 2 * p.Hkv;
    const int item = b * 4 + w, t = item / per, h = (item - t * per) >> 1;
    if (t >= p.singles) return;
    for_runs(p, t, 1, [&](int, bool, const Places& places, int t, int n, int64_t blk, int off) {
      if (item & 1) append_values(p, h, t, n, blk, off);
      else append_keys(p, places, h, t, n, blk, off);
    });
    return;
  }
  b -= single_blocks;
  if (b < run_blocks) {
    const int span = b / p.Hkv, h = b - span * p.Hkv;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for_runs(p, p.singles + rows * span, rows, [&](int i, bool few, const Places& places, int t, int n, int64_t blk,
                                                            int off) {
      if (few) {
        append_run<HELD>(p, places, h, t, n, blk, off, red);
        return;
      }
      // Many runs, or short ones: a wave to the keys or the values of each.  64 sequences of 3 tokens, 8 kv heads, in
      // spans of 32 rows: 12 us, one run after the other 31; 3 of 2 tokens 5.4, else 10.4.  (Three may be long: 8
      // prompts of ~100 behind 40 11.8 us, by waves 15.8.)
      const int job = 2 * i + (i >> 1);
      if ((job & 3) == w) append_keys(p, places, h, t, n, blk, off);
      if ((job + 1 & 3) == w) append_values(p, h, t, n, blk, off);
    });
    return;
  }
  append_q(p, b - run_blocks);
}

}  // namespace

void launch_scaled_append(const ScaledAppend& p, hipStream_t s) {
  const long per = 2 * p.Hkv;
  const long single = (p.singles * per + 3) / 4;
  // Runs begin anywhere, and a span's are taken in turn: spans of 8 rows where their workgroups are at most 512, two to a
  // unit, of 16 up to 1300, else of 32.  The shape decides as well, which the host does not know: short and ragged runs
  // gain by small spans, a prompt that begins its own pages loses (every other span of 16 finds no leader).  8 kv heads,
  // spans of 8, 16 and 32, us, ten sets of rows in turn or (*) one:
  //   up to 512     49 sequences of 3 tokens behind some 7.4, 9.9, 15.0; 20 of 24 9.0, 9.4, 12.3; but one of 500 6.2, 5.6, 5.7
  //   up to 1300    8 of ~130 9.0, 9.8, 10.6; 200 of ~8 13.9, 12.9, 16.0; 4 of ~270 8.6, 8.7, 10.0; 4 of ~585 12.9, 10.1,
  //                 10.6; but one of 1000 8.0, 6.5, 5.9, of 2048 13.7, 8.4, 7.0; 2 of 1000 12.8, 9.2, 8.6; 4 kv heads, blocks
  //                 of 64, 24 of ~200 from their pages' first tokens on 15.4, 13.5, 13.1, behind ~30 15.2, 14.1, 14.5
  //   1340 to 1660  12 of ~220 13.5, 11.9, 12.4; 12 of ~270* 13.6, 13.0, 13.2; 80 of ~40* 17.1, 14.6, 13.8
  //   from 2000 on  40 of ~100* 17.4, 17.6, 14.7; 20 of ~300* 22.7, 18.7, 17.8; 60 of ~200* 38.3, 28.2, 23.6
  const long rest = p.T - p.singles;
  auto spans = [&](int rows) { return (rest + rows - 1) / rows * p.Hkv; };
  const int rows = spans(8) <= 512 ? 8 : spans(16) <= 1300 ? 16 : 32;
  const long runs = spans(rows);
  const long q = ((long)p.q_rows * ((p.Hq + kQHeads - 1) / kQHeads) + 15) / 16;
  if (single + runs + q == 0) return;
  const dim3 grid((unsigned)(single + runs + q));
  if (p.BS <= 32) scaled_append_kernel<1><<<grid, 256, 0, s>>>(p, (int)single, (int)runs, rows);
  else scaled_append_kernel<2><<<grid, 256, 0, s>>>(p, (int)single, (int)runs, rows);
}

}  // namespace akap
