// Attention over the scaled 8-bit cache (scaled_cache.h): single rows of running sequences (decode) and rows of
// prompts.  S^T = K Q^T and O^T = V^T P^T on the matrix cores, keys as rows and queries as columns, so that a
// query's maximum and sum stay in one lane column; queries and softmax weights are bf16, codes are widened to
// bf16 with their scale, which is exact, sums and statistics are fp32.  Weights are rounded because the matrix
// cores take bf16 at sixteen times the rate of fp32, as the attention over the other caches does it: half a step,
// 2^-8 of each.  Against 64 bits a step of 128 rows is off by 0.0022 of its outputs' size, with fp32 weights, where
// the outputs' own rounding is left, by 0.0017.
//
// A key is seen if it lies inside the sequence's length, the block table and a page of the cache (a table entry
// outside the cache: its keys are left out).  A row that sees none is zero.
#include <algorithm>

#include "scaled_cache.h"
#include "kernels.h"

namespace akap {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
constexpr int D = 128;

// keys of a sequence that its block table can hold
__device__ __forceinline__ int keys_of(const ScaledAttn& p, int seq) {
  const int64_t most = (int64_t)p.bt_cols * p.BS;
  const int n = p.seq_lens[seq];
  return n < 0 ? 0 : n < most ? n : (int)most;
}

// ------------------------------------------------------------------------------------------------- decode
// grid (sequences, kv heads, partitions), four or eight waves that take a partition's 32-token chunks in turn; the columns of
// the 16 x 16 x 32 products are the kv head's query heads.  A chunk is 8 loads of 16 bytes to a lane: of K the dims
// 64 p + 16 g .. + 15 of a token (its k-steps 2 p and 2 p + 1 contract over the first and second 8, q in the same
// order), of V two dims of an 8-token group.  The next chunk's K is asked for when this one's scores are formed, its
// V when this one's is used up: a whole chunk on the way in the registers of one.
// Rows that fill the card are bound by their codes' bytes: 200 rows of up to 4000 keys (16 / 8 heads) 221 us, 6.1 TB/s,
// 64 of up to 2048 (32 / 8) 35.3, 5.6; few by a chain of loads: one at 333 5.1 us in a graph, 3 of up to 30000 of one kv
// head 13.8, of which the merge within the launch 2 to 3.
struct Chunk {
  u32x4 k[2][2];   // [16-token tile][p]
  u32x4 v[4];      // dims 32 n + 2 r and + 1 of group g
};
constexpr int kStream = 2;     // buffer instructions: read once a step, not kept in the caches

// the 32-token chunk of a cache that begins at byte `at`; 0 and nothing read where there is none
__device__ __forceinline__ __amdgpu_buffer_rsrc_t chunk_rsrc(const uint8_t* cache, int64_t at, bool some) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)(cache + at), (short)0, some ? 32 * D : 0, 0x00020000);
}
__device__ __forceinline__ void load_k(Chunk& c, __amdgpu_buffer_rsrc_t rs) {
  const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
  const int at = (g >> 1) * 512 + r * 32 + (g & 1) * 16;
#pragma unroll
  for (int tt = 0; tt < 2; ++tt)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      c.k[tt][i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, at + tt * 2048 + i * 1024, 0, kStream));
}
__device__ __forceinline__ void load_v(Chunk& c, __amdgpu_buffer_rsrc_t rs) {
  const int lane = threadIdx.x & 63, at = (lane >> 4) * D * 8 + (lane & 15) * 16;
#pragma unroll
  for (int n = 0; n < 4; ++n)
    c.v[n] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, at + n * 256, 0, kStream));
}

struct Row {
  f32x4 o[8];      // dims 32 (i >> 1) + 8 g + 2 j + (i & 1), j = 0..3
  float m, l;      // running maximum (log2), this lane's part of the sum
};

// scores of tokens 8 g + 0..7 of the chunk
__device__ __forceinline__ void chunk_scores(float (&x)[8], const bf16x8 (&q)[4], const Chunk& c, float kscale) {
  f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      s[tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes_wide(c.k[tt][i][0], c.k[tt][i][1], 1.f), q[2 * i], s[tt], 0, 0, 0);
      s[tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes_wide(c.k[tt][i][2], c.k[tt][i][3], 1.f), q[2 * i + 1], s[tt], 0, 0, 0);
    }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = s[i >> 2][i & 3] * kscale;
}

// left: the chunk's keys that are seen; the others may hold any codes.  (One body with small branches: a second one
// for whole chunks took the kernel from 126 registers to 202, from four waves a SIMD to two.)
__device__ __forceinline__ void chunk_rows(Row& st, float (&x)[8], Chunk& c, float vscale, int left) {
  const int g = (threadIdx.x & 63) >> 4;
  if (left < 32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 8 * g + i < left ? x[i] : -INFINITY;
  }
  float top = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) top = fmaxf(top, x[i]);
  top = fmaxf(top, __shfl_xor(top, 16, 64));
  top = fmaxf(top, __shfl_xor(top, 32, 64));
  const float m = fmaxf(st.m, top), a = __builtin_amdgcn_exp2f(st.m - m);
  st.m = m;
  float sum = 0.f;
  bf16x8 w;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float e = __builtin_amdgcn_exp2f(x[i] - m);
    sum += e;
    w[i] = f2bf(e);
  }
  st.l = st.l * a + sum;
  if (left < 32) {                   // values that are not seen may be no numbers: zeros
    const int mine = left - 8 * g;
    const uint32_t lo = mine >= 4 ? ~0u : mine <= 0 ? 0u : (1u << (8 * mine)) - 1;
    const uint32_t hi = mine >= 8 ? ~0u : mine <= 4 ? 0u : (1u << (8 * (mine - 4))) - 1;
#pragma unroll
    for (int n = 0; n < 4; ++n) c.v[n] = u32x4{c.v[n][0] & lo, c.v[n][1] & hi, c.v[n][2] & lo, c.v[n][3] & hi};
  }
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      f32x4& o = st.o[2 * n + e];
      o *= a;
      o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes_wide(c.v[n][2 * e], c.v[n][2 * e + 1], vscale), w, o, 0, 0, 0);
    }
}

// Partial rows: those of a launch that merges its own go past the XCDs' caches.
constexpr int kPast = 16;
template <bool SHARED>
__device__ __forceinline__ float part_load(const float* at) {
  return SHARED ? __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : *at;
}

// The partitions of a (sequence, kv head) into its rows: 16 threads to a row, 8 dims to a thread, 16 / (G rounded
// up to a power of two; of eight waves 32) groups of threads that take every so many-th partition, eight of them
// requested together.  lds: 16 (32) rows of D + 4.
template <bool SHARED, int NW>
__device__ __forceinline__ void merge(const ScaledAttn& p, int seq, int kvh, int nparts, int q_tok, float* lds) {
  constexpr int U = 8;
  const int G = p.G, wide = G <= 1 ? 1 : 1 << (32 - __builtin_clz(G - 1));
  const int at16 = threadIdx.x >> 4, row = at16 & (wide - 1), first = at16 / wide, groups = 4 * NW / wide;
  const int d0 = (threadIdx.x & 15) * 8;
  const int64_t base = (int64_t)(seq * p.Hkv + kvh) * p.num_parts * G;
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(p.part_o + base * D), (short)0, SHARED ? p.num_parts * G * D * 4 : 0, 0x00020000);
  float M = -1e30f, L = 0.f, acc[8] = {};
  if (row < G) {
    for (int i0 = first; i0 < nparts; i0 += U * groups) {
      float m[U], l[U];
      f32x4 o[U][2];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = min(i0 + u * groups, nparts - 1) * G + row;
        m[u] = part_load<SHARED>(p.part_m + base + at);
        l[u] = part_load<SHARED>(p.part_l + base + at);
        if constexpr (SHARED) {
          const int b = (at * D + d0) * 4;
          o[u][0] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, b, 0, kPast));
          o[u][1] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, b + 16, 0, kPast));
        } else {
          const float* po = p.part_o + (base + at) * D + d0;
#pragma unroll
          for (int k = 0; k < 2; ++k) o[u][k] = f32x4{po[4 * k], po[4 * k + 1], po[4 * k + 2], po[4 * k + 3]};
        }
      }
      float top = M;
#pragma unroll
      for (int u = 0; u < U; ++u) top = fmaxf(top, m[u]);     // (the last partition again changes nothing)
      const float a = __builtin_amdgcn_exp2f(M - top);
      M = top;
      L *= a;
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] *= a;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i0 + u * groups >= nparts) break;
        const float f = __builtin_amdgcn_exp2f(m[u] - M) * l[u];
        L += f;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += f * o[u][j >> 2][j & 3];
      }
    }
  }
  if (groups > 1 && nparts > 1) {
    float* mine = lds + at16 * (D + 4);
    *reinterpret_cast<f32x4*>(mine + d0) = f32x4{acc[0], acc[1], acc[2], acc[3]};
    *reinterpret_cast<f32x4*>(mine + d0 + 4) = f32x4{acc[4], acc[5], acc[6], acc[7]};
    if (d0 == 0) {
      mine[D] = M;
      mine[D + 1] = L;
    }
    __syncthreads();
    if (first > 0) return;
    for (int i = 1; i < groups; ++i) {
      const float* other = lds + (i * wide + row) * (D + 4);
      const float top = fmaxf(M, other[D]), a = __builtin_amdgcn_exp2f(M - top), b = __builtin_amdgcn_exp2f(other[D] - top);
      M = top;
      L = L * a + other[D + 1] * b;
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = acc[j] * a + other[d0 + j] * b;
    }
  }
  if (row >= G || first > 0) return;
  const float inv = L > 0.f ? 1.f / L : 0.f;
  bf16x8 o;
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = f2bf(acc[j] * inv);
  *reinterpret_cast<bf16x8*>(p.out + ((size_t)q_tok * p.Hq + kvh * G + row) * D + d0) = o;
}

__global__ __launch_bounds__(256) void scaled_merge_kernel(ScaledAttn p) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int seq = blockIdx.x, keys = keys_of(p, seq);
  merge<false, 4>(p, seq, blockIdx.y, min(p.num_parts, (keys + p.part_size - 1) / p.part_size),
               p.q_start ? p.q_start[seq] : seq, lds);
}

// The fused form's rows, 16 threads to a row and 8 dims to a thread: the kv head's G query heads, its key, its value.
// Asked for ahead of the first chunk.
struct NewRow {
  bf16x8 x, w;
  f32x4 c[2], s[2];
  int64_t slot;    // -1: none
  int page;
  float was;       // the scale of the slot's page, of keys in the rows up to the key's, of values in the value's
};
__device__ __forceinline__ void new_row_load(NewRow& n, const ScaledAttn& p, int seq, int kvh) {
  const int G = p.G, row = min((int)threadIdx.x >> 4, G + 1), j = threadIdx.x & 15;
  const int head = row < G ? kvh * G + row : row == G ? p.Hq + kvh : p.Hq + p.Hkv + kvh;
  n.x = *reinterpret_cast<const bf16x8*>(p.qkv + (size_t)seq * p.qkv_stride + head * D + 8 * j);
  const bf16* w = row < G ? p.q_w : row == G ? p.k_w : nullptr;
  n.w = w != nullptr ? *reinterpret_cast<const bf16x8*>(w + 8 * j) : bf16x8{};
  const int64_t pos = p.positions[seq], slot = p.slots[seq];
  const f32x4* cs = reinterpret_cast<const f32x4*>(
      p.cos_sin + (size_t)(pos < 0 ? 0 : pos < p.max_pos ? pos : p.max_pos - 1) * D + 8 * (j & 7));
  n.slot = slot < (int64_t)p.num_blocks * p.BS ? slot : -1;
  const int64_t page = n.slot < 0 ? 0 : (int64_t)p.num_blocks * p.BS < (1ll << 31) ? (uint32_t)n.slot / (uint32_t)p.BS : n.slot / p.BS;
  n.page = (int)page;
  n.was = (row > G ? p.v_scale : p.k_scale)[page * p.Hkv + kvh];
  n.c[0] = cs[0];
  n.c[1] = cs[1];
  n.s[0] = cs[16];
  n.s[1] = cs[17];
}
__device__ __forceinline__ float row16_max(float v) {
  v = fmaxf(v, dpp_mov<0xB1>(v));
  v = fmaxf(v, dpp_mov<0x4E>(v));
  v = fmaxf(v, dpp_mov<0x141>(v));
  return fmaxf(v, dpp_mov<0x140>(v));
}
// What the workgroup that holds the row's last key keeps of it in LDS: the codes (for the chunk that has it: nobody waits
// for what is stored), the page's scales (of no slot -1), and whether its other codes were rounded anew.
struct NewKey {
  uint8_t k[D], v[D];
  float scale[2];
  int grown[2];
};
// q to LDS; `writes`: the new key and value into their page, as the append kernel does it, by 16 threads.
__device__ __forceinline__ void new_row_put(NewRow& n, const ScaledAttn& p, int kvh, bool writes, bf16* q_s, NewKey* key) {
  const int G = p.G, row = threadIdx.x >> 4, j = threadIdx.x & 15;
  if (row >= G + 2) return;
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = bf2f(n.x[e]);
  if (row <= G) norm_rotate(x, (row < G ? p.q_w : p.k_w) != nullptr, n.w, true, n.c, n.s, j, p.eps);
  if (row < G) {
    bf16x8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = f2bf(x[e]);
    *reinterpret_cast<bf16x8*>(q_s + row * D + 8 * j) = o;
    return;
  }
  if (!writes) return;
  const int value = row > G;
  if (n.slot < 0) {
    if (j == 0) {
      key->scale[value] = -1.f;
      key->grown[value] = 0;
    }
    return;
  }
  const int64_t at = (int64_t)n.page * p.Hkv + kvh;
  const int off = (int)(n.slot - (int64_t)n.page * p.BS);
  uint8_t* codes = (value ? p.v_cache : p.k_cache) + at * p.BS * D;
  float most = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) most = fmaxf(most, scale_mag(x[e]));
  const int need = scale_exp(row16_max(most)), was = off > 0 ? stored_exp(n.was) : -100, exp = max(need, was);
  const bool grown = off > 0 && need > was;
  if (grown) {
    codes_grow<16>(codes, was - need, p.BS);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  const float inv = exp_scale(-exp);
  const u32x2 c = {codes4(x[0], x[1], x[2], x[3], inv), codes4(x[4], x[5], x[6], x[7], inv)};
  *reinterpret_cast<u32x2*>((value ? key->v : key->k) + 8 * j) = c;
  if (!value) {
    *reinterpret_cast<u32x2*>(codes + k_swz_offset(off) + k_dim_offset(8 * j)) = c;
  } else {
    uint8_t* to = codes + (size_t)(off >> 3) * D * 8 + 64 * j + (off & 7);
#pragma unroll
    for (int e = 0; e < 8; ++e) to[8 * e] = (uint8_t)(c[e >> 2] >> (8 * (e & 3)));
  }
  if (j == 0) {
    (value ? p.v_scale : p.k_scale)[at] = exp_scale(exp);
    key->scale[value] = exp_scale(exp);
    key->grown[value] = grown;
  }
  if (grown) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}
// the new key into its chunk's registers: token `tok` of the 32
__device__ __forceinline__ void put_k(Chunk& c, const NewKey* key, int tok) {
  const int lane = threadIdx.x & 63, g = lane >> 4;
  const bool mine = (lane & 15) == ((tok >> 3) << 2 | (tok & 3));
  const bool upper = (tok >> 2) & 1;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const u32x4 x = *reinterpret_cast<const u32x4*>(key->k + 64 * i + 16 * g);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      c.k[0][i][e] = mine && !upper ? x[e] : c.k[0][i][e];
      c.k[1][i][e] = mine && upper ? x[e] : c.k[1][i][e];
    }
  }
}
__device__ __forceinline__ void put_v(Chunk& c, const NewKey* key, int tok) {
  const int lane = threadIdx.x & 63, r = lane & 15;
  const bool mine = (lane >> 4) == tok >> 3, upper = tok & 4;
  const int at = 8 * (tok & 3);
  const uint32_t keep = ~(0xffu << at);
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const uint32_t x = *reinterpret_cast<const uint16_t*>(key->v + 32 * n + 2 * r);
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const uint32_t b = ((x >> (8 * d)) & 0xff) << at;
      const uint32_t lo = c.v[n][2 * d], hi = c.v[n][2 * d + 1];
      c.v[n][2 * d] = mine && !upper ? (lo & keep) | b : lo;
      c.v[n][2 * d + 1] = mine && upper ? (hi & keep) | b : hi;
    }
  }
}

template <bool FUSED, int NW>
__global__ __launch_bounds__(64 * NW, 4) void scaled_decode_kernel(ScaledAttn p) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int seq = blockIdx.x, kvh = blockIdx.y, part = blockIdx.z;
  const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = p.G, BS = p.BS;
  const int first = part * p.part_size, t0 = first + 32 * w, tok = t0 + 32 * NW * lane;
  // page and scales of the wave's chunk `lane` (the host bounds a partition to 64 chunks a wave); the table's entry
  // is asked for beside the length
  const int column = tok / BS;
  int page = p.block_tables[(size_t)seq * p.bt_stride + min(column, p.bt_cols - 1)];
  const int keys = keys_of(p, seq), end = min(keys, first + p.part_size);
  const int q_tok = p.q_start ? p.q_start[seq] : seq;
  const int nparts = min(p.num_parts, (keys + p.part_size - 1) / p.part_size);
  if (p.num_parts > 1 && first >= keys) {      // (the merge leaves it out)
    if (p.tickets != nullptr && part == 0) merge<true, NW>(p, seq, kvh, 0, q_tok, lds);
    return;
  }
  NewRow fresh;
  if constexpr (FUSED) new_row_load(fresh, p, seq, kvh);
  if (tok >= end || (uint32_t)page >= (uint32_t)p.num_blocks) page = -1;
  const int64_t sc = (int64_t)max(page, 0) * p.Hkv + kvh;
  float ks = p.k_scale[sc] * p.scale_log2, vs = p.v_scale[sc];
  const int in_page = (tok - column * BS) * D;
  // chunk i of the wave: asked for without a branch, so that what each wait is for is known
  auto page_of = [&](int i) { return i < 64 ? __builtin_amdgcn_readlane(page, i & 63) : -1; };
  auto rsrc_of = [&](const uint8_t* cache, int i) {
    const int blk = page_of(i);
    return chunk_rsrc(cache, ((int64_t)max(blk, 0) * p.Hkv + kvh) * BS * D + (blk < 0 ? 0 : __builtin_amdgcn_readlane(in_page, i & 63)),
                      blk >= 0);
  };
  Chunk c;
  load_k(c, rsrc_of(p.k_cache, 0));
  load_v(c, rsrc_of(p.v_cache, 0));
  bf16x8 q[4];
  NewKey* key = nullptr;             // where the row's last key is new and this partition's
  if constexpr (FUSED) {
    bf16* q_s = reinterpret_cast<bf16*>(lds);            // [G][D]
    key = reinterpret_cast<NewKey*>(lds + p.new_key);
    const bool writes = keys > 0 && part == nparts - 1;
    new_row_put(fresh, p, kvh, writes, q_s, key);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // LDS alone: the first chunk stays on its way
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (!writes || key->scale[0] < 0.f) key = nullptr;
    if (key != nullptr) {
      const int last = (keys - 1) / BS;
      if (column == last) {
        ks = key->scale[0] * p.scale_log2;
        vs = key->scale[1];
      }
      // a page rounded anew lies in this partition whole: what was read of it before is read again
      if ((key->grown[0] | key->grown[1]) != 0 && t0 < end && t0 / BS == last) {
        load_k(c, rsrc_of(p.k_cache, 0));
        load_v(c, rsrc_of(p.v_cache, 0));
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      q[i] = *reinterpret_cast<const bf16x8*>(q_s + min(r, G - 1) * D + 16 * g + 64 * (i >> 1) + 8 * (i & 1));
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();                        // (the rows' sums go where q is)
  } else {
    const bf16* qp = p.q + ((size_t)q_tok * p.Hq + kvh * G + min(r, G - 1)) * D + 16 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const bf16x8*>(qp + 64 * (i >> 1) + 8 * (i & 1));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = r < G ? q[i] : bf16x8{};
  Row st;
#pragma unroll
  for (int i = 0; i < 8; ++i) st.o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  st.m = -1e30f;
  st.l = 0.f;
  for (int t = t0, i = 0; t < end; t += 32 * NW, ++i) {
    const bool some = page_of(i) >= 0;
    float x[8];
    const bool has = FUSED && key != nullptr && (uint32_t)(keys - 1 - t) < 32;
    if (has) put_k(c, key, keys - 1 - t);
    if (some) chunk_scores(x, q, c, lane_f(ks, i));
    load_k(c, rsrc_of(p.k_cache, i + 1));
    if (has) put_v(c, key, keys - 1 - t);
    if (some) chunk_rows(st, x, c, lane_f(vs, i), end - t);
    load_v(c, rsrc_of(p.v_cache, i + 1));
  }
  float l = st.l;
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  float* o_s = lds;                               // [NW][G][D + 4]
  float* m_s = lds + NW * G * (D + 4);            // [NW][G]
  float* l_s = m_s + NW * G;
  if (r < G) {
    float* to = o_s + (w * G + r) * (D + 4) + 8 * g;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<f32x2*>(to + 32 * n + 2 * j) = f32x2{st.o[2 * n][j], st.o[2 * n + 1][j]};
    if (g == 0) {
      m_s[w * G + r] = st.m;
      l_s[w * G + r] = l;
    }
  }
  __syncthreads();
  const bool alone = p.num_parts == 1 || (p.tickets != nullptr && nparts <= 1);
  const bool past = p.tickets != nullptr && !alone;
  // a thread's dims: 8 in a row, of partial rows that go past the caches 4 and 4, whole lines to a store
  const int row = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * (past ? 4 : 8), d4 = past ? 64 : 4;
  if (row < G) {
    float M = -1e30f, L = 0.f, acc[8] = {};
#pragma unroll
    for (int i = 0; i < NW; ++i) M = fmaxf(M, m_s[i * G + row]);
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      const float f = __builtin_amdgcn_exp2f(m_s[i * G + row] - M);
      L += f * l_s[i * G + row];
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] += f * o_s[(i * G + row) * (D + 4) + d0 + (j >> 2) * d4 + (j & 3)];
    }
    const float inv = L > 0.f ? 1.f / L : 0.f;
    const int64_t at = ((int64_t)(seq * p.Hkv + kvh) * p.num_parts + part) * G + row;
    if (alone) {
      bf16x8 o;
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = f2bf(acc[j] * inv);
      *reinterpret_cast<bf16x8*>(p.out + ((size_t)q_tok * p.Hq + kvh * G + row) * D + d0) = o;
    } else if (past) {
      const __amdgpu_buffer_rsrc_t rs =
          __builtin_amdgcn_make_buffer_rsrc((void*)(p.part_o + (at - row) * D), (short)0, G * D * 4, 0x00020000);
#pragma unroll
      for (int k = 0; k < 2; ++k)
        __builtin_amdgcn_raw_buffer_store_b128(
            u32x4{__float_as_uint(acc[4 * k] * inv), __float_as_uint(acc[4 * k + 1] * inv),
                  __float_as_uint(acc[4 * k + 2] * inv), __float_as_uint(acc[4 * k + 3] * inv)},
            rs, (row * D + d0 + 64 * k) * 4, 0, kPast);
      if (d0 == 0) {
        __hip_atomic_store(p.part_m + at, M, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(p.part_l + at, L, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) p.part_o[at * D + d0 + j] = acc[j] * inv;
      if (d0 == 0) {
        p.part_m[at] = M;
        p.part_l[at] = L;
      }
    }
  }
  if (!past) return;
  // The last of the row's partitions to get here merges them.  Its stores acknowledged, a workgroup adds its share to
  // the row's ticket: 1, the first partition 1 - nparts, so that all of them together leave the zero that was there.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  int* flag = reinterpret_cast<int*>(m_s);
  if (threadIdx.x == 0) {
    const int share = part == 0 ? 1 - nparts : 1;
    *flag = __hip_atomic_fetch_add(p.tickets + (int64_t)(seq * p.Hkv + kvh) * kCtrStride, share, __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT) + share == 0;
  }
  __syncthreads();
  const bool last = *flag != 0;
  __syncthreads();
  if (last) merge<true, NW>(p, seq, kvh, nparts, q_tok, lds);
}

// ------------------------------------------------------------------------------------------------- prompts
// A workgroup takes a tile of 32 NW flattened rows (token and head of the kv head's group), a wave 32 of them, and
// 64 keys at a time, which all waves have widened into LDS, while the next ones' codes are on their way to
// registers.  Products 32 x 32 x 16; a lane column is a query row.
__device__ __forceinline__ float half_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// row r of a 32-key product holds this key: then the 8 accumulator registers that a lane half hands on as
// weights are the keys of one 8-token group
__device__ __forceinline__ int row_key(int r) { return 16 * (r >> 4) + 8 * ((r >> 2) & 1) + 4 * ((r >> 3) & 1) + (r & 3); }

constexpr int kKeys = 64;
// Fragments asked for ahead of the product that takes them.  (Left to the compiler each was read right before its
// product and waited for: 1000 tokens behind 9000 in one part, a wave to a SIMD, 292 us; 3 ahead 235, 4 and 6 too.)
constexpr int kAhead = 3;
// Vector and matrix instructions and LDS stay on their side; scalar ones and loads may cross.
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0x14); }
// Key tiles that a part of a split tile takes at least (with 8, and all at once before the products: 700 tokens behind
// 300, 16 / 8 heads, 36.5 us for 28).
constexpr int kSplitTiles = 4;

// key tiles of a tile's rows, and the parts that they are cut into
struct Tile {
  int seq, row0, q0, q_len, ctx, keys, ntiles, parts;
};
template <int ROWS>
__device__ __forceinline__ Tile tile_of(const ScaledAttn& p, int seq, int row0) {
  Tile t;
  t.seq = seq;
  t.row0 = row0;
  t.q0 = p.q_start[seq];
  t.q_len = p.q_start[seq + 1] - t.q0;
  t.ctx = p.seq_lens[seq] - t.q_len;
  t.keys = keys_of(p, seq);
  const int last = row0 >= t.q_len * p.G ? -1 : min(t.q_len - 1, (row0 + ROWS - 1) / p.G);
  t.ntiles = last < 0 ? 0 : max(0, min(t.ctx + last, t.keys - 1)) / kKeys + 1;
  t.parts = max(1, min(p.num_parts, t.ntiles / kSplitTiles));
  return t;
}

// A wave's step, a barrier behind it: 16 products for the outputs by tile u - 1's weights, between them the maximum of
// tile u's scores, and K of tile u + 2 and V of tile u widened into LDS, where their buffers are free; then 16
// products for the scores of tile u + 1, between them the weights of tile u.  Products and what stands between them are
// laid down one by one (fence): a SIMD issues in order, and a product runs 32 cycles beside the next vector work.
// Before, with all products of a step and then all weights, and eight waves' later four half a step behind: 1000 behind
// 9000 in one part, four waves 292 us (now 198), eight 264 (241); 2 of ~759 (20 / 4 heads) 30.5 (23.3); 4 of 4096 (32 /
// 8) 569 (528).  One wave of 64 rows, whose fragments serve two products (tried when a fragment's wait still stood right
// behind its read): 448 for the 264.
// Bound by how far products, vector work and LDS run beside each other.  8 prompts of 2048 (32 / 8 heads) 307 us, 0.89
// PFLOP/s at the 2.2 GHz that the card settles at (lower in the first tens of calls: up to 400 us).  Of a CU's 646 K
// cycles its matrix units are at work in 43 %, its vector units in 50 %, both together in 21 %, neither in 28 % (a wave
// waits for LDS, loads or the barrier 30 % of its time); LDS is busy in 33 %, a sixth of that bank conflicts.
template <int NW>
__global__ __launch_bounds__(64 * NW, NW == 4 ? 2 : 1) void scaled_prefill_kernel(ScaledAttn p, int subs) {
  constexpr int ROWS = 32 * NW, NT = 64 * NW, PW = 512 / NT;    // 16-byte pieces of K (and of V) to a thread
  __shared__ __attribute__((aligned(16))) bf16 lds[2][2][kKeys * D];    // [K | V][buffer]
  const int flat = gridDim.x - 1 - blockIdx.x;     // the map rises by work: longest tiles first
  const int item = __builtin_amdgcn_readfirstlane(flat / p.Hkv), kvh = flat - item * p.Hkv;
  const int tile = __builtin_amdgcn_readfirstlane(item / p.num_parts), part = item - tile * p.num_parts;
  const int named = __builtin_amdgcn_readfirstlane(tile / subs);      // the map's tile, which subs workgroups share
  const int seq = __builtin_amdgcn_readfirstlane(p.tile_seq[named]);
  const int first_row = __builtin_amdgcn_readfirstlane(p.tile_row[named]) + (tile - named * subs) * ROWS;
  const Tile T = tile_of<ROWS>(p, seq, first_row);
  if (part >= T.parts || T.ntiles == 0) return;
  const int ta = __builtin_amdgcn_readfirstlane(T.ntiles * part / T.parts);
  const int tb = __builtin_amdgcn_readfirstlane(T.ntiles * (part + 1) / T.parts);
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, h = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = p.G, BS = p.BS, row0 = T.row0, q0 = T.q0, keys = T.keys;
  const int R = row0 + 32 * w + r, pos = R / G, hig = R - pos * G;
  const bool valid = pos < T.q_len;
  const int limit = valid ? min(T.ctx + pos, keys - 1) : -1;
  const int w_first = (row0 + 32 * w) / G;
  const int w_min = min(T.ctx + w_first, keys - 1);

  // pieces: 512 of K and 512 of V to a tile; a wave's lie in one 32-key chunk
  const int chunk = (w * PW * 64) >> 8;
  // Pages and scales of 64 chunks, one to a lane, from tile `held` on; read by readlane, so that no step waits for
  // the table.  A page is -1 where the chunk lies behind the keys or outside the cache.
  int held = ta, page_l, off_l;
  float ks_l, vs_l;
  auto hold = [&](int t) {
    held = t;
    const int c = 2 * t + lane;
    const bool some = 32 * c < keys && c < 2 * tb;
    const int column = some ? 32 * c / BS : 0;
    const int b = p.block_tables[(size_t)T.seq * p.bt_stride + column];
    off_l = some ? (32 * c - column * BS) * D : 0;
    page_l = some && (uint32_t)b < (uint32_t)p.num_blocks ? b : -1;
    const int64_t at = (int64_t)max(page_l, 0) * p.Hkv + kvh;
    ks_l = p.k_scale[at];
    vs_l = p.v_scale[at];
  };
  hold(ta);
  auto page_of = [&](int t, int k) { return __builtin_amdgcn_readlane(page_l, 2 * (t - held) + k); };
  auto kscale_of = [&](int t) { return lane_f(ks_l, 2 * (t - held) + chunk); };
  auto vscale_of = [&](int t) { return lane_f(vs_l, 2 * (t - held) + chunk); };
  u32x4 kc[PW], vc[PW];
  auto fetch = [&](u32x4 (&to)[PW], const uint8_t* cache, int t) {
    const int i0 = 2 * (t - held) + chunk, b = __builtin_amdgcn_readlane(page_l, i0);
    const __amdgpu_buffer_rsrc_t rs = chunk_rsrc(cache, ((int64_t)max(b, 0) * p.Hkv + kvh) * BS * D +
                                                            __builtin_amdgcn_readlane(off_l, i0), b >= 0);    // (of no page: zeros)
#pragma unroll
    for (int i = 0; i < PW; ++i)
      to[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, ((tid * PW + i) & 255) * 16, 0, 0));
  };
  // K image: token rows of 256 bytes, 16-byte column c of row k at c ^ (k & 15); V image: the groups as they are
  auto put_k = [&](int buf, float scale, int n) {      // n: half a piece
    const int i = n >> 1, pc = (tid * PW + i) & 255;       // K: [half 2][dims / 32 4][row 16][2]
    const int col = 4 * ((pc >> 5) & 3) + 2 * (pc & 1) + (n & 1), r16 = (pc >> 1) & 15;
    const int key = 32 * chunk + 8 * (r16 >> 2) + 4 * (pc >> 7) + (r16 & 3);
    *reinterpret_cast<bf16x8*>(lds[0][buf] + key * D + (col ^ (key & 15)) * 8) =
        codes_wide(kc[i][2 * (n & 1)], kc[i][2 * (n & 1) + 1], scale);
  };
  // values behind the last key may be no numbers: zeros
  auto clear_v = [&](int t) {
    const int c = 2 * t + chunk;
    if (32 * c + 32 <= keys) return;
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      const int left = keys - 32 * c - 8 * (((tid * PW + i) & 255) >> 6);
      const uint32_t lo = left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1;
      const uint32_t hi = left >= 8 ? ~0u : left <= 4 ? 0u : (1u << (8 * (left - 4))) - 1;
      vc[i] = u32x4{vc[i][0] & lo, vc[i][1] & hi, vc[i][2] & lo, vc[i][3] & hi};
    }
  };
  auto put_v = [&](int buf, float scale, int n) {
    const int i = n >> 1;
    *reinterpret_cast<bf16x8*>(lds[1][buf] + (chunk * 256 + ((tid * PW + i) & 255)) * 16 + 8 * (n & 1)) =
        codes_wide(vc[i][2 * (n & 1)], vc[i][2 * (n & 1) + 1], scale);
  };

  fetch(kc, p.k_cache, ta);
  fetch(vc, p.v_cache, ta);
  u32x4 kc2[PW];
  fetch(kc2, p.k_cache, ta + 1);
  // Q^T: lane (r, h) holds dims 16 s + 8 h .. + 7 of its row
  bf16x8 qf[8];
  {
    const int t = valid ? pos : 0;
    const bool prep = p.qkv != nullptr;
    const bf16* src = (prep ? p.qkv + (size_t)(q0 + t) * p.qkv_stride : p.q + (size_t)(q0 + t) * p.Hq * D) +
                      (kvh * G + hig) * D + 8 * h;
#pragma unroll
    for (int s = 0; s < 8; ++s) qf[s] = *reinterpret_cast<const bf16x8*>(src + 16 * s);
    if (prep) {       // (as norm_rotate does it, in the same order)
#pragma clang fp contract(off)
      float x[8][8];
#pragma unroll
      for (int s = 0; s < 8; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[s][j] = bf2f(qf[s][j]);
      if (p.q_w != nullptr) {
        float ss[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) ss[s] = half_sum(squares(x[s]));
        const float inv = inv_sqrt((((ss[0] + ss[1]) + (ss[2] + ss[3])) + ((ss[4] + ss[5]) + (ss[6] + ss[7]))) * (1.f / D) + p.eps);
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          const bf16x8 nw = *reinterpret_cast<const bf16x8*>(p.q_w + 16 * s + 8 * h);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[s][j] = x[s][j] * inv * bf2f(nw[j]);
        }
      }
      const int64_t at = p.positions[q0 + t];
      const float* cs = p.cos_sin + (size_t)(at < 0 ? 0 : at < p.max_pos ? at : p.max_pos - 1) * D + 8 * h;
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float c = cs[16 * s + j], sn = cs[64 + 16 * s + j];
          qf[s][j] = f2bf(x[s][j] * c - x[s + 4][j] * sn);
          qf[s + 4][j] = f2bf(x[s + 4][j] * c + x[s][j] * sn);
        }
    }
  }
#pragma unroll
  for (int n = 0; n < 2 * PW; ++n) put_k(ta & 1, kscale_of(ta), n);
#pragma unroll
  for (int i = 0; i < PW; ++i) kc[i] = kc2[i];
#pragma unroll
  for (int n = 0; n < 2 * PW; ++n) put_k((ta + 1) & 1, kscale_of(ta + 1), n);
  fetch(kc, p.k_cache, ta + 2);
  // (no tile before the first: weights and values of zero)
#pragma unroll
  for (int i = 0; i < 2 * PW; ++i) *reinterpret_cast<u32x4*>(lds[1][(ta + 1) & 1] + (tid * 2 * PW + i) * 8) = u32x4{};

  f32x16 o[4], sa[2], sb[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = f32x16{};
  float m = -1e30f, l = 0.f;
  bf16x8 pb[4] = {};                    // weights: keys 16 g + 8 h .. + 7
  auto k_frag = [&](int buf, int i, int k) {
    const int key = 32 * k + row_key(r);
    return *reinterpret_cast<const bf16x8*>(lds[0][buf] + key * D + ((2 * i + h) ^ (key & 15)) * 8);
  };
  auto v_frag = [&](int buf, int g, int dt) {
    return *reinterpret_cast<const bf16x8*>(lds[1][buf] + ((2 * g + h) * D + 32 * dt + r) * 8);
  };
  // (LDS alone: what is on its way from memory stays so)
  auto half = [&]() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  auto mask = [&](f32x16 (&s)[2], int t) {
    const int key0 = t * kKeys;
    const bool lost0 = page_of(t, 0) < 0, lost1 = page_of(t, 1) < 0;
    if (key0 + kKeys - 1 > w_min || lost0 || lost1) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (key0 + 32 * k + 16 * (j >> 3) + 8 * h + (j & 7) > limit || (k ? lost1 : lost0)) s[k][j] = -INFINITY;
    }
  };
  float a = 1.f;
  // 16 products each, behind the n-th beside(n)
  auto rows = [&](int buf, const auto& beside) {
    bf16x8 f[kAhead];
#pragma unroll
    for (int n = 0; n < kAhead; ++n) f[n] = v_frag(buf, n >> 2, n & 3);
#pragma unroll
    for (int n = 0; n < 16; ++n) {
      fence();
      o[n & 3] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[n % kAhead], pb[n >> 2], o[n & 3], 0, 0, 0);
      if (n + kAhead < 16) f[n % kAhead] = v_frag(buf, (n + kAhead) >> 2, (n + kAhead) & 3);
      beside(n);
    }
    fence();
  };
  auto scores = [&](f32x16 (&s)[2], int buf, const auto& beside) {
    bf16x8 f[kAhead];
#pragma unroll
    for (int n = 0; n < kAhead; ++n) f[n] = k_frag(buf, n >> 1, n & 1);
    s[0] = f32x16{};
    s[1] = f32x16{};
#pragma unroll
    for (int n = 0; n < 16; ++n) {
      fence();
      s[n & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[n % kAhead], qf[n >> 1], s[n & 1], 0, 0, 0);
      if (n + kAhead < 16) f[n % kAhead] = k_frag(buf, (n + kAhead) >> 1, (n + kAhead) & 1);
      beside(n);
    }
    fence();
  };
  // a tile's maximum, four scores at a time, then what its weights are relative to
  float tp[4];
  bool moved = false;
  auto tops = [&](const f32x16 (&s)[2], int n) {
    if (n < 8) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x = s[n >> 2][4 * (n & 3) + j];
        tp[j] = n == 0 ? x : fmaxf(tp[j], x);
      }
    } else if (n == 8) {
      const float top = fmaxf(fmaxf(tp[0], tp[1]), fmaxf(tp[2], tp[3]));
      // the maximum moves, and sums are scaled, only where it is exceeded by 2^8: weights up to that are as good
      const float cand = fmaxf(m, half_max(top) * p.scale_log2), mn = cand > m + 8.f ? cand : m;
      a = __builtin_amdgcn_exp2f(m - mn);
      moved = mn != m;
      m = mn;
    }
  };
  float sum[4], x0[2], e0[2];
  // two weights of 32: arguments one call ahead of the exponentials, sums one behind
  auto weigh = [&](const f32x16 (&s)[2], int n) {
    if (n == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] = 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j) x0[j] = fmaf(s[0][j], p.scale_log2, -m);
    }
    if (n > 0) {
      const int e = 2 * (n - 1);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        sum[(e + j) & 3] += e0[j];
        pb[e >> 3][(e & 7) + j] = f2bf(e0[j]);
      }
    }
    if (n < 16) {
#pragma unroll
      for (int j = 0; j < 2; ++j) e0[j] = __builtin_amdgcn_exp2f(x0[j]);
      if (n < 15) {
        const int e = 2 * (n + 1);
#pragma unroll
        for (int j = 0; j < 2; ++j) x0[j] = fmaf(s[e >> 4][(e & 15) + j], p.scale_log2, -m);
      }
    } else {
      l = l * a + half_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
    }
  };
  auto settle = [&]() {
    if (__any(moved)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] *= a;
    }
  };
  auto none = [](int) {};
  half();
  scores(sa, ta & 1, none);
  half();
  auto step = [&](int u, f32x16 (&s)[2], f32x16 (&sn)[2]) {
    mask(s, u);
    clear_v(u);
    if (u + 3 - held > 31) hold(u);
    const float ksc = kscale_of(u + 2), vsc = vscale_of(u);
    rows((u + 1) & 1, [&](int n) {
      tops(s, n);
      if (n >= 16 - 4 * PW && n < 16 - 2 * PW) put_k(u & 1, ksc, n - 16 + 4 * PW);
      if (n >= 16 - 2 * PW) put_v(u & 1, vsc, n - 16 + 2 * PW);
    });
    fetch(kc, p.k_cache, u + 3);
    fetch(vc, p.v_cache, u + 1);
    settle();
    scores(sn, (u + 1) & 1, [&](int n) { weigh(s, n); });
    weigh(s, 16);
    half();
  };
  int u = ta;
  for (; u + 2 < tb; u += 2) {
    step(u, sa, sb);
    step(u + 1, sb, sa);
  }
  if (u + 1 < tb) {
    step(u, sa, sb);
    sa[0] = sb[0];
    sa[1] = sb[1];
  }
  mask(sa, tb - 1);
  clear_v(tb - 1);
  rows(tb & 1, [&](int n) {
    tops(sa, n);
    if (n >= 8 && n < 8 + 2 * PW) put_v((tb - 1) & 1, vscale_of(tb - 1), n - 8);
  });
  settle();
#pragma unroll
  for (int n = 0; n <= 16; ++n) weigh(sa, n);
  half();
  rows((tb - 1) & 1, none);
  // dims 32 dt + 8 i + 4 h .. + 3 of a row to a lane
  if (T.parts > 1) {
    const int64_t at = ((int64_t)(tile * p.num_parts + part) * p.Hkv + kvh) * ROWS + 32 * w + r;
    float* to = p.part_o + at * D + 4 * h;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4*>(to + 32 * dt + 8 * i) =
            f32x4{o[dt][4 * i], o[dt][4 * i + 1], o[dt][4 * i + 2], o[dt][4 * i + 3]};
    if (h == 0) {
      p.part_m[at] = m;
      p.part_l[at] = l;
    }
    return;
  }
  if (!valid) return;
  const float inv = l > 0.f ? 1.f / l : 0.f;
  bf16* to = p.out + ((size_t)(q0 + pos) * p.Hq + kvh * G + hig) * D + 4 * h;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bf16x4 x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = f2bf(o[dt][4 * i + j] * inv);
      *reinterpret_cast<bf16x4*>(to + 32 * dt + 8 * i) = x;
    }
}

// The parts of split tiles: 32 threads to a row, 8 rows to a workgroup.  Bound by the parts' bytes: 16000 rows in four
// parts 8.0 us, 4.2 TB/s (one part after the other 8.3).
template <int ROWS>
__global__ __launch_bounds__(256) void scaled_prefill_merge_kernel(ScaledAttn p, int subs) {
  const int item = blockIdx.x / (ROWS / 8), sub = blockIdx.x - item * (ROWS / 8);
  const int tile = item / p.Hkv, kvh = item - tile * p.Hkv, named = tile / subs;
  const Tile T = tile_of<ROWS>(p, p.tile_seq[named], p.tile_row[named] + (tile - named * subs) * ROWS);
  if (T.parts <= 1) return;
  const int row = sub * 8 + (threadIdx.x >> 5), d0 = (threadIdx.x & 31) * 4;
  const int R = T.row0 + row, pos = R / p.G;
  if (pos >= T.q_len) return;
  float M = -1e30f, L = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  constexpr int U = 4;             // parts asked for together
  for (int i0 = 0; i0 < T.parts; i0 += U) {
    float m[U], l[U], top = M;
    f32x4 o[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = ((int64_t)(tile * p.num_parts + min(i0 + u, T.parts - 1)) * p.Hkv + kvh) * ROWS + row;
      m[u] = p.part_m[at];
      l[u] = p.part_l[at];
      o[u] = *reinterpret_cast<const f32x4*>(p.part_o + at * D + d0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) top = fmaxf(top, m[u]);     // (the last part again changes nothing)
    const float a = __builtin_amdgcn_exp2f(M - top);
    M = top;
    L *= a;
    acc *= a;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float b = i0 + u < T.parts ? __builtin_amdgcn_exp2f(m[u] - M) : 0.f;
      L += b * l[u];
      acc += b * o[u];
    }
  }
  const float inv = L > 0.f ? 1.f / L : 0.f;
  bf16x4 x;
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = f2bf(acc[j] * inv);
  *reinterpret_cast<bf16x4*>(p.out + ((size_t)(T.q0 + pos) * p.Hq + kvh * p.G + R - pos * p.G) * D + d0) = x;
}

}  // namespace

void launch_scaled_decode(const ScaledAttn& p, int num_seqs, hipStream_t s) {
  if (num_seqs == 0) return;
  // Coarser partitions than asked for, in whole ones.  One for up to 512 keys (1 row at 333, 16 / 8 heads, 5.1 us, in two
  // 7.0), at most 64 (3 rows at ~25000, 8 / 1 heads, 13.9 us, in 118 19.7), else 256 keys or more (1 row at 4000 8.7 us,
  // 512 10.3); and rows that fill the card by themselves need none, up to 2048 keys (beyond, a long row among short ones
  // would hold up the step): 64 rows at ~1500 keys of 32 / 8 heads in partitions of 512, 1024, 2048 44, 42, 36 us, 128
  // at ~1050 65, 60, 53; 16 at ~2250 in 768 and 1024 17.9 and 19.0, 1 at 30000 of 16 / 8 heads in 512 and 768 16.5 and
  // 17.8 (but 15 at ~5500 of one kv head in 256 and 512 13.2 and 11.8).
  // All of it goes by the keys that a caller has room for, which in an engine are those of its longest allowed sequence:
  // short rows there are cut, and take four waves, as long ones would (16 / 8 heads, us, room for the longest row, for
  // 4096, for 32768 keys: 1 row at 333 5.2, 7.1, 5.6, 1 at 1000 7.8, 7.7, 9.7, 16 at ~340 6.7, 8.0, 8.0, 16 at ~1750 13.0,
  // 15.9, 22.2; rows that fill the card alike).
  ScaledAttn q = p;
  const int64_t rows = (int64_t)num_seqs * p.Hkv;
  const int held = p.num_parts * p.part_size, size = p.part_size;      // (below 2^30)
  const int fill = (int)std::min<int64_t>((p.num_parts * rows + 511) / 512, (2047 + size) / size);
  const int least = ((held <= 512 ? 511 : 255) + size) / size;
  const int by = std::min(std::max({least, (p.num_parts + 63) / 64, fill}), kDecodeMaxPart / size);
  q.part_size = size * by;
  q.num_parts = (p.num_parts + by - 1) / by;
  // Eight waves where a workgroup has a unit to itself and more than a chunk for each: 1 row at 333 5.1 us, by four 5.5,
  // 16 at ~340 with the append 8.0 and 8.7, 3 at ~25000 13.9 and 16.3; but 1 at 1000 of one kv head, in 256s, 7.9 and 7.1.
  auto lds = [&](int waves) {
    return std::max<size_t>(waves * (p.G * (D + 4) + 2 * p.G), q.num_parts > 1 ? 4 * waves * (D + 4) : 0);
  };
  const bool wide = rows * q.num_parts <= 256 && std::min(q.part_size, held) > 256 &&
                    lds(8) * sizeof(float) + sizeof(NewKey) + 16 <= 65536;
  const size_t rows_s = lds(wide ? 8 : 4);
  q.new_key = (int)(rows_s + 3) / 4 * 4;
  const size_t smem = p.qkv != nullptr ? q.new_key * sizeof(float) + sizeof(NewKey) : rows_s * sizeof(float);
  const dim3 grid(num_seqs, p.Hkv, q.num_parts);
  if (p.qkv != nullptr) {
    if (wide) scaled_decode_kernel<true, 8><<<grid, 512, smem, s>>>(q);
    else scaled_decode_kernel<true, 4><<<grid, 256, smem, s>>>(q);
  } else {
    if (wide) scaled_decode_kernel<false, 8><<<grid, 512, smem, s>>>(q);
    else scaled_decode_kernel<false, 4><<<grid, 256, smem, s>>>(q);
  }
  if (q.num_parts > 1 && p.tickets == nullptr)
    scaled_merge_kernel<<<dim3(num_seqs, p.Hkv), 256, 16 * (D + 4) * sizeof(float), s>>>(q);
}

void launch_scaled_prefill(const ScaledAttn& p, int num_tiles, int tile_rows, int waves, hipStream_t s) {
  if (num_tiles == 0) return;
  const int subs = tile_rows / (32 * waves), tiles = num_tiles * subs, grid = tiles * p.Hkv * p.num_parts;
  const int merge = tiles * p.Hkv * (4 * waves);
  if (waves == 8) {
    scaled_prefill_kernel<8><<<grid, 512, 0, s>>>(p, subs);
    if (p.num_parts > 1) scaled_prefill_merge_kernel<256><<<merge, 256, 0, s>>>(p, subs);
  } else {
    scaled_prefill_kernel<4><<<grid, 256, 0, s>>>(p, subs);
    if (p.num_parts > 1) scaled_prefill_merge_kernel<128><<<merge, 256, 0, s>>>(p, subs);
  }
}

}  // namespace akap
