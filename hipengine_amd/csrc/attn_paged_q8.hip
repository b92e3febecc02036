// Attention of ragged queries over the 8-bit paged KV cache:  o = softmax(scale * q K^T + mask) V.
//
// Rows.  The queries of one KV head are flattened to rows r = query * group + member, so that grouped heads share every
// load of K and V and a tile has no empty rows between queries.  Row r's query sits at place kv_len - q_len + query and
// sees the keys up to it (and, with a window, no further back than window - 1); a row that sees none gives zeros.
//
// One wave holds 32 (or 64) rows and walks over blocks of 32 keys, keeping for each row the running maximum and sum of
// the softmax.  It computes transposed products on v_mfma_f32_32x32x16_f16: S^T = K Q^T (rows keys, columns queries) and
// O^T += V^T P^T.  A lane then owns one query column: maximum, sum and rescaling are per lane, the accumulator of S^T is
// already P^T's operand (the cache's V layout is in the accumulator's key order), and K, V and P never pass through LDS.
//
// Numbers.  K and V are whole numbers up to 127, exact in fp16.  q is bf16 or fp16: bf16 rows are divided by the power
// of two of their largest magnitude, which makes them exact in fp16 down to 2^-24 of it.  Products and sums are float32.
// P is rounded to fp16 (relative 2^-11): it lies in 0 .. 2^15 around a reference that follows the running maximum, and
// the sum of the softmax adds the rounded values, so the rounding does not move the weights' total.
//
// Scales.  K's block scale goes into the softmax's argument.  V's goes into P: with w = p * v_scale, w = exp2(s + log2
// v_scale - m) for a maximum m over that sum, O = (sum w v_int) / (sum w / v_scale) - one more constant per block in an
// addition that is there anyway, and P keeps its range whatever the scales are.  (Where scales lie far apart a block's w
// can vanish while its p counts in the sum: `far` below.)
//
// Splits.  Where rows are few, the keys of a sequence are cut into chunks for workgroups of their own, whose partial
// maxima, sums and outputs go to a workspace and are joined by a second kernel in chunk order (no atomics).

#include "attn_common.hpp"

#include "gguf_init.hpp"

#include "../../include/hipengine_gfx950.h"

namespace {

using namespace hipengine_gfx950;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f2v __attribute__((ext_vector_type(2)));
typedef float f16v __attribute__((ext_vector_type(16)));

constexpr int WAVES = 4;
constexpr int MAX_KV = 1 << 30;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float NEVER = -1e30f;        // a maximum before any key: finite, so that differences to it are no NaN
constexpr float HEADROOM = 8.0f;       // log2 by which a row's maximum may pass its reference before rows are rescaled
constexpr float OFFSET = 7.0f;         // log2 of P at the reference: P <= 2^15, and fp16's least step is 2^-31 of it

struct AttnArgs {
  KvCacheQ8 cache;
  const void* q;
  void* out;
  int64_t q_stride, out_stride;
  const int32_t* q_start;
  const int32_t* kv_lens;
  int64_t tokens;
  float scale;            // of the softmax, times log2(e)
  int group;              // query heads per KV head
  int q_heads;
  int window;
  int splits;             // chunks of keys
  int chunk;              // blocks of 32 keys in a chunk
  float* part_acc;        // [splits][tokens * q_heads][D]
  float* part_ml;         // [splits][tokens * q_heads][2]
};

// Four excess-128 bytes -> four fp16 whole numbers.  0x6400 | b is 1024 + b in fp16.
__device__ __forceinline__ void bytes_to_half(uint32_t w, h2& lo, h2& hi) {
  const h2 bias = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
  lo = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x07010700u)) - bias;
  hi = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x07030702u)) - bias;
}
__device__ __forceinline__ h8 bytes8_to_half(uint32_t a, uint32_t b) {
  h2 p[4];
  bytes_to_half(a, p[0], p[1]);
  bytes_to_half(b, p[2], p[3]);
  return __builtin_bit_cast(h8, p);
}

// The other half of the wave's value of the same column.
__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32); }

__device__ __forceinline__ float read_lane_f(float v, int lane) {
  return bits_to_float(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(float_to_bits(v)), lane)));
}

// KEYS: the four waves of a workgroup share its rows and take blocks of keys in turn (decode); else every wave has rows
// of its own and walks over all keys (prompts).  NT: columns of 32 rows that a wave holds.
// grid (KV heads, row tiles, batch * splits): heads in front, so that with 8 of them each XCD keeps one head's cache in
// its L2; the tiles of the latest queries, which see the most keys, start first.
template <int D, int KIND, int NT, bool KEYS>
__global__ void __launch_bounds__(WAVES * 64, NT == 1 && D <= 128 ? 2 : 1) paged_attention_kernel(AttnArgs a) {
  constexpr int KC = D / 32;           // 16-byte loads of K a lane, and tiles of 32 dims of V
  constexpr int TILE = KEYS ? 32 * NT : 32 * NT * WAVES;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int head = blockIdx.x;
  const int seq = blockIdx.z / a.splits, split = blockIdx.z - seq * a.splits;
  const SeqRows rows = seq_rows(a.q_start, seq, a.tokens);
  const int n_rows = static_cast<int>(rows.count) * a.group;
  const int tile = gridDim.y - 1 - blockIdx.y;
  const int row0 = tile * TILE + (KEYS ? 0 : wave * 32 * NT);
  if (tile * TILE >= n_rows) return;
  const bool idle = row0 >= n_rows;                    // (prompts) this wave has no rows, but the barriers are not its own
  if (!KEYS && idle) return;
  const int kv_len = min(max(a.kv_lens[seq], 0), MAX_KV);
  const int q_len = static_cast<int>(rows.count);

  // Keys that the wave's rows see: [lo of the first row, lim of the last one).
  auto limit = [&](int query) { return min(max(kv_len - q_len + query + 1, 0), kv_len); };
  auto lower = [&](int query) { return a.window > 0 ? max(kv_len - q_len + query + 1 - a.window, 0) : 0; };
  const int last_row = min(row0 + 32 * NT, n_rows) - 1;
  const int first_q = row0 / a.group, last_q = last_row / a.group;
  const int lim_first = limit(first_q), lim_last = limit(last_q);
  const int lo_first = lower(first_q), lo_last = lower(last_q);
  // Chunks are laid from the first block that the first query of the tile sees.
  const int tile_lo = KEYS ? lo_first : lower(tile * TILE / a.group);
  int blk = lo_first >> 5;
  int blk_end = (lim_last + 31) >> 5;
  if (a.splits > 1) {
    const int from = (tile_lo >> 5) + split * a.chunk;
    blk = max(blk, from);
    if (split + 1 < a.splits) blk_end = min(blk_end, from + a.chunk);   // the last chunk takes what a longer cache than announced holds
  }

  // Q^T as the MFMA's second operand: lane (column, half) holds dims 32 i + 16 half + 8 b .. + 7.
  h8 q[NT][2 * KC];
  float q_exp[NT];
  int lim[NT], lo[NT];
  bool valid[NT];
  int64_t out_at[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = row0 + 32 * n + col;
    valid[n] = r < n_rows;
    const int query = valid[n] ? r / a.group : 0, member = valid[n] ? r - query * a.group : 0;
    lim[n] = limit(query);
    lo[n] = lower(query);
    const int64_t row = rows.first + query;
    const int64_t at = static_cast<int64_t>(head * a.group + member) * D;
    out_at[n] = row * a.out_stride + at;
    float x[2 * KC][8];
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 2 * KC; ++i) {
      load8_f32<KIND>(a.q, row * a.q_stride + at + 32 * (i >> 1) + 16 * half + 8 * (i & 1), x[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[i][j]));
    }
    int e = 0;
    if constexpr (KIND == KIND_BF16) {
      amax = fmaxf(amax, other_half(amax));
      e = max(static_cast<int>(float_to_bits(amax) >> 23), 1) - 127;
    }
    q_exp[n] = ldexpf(1.0f, e) * a.scale;
#pragma unroll
    for (int i = 0; i < 2 * KC; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) q[n][i][j] = static_cast<_Float16>(KIND == KIND_BF16 ? ldexpf(x[i][j], -e) : x[i][j]);
  }

  f16v acc[KC][NT];
  float m[NT], l[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n] = NEVER;
    l[n] = 0.0f;
#pragma unroll
    for (int t = 0; t < KC; ++t) acc[t][n] = f16v{0};
  }

  const int step = KEYS ? WAVES : 1;
  int j = blk + (KEYS ? wave : 0);
  // Block numbers and scales of the next 64 of the wave's blocks, one a lane.
  int base = j;
  int64_t block_of = -1;
  float ks_of = 0.0f, lv_of = 0.0f, iv_of = 0.0f;
  auto lookup = [&] {
    base = j;
    const int mine = j + lane * step;
    block_of = mine < blk_end ? kv_block_index(a.cache, seq, mine, head) : -1;
    if (block_of >= 0) {
      const float vs = a.cache.v_scale[block_of];
      const float v_clean = fmaxf(vs, KV_SCALE_FLOOR);          // of a NaN: the floor
      ks_of = a.cache.k_scale[block_of];
      lv_of = vs == vs ? log2f(v_clean) : vs;
      iv_of = 1.0f / v_clean;
    }
  };
  auto block_at = [&](int which) -> int64_t {
    const int k = (which - base) / step;
    const uint32_t lo32 = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(block_of), k));
    const uint32_t hi32 = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(block_of >> 32), k));
    return static_cast<int64_t>((static_cast<uint64_t>(hi32) << 32) | lo32);
  };
  float lv_top = -__builtin_inff();
  const int k_off = lane * 16, v_off = col * 32 + half * 16;

  while (j < blk_end) {
    if (j == blk + (KEYS ? wave : 0) || j - base >= 64 * step) lookup();
    const int slot = (j - base) / step;
    const int64_t block = block_at(j);
    if (block < 0) { j += step; continue; }              // a bad page: its keys are not there
    const uint8_t* kp = a.cache.k + block * (D * KV_BLOCK);
    const uint8_t* vp = a.cache.v + block * (D * KV_BLOCK);
    uint4 kr[KC], vr[KC];
#pragma unroll
    for (int i = 0; i < KC; ++i) kr[i] = *reinterpret_cast<const uint4*>(kp + i * 1024 + k_off);
#pragma unroll
    for (int i = 0; i < KC; ++i) vr[i] = *reinterpret_cast<const uint4*>(vp + i * 1024 + v_off);
    const float ks = read_lane_f(ks_of, slot), lv = read_lane_f(lv_of, slot), iv = read_lane_f(iv_of, slot);

    f16v s[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n] = f16v{0};
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      const h8 k0 = bytes8_to_half(kr[i].x, kr[i].y), k1 = bytes8_to_half(kr[i].z, kr[i].w);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        s[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0, q[n][2 * i], s[n], 0, 0, 0);
        s[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k1, q[n][2 * i + 1], s[n], 0, 0, 0);
      }
    }

    // A block whose V scale is less than a quarter of the largest so far: its w may be lost in fp16 although its p counts
    // in the sum, which then takes p itself, at the price of 16 more exponentials.
    lv_top = fmaxf(lv_top, lv);
    const bool far = lv < lv_top - 2.0f;
    const int key0 = j * KV_BLOCK;
    const bool masked = key0 + KV_BLOCK > lim_first || key0 < lo_last;   // some row does not see the whole block
    h8 p[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float c = ks * q_exp[n];
      // s is raw here; the argument of row n is fma(s, c, lv), and c > 0 keeps the order.
      float top = -__builtin_inff();
      if (masked) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = key0 + 8 * (i >> 2) + 4 * half + (i & 3);
          if (key < lim[n] && key >= lo[n]) top = fmaxf(top, s[n][i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[n][i]);
      }
      top = fmaxf(top, other_half(top));
      const float high = fmaf(top, c, lv);                // NaN (a poisoned block, or nothing seen at a zero c) moves nothing
      if (__any(high > m[n] + HEADROOM)) {
        const float to = fmaxf(m[n], high);
        const float f = __builtin_amdgcn_exp2f(m[n] - to);
        m[n] = to;
        l[n] *= f;
#pragma unroll
        for (int t = 0; t < KC; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[t][n][i] *= f;
      }
      const float shift = lv - m[n] + OFFSET;
      float w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = __builtin_amdgcn_exp2f(fmaf(s[n][i], c, shift));
      if (masked) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = key0 + 8 * (i >> 2) + 4 * half + (i & 3);
          w[i] = key < lim[n] && key >= lo[n] ? w[i] : 0.0f;
        }
      }
      if (far) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = key0 + 8 * (i >> 2) + 4 * half + (i & 3);
          const float e = __builtin_amdgcn_exp2f(fmaf(s[n][i], c, OFFSET - m[n]));
          l[n] += !masked || (key < lim[n] && key >= lo[n]) ? e : 0.0f;
        }
      }
      float sum = 0.0f;
      const h2 one = {static_cast<_Float16>(1.0f), static_cast<_Float16>(1.0f)};
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const h2 r = __builtin_convertvector((f2v{w[i], w[i + 1]}), h2);
        p[n][i >> 3][i & 7] = r.x;
        p[n][i >> 3][(i & 7) + 1] = r.y;
        sum = __builtin_amdgcn_fdot2(r, one, sum, false);
      }
      if (!far) l[n] = fmaf(sum, iv, l[n]);
    }

#pragma unroll
    for (int t = 0; t < KC; ++t) {
      const h8 v0 = bytes8_to_half(vr[t].x, vr[t].y), v1 = bytes8_to_half(vr[t].z, vr[t].w);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        acc[t][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v0, p[n][0], acc[t][n], 0, 0, 0);
        acc[t][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v1, p[n][1], acc[t][n], 0, 0, 0);
      }
    }
    j += step;
  }

#pragma unroll
  for (int n = 0; n < NT; ++n) l[n] += other_half(l[n]);

  if constexpr (KEYS) {
    // Join the four waves: 2 and 3 into 0 and 1, then 1 into 0; through at most 32 KB of LDS.
    constexpr int PART = KC < 4 ? KC : 4;
    __shared__ float lds_acc[2][PART][NT][16][64];
    __shared__ float lds_ml[2][NT][2][64];
#pragma unroll
    for (int other = WAVES / 2; other >= 1; other >>= 1) {
      const bool gives = wave >= other && wave < 2 * other;
      float f[NT], f2[NT];
#pragma unroll
      for (int t0 = 0; t0 < KC; t0 += PART) {
        if (gives) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            lds_ml[wave - other][n][0][lane] = m[n];
            lds_ml[wave - other][n][1][lane] = l[n];
#pragma unroll
            for (int t = 0; t < PART; ++t)
#pragma unroll
              for (int i = 0; i < 16; ++i) lds_acc[wave - other][t][n][i][lane] = acc[t0 + t][n][i];
          }
        }
        __syncthreads();
        if (wave < other) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (t0 == 0) {
              const float m2 = lds_ml[wave][n][0][lane], l2 = lds_ml[wave][n][1][lane], to = fmaxf(m[n], m2);
              f[n] = __builtin_amdgcn_exp2f(m[n] - to);
              f2[n] = __builtin_amdgcn_exp2f(m2 - to);
              m[n] = to;
              l[n] = l[n] * f[n] + l2 * f2[n];
            }
#pragma unroll
            for (int t = 0; t < PART; ++t)
#pragma unroll
              for (int i = 0; i < 16; ++i)
                acc[t0 + t][n][i] = acc[t0 + t][n][i] * f[n] + lds_acc[wave][t][n][i][lane] * f2[n];
          }
        }
        __syncthreads();
      }
    }
    if (wave != 0) return;
  }

#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (!valid[n]) continue;
    if (a.splits > 1) {
      const int64_t query = (row0 + 32 * n + col) / a.group, member = (row0 + 32 * n + col) - query * a.group;
      const int64_t at = (static_cast<int64_t>(split) * a.tokens + rows.first + query) * a.q_heads + head * a.group + member;
      if (half == 0) {
        a.part_ml[2 * at] = m[n];
        a.part_ml[2 * at + 1] = l[n];
      }
#pragma unroll
      for (int t = 0; t < KC; ++t)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<float4*>(a.part_acc + at * D + 32 * t + 2 * i + 4 * half) =
              make_float4(acc[t][n][i], acc[t][n][i + 1], acc[t][n][i + 2], acc[t][n][i + 3]);
    } else {
      const float r = l[n] == 0.0f ? 0.0f : 1.0f / l[n];   // a row that saw no key gives zeros
#pragma unroll
      for (int t = 0; t < KC; ++t)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          uint32_t w[2];
#pragma unroll
          for (int b = 0; b < 2; ++b)
            w[b] = half_bits<KIND>(acc[t][n][i + 2 * b] * r) | (half_bits<KIND>(acc[t][n][i + 2 * b + 1] * r) << 16);
          __builtin_memcpy(__builtin_assume_aligned(static_cast<uint16_t*>(a.out) + out_at[n] + 32 * t + 2 * i + 4 * half, 2), w, 8);
        }
    }
  }
}

// Joins the chunks of one output row: grid (rows a sequence, batch), one wave a row, D / 64 dims a lane.
template <int D, int KIND>
__global__ void __launch_bounds__(256) join_kernel(AttnArgs a, int tile_rows) {
  constexpr int V = D / 64;
  const int seq = blockIdx.y, lane = threadIdx.x & 63;
  const SeqRows rows = seq_rows(a.q_start, seq, a.tokens);
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (r >= rows.count * a.q_heads) return;
  const int query = static_cast<int>(r / a.q_heads), q_head = static_cast<int>(r - static_cast<int64_t>(query) * a.q_heads);
  // The chunks that a workgroup ran for this row: as the attention kernel laid them for the row's tile.
  const int kv_len = min(max(a.kv_lens[seq], 0), MAX_KV), q_len = static_cast<int>(rows.count);
  const int row = query * a.group + q_head % a.group;
  const int tile_query = row / tile_rows * tile_rows / a.group;
  const int lo = a.window > 0 ? max(kv_len - q_len + tile_query + 1 - a.window, 0) : 0;
  const int lim = min(max(kv_len - q_len + query + 1, 0), kv_len);
  const int blocks = max(((lim + 31) >> 5) - (lo >> 5), 0);
  const int splits = min((blocks + a.chunk - 1) / a.chunk, a.splits);
  const int64_t at = (rows.first + query) * a.q_heads + q_head, pitch = a.tokens * a.q_heads;
  float m = NEVER;
  for (int s = lane; s < splits; s += 64) m = fmaxf(m, a.part_ml[2 * (s * pitch + at)]);
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) m = fmaxf(m, __shfl_xor(m, off));
  float l = 0.0f, o[V] = {};
  for (int s0 = 0; s0 < splits; s0 += 64) {
    const int s = s0 + lane;
    float f = 0.0f;
    if (s < splits) {
      const int64_t i = 2 * (s * pitch + at);
      f = __builtin_amdgcn_exp2f(a.part_ml[i] - m);
      l += a.part_ml[i + 1] * f;
    }
    const int n = min(splits - s0, 64);
#pragma unroll 4
    for (int k = 0; k < n; ++k) {
      const float w = read_lane_f(f, k);
      const float* src = a.part_acc + ((s0 + k) * pitch + at) * D + lane * V;
#pragma unroll
      for (int v = 0; v < V; ++v) o[v] = fmaf(src[v], w, o[v]);
    }
  }
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) l += __shfl_xor(l, off);
  const float f = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* dst = static_cast<uint16_t*>(a.out) + (rows.first + query) * a.out_stride + static_cast<int64_t>(q_head) * D + lane * V;
#pragma unroll
  for (int v = 0; v < V; ++v) dst[v] = static_cast<uint16_t>(half_bits<KIND>(o[v] * f));
}

// How a call is cut: decided from sizes alone, so that the workspace can be sized before the call.
struct Plan {
  bool keys;          // the waves of a workgroup share rows and split keys
  int nt;
  int tile_rows;
  int64_t tiles;
  int most_splits;    // what the workspace is sized for: no fewer for fewer keys
  int splits, chunk;
};

constexpr int CUS = 256;

Plan plan_of(int64_t batch, int64_t max_q, int64_t max_kv, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t window) {
  Plan p;
  const int64_t rows = max_q * (q_heads / kv_heads);
  p.keys = rows <= 64;
  p.nt = 1;
  p.tile_rows = p.keys ? 32 * p.nt : 32 * p.nt * WAVES;
  p.tiles = (rows + p.tile_rows - 1) / p.tile_rows;
  // Keys that a tile can see.
  int64_t span = max_kv;
  if (window > 0 && window + max_q + 31 < span) span = window + max_q + 31;
  const int64_t blocks = (span + 31) / 32 + (window > 0 ? 1 : 0);
  const int64_t groups = batch * kv_heads * p.tiles, want = 2 * CUS;
  int64_t splits = (want + groups - 1) / groups;
  const int64_t least = p.keys ? 16 : 32;               // blocks worth a workgroup of its own
  const int64_t most = (blocks + least - 1) / least;
  if (splits > most) splits = most;
  if (splits < 1) splits = 1;
  p.most_splits = static_cast<int>(splits);
  p.chunk = static_cast<int>((blocks + splits - 1) / splits);
  p.splits = static_cast<int>((blocks + p.chunk - 1) / p.chunk);
  return p;
}

constexpr int BAD = static_cast<int>(hipErrorInvalidValue);

bool shape_ok(int64_t tokens, int64_t batch, int64_t max_q, int64_t max_kv, int64_t q_heads, int64_t kv_heads, int64_t dim,
              int64_t window) {
  return tokens > 0 && batch > 0 && batch <= 65535 && max_q > 0 && max_kv >= 0 && max_kv <= MAX_KV && kv_heads > 0 &&
         kv_heads <= 65535 && q_heads > 0 && q_heads % kv_heads == 0 && q_heads <= 4096 &&
         (dim == 64 || dim == 128 || dim == 256) && window >= 0 && window <= (1 << 30) && tokens <= (1 << 26) &&
         max_q * (q_heads / kv_heads) <= (1 << 30);
}

int64_t workspace_of(int splits, int64_t tokens, int64_t q_heads, int64_t dim) {
  return splits > 1 ? static_cast<int64_t>(splits) * tokens * q_heads * (dim + 2) * 4 : 0;
}

template <int D, int KIND>
int launch(const AttnArgs& a, const Plan& p, int64_t batch, int64_t max_q, int64_t kv_heads, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(kv_heads), static_cast<unsigned>(p.tiles), static_cast<unsigned>(batch * p.splits));
  const dim3 threads(WAVES * 64);
  if (p.keys) hipLaunchKernelGGL((paged_attention_kernel<D, KIND, 1, true>), grid, threads, 0, stream, a);
  else hipLaunchKernelGGL((paged_attention_kernel<D, KIND, 1, false>), grid, threads, 0, stream, a);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess || p.splits == 1) return static_cast<int>(err);
  const dim3 join(static_cast<unsigned>((max_q * a.q_heads + 3) / 4), static_cast<unsigned>(batch));
  hipLaunchKernelGGL((join_kernel<D, KIND>), join, dim3(256), 0, stream, a, p.tile_rows);
  return static_cast<int>(hipGetLastError());
}

}  // namespace

extern "C" int hipengine_gfx950_paged_attention_q8_workspace_bytes(int64_t tokens, int64_t batch, int64_t max_q_len,
                                                                   int64_t max_kv_len, int64_t q_heads, int64_t kv_heads,
                                                                   int64_t head_dim, int64_t* bytes) {
  if (!bytes || !shape_ok(tokens, batch, max_q_len, max_kv_len, q_heads, kv_heads, head_dim, 0)) return BAD;
  const int64_t longest = max_q_len < tokens ? max_q_len : tokens;
  *bytes = workspace_of(plan_of(batch, longest, max_kv_len, q_heads, kv_heads, head_dim, 0).most_splits, tokens, q_heads, head_dim);
  return 0;
}

extern "C" int hipengine_gfx950_paged_attention_q8(const void* q, void* out, int32_t kind, int64_t q_stride,
                                                   int64_t out_stride, const uint8_t* k_cache, const uint8_t* v_cache,
                                                   const float* k_scale, const float* v_scale, const int32_t* page_table,
                                                   int64_t table_stride, const int32_t* q_start, const int32_t* kv_lens,
                                                   int64_t tokens, int64_t batch, int64_t max_q_len, int64_t max_kv_len,
                                                   int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t pages,
                                                   int64_t page_size, float softmax_scale, int64_t window, void* workspace,
                                                   int64_t workspace_bytes, hipStream_t stream) {
  if (!q || !out || q == out || !k_cache || !v_cache || !k_scale || !v_scale || !page_table || !q_start || !kv_lens ||
      !(kind == KIND_BF16 || kind == KIND_F16) ||
      !shape_ok(tokens, batch, max_q_len, max_kv_len, q_heads, kv_heads, head_dim, window) || table_stride <= 0 ||
      pages <= 0 || pages > 0x7FFFFFFF || page_size < KV_BLOCK || page_size > (1 << 20) ||
      (page_size & (page_size - 1)) != 0 || !(softmax_scale > 0.0f) || !(softmax_scale <= 3.4028234663852886e+38f) ||
      ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15) != 0)
    return BAD;
  const int64_t width = q_heads * head_dim;
  if (q_stride == 0) q_stride = width;
  if (out_stride == 0) out_stride = width;
  if (q_stride < width || out_stride < width) return BAD;
  const int64_t longest = max_q_len < tokens ? max_q_len : tokens;
  const Plan p = plan_of(batch, longest, max_kv_len, q_heads, kv_heads, head_dim, window);
  const int64_t need = workspace_of(p.splits, tokens, q_heads, head_dim);
  if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0)) return BAD;
  if (p.tiles > 65535 || batch * p.splits > 65535) return BAD;
  const KvCacheQ8 cache{const_cast<uint8_t*>(k_cache), const_cast<uint8_t*>(v_cache), const_cast<float*>(k_scale),
                        const_cast<float*>(v_scale), page_table, table_stride, pages, static_cast<int>(kv_heads),
                        63 - __builtin_clzll(static_cast<unsigned long long>(page_size))};
  float* acc = static_cast<float*>(workspace);
  const AttnArgs a{cache, q, out, q_stride, out_stride, q_start, kv_lens, tokens, softmax_scale * LOG2E,
                   static_cast<int>(q_heads / kv_heads), static_cast<int>(q_heads), static_cast<int>(window), p.splits,
                   p.chunk, acc, acc ? acc + static_cast<int64_t>(p.splits) * tokens * q_heads * head_dim : nullptr};
  switch (head_dim * 4 + kind) {
    case 64 * 4 + KIND_BF16: return launch<64, KIND_BF16>(a, p, batch, longest, kv_heads, stream);
    case 64 * 4 + KIND_F16: return launch<64, KIND_F16>(a, p, batch, longest, kv_heads, stream);
    case 128 * 4 + KIND_BF16: return launch<128, KIND_BF16>(a, p, batch, longest, kv_heads, stream);
    case 128 * 4 + KIND_F16: return launch<128, KIND_F16>(a, p, batch, longest, kv_heads, stream);
    case 256 * 4 + KIND_BF16: return launch<256, KIND_BF16>(a, p, batch, longest, kv_heads, stream);
    default: return launch<256, KIND_F16>(a, p, batch, longest, kv_heads, stream);
  }
}

int hipengine_gfx950::paged_attention_load() {
  hipFuncAttributes attr;
  return static_cast<int>(hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(paged_attention_kernel<128, KIND_BF16, 1, true>)));
}
