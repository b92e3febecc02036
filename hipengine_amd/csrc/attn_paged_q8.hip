// Attention of ragged queries over the 8-bit paged KV cache:  o = softmax(scale * q K^T + mask) V.
//
// Rows.  The queries of one KV head are flattened to rows r = query * group + member, so that grouped heads share every
// load of K and V and a tile has no empty rows between queries.  Row r's query sits at place kv_len - q_len + query and
// sees the keys up to it (and, with a window, no further back than window - 1); a row that sees none gives zeros.
//
// One wave holds 32 rows and walks once over blocks of 32 keys, keeping for each row a reference near its maximum and the
// sum of the softmax.  It computes transposed products on v_mfma_f32_32x32x16_f16: S^T = K Q^T (rows keys, columns
// queries) and O^T += V^T P^T.  A lane then owns one query column: maximum, sum and rescaling are per lane, the
// accumulator of S^T is already P^T's operand (the cache's V layout is in the accumulator's key order), and P never
// passes through LDS.
//
// Numbers.  K and V are whole numbers up to 127, exact in fp16.  q is bf16 or fp16: bf16 rows are divided by the power
// of two of their largest magnitude, which makes them exact in fp16 down to 2^-24 of it.  Products and sums are float32.
// P is rounded to fp16 (relative 2^-11): it lies in 0 .. 2^15, 2^7 at the reference, and the sum of the softmax adds the
// rounded values, so the rounding does not move the weights' total.
//
// Scales.  K's block scale goes into the softmax's argument.  V's goes into P: with w = p * v_scale, w = exp2(s + log2
// v_scale - m) for a maximum m over that sum, O = (sum w v_int) / (sum w / v_scale) - one more constant per block in an
// addition that is there anyway, and P keeps its range whatever the scales are.  (Where scales lie far apart a block's w
// can vanish while its p counts in the sum: `far` below.  What fp16 holds to its 11 bits counts as rounded there too: with p
// in its place a row whose weight lies on such a block was off by another 2^-11 of its value.)
//
// Splits.  Where rows are few, the keys of a sequence are cut into chunks for workgroups of their own, whose partial
// maxima, sums and outputs go to a workspace and are joined by a second kernel in chunk order (no atomics).

#include <type_traits>

#include "attn_common.hpp"

#include "gguf_init.hpp"

#include "../../include/hipengine_gfx950.h"

namespace {

using namespace hipengine_gfx950;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f2v __attribute__((ext_vector_type(2)));
typedef float f16v __attribute__((ext_vector_type(16)));

constexpr int WAVES = 4;               // of a workgroup (of attention_rows_kernel also twice as many)
constexpr int MAX_KV = 1 << 30;
constexpr int least_rows(int dim) { return 2048 / dim; }   // fewest blocks in a part of a prompt's keys
constexpr float LOG2E = 1.4426950408889634f;
constexpr float NEVER = -3e38f;        // a maximum before any key: finite, so that differences to it are no NaN
constexpr float HEADROOM = 8.0f;       // attention_keys_kernel: log2 by which a row's maximum may pass its reference
constexpr float RANGE = 32768.0f;      // attention_rows_kernel: sum of P above which it is moved (fp16 ends at 65504)
constexpr _Float16 FULL = 6.103515625e-5f16;   // 2^-14: fp16 holds what is less to fewer than 11 bits
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
  int splits;             // most chunks of keys
  int chunk;              // fewest blocks of 32 keys in a chunk; 0: of a prompt by itself, see chunk_of
  // Of several prompts in parts:
  int32_t* parts;         // [batch] chunks of each sequence; else null
  int items, tiles;       // workgroups for a KV head, and for a sequence's rows at most
  int batch;
  int least;              // blocks that a part has if there are as many
  float* part_acc;        // [splits][tokens * q_heads][D]
  float* part_ml;         // [splits][tokens * q_heads][2]
};

// Four excess-128 bytes -> four fp16 whole numbers.  0x6400 | b is 1024 + b in fp16.
// (Half of these instructions could go: a byte under zeros is the subnormal b * 2^-24, and the excess could come off the
// sums. But the matrix instruction drops the low bits of what it adds, in one direction, and with an excess of 128 in
// every value that showed: O was off by 2^-19 of 128 steps of V.)
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

// A barrier for what goes through LDS: unlike __syncthreads() it does not wait for loads from memory, which are on their
// way across it on purpose.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// The other half of the wave's value of the same column.
__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32); }

__device__ __forceinline__ float read_lane_f(float v, int lane) {
  return bits_to_float(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(float_to_bits(v)), lane)));
}

// Blocks that some tile of a sequence can see, at most.
template <typename T>
__host__ __device__ __forceinline__ T blocks_of(T kv_len, T q_len, T window) {
  const T all = (kv_len + 31) / 32, near = (window + q_len + 62) / 32 + 1;      // (a window may begin anywhere in a block)
  return window > 0 && near < all ? near : all;
}

// The keys that a query sees: places [lower, limit).
struct Sight {
  int kv_len, q_len, window;
  __device__ __forceinline__ int limit(int query) const { return min(max(kv_len - q_len + query + 1, 0), kv_len); }
  __device__ __forceinline__ int lower(int query) const { return window > 0 ? max(kv_len - q_len + query + 1 - window, 0) : 0; }
};

// Blocks in each of a tile's chunks, at most `parts` of them, from the keys that there are: the announced lengths only say how
// many chunks there may be, so that a call captured for the longest cache cuts a short one as finely.  All tiles of a prompt by
// itself have the same chunks, so that they read a block at the same time, and no more of them than have least_rows() blocks each
// (512 tokens behind 8000, D 128, announced for 131072: 129 us, as announced for 8512; with chunks of the announced length 231).
// (Made uniform by hand: the quotient comes from vector registers, of which D 256 has none to spare.)
template <int D, bool KEYS = false>
__device__ __forceinline__ int chunk_of(const AttnArgs& a, const Sight& sight, int parts, int blocks) {
  if (!KEYS && a.chunk == 0) {
    blocks = blocks_of(sight.kv_len, sight.q_len, a.window);
    parts = max(min(parts, (blocks + least_rows(D) - 1) / least_rows(D)), 1);
  }
  return __builtin_amdgcn_readfirstlane(max((blocks + parts - 1) / parts, KEYS ? a.chunk : max(a.chunk, 1)));
}

// Which part of which tile a workgroup works on.
struct Share {
  int seq, tile, split, parts;   // seq < 0: none
};

// Several prompts differ in rows and keys, so each is cut into parts of its own: all parts have about c blocks, with the
// least c that needs no more workgroups than there are.  3 chunks of about 400 tokens of D 256 behind 2000 to 6000 others,
// as 242 workgroups of up to 47 blocks, take 110 us; as 160 of up to 63, by a chunk from the announced length, 132 us.
// Every wave computes it for itself, a sequence a lane, up to four times 64.
template <int TILE>
__device__ Share share_of(const AttnArgs& a, int item) {
  constexpr int MORE = 4;
  const int lane = threadIdx.x & 63;
  int tiles[MORE], blocks[MORE], longest = 0;
  float work = 0.0f;
#pragma unroll
  for (int i = 0; i < MORE; ++i) {
    const int b = lane + 64 * i;
    tiles[i] = blocks[i] = 0;
    if (64 * i >= a.batch) continue;
    if (b < a.batch) {
      tiles[i] = static_cast<int>(min((seq_rows(a.q_start, b, a.tokens).count * a.group + TILE - 1) / TILE, static_cast<int64_t>(a.tiles)));
      blocks[i] = (min(max(a.kv_lens[b], 0), MAX_KV) + 31) >> 5;
      if (a.window > 0) blocks[i] = min(blocks[i], ((a.window + TILE / a.group + 1) >> 5) + 2);
    }
    work += static_cast<float>(tiles[i]) * static_cast<float>(blocks[i]);
    if (tiles[i] > 0) longest = max(longest, blocks[i]);
  }
  auto sum = [](auto v) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) v += __shfl_xor(v, off);
    return v;
  };
  work = sum(work);
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) longest = max(longest, __shfl_xor(longest, off));
  int c = max(max(static_cast<int>(work / static_cast<float>(a.items)), a.least), (longest + a.splits - 1) / a.splits);
  int parts[MORE];
  for (;; c += (c >> 4) + 1) {       // ends: with c = longest there are no more than a.tiles * a.batch <= a.items
    int all = 0;
#pragma unroll
    for (int i = 0; i < MORE; ++i) {
      if (64 * i >= a.batch) continue;
      parts[i] = max((blocks[i] + c - 1) / c, 1);
      all += tiles[i] * parts[i];
    }
    if (c >= longest || sum(all) <= a.items) break;
  }
  Share r{-1, 0, 0, 1};
#pragma unroll
  for (int i = 0; i < MORE; ++i) {
    if (64 * i >= a.batch) continue;
    const int own = tiles[i] * parts[i];
    int up_to = own;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int o = __shfl_up(up_to, off);
      if (lane >= off) up_to += o;
    }
    const unsigned long long here = __ballot(item >= up_to - own && item < up_to);
    if (r.seq < 0 && here) {
      const int l = __builtin_ctzll(here), n = __builtin_amdgcn_readlane(tiles[i], l);
      const int at = item - __builtin_amdgcn_readlane(up_to - own, l);
      r = {l + 64 * i, n - 1 - at % n, at / n, __builtin_amdgcn_readlane(parts[i], l)};
    }
    item -= __builtin_amdgcn_readlane(up_to, 63);
    if (blockIdx.x == 0 && blockIdx.y == 0 && lane + 64 * i < a.batch) a.parts[lane + 64 * i] = parts[i];
  }
  auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  return {uniform(r.seq), uniform(r.tile), uniform(r.split), uniform(r.parts)};
}

// One column: a row of queries as the matrix instruction's second operand (lane (column, half) holds dims 32 i + 16 half +
// 8 b .. + 7 of piece 2 i + b), and what goes with it.
template <int D>
struct Column {
  h8 q[D / 16];
  float c;             // argument of the softmax, in log2, per raw product and unit of K's scale
  int lim, lo;
};

template <int D, int KIND>
__device__ __forceinline__ Column<D> load_column(const AttnArgs& a, const SeqRows& rows, const Sight& sight, int r, int n_rows, int head) {
  constexpr int P = D / 16;
  const int half = (threadIdx.x & 63) >> 5;
  Column<D> k;
  if (r >= n_rows) r = 0;              // (some row, never stored)
  const int query = r / a.group, member = r - query * a.group;
  k.lim = sight.limit(query);
  k.lo = sight.lower(query);
  const int64_t at = (rows.first + query) * a.q_stride + (head * a.group + member) * static_cast<int64_t>(D);
  auto dims = [&](int i) { return at + 32 * (i >> 1) + 16 * half + 8 * (i & 1); };
  float x[8];
  int e = 0;
  if constexpr (KIND == KIND_BF16) {   // read twice, the second time from L1: kept, the row would be D registers
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      load8_f32<KIND>(a.q, dims(i), x);
#pragma unroll
      for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[j]));
    }
    amax = fmaxf(amax, other_half(amax));
    e = max(static_cast<int>(float_to_bits(amax) >> 23), 1) - 127;
    asm volatile("" ::: "memory");
  }
  k.c = ldexpf(1.0f, e) * a.scale;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    load8_f32<KIND>(a.q, dims(i), x);
#pragma unroll
    for (int j = 0; j < 8; ++j) k.q[i][j] = static_cast<_Float16>(KIND == KIND_BF16 ? ldexpf(x[j], -e) : x[j]);
    // (keeps the conversion in front of the loop: the compiler sinks it into the loop otherwise, 97 instructions a block)
    asm volatile("" : "+v"(k.q[i]));
  }
  return k;
}

// Numbers and scales of 64 of a sequence's blocks, `step` apart, one a lane.  A block that is not there (a bad page, or
// behind the end) is block 0 with a V scale of zero: it adds nothing, and nothing branches on it.
struct Blocks {
  int base, step;
  int64_t number;
  float ks, lv, iv;    // scale of K, log2 of V's, 1 / V's
  bool found;
  __device__ __forceinline__ void find(const KvCacheQ8& c, int seq, int head, int from, int end) {
    base = from;
    const int mine = from + static_cast<int>(threadIdx.x & 63) * step;
    number = mine < end ? kv_block_index(c, seq, mine, head) : -1;
    found = number >= 0;
    number = max(number, int64_t{0});
  }
  // Apart, so that the blocks themselves can be asked for first.
  __device__ __forceinline__ void scales(const KvCacheQ8& c) {
    const float v = c.v_scale[number], k = c.k_scale[number];
    const float v_clean = fmaxf(v, KV_SCALE_FLOOR);          // of a NaN: the floor
    ks = !found ? 0.0f : kv_scale(k);
    lv = !found ? -__builtin_inff() : v == v ? __builtin_amdgcn_logf(v_clean) : v;
    iv = !found ? 0.0f : 1.0f / v_clean;
  }
  __device__ __forceinline__ void lookup(const KvCacheQ8& c, int seq, int head, int from, int end) {
    find(c, seq, head, from, end);
    scales(c);
  }
  __device__ __forceinline__ int slot(int which) const { return (which - base) / step; }
  __device__ __forceinline__ int64_t at(int which) const {
    const int k = slot(which);
    const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(number), k));
    const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(number >> 32), k));
    return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
  }
};

struct Scales {
  float ks, lv, iv;
  bool far;            // V's is less than a quarter of the largest so far
};
__device__ __forceinline__ Scales scales_of(const Blocks& b, int which, float& lv_top) {
  const int slot = b.slot(which);
  Scales r{read_lane_f(b.ks, slot), read_lane_f(b.lv, slot), read_lane_f(b.iv, slot), false};
  lv_top = fmaxf(lv_top, r.lv);
  r.far = r.lv < lv_top - 2.0f && r.lv > -__builtin_inff();
  return r;
}

__device__ __forceinline__ _Float16 least_of(const h8 (&w)[2]) {
  const auto a = __builtin_elementwise_min(w[0], w[1]);
  const auto b = __builtin_elementwise_min(__builtin_shufflevector(a, a, 0, 1, 2, 3), __builtin_shufflevector(a, a, 4, 5, 6, 7));
  const h2 c = __builtin_elementwise_min(__builtin_shufflevector(b, b, 0, 1), __builtin_shufflevector(b, b, 2, 3));
  return __builtin_elementwise_min(c.x, c.y);
}

// One block of the softmax of a column: raw products s of its 32 keys -> P, as the operand of O += V P, with the running
// reference m and sum l.  rescale(f) multiplies O where the reference moves.
template <int D, typename F>
__device__ __forceinline__ void softmax_block(f16v& s, const Column<D>& k, const Scales& b, bool masked, int key0, float one,
                                              float& m, float& l, h8 (&p)[2], F rescale) {
  const int half = (threadIdx.x & 63) >> 5;
  const float c = b.ks * k.c;
  auto sees = [&](int i) {
    const int key = key0 + 8 * (i >> 2) + 4 * half + (i & 3);
    return key < k.lim && key >= k.lo;
  };
  // The argument of a key is fma(s, c, lv), and c > 0 keeps the order.
  float top = -__builtin_inff();
  if (masked) {
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, sees(i) ? s[i] : -__builtin_inff());
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, s[i]);
  }
  top = fmaxf(top, other_half(top));
  const float high = fmaf(top, c, b.lv);       // a NaN (a poisoned block, or nothing seen at a zero c) moves nothing
  if (__any(high > m + HEADROOM)) {
    const float to = fmaxf(m, high);
    const float f = __builtin_amdgcn_exp2f(m - to);
    m = to;
    l *= f;
    rescale(f);
  }
  // P is summed as rounded, its subnormals too (the dot product instruction would take those as 0): v_fma_mix_f32 with a
  // `one` that the compiler does not see through.
  float sum = 0.0f;
  if (b.far) {
    // Where w is lost in fp16 although p counts in the sum, that takes p itself; both from one exponential.
    const float v = __builtin_amdgcn_exp2f(b.lv), shift = OFFSET - m;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, shift));
      if (masked) s[i] = sees(i) ? s[i] : 0.0f;
      const _Float16 r = static_cast<_Float16>(s[i] * v);
      p[i >> 3][i & 7] = r;
      sum += r >= FULL ? static_cast<float>(r) * b.iv : s[i];      // (a NaN takes s, which is one too)
    }
    l += sum;
  } else {
    const float shift = b.lv - m + OFFSET;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, shift));
    if (masked) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = sees(i) ? s[i] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const h2 r = __builtin_convertvector((f2v{s[i], s[i + 1]}), h2);
      p[i >> 3][i & 7] = r.x;
      p[i >> 3][(i & 7) + 1] = r.y;
      sum = fmaf(static_cast<float>(r.x), one, sum);
      sum = fmaf(static_cast<float>(r.y), one, sum);
    }
    l = fmaf(sum, b.iv, l);
  }
}

__device__ __forceinline__ float opaque_one() {
  float one = 1.0f;
  asm volatile("" : "+v"(one));
  return one;
}

// A column's result: to the output, or with splits to the workspace.
template <int D, int KIND>
__device__ __forceinline__ void store_column(const AttnArgs& a, const SeqRows& rows, int r, int n_rows, int head, int split,
                                             int parts, float m, float l, const f16v (&acc)[D / 32]) {
  if (r >= n_rows) return;
  const int half = (threadIdx.x & 63) >> 5, query = r / a.group;
  const int64_t q_head = head * a.group + (r - query * a.group), row = rows.first + query;
  if (parts > 1) {
    const int64_t at = (static_cast<int64_t>(split) * a.tokens + row) * a.q_heads + q_head;
    if (half == 0) {
      a.part_ml[2 * at] = m;
      a.part_ml[2 * at + 1] = l;
    }
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<float4*>(a.part_acc + at * D + 32 * t + 2 * i + 4 * half) =
            make_float4(acc[t][i], acc[t][i + 1], acc[t][i + 2], acc[t][i + 3]);
    return;
  }
  const float f = l == 0.0f ? 0.0f : 1.0f / l;   // a row that saw no key gives zeros
  uint16_t* out = static_cast<uint16_t*>(a.out) + row * a.out_stride + q_head * D + 4 * half;
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      uint32_t w[2];
#pragma unroll
      for (int b = 0; b < 2; ++b)
        w[b] = half_bits2<KIND>(acc[t][i + 2 * b] * f, acc[t][i + 2 * b + 1] * f);
      __builtin_memcpy(__builtin_assume_aligned(out + 32 * t + 2 * i, 2), w, 8);
    }
}

// ---- few rows: the four waves of a workgroup share 32 rows and take blocks of keys in turn --------------------------
// grid (KV heads, row tiles, batch * splits).  Nothing passes through LDS but the waves' join at the end.  With work for
// every CU it is bound by the cache's bytes, K's and V's next blocks being on their way while one is worked on: 8
// sequences of 900 to 32767 tokens (16800 on average), 8 heads of 128, 276 MB in 59 us, 4.7 TB/s (a large copy: 4.8), and 5
// for the join; 64 of 300 to 8192 of D 64, 278 MB in 64 us.  A short call is bound by its chain of loads (lengths, page,
// block) and the steps behind it, one after the other: 600 tokens, 19 blocks in five steps of the waves, 10.3 us.
// All sequences get as many parts, whatever their lengths, and one each where sequences times KV heads are 512 or more: 64 of 8
// heads of 128, one of 32768 tokens and 63 of 200 to 296, take 201 us, ten times what their bytes do.
template <int D, int KIND>
__global__ void __launch_bounds__(WAVES * 64, D <= 128 ? 2 : 1) attention_keys_kernel(AttnArgs a) {
  constexpr int KC = D / 32;           // 16-byte loads of K a lane, and tiles of 32 dims of V
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = blockIdx.x;
  const int seq = blockIdx.z / a.splits, split = blockIdx.z - seq * a.splits;
  const SeqRows rows = seq_rows(a.q_start, seq, a.tokens);
  const int n_rows = static_cast<int>(rows.count) * a.group, row0 = blockIdx.y * 32;
  if (row0 >= n_rows) return;
  const Sight sight{min(max(a.kv_lens[seq], 0), MAX_KV), static_cast<int>(rows.count), a.window};
  const int first_q = row0 / a.group, last_q = (min(row0 + 32, n_rows) - 1) / a.group;
  const int lim_first = sight.limit(first_q), lo_last = sight.lower(last_q);
  int blk = sight.lower(first_q) >> 5, blk_end = (sight.limit(last_q) + 31) >> 5;
  if (a.splits > 1) {
    const int chunk = chunk_of<D, true>(a, sight, a.splits, blk_end - blk);
    blk += split * chunk;
    blk_end = min(blk_end, blk + chunk);
  }
  f16v acc[KC];
#pragma unroll
  for (int t = 0; t < KC; ++t) acc[t] = f16v{0};
  float m = NEVER, l = 0.0f, lv_top = -__builtin_inff();
  const float one = opaque_one();
  int j = blk + wave;
  Blocks blocks;
  blocks.step = WAVES;
  const int k_off = lane * 16, v_off = (lane & 31) * 32 + (lane >> 5) * 16;
  auto load = [&](const uint8_t* from, int which, int off, uint4 (&r)[KC]) {
    const uint8_t* p = from + blocks.at(which) * (D * KV_BLOCK);
#pragma unroll
    for (int i = 0; i < KC; ++i) r[i] = *reinterpret_cast<const uint4*>(p + i * 1024 + off);
  };
  // The chain of a short call: lengths, page, block; everything else is asked for beside it.
  uint4 kr[KC], vr[KC];
  blocks.find(a.cache, seq, head, j, blk_end);
  load(a.cache.k, j, k_off, kr);
  load(a.cache.v, j, v_off, vr);
  blocks.scales(a.cache);
  const Column<D> k = load_column<D, KIND>(a, rows, sight, row0 + (lane & 31), n_rows, head);
  if (j < blk_end) {
    // K's registers are loaded with the next block as soon as the products with them are issued, V's likewise: each load
    // has the other half of a step to arrive in.
    for (; j < blk_end; j += WAVES) {
      const Scales b = scales_of(blocks, j, lv_top);
      f16v s = f16v{0};
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        s = __builtin_amdgcn_mfma_f32_32x32x16_f16(bytes8_to_half(kr[i].x, kr[i].y), k.q[2 * i], s, 0, 0, 0);
        s = __builtin_amdgcn_mfma_f32_32x32x16_f16(bytes8_to_half(kr[i].z, kr[i].w), k.q[2 * i + 1], s, 0, 0, 0);
      }
      const int next = j + WAVES, key0 = j * KV_BLOCK;
      if (blocks.slot(next) >= 64) blocks.lookup(a.cache, seq, head, next, blk_end);
      load(a.cache.k, next, k_off, kr);
      h8 p[2];
      softmax_block<D>(s, k, b, key0 + KV_BLOCK > lim_first || key0 < lo_last, key0, one, m, l, p, [&](float f) {
#pragma unroll
        for (int t = 0; t < KC; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[t][i] *= f;
      });
#pragma unroll
      for (int t = 0; t < KC; ++t) {
        acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bytes8_to_half(vr[t].x, vr[t].y), p[0], acc[t], 0, 0, 0);
        acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bytes8_to_half(vr[t].z, vr[t].w), p[1], acc[t], 0, 0, 0);
      }
      load(a.cache.v, next, v_off, vr);
    }
  }
  l += other_half(l);

  // Join the four waves: 2 and 3 into 0 and 1, then 1 into 0; through at most 32 KB of LDS.
  constexpr int PART = KC < 4 ? KC : 4;
  __shared__ float4 lds_acc[2][PART][4][64];
  __shared__ float lds_ml[2][2][64];
#pragma unroll
  for (int other = WAVES / 2; other >= 1; other >>= 1) {
    float f = 1.0f, f2 = 0.0f;
#pragma unroll
    for (int t0 = 0; t0 < KC; t0 += PART) {
      if (wave >= other && wave < 2 * other) {
        lds_ml[wave - other][0][lane] = m;
        lds_ml[wave - other][1][lane] = l;
#pragma unroll
        for (int t = 0; t < PART; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            lds_acc[wave - other][t][i][lane] = make_float4(acc[t0 + t][4 * i], acc[t0 + t][4 * i + 1], acc[t0 + t][4 * i + 2],
                                                            acc[t0 + t][4 * i + 3]);
      }
      __syncthreads();
      if (wave < other) {
        if (t0 == 0) {
          const float m2 = lds_ml[wave][0][lane], l2 = lds_ml[wave][1][lane], to = fmaxf(m, m2);
          f = __builtin_amdgcn_exp2f(m - to);
          f2 = __builtin_amdgcn_exp2f(m2 - to);
          m = to;
          l = l * f + l2 * f2;
        }
#pragma unroll
        for (int t = 0; t < PART; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 o = lds_acc[wave][t][i][lane];
            acc[t0 + t][4 * i] = acc[t0 + t][4 * i] * f + o.x * f2;
            acc[t0 + t][4 * i + 1] = acc[t0 + t][4 * i + 1] * f + o.y * f2;
            acc[t0 + t][4 * i + 2] = acc[t0 + t][4 * i + 2] * f + o.z * f2;
            acc[t0 + t][4 * i + 3] = acc[t0 + t][4 * i + 3] * f + o.w * f2;
          }
      }
      __syncthreads();
    }
  }
  if (wave == 0) store_column<D, KIND>(a, rows, row0 + (lane & 31), n_rows, head, split, a.splits, m, l, acc);
}

// ---- many rows: the waves of a workgroup have 32 rows each and walk over the keys together --------------------------
// grid (KV heads, row tiles, batch * splits): heads in front, so that with 8 of them each XCD keeps one head's cache in
// its L2; the tiles of the latest queries, which see the most keys, start first.
//
// Converting a block to fp16 costs a wave more than its matrix products (packed fp16 subtractions run at half rate), so
// the waves convert a block once, each its share, into LDS, in operand order: a lane reads its 16 bytes of every operand
// at lane * 16.  Two buffers and one barrier a step: at its end a wave converts its share of block j + 1 from registers
// into the other buffer and asks memory for block j + 2.
// There is no running maximum: P is taken against the reference as it is, and only where a column's sum says that P has
// grown out of its range is the maximum looked for, the reference moved and P taken again.
//
// What bounds it: 8192 tokens, 40 / 8 heads of 128, 674 to 720 us (0.95 to 1.02 PFLOP/s; a large bf16 product: 1.37): vector
// instructions 66 % and matrix instructions 53 % of the cycles, at 2.05 GHz.  Of D 256 it is the occupancy, two waves a SIMD,
// which wait for each other at the barrier (45 % of a wave's time; matrix instructions 44 % of the cycles): 0.6 PFLOP/s.
// Four waves, three such workgroups a CU, let one wave's softmax run in another's products.  Measured and not taken: eight
// waves (half the conversions a wave, but two waves a SIMD) 717 to 735 us, with half of them half a step behind the others
// 786 to 802; products of the next block behind the softmax of this one (250 registers, two waves a SIMD) 765 to 780; 64
// rows a wave 1053; K and V converted by every wave from registers 899; a running maximum looked for ahead of the
// exponentials 716; wave priorities around the products or the softmax, no difference.
template <int D, int KIND, int W>
__global__ void __launch_bounds__(W * 64, D <= 128 ? 3 : 2) attention_rows_kernel(AttnArgs a) {
  constexpr int TILE = 32 * W;
  constexpr int KC = D / 32, PIECES = 2 * KC;          // operand pieces of K, and of V; a 16-byte load gives two of them
  constexpr int LOADS = 2 * KC, MINE = LOADS / W;      // of a block: K's, then V's
  // Operands that are on their way from LDS while others are multiplied, V's first ones during the softmax; the order is
  // pinned, the compiler would ask for two and wait for them (8192 tokens 712 us and in this order 699, 2048 tokens 74 and
  // 71).  More would take more registers than there are.
  constexpr int K_AHEAD = D == 256 ? 3 : 4, V_AHEAD = D == 256 ? 1 : 2;
  __shared__ h8 lds_k[2][PIECES][64];
  __shared__ h8 lds_v[2][PIECES][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = blockIdx.x;
  Share share{static_cast<int>(blockIdx.z / a.splits), static_cast<int>(gridDim.y - 1 - blockIdx.y),
              static_cast<int>(blockIdx.z % a.splits), a.splits};
  if (a.parts) share = share_of<TILE>(a, blockIdx.y);
  if (share.seq < 0) return;
  const int seq = share.seq;
  const SeqRows rows = seq_rows(a.q_start, seq, a.tokens);
  const int n_rows = static_cast<int>(rows.count) * a.group;
  const int tile0 = share.tile * TILE, row0 = tile0 + wave * 32;
  if (tile0 >= n_rows) return;
  const Sight sight{min(max(a.kv_lens[seq], 0), MAX_KV), static_cast<int>(rows.count), a.window};
  // Blocks that the tile sees; a wave's own rows may see fewer, it masks the rest.
  int blk = sight.lower(tile0 / a.group) >> 5;
  int blk_end = (sight.limit((min(tile0 + TILE, n_rows) - 1) / a.group) + 31) >> 5;
  if (share.parts > 1) {
    const int chunk = chunk_of<D>(a, sight, share.parts, blk_end - blk);
    blk += share.split * chunk;
    blk_end = min(blk_end, blk + chunk);
  }
  const int lim_first = sight.limit(min(row0, n_rows - 1) / a.group);
  const int lo_last = sight.lower((min(row0 + 32, n_rows) - 1) / a.group);

  const Column<D> k = load_column<D, KIND>(a, rows, sight, row0 + (lane & 31), n_rows, head);
  f16v acc[KC];
#pragma unroll
  for (int t = 0; t < KC; ++t) acc[t] = f16v{0};
  float m = NEVER, l = 0.0f, lv_top = -__builtin_inff();
  const float one = opaque_one();
  Blocks blocks;
  blocks.step = 1;
  Scales s1{}, s2{};               // of the two blocks that were asked for last
  uint4 raw[MINE];
  auto load_of = [&](int r) { return wave + W * r; };
  auto fetch = [&](int which) {
    if (blocks.slot(which) >= 64) blocks.lookup(a.cache, seq, head, which, blk_end);
    const int slot = blocks.slot(which);
    const int64_t at = blocks.at(which) * (D * KV_BLOCK);
    s1 = s2;
    s2 = Scales{read_lane_f(blocks.ks, slot), read_lane_f(blocks.lv, slot), read_lane_f(blocks.iv, slot), false};
#pragma unroll
    for (int r = 0; r < MINE; ++r) {
      const int i = load_of(r);
      const uint8_t* from = i < KC ? a.cache.k + at + i * 1024 + lane * 16
                                   : a.cache.v + at + (i - KC) * 1024 + (lane & 31) * 32 + (lane >> 5) * 16;
      raw[r] = *reinterpret_cast<const uint4*>(from);
    }
  };
  auto convert = [&](int buffer) {
#pragma unroll
    for (int r = 0; r < MINE; ++r) {
      const int i = load_of(r);
      h8(*to)[64] = i < KC ? &lds_k[buffer][2 * i] : &lds_v[buffer][2 * (i - KC)];
      to[0][lane] = bytes8_to_half(raw[r].x, raw[r].y);
      to[1][lane] = bytes8_to_half(raw[r].z, raw[r].w);
    }
  };
  const int half = lane >> 5;
  // P of a block from its raw products s (see above), and what it adds to the sum.
  auto weigh = [&](const f16v& s, float c, float shift, h8 (&p)[2]) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const float w0 = __builtin_amdgcn_exp2f(fmaf(s[i], c, shift)), w1 = __builtin_amdgcn_exp2f(fmaf(s[i + 1], c, shift));
      const h2 r = __builtin_convertvector((f2v{w0, w1}), h2);
      p[i >> 3][i & 7] = r.x;
      p[i >> 3][(i & 7) + 1] = r.y;
      // summed as rounded, subnormals too (the dot product instruction takes those as 0): v_fma_mix_f32 with a 1 that the
      // compiler does not see through
      sum = fmaf(static_cast<float>(r.x), one, sum);
      sum = fmaf(static_cast<float>(r.y), one, sum);
    }
    return sum;
  };
  if (blk < blk_end) {
    blocks.lookup(a.cache, seq, head, blk, blk_end);
    fetch(blk);
    convert(0);
    fetch(blk + 1);                // (behind the end: block 0's bytes, not worked on)
    for (int j = blk; j < blk_end; ++j) {
      const int here = (j - blk) & 1;
      lds_barrier();               // block j is in LDS, and nobody reads the other buffer any more
      const Scales b = s1;
      f16v s = f16v{0};
      {
        h8 o[K_AHEAD];
#pragma unroll
        for (int i = 0; i < K_AHEAD; ++i) o[i] = lds_k[here][i][lane];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          s = __builtin_amdgcn_mfma_f32_32x32x16_f16(o[i % K_AHEAD], k.q[i], s, 0, 0, 0);
          if (i + K_AHEAD < PIECES) o[i % K_AHEAD] = lds_k[here][i + K_AHEAD][lane];
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      auto v_piece = [&](int i) { return lds_v[here][2 * (i % KC) + i / KC][lane]; };
      h8 vo[V_AHEAD];
#pragma unroll
      for (int i = 0; i < V_AHEAD; ++i) vo[i] = v_piece(i);
      const int key0 = j * KV_BLOCK;
      float c = b.ks * k.c;
      c = c < 1e-37f ? 1e-37f : c;   // (a NaN stays)
      float lv = b.lv;
      bool none = false;
      if (key0 + KV_BLOCK > lim_first || key0 < lo_last) {
        // Keys that the column does not see count as -infinity; where it sees none, everything as 0 under a weight of 0: a
        // NaN scale must not reach it.
        none = key0 >= k.lim || key0 + KV_BLOCK <= k.lo;
        c = none ? 0.0f : c;
        lv = none ? -__builtin_inff() : lv;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = key0 + 8 * (i >> 2) + 4 * half + (i & 3);
          s[i] = key < k.lim && key >= k.lo ? s[i] : none ? 0.0f : -__builtin_inff();
        }
      }
      h8 p[2];
      float sum = weigh(s, c, lv - m + OFFSET, p);
      if (__any(sum > RANGE)) {
        float top = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
        top = fmaxf(top, other_half(top));
        const float to = fmaxf(m, fmaf(top, c, lv)), f = __builtin_amdgcn_exp2f(m - to);
        m = to;
        l *= f;
#pragma unroll
        for (int t = 0; t < KC; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[t][i] *= f;
        sum = weigh(s, c, lv - m + OFFSET, p);
      }
      lv_top = fmaxf(lv_top, b.lv);
      // Where V's scale is less than a quarter of the largest so far, some w may be lost in fp16 although p counts in the sum,
      // which then takes p itself in their place, at the price of 16 more exponentials (8192 tokens whose scales lie up to 2^6
      // apart: 703 us against 671).  Of D 256 there are no registers to look for such w first, nor to take them off the sum
      // afterwards (512 tokens 39.4 us against 38.3, whatever the scales).
      const bool far = b.lv < lv_top - 2.0f && b.lv > -__builtin_inff();
      const float p_shift = none ? -__builtin_inff() : OFFSET - m;
      if constexpr (D == 256) {
        if (far) {
          float add = 0.0f;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const _Float16 w = p[i >> 3][i & 7];
            const float p_i = __builtin_amdgcn_exp2f(fmaf(s[i], c, p_shift));
            add += w < FULL ? p_i : static_cast<float>(w) * b.iv;
          }
          l += add;
        } else {
          l = fmaf(sum, b.iv, l);
        }
      } else {
        l = fmaf(sum, b.iv, l);
        if (far && __any(least_of(p) < FULL)) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const _Float16 w = p[i >> 3][i & 7];
            const float more = fmaf(-static_cast<float>(w), b.iv, __builtin_amdgcn_exp2f(fmaf(s[i], c, p_shift)));
            l += w < FULL ? more : 0.0f;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        acc[i % KC] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vo[i % V_AHEAD], p[i / KC], acc[i % KC], 0, 0, 0);
        if (i + V_AHEAD < PIECES) vo[i % V_AHEAD] = v_piece(i + V_AHEAD);
        __builtin_amdgcn_sched_barrier(0);
      }
      convert(here ^ 1);
      fetch(j + 2);
    }
  }
  l += other_half(l);
  store_column<D, KIND>(a, rows, row0 + (lane & 31), n_rows, head, share.split, share.parts, m, l, acc);
}

// Joins the chunks of output rows: grid (rows a sequence / (4 / TEAM), batch); TEAM waves have a row and take its chunks in
// turn, D / 64 dims a lane.  What bounds it is the time that a load takes, so for few rows, or many chunks, a row has four
// waves: 40 rows of 64 chunks 4.0 us, 320 of up to 8 chunks 4.9 us, with a wave a row 11 and 5.8.  Many rows of few chunks
// have enough loads on their way: 2560 rows of 2 or 3 chunks 5.2 us, 24576 of D 256 14.4 us, with four waves 9.9 and 39.
template <int D, int KIND, int TEAM>
__global__ void __launch_bounds__(256) join_kernel(AttnArgs a, int tile_rows) {
  constexpr int V = D / 64;
  __shared__ float part[4][D];
  const int seq = blockIdx.y, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int parts = a.parts ? a.parts[seq] : a.splits;
  if (parts <= 1) return;
  const SeqRows rows = seq_rows(a.q_start, seq, a.tokens);
  const int64_t r = static_cast<int64_t>(blockIdx.x) * (4 / TEAM) + wave / TEAM;
  if (r >= rows.count * a.q_heads) return;             // (of a team all waves or none: the barrier below is for TEAM 4)
  const int query = static_cast<int>(r / a.q_heads), q_head = static_cast<int>(r - static_cast<int64_t>(query) * a.q_heads);
  // The chunks that a workgroup ran for this row: as the attention kernel laid them for the row's tile.
  const Sight sight{min(max(a.kv_lens[seq], 0), MAX_KV), static_cast<int>(rows.count), a.window};
  const int row = query * a.group + q_head % a.group;
  const int tile0 = row / tile_rows * tile_rows, last_q = (min(tile0 + tile_rows, static_cast<int>(rows.count) * a.group) - 1) / a.group;
  const int first = sight.lower(tile0 / a.group) >> 5, chunk = chunk_of<D>(a, sight, parts, ((sight.limit(last_q) + 31) >> 5) - first);
  const int blocks = max(((sight.limit(query) + 31) >> 5) - first, 0), splits = (blocks + chunk - 1) / chunk;
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
    // A team's last chunks are asked for at once too (those behind the end are the last one again, at no weight); a wave that
    // is one of thousands does better without.
    constexpr int AHEAD = TEAM == 1 ? 1 : 8;
#pragma unroll(TEAM == 1 ? 8 : 1)
    for (int k0 = wave % TEAM; k0 < n; k0 += AHEAD * TEAM) {
      float x[AHEAD][V];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        __builtin_memcpy(x[i], __builtin_assume_aligned(a.part_acc + ((s0 + min(k0 + i * TEAM, n - 1)) * pitch + at) * D + lane * V, 4 * V), 4 * V);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const bool there = k0 + i * TEAM < n;
        const float w = there ? read_lane_f(f, k0 + i * TEAM) : 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) o[v] = fmaf(there ? x[i][v] : 0.0f, w, o[v]);
      }
    }
  }
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) l += __shfl_xor(l, off);
  const float f = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* dst = static_cast<uint16_t*>(a.out) + (rows.first + query) * a.out_stride + static_cast<int64_t>(q_head) * D;
  if constexpr (TEAM == 1) {
    uint32_t w[(V + 1) / 2];
#pragma unroll
    for (int v = 0; v < V; v += 2) w[v / 2] = half_bits2<KIND>(o[v] * f, v + 1 < V ? o[v + 1] * f : 0.0f);
    __builtin_memcpy(__builtin_assume_aligned(dst + lane * V, 2), w, 2 * V);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) part[wave][lane * V + v] = o[v];
    __syncthreads();
    const int d = 2 * threadIdx.x;
    if (d >= D) return;
    const uint32_t w = half_bits2<KIND>((part[0][d] + part[1][d] + part[2][d] + part[3][d]) * f,
                                        (part[0][d + 1] + part[1][d + 1] + part[2][d + 1] + part[3][d + 1]) * f);
    __builtin_memcpy(__builtin_assume_aligned(dst + d, 2), &w, 4);
  }
}

// How a call is cut: decided from sizes alone, so that the workspace can be sized before the call.
struct Plan {
  bool keys;          // few rows: the waves of a workgroup share them and split keys
  int waves;
  int tile_rows;
  int64_t tiles;
  int splits;         // most parts of a tile's keys
  int most_splits;    // what the workspace is sized for: no fewer for fewer keys
  int typical;        // parts where all sequences are as long as announced
  int chunk, least;   // as in AttnArgs
  bool shares;        // several prompts in parts
  int64_t items;      // their workgroups a KV head
};

constexpr int CUS = 256;

// What rows are cut into, and keys where the rows alone are too few.
void cut(Plan& p, int64_t rows, int64_t blocks, int64_t batch, int64_t kv_heads, int64_t slots, int64_t least) {
  p.tiles = (rows + p.tile_rows - 1) / p.tile_rows;
  const int64_t groups = batch * kv_heads * p.tiles, most = blocks > least ? (blocks + least - 1) / least : 1;
  const int64_t splits = !p.keys && groups >= CUS ? 1 : (slots + groups - 1) / groups;
  // Of prompts that differ in length the longer ones get more parts than that.
  const int64_t up_to = p.keys || batch == 1 || splits == 1 ? splits : 2 * splits;
  p.typical = static_cast<int>(splits < most ? splits : most);
  p.splits = p.most_splits = static_cast<int>(up_to < most ? up_to : most);
  p.shares = !p.keys && batch > 1 && p.splits > 1;
  p.least = static_cast<int>(least);
  p.chunk = p.keys ? p.least : p.shares ? 1 : 0;
  p.items = slots / kv_heads > batch * p.tiles ? slots / kv_heads : batch * p.tiles;
}

Plan plan_of(int64_t batch, int64_t max_q, int64_t max_kv, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t window) {
  Plan p;
  const int64_t rows = max_q * (q_heads / kv_heads);
  p.keys = rows <= 64;
  const int64_t blocks = blocks_of(max_kv, max_q, window);
  // Two workgroups a CU.  With a workgroup a CU from the rows alone, prompts are not split (they would be joined for less
  // than they gain: 2048 tokens, 640 tiles, 72 us as they are and 97 us in two parts).  A part of a prompt has at least
  // LEAST_ROWS and one of few rows, whose keys four waves share, at least LEAST_KEYS: a single token behind 600 others (19
  // blocks of 128) takes 14.4 us undivided and 17.3 us in two parts and the joining of them, behind 32768 others 22 us in
  // 32 parts and 26 us in 64; 512 tokens of D 128 (16 blocks) 23 us undivided and 35 us in two, of D 256 40 and 38 us.
  const int64_t LEAST_KEYS = 4096 / dim, LEAST_ROWS = least_rows(static_cast<int>(dim));
  p.waves = WAVES;
  p.tile_rows = p.keys ? 32 : 32 * WAVES;
  cut(p, rows, blocks, batch, kv_heads, 2 * CUS, p.keys ? LEAST_KEYS : LEAST_ROWS);
  if (!p.keys && dim == 256) {
    // Eight waves convert a block for twice the rows. Of D 256 a CU holds as many of them either way (of smaller D not: 3
    // workgroups of four), and they win once there is nearly a workgroup for every CU: 3 chunks of 512 tokens 129 us
    // against 154, 1024 tokens 48 against 52, but 512 tokens 42 against 38.
    Plan wide = p;
    wide.waves = 2 * WAVES;
    wide.tile_rows = 64 * WAVES;
    cut(wide, rows, blocks, batch, kv_heads, CUS, LEAST_ROWS);
    const int most = p.most_splits > wide.most_splits ? p.most_splits : wide.most_splits;   // (a window may decide otherwise)
    if (batch * kv_heads * wide.tiles * wide.typical >= CUS * 3 / 4) p = wide;
    p.most_splits = most;
  }
  return p;
}

constexpr int BAD = static_cast<int>(hipErrorInvalidValue);
constexpr int64_t MAX_TILES = 65535;   // of a sequence: the grid's second dimension

// The rows of D 256 that are more than MAX_TILES tiles of four waves are tiles of eight (they fill the chip).
bool shape_ok(int64_t tokens, int64_t batch, int64_t max_q, int64_t max_kv, int64_t q_heads, int64_t kv_heads, int64_t dim,
              int64_t window) {
  return tokens > 0 && batch > 0 && batch <= 65535 && max_q > 0 && max_kv >= 0 && max_kv <= MAX_KV && kv_heads > 0 &&
         kv_heads <= 65535 && q_heads > 0 && q_heads % kv_heads == 0 && q_heads <= 4096 &&
         (dim == 64 || dim == 128 || dim == 256) && window >= 0 && window <= (1 << 30) && tokens <= (1 << 26) &&
         (max_q < tokens ? max_q : tokens) * (q_heads / kv_heads) <= MAX_TILES * 32 * (dim == 256 ? 2 * WAVES : WAVES);
}

int64_t workspace_of(bool keys, int splits, int64_t tokens, int64_t batch, int64_t q_heads, int64_t dim) {
  return splits > 1 ? static_cast<int64_t>(splits) * tokens * q_heads * (dim + 2) * 4 + (keys || batch == 1 ? 0 : 4 * batch) : 0;
}

template <int D, int KIND>
int launch(const AttnArgs& a, const Plan& p, int64_t batch, int64_t max_q, int64_t kv_heads, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(kv_heads), static_cast<unsigned>(p.shares ? p.items : p.tiles),
                  static_cast<unsigned>(p.shares ? 1 : batch * p.splits));
  if (p.keys) {
    hipLaunchKernelGGL((attention_keys_kernel<D, KIND>), grid, dim3(WAVES * 64), 0, stream, a);
  } else if (p.waves == WAVES) {
    hipLaunchKernelGGL((attention_rows_kernel<D, KIND, WAVES>), grid, dim3(WAVES * 64), 0, stream, a);
  } else if constexpr (D == 256) {
    hipLaunchKernelGGL((attention_rows_kernel<D, KIND, 2 * WAVES>), grid, dim3(2 * WAVES * 64), 0, stream, a);
  }
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess || p.splits == 1) return static_cast<int>(err);
  const int64_t out_rows = max_q * a.q_heads;
  const unsigned each = static_cast<unsigned>(out_rows), of_four = static_cast<unsigned>((out_rows + 3) / 4), b = static_cast<unsigned>(batch);
  if (p.typical > 8 || batch * out_rows <= 2048)
    hipLaunchKernelGGL((join_kernel<D, KIND, 4>), dim3(each, b), dim3(256), 0, stream, a, p.tile_rows);
  else
    hipLaunchKernelGGL((join_kernel<D, KIND, 1>), dim3(of_four, b), dim3(256), 0, stream, a, p.tile_rows);
  return static_cast<int>(hipGetLastError());
}

}  // namespace

extern "C" int hipengine_gfx950_paged_attention_q8_workspace_bytes(int64_t tokens, int64_t batch, int64_t max_q_len,
                                                                   int64_t max_kv_len, int64_t q_heads, int64_t kv_heads,
                                                                   int64_t head_dim, int64_t* bytes) {
  if (!bytes || !shape_ok(tokens, batch, max_q_len, max_kv_len, q_heads, kv_heads, head_dim, 0)) return BAD;
  const int64_t longest = max_q_len < tokens ? max_q_len : tokens;
  const Plan p = plan_of(batch, longest, max_kv_len, q_heads, kv_heads, head_dim, 0);
  *bytes = workspace_of(p.keys, p.most_splits, tokens, batch, q_heads, head_dim);
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
  const int64_t need = workspace_of(p.keys, p.splits, tokens, batch, q_heads, head_dim);
  if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0)) return BAD;
  const KvCacheQ8 cache{const_cast<uint8_t*>(k_cache), const_cast<uint8_t*>(v_cache), const_cast<float*>(k_scale),
                        const_cast<float*>(v_scale), page_table, table_stride, pages, static_cast<int>(kv_heads),
                        63 - __builtin_clzll(static_cast<unsigned long long>(page_size))};
  const int64_t out_rows = p.splits > 1 ? static_cast<int64_t>(p.splits) * tokens * q_heads : 0;
  float* acc = p.splits > 1 ? static_cast<float*>(workspace) : nullptr;
  float* ml = acc ? acc + out_rows * head_dim : nullptr;
  int32_t* parts = p.shares ? reinterpret_cast<int32_t*>(ml + 2 * out_rows) : nullptr;
  const AttnArgs a{cache, q, out, q_stride, out_stride, q_start, kv_lens, tokens, softmax_scale * LOG2E,
                   static_cast<int>(q_heads / kv_heads), static_cast<int>(q_heads), static_cast<int>(window), p.splits,
                   p.chunk, parts, static_cast<int>(p.items), static_cast<int>(p.tiles), static_cast<int>(batch), p.least, acc, ml};
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
  return static_cast<int>(hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(attention_keys_kernel<128, KIND_BF16>)));
}
