// The paged KV cache in 8 bits: appending tokens (with the keys' norm and rotation on the way) and reading them back.
//
// One float32 scale for each block of 32 tokens and head, K and V apart:
//   scale' = max(scale of the tokens that stay, amax / 127, 2^-64),   byte = 128 + clamp(rint(x / scale'), -127, 127)
// and where that is more than the old scale the tokens that stay are brought to it, q' = rint(q * scale / scale').
// A block whose first token is among the appended ones starts anew: whatever it held, its old scale is not looked at.
// A NaN or infinity among a block's new tokens makes its scale NaN, and with it everything that the block yields (8-bit
// values have no place for one); it stays so until the block starts anew.  Bytes behind the appended tokens stay.
//
// Work is cut by (sequence, block, head, K or V), and one workgroup owns that piece: the only writer of the block's
// scale and bytes, so there are no atomics and results do not depend on timing.
//
// What bounds it.  A single token waits for its chain of loads (row, page, scale, block): 8 sequences, append 4.6 and read
// 4.0 us.  Of prompts, 8244 tokens of 8 heads of 128 (50 MB in and out), reading back takes 11 us (4.6 TB/s, a large copy
// 4.8; with K through LDS as well 13.9); appending takes 21, not by its bytes but by its stages: rows, norm and rotation,
// the largest magnitude, and only then the bytes (K alone 18, V alone 11, both without the rotation 18; with the tokens in
// LDS as float32 and the angles shared, 26).

#include <hip/hip_runtime.h>

#include "attn_common.hpp"

#include "gguf_init.hpp"

#include "../../include/hipengine_gfx950.h"

namespace {

using namespace hipengine_gfx950;

constexpr int THREADS = 256;

// Byte offset of the 16-byte item in a block, K or V: item i of K is dims 16 (i / 32) .. of token i % 32, item i of V is
// places 16 (i % 2) .. of dim i / 2; in both layouts the items follow each other.
__device__ __forceinline__ int item_offset(int item) { return item * 16; }

// Which block of which sequence a workgroup works on.  With `per_seq` > 0 every sequence has that many blocks in the
// grid; with 0 sequence b has floor(q_start[b] / 32) + 2b blocks in front of it, which leaves room for the most that its
// tokens can touch (n tokens touch at most floor(n / 32) + 2 blocks) without a prefix sum over the batch.
struct Piece {
  int seq;
  int64_t block;       // in its sequence
  int first, last;     // tokens of the block that this call is about: [first, last), 0..32
  int64_t row;         // row of the batch that token `first` is
};

// Every wave finds it for itself, 64 sequences at a time and without a barrier.
__device__ __forceinline__ bool find_piece(const int32_t* __restrict__ q_start, const int32_t* __restrict__ kv_lens,
                                           int64_t tokens, int batch, int per_seq, int64_t unit, Piece& p) {
  int seq = -1;
  int64_t local;
  if (per_seq > 0) {
    seq = static_cast<int>(unit / per_seq);
    local = unit - static_cast<int64_t>(seq) * per_seq;
  } else {
    const int lane = threadIdx.x & 63;
    for (int b0 = 0; b0 < batch; b0 += 64) {
      const int b = b0 + lane;
      const bool before = b < batch && (max(q_start[b], 0) >> 5) + 2 * static_cast<int64_t>(b) <= unit;
      const unsigned long long all = __ballot(before);
      if (all) seq = b0 + 63 - __builtin_clzll(all);
      if (all != ~0ull) break;                        // (blocks in front grow from sequence to sequence)
    }
    if (seq < 0) return false;
    local = unit - ((max(q_start[seq], 0) >> 5) + 2 * static_cast<int64_t>(seq));
  }
  const SeqRows rows = seq_rows(q_start, seq, tokens);
  const int64_t end = kv_lens[seq];                  // place behind the last token
  const int64_t begin = end - rows.count;            // place of the first row; rows at negative places are left out
  const int64_t from = max(begin, int64_t{0});
  p.seq = seq;
  p.block = (from >> 5) + local;
  const int64_t base = p.block << 5;
  if (local < 0 || base >= end || rows.count <= 0) return false;
  p.first = static_cast<int>(max(from - base, int64_t{0}));
  p.last = static_cast<int>(min(end - base, int64_t{KV_BLOCK}));
  p.row = rows.first + (base + p.first - begin);
  return p.first < p.last;
}

struct AppendArgs {
  KvCacheQ8 cache;
  const void* k;
  const void* v;
  int64_t k_stride, v_stride;
  const float* k_weight;
  const int64_t* positions;
  const float* inv_freq;
  const int32_t* q_start;
  const int32_t* kv_lens;
  int64_t tokens;
  int batch, per_seq, rotary_dim, interleaved;
  float eps, rope_scale;
};

// 128 + rint(x / scale) in the low byte: the quotient by the reciprocal, corrected by its exact remainder (rounded as the
// division is), and the rounding by adding 1.5 * 2^23.  |x| is at most 127 scales up to the scale's own rounding, which rint
// takes off again: nothing is to be clamped.
__device__ __forceinline__ uint32_t quantize(float x, float scale, float reciprocal) {
  const float q = x * reciprocal, exact = fmaf(fmaf(-scale, q, x), reciprocal, q);
  return float_to_bits(exact + 12583040.0f);
}
// The low bytes of four.
__device__ __forceinline__ uint32_t pack_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0C0C0400u), __builtin_amdgcn_perm(b, a, 0x0C0C0400u), 0x05040100u);
}
__device__ __forceinline__ uint32_t requantize(uint32_t byte, float ratio) {
  return static_cast<uint32_t>(static_cast<int>(rintf(static_cast<float>(static_cast<int>(byte) - 128) * ratio)) + 128);
}

// The largest of a wave.
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t u) {
  u = max(u, static_cast<uint32_t>(dpp_i<DPP_QUAD_XOR1>(static_cast<int>(u))));
  u = max(u, static_cast<uint32_t>(dpp_i<DPP_QUAD_XOR2>(static_cast<int>(u))));
  u = max(u, static_cast<uint32_t>(dpp_i<DPP_ROW_HALF_MIRROR>(static_cast<int>(u))));
  u = max(u, static_cast<uint32_t>(dpp_i<0x140>(static_cast<int>(u))));     // row_mirror
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  u = max(r[0], r[1]);
  const auto h = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return max(h[0], h[1]);
}

constexpr int V_ROW = KV_BLOCK + 4;      // bytes of a V block's row in LDS: 8 lanes work on rows 8 apart

template <int D>
struct AppendLds {
  __align__(16) uint8_t v[D * V_ROW];
  uint32_t amax_of[THREADS / 64];
  float old;
};

// The new tokens stay in registers, 8 values of a token a lane, from their loads to their bytes: normed and rotated (angles
// are computed by every lane for itself), their largest magnitude joined through LDS, quantized.  A token's bytes of K lie
// together and go straight to the cache; those of V pass through LDS as bytes, to leave as the rows of the V block.
template <int KIND, int D, bool is_v>
__device__ __forceinline__ void append_piece(const AppendArgs& a, AppendLds<D>& lds) {
  constexpr int LANES = D / 8, ROWS = THREADS / LANES, PASSES = KV_BLOCK / ROWS, ITEMS = (2 * D + THREADS - 1) / THREADS;
  const int head = blockIdx.y;
  Piece p;
  if (!find_piece(a.q_start, a.kv_lens, a.tokens, a.batch, a.per_seq, blockIdx.x, p)) return;
  // Everything that is to be read is asked for as early as it can be: the rows before the page is known.
  const int slot = threadIdx.x % LANES, sub = threadIdx.x / LANES;
  const void* src = is_v ? a.v : a.k;
  const int64_t stride = is_v ? a.v_stride : a.k_stride;
  const bool turns = !is_v && 8 * slot < a.rotary_dim, interleaved = a.interleaved != 0;
  float y[PASSES][8];
  int64_t position[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int t = p.first + i * ROWS + sub;
    if (t >= p.last) break;
    load8_f32<KIND>(src, (p.row + (t - p.first)) * stride + static_cast<int64_t>(head) * D + 8 * slot, y[i]);
    position[i] = (p.block << 5) + t;
    if (turns && a.positions) position[i] = a.positions[p.row + (t - p.first)];
  }
  const int64_t block = kv_block_index(a.cache, p.seq, p.block, head);
  if (block < 0) return;
  const bool whole = p.first == 0 && p.last == KV_BLOCK;
  uint8_t* bytes = (is_v ? a.cache.v : a.cache.k) + block * (D * KV_BLOCK);
  float* scale_at = (is_v ? a.cache.v_scale : a.cache.k_scale) + block;
  float old = 0.0f;
  if (threadIdx.x == 0 && p.first > 0) old = kv_scale(*scale_at);      // by the thread that will write it
  uint4 kept[ITEMS];
  if (is_v && !whole) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int item = threadIdx.x + i * THREADS;
      if (item < 2 * D) kept[i] = *reinterpret_cast<const uint4*>(bytes + item_offset(item));
    }
  }
  uint32_t amax_bits = 0;         // magnitudes order like their bits, infinity and NaN above all numbers
  double freq[8];
  if (turns) {
    const float* from = a.inv_freq + first_pair(slot, a.rotary_dim, interleaved);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < 4 || !interleaved) freq[k] = turns_of(from[k]);
  }
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int t = p.first + i * ROWS + sub;
    if (t >= p.last) break;
    if constexpr (!is_v) {
      float2 cs[8];
      if (turns) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < 4 || !interleaved) cs[k] = rotation(position[i], freq[k], a.rope_scale);
      }
      norm_rotate8<D>(y[i], slot, a.k_weight, a.eps, [&](int k) { return cs[k]; }, a.rotary_dim, interleaved);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) amax_bits = max(amax_bits, float_to_bits(y[i][k]) & 0x7FFFFFFFu);
  }
  amax_bits = wave_max_u32(amax_bits);
  if ((threadIdx.x & 63) == 0) lds.amax_of[threadIdx.x >> 6] = amax_bits;
  if (threadIdx.x == 0) lds.old = old;
  __syncthreads();
  amax_bits = max(max(lds.amax_of[0], lds.amax_of[1]), max(lds.amax_of[2], lds.amax_of[3]));
  old = lds.old;
  const bool poisoned = amax_bits >= 0x7F800000u || old != old;
  const float scale = fmaxf(fmaxf(old, bits_to_float(amax_bits) / 127.0f), KV_SCALE_FLOOR);
  const float ratio = old / scale, reciprocal = 1.0f / scale;      // ratio: 1 where the scale stays
  if (threadIdx.x == 0) *scale_at = poisoned ? __builtin_nanf("") : scale;
  const bool grown = ratio != 1.0f && !poisoned;

#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int t = p.first + i * ROWS + sub;
    if (t >= p.last) break;
    uint32_t q[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) q[k] = poisoned ? 128u : quantize(y[i][k], scale, reciprocal);
    if constexpr (is_v) {
#pragma unroll
      for (int k = 0; k < 8; ++k) lds.v[(8 * slot + k) * V_ROW + v_place(t)] = static_cast<uint8_t>(q[k]);
    } else {
      *reinterpret_cast<uint2*>(bytes + ((slot >> 1) * KV_BLOCK + t) * 16 + 8 * (slot & 1)) =
          make_uint2(pack_bytes(q[0], q[1], q[2], q[3]), pack_bytes(q[4], q[5], q[6], q[7]));
    }
  }
  if constexpr (!is_v) {
    if (!grown || p.first == 0) return;
    for (int item = threadIdx.x; item < 2 * D; item += THREADS) {      // 16 dims of one of the earlier tokens
      if ((item & 31) >= p.first) continue;
      uint4 u = *reinterpret_cast<const uint4*>(bytes + item_offset(item));
      uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t r = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) r |= requantize((w[i] >> (8 * j)) & 0xFFu, ratio) << (8 * j);
        w[i] = r;
      }
      *reinterpret_cast<uint4*>(bytes + item_offset(item)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  } else {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {      // 16 tokens of a dim
      const int item = threadIdx.x + i * THREADS;
      if (item >= 2 * D) break;
      const uint32_t* from = reinterpret_cast<const uint32_t*>(lds.v + (item >> 1) * V_ROW + (item & 1) * 16);
      uint32_t w[4] = {from[0], from[1], from[2], from[3]};
      if (!whole) {
        const uint32_t there[4] = {kept[i].x, kept[i].y, kept[i].z, kept[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t r = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int t = v_token((item & 1) * 16 + 4 * j + b);
            uint32_t byte = ((t >= p.first && t < p.last ? w[j] : there[j]) >> (8 * b)) & 0xFFu;
            if (t < p.first && grown) byte = requantize(byte, ratio);
            r |= byte << (8 * b);
          }
          w[j] = r;
        }
      }
      *reinterpret_cast<uint4*>(bytes + item_offset(item)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// grid (units, heads, 2): z 0 is K, z 1 is V.
template <int KIND, int D>
__global__ void __launch_bounds__(THREADS) kv_append_kernel(AppendArgs a) {
  __shared__ AppendLds<D> lds;
  if (blockIdx.z == 0) append_piece<KIND, D, false>(a, lds);
  else append_piece<KIND, D, true>(a, lds);
}

struct ReadArgs {
  KvCacheQ8 cache;
  void* k;
  void* v;
  int64_t k_stride, v_stride;
  const int32_t* start;
  const int32_t* kv_lens;
  int64_t tokens;
  int batch, per_seq;
};

// 8 values of a token a lane, as in the append.  Those of K lie together; V's block passes through LDS as bytes, so that a
// row's values leave as whole lines.  A block that is not in the cache (a bad page) yields zeros.
template <int KIND, int D, bool is_v>
__device__ __forceinline__ void read_piece(const ReadArgs& a, uint8_t* lds) {
  constexpr int LANES = D / 8, ROWS = THREADS / LANES, PASSES = KV_BLOCK / ROWS;
  void* dst = is_v ? a.v : a.k;
  if (!dst) return;
  const int head = blockIdx.y;
  Piece p;
  if (!find_piece(a.start, a.kv_lens, a.tokens, a.batch, a.per_seq, blockIdx.x, p)) return;
  const int64_t block = kv_block_index(a.cache, p.seq, p.block, head);
  const float scale = block < 0 ? 0.0f : kv_scale((is_v ? a.cache.v_scale : a.cache.k_scale)[block]);
  const uint8_t* bytes = (is_v ? a.cache.v : a.cache.k) + max(block, int64_t{0}) * (D * KV_BLOCK);
  const int slot = threadIdx.x % LANES, sub = threadIdx.x / LANES;
  uint2 direct[PASSES];
  if constexpr (is_v) {
    for (int item = threadIdx.x; item < 2 * D; item += THREADS) {
      const uint4 u = *reinterpret_cast<const uint4*>(bytes + item_offset(item));
      uint32_t* to = reinterpret_cast<uint32_t*>(lds + (item >> 1) * V_ROW + (item & 1) * 16);
      to[0] = u.x; to[1] = u.y; to[2] = u.z; to[3] = u.w;
    }
    __syncthreads();
  } else {
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int t = p.first + i * ROWS + sub;
      if (t < p.last) direct[i] = *reinterpret_cast<const uint2*>(bytes + ((slot >> 1) * KV_BLOCK + t) * 16 + 8 * (slot & 1));
    }
  }
  const int64_t stride = is_v ? a.v_stride : a.k_stride;
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int t = p.first + i * ROWS + sub;
    if (t >= p.last) break;
    float y[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t byte = is_v ? lds[(8 * slot + k) * V_ROW + v_place(t)] : ((k < 4 ? direct[i].x : direct[i].y) >> (8 * (k & 3))) & 0xFFu;
      y[k] = block < 0 ? 0.0f : (static_cast<float>(byte) - 128.0f) * scale;
    }
    store8_f32<KIND>(dst, (p.row + (t - p.first)) * stride + static_cast<int64_t>(head) * D + 8 * slot, y);
  }
}

// grid (units, heads, 2)
template <int KIND, int D>
__global__ void __launch_bounds__(THREADS) kv_read_kernel(ReadArgs a) {
  __shared__ __align__(16) uint8_t lds[D * V_ROW];
  if (blockIdx.z == 0) read_piece<KIND, D, false>(a, lds);
  else read_piece<KIND, D, true>(a, lds);
}

// The cheaper of the two ways of cutting a batch into units (see Piece): `per_seq` blocks for every sequence where all
// are short, else 32-token steps over the whole batch.  0 per sequence means the second.
struct Units {
  int64_t units;
  int per_seq;
};
Units units_of(int64_t tokens, int64_t batch, int64_t longest) {
  const int64_t per_seq = longest > 0 ? (longest + 30) / 32 + 1 : 0;   // n tokens, at worst from place 31 of a block on
  const int64_t even = longest == 1 ? batch : per_seq * batch, steps = tokens / 32 + 2 * batch;
  if (longest > 0 && even <= steps) return {even, static_cast<int>(longest == 1 ? 1 : per_seq)};
  return {steps, 0};
}

bool cache_ok(const void* k, const void* v, const float* ks, const float* vs, const int32_t* table, int64_t table_stride,
              const int32_t* q_start, const int32_t* kv_lens, int64_t pages, int64_t page_size, int64_t kv_heads,
              int64_t head_dim) {
  return k && v && ks && vs && table && q_start && kv_lens && table_stride > 0 && pages > 0 && pages <= 0x7FFFFFFF &&
         page_size >= KV_BLOCK && page_size <= (1 << 20) && (page_size & (page_size - 1)) == 0 && kv_heads > 0 &&
         kv_heads <= 65535 && (head_dim == 64 || head_dim == 128 || head_dim == 256) &&
         ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
}

KvCacheQ8 cache_of(void* k, void* v, float* ks, float* vs, const int32_t* table, int64_t table_stride, int64_t pages,
                   int64_t page_size, int64_t kv_heads) {
  return {static_cast<uint8_t*>(k), static_cast<uint8_t*>(v), ks, vs, table, table_stride, pages, static_cast<int>(kv_heads),
          63 - __builtin_clzll(static_cast<unsigned long long>(page_size))};
}

constexpr int64_t MAX_UNITS = 8388607;   // a grid holds fewer than 2^32 threads a dimension
constexpr int BAD = static_cast<int>(hipErrorInvalidValue);

template <int KIND>
int launch_append(const AppendArgs& a, int dim, dim3 grid, hipStream_t stream) {
  switch (dim) {
    case 64: hipLaunchKernelGGL((kv_append_kernel<KIND, 64>), grid, dim3(THREADS), 0, stream, a); break;
    case 128: hipLaunchKernelGGL((kv_append_kernel<KIND, 128>), grid, dim3(THREADS), 0, stream, a); break;
    default: hipLaunchKernelGGL((kv_append_kernel<KIND, 256>), grid, dim3(THREADS), 0, stream, a); break;
  }
  return static_cast<int>(hipGetLastError());
}

template <int KIND>
int launch_read(const ReadArgs& a, int dim, dim3 grid, hipStream_t stream) {
  switch (dim) {
    case 64: hipLaunchKernelGGL((kv_read_kernel<KIND, 64>), grid, dim3(THREADS), 0, stream, a); break;
    case 128: hipLaunchKernelGGL((kv_read_kernel<KIND, 128>), grid, dim3(THREADS), 0, stream, a); break;
    default: hipLaunchKernelGGL((kv_read_kernel<KIND, 256>), grid, dim3(THREADS), 0, stream, a); break;
  }
  return static_cast<int>(hipGetLastError());
}

}  // namespace

extern "C" int hipengine_gfx950_kv_append_q8(const void* k, const void* v, int32_t in_kind, int64_t k_stride,
                                             int64_t v_stride, const float* k_weight, const int64_t* positions,
                                             const float* inv_freq, int64_t rotary_dim, int32_t interleaved, float eps,
                                             float rope_scale, uint8_t* k_cache, uint8_t* v_cache, float* k_scale,
                                             float* v_scale, const int32_t* page_table, int64_t table_stride,
                                             const int32_t* q_start, const int32_t* kv_lens, int64_t tokens, int64_t batch,
                                             int64_t max_q_len, int64_t pages, int64_t page_size, int64_t kv_heads,
                                             int64_t head_dim, hipStream_t stream) {
  if (!cache_ok(k_cache, v_cache, k_scale, v_scale, page_table, table_stride, q_start, kv_lens, pages, page_size, kv_heads,
                head_dim))
    return BAD;
  if (!k || !v || in_kind < KIND_F32 || in_kind > KIND_F16 || tokens <= 0 || tokens > 0x7FFFFFFF || batch <= 0 ||
      batch > 65535 || max_q_len <= 0 || !(eps >= 0.0f))
    return BAD;
  if (inv_freq ? (rotary_dim < 16 || rotary_dim > head_dim || rotary_dim % 16 != 0) : rotary_dim != 0) return BAD;
  const int64_t width = kv_heads * head_dim;
  if (k_stride == 0) k_stride = width;
  if (v_stride == 0) v_stride = width;
  if (k_stride < width || v_stride < width) return BAD;
  const Units u = units_of(tokens, batch, max_q_len < tokens ? max_q_len : tokens);
  if (u.units > MAX_UNITS) return BAD;
  const AppendArgs a{cache_of(k_cache, v_cache, k_scale, v_scale, page_table, table_stride, pages, page_size, kv_heads),
                     k, v, k_stride, v_stride, k_weight, positions, inv_freq, q_start, kv_lens, tokens,
                     static_cast<int>(batch), u.per_seq, static_cast<int>(rotary_dim), interleaved, eps, rope_scale};
  const dim3 grid(static_cast<unsigned>(u.units), static_cast<unsigned>(kv_heads), 2);
  const int dim = static_cast<int>(head_dim);
  switch (in_kind) {
    case KIND_F32: return launch_append<KIND_F32>(a, dim, grid, stream);
    case KIND_BF16: return launch_append<KIND_BF16>(a, dim, grid, stream);
    default: return launch_append<KIND_F16>(a, dim, grid, stream);
  }
}

extern "C" int hipengine_gfx950_kv_read_q8(const uint8_t* k_cache, const uint8_t* v_cache, const float* k_scale,
                                           const float* v_scale, const int32_t* page_table, int64_t table_stride,
                                           const int32_t* row_start, const int32_t* kv_lens, void* k_out, void* v_out,
                                           int32_t out_kind, int64_t k_out_stride, int64_t v_out_stride, int64_t tokens,
                                           int64_t batch, int64_t pages, int64_t page_size, int64_t kv_heads,
                                           int64_t head_dim, hipStream_t stream) {
  if (!cache_ok(k_cache, v_cache, k_scale, v_scale, page_table, table_stride, row_start, kv_lens, pages, page_size, kv_heads,
                head_dim))
    return BAD;
  if ((!k_out && !v_out) || out_kind < KIND_F32 || out_kind > KIND_F16 || tokens <= 0 || tokens > 0x7FFFFFFF || batch <= 0 ||
      batch > 65535)
    return BAD;
  const int64_t width = kv_heads * head_dim;
  if (k_out_stride == 0) k_out_stride = width;
  if (v_out_stride == 0) v_out_stride = width;
  if (k_out_stride < width || v_out_stride < width) return BAD;
  const Units u = units_of(tokens, batch, 0);
  if (u.units > MAX_UNITS) return BAD;
  const ReadArgs a{cache_of(const_cast<uint8_t*>(k_cache), const_cast<uint8_t*>(v_cache), const_cast<float*>(k_scale),
                            const_cast<float*>(v_scale), page_table, table_stride, pages, page_size, kv_heads),
                   k_out, v_out, k_out_stride, v_out_stride, row_start, kv_lens, tokens, static_cast<int>(batch), u.per_seq};
  const dim3 grid(static_cast<unsigned>(u.units), static_cast<unsigned>(kv_heads), 2);
  const int dim = static_cast<int>(head_dim);
  switch (out_kind) {
    case KIND_F32: return launch_read<KIND_F32>(a, dim, grid, stream);
    case KIND_BF16: return launch_read<KIND_BF16>(a, dim, grid, stream);
    default: return launch_read<KIND_F16>(a, dim, grid, stream);
  }
}

int hipengine_gfx950::kv_cache_load() {
  hipFuncAttributes attr;
  return static_cast<int>(hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(kv_append_kernel<KIND_BF16, 128>)));
}
