// What the kernels of the attention half share: vector loads of activations, the position rotation, the geometry of
// the 8-bit paged KV cache and the mapping of a ragged batch onto blocks of its tokens.
//
// KV cache. A page holds page_size tokens (a power of two, 32 or more) of every KV head; inside a (page, head) the
// tokens lie in blocks of 32, and a block has one float32 scale for K and one for V. Values are bytes 128 + q with q in
// -127..127 (excess-128 needs no sign extension on the way to fp16: byte b under 0x64 is the fp16 number 1024 + b). Both
// block layouts are the operand order of v_mfma_f32_32x32x16_f16, so that a wave's 16-byte loads are contiguous and
// nothing has to be reordered:
//   K block  [D/16][32 tokens][16 dims]   lane (token, half) reads dims 16 (2i + half) .. + 15 as one load
//   V block  [D][32 places]               token t at place (t & 3) | (t >> 3 & 3) << 2 | (t >> 2 & 1) << 4:
//                                         lane (dim, half) reads the 16 tokens that the 32x32 accumulator of
//                                         K Q^T leaves in that half of the wave, in the accumulator's register order
#pragma once

#include "gguf_common.hpp"

namespace hipengine_gfx950 {

constexpr int KV_BLOCK = 32;
constexpr float KV_SCALE_FLOOR = 5.421010862427522e-20f;   // 2^-64: what is less counts as this

struct KvCacheQ8 {
  uint8_t* k;          // [pages, heads, page_size / 32, D * 32]
  uint8_t* v;
  float* k_scale;      // [pages, heads, page_size / 32]
  float* v_scale;
  const int32_t* table;   // [batch, table_stride] page numbers
  int64_t table_stride;
  int64_t pages;
  int heads;
  int page_log2;       // log2(page_size)
};

// A block's scale as it counts; a NaN stays one.
__device__ __forceinline__ float kv_scale(float s) { return s < KV_SCALE_FLOOR ? KV_SCALE_FLOOR : s; }

__device__ __forceinline__ int v_place(int t) { return (t & 3) | ((t >> 3 & 3) << 2) | ((t >> 2 & 1) << 4); }
__device__ __forceinline__ int v_token(int p) { return (p & 3) | ((p >> 2 & 3) << 3) | ((p >> 4 & 1) << 2); }

// Number of the 32-token block `blk` (of its sequence `seq`) of KV head `head` in the cache, or -1: behind the page
// table, or on a page number outside the cache. Whatever a table holds, nothing outside the cache is addressed.
__device__ __forceinline__ int64_t kv_block_index(const KvCacheQ8& c, int seq, int64_t blk, int head) {
  const int per_page_log2 = c.page_log2 - 5;
  const int64_t slot = blk >> per_page_log2;
  if (slot >= c.table_stride) return -1;
  const int64_t page = c.table[seq * c.table_stride + slot];
  if (page < 0 || page >= c.pages) return -1;
  return ((page * c.heads + head) << per_page_log2) + (blk & ((1 << per_page_log2) - 1));
}

// Rows [first, first + count) of sequence `seq` of a ragged batch, kept inside the batch whatever q_start holds.
struct SeqRows {
  int64_t first;
  int64_t count;
};
__device__ __forceinline__ SeqRows seq_rows(const int32_t* __restrict__ q_start, int seq, int64_t tokens) {
  const int64_t a = min(max(static_cast<int64_t>(q_start[seq]), int64_t{0}), tokens);
  const int64_t b = min(max(static_cast<int64_t>(q_start[seq + 1]), a), tokens);
  return {a, b - a};
}

// ---- vector loads and stores of 8 activations (element alignment is enough) ----------------------------------

template <int KIND>
__device__ __forceinline__ void load8_f32(const void* base, int64_t idx, float (&v)[8]) {
  if constexpr (KIND == KIND_F32) {
    __builtin_memcpy(v, __builtin_assume_aligned(static_cast<const float*>(base) + idx, 4), 32);
  } else {
    uint4 u;
    __builtin_memcpy(&u, __builtin_assume_aligned(static_cast<const uint16_t*>(base) + idx, 2), 16);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (KIND == KIND_BF16) {
        v[2 * i] = bits_to_float(w[i] << 16);
        v[2 * i + 1] = bits_to_float(w[i] & 0xFFFF0000u);
      } else {
        v[2 * i] = f16_bits_to_float(w[i] & 0xFFFFu);
        v[2 * i + 1] = f16_bits_to_float(w[i] >> 16);
      }
    }
  }
}

// Two values as bf16 or fp16, rounded to nearest even, in one conversion instruction; a NaN stays one.
template <int KIND>
__device__ __forceinline__ uint32_t half_bits2(float a, float b) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  if constexpr (KIND == KIND_BF16) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), b2));
  } else {
    typedef half_t h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), h2));
  }
}

template <int KIND>
__device__ __forceinline__ void store8_f32(void* base, int64_t idx, const float (&v)[8]) {
  if constexpr (KIND == KIND_F32) {
    __builtin_memcpy(__builtin_assume_aligned(static_cast<float*>(base) + idx, 4), v, 32);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = half_bits2<KIND>(v[2 * i], v[2 * i + 1]);
    __builtin_memcpy(__builtin_assume_aligned(static_cast<uint16_t*>(base) + idx, 2), w, 16);
  }
}

// ---- position rotation ---------------------------------------------------------------------------------------

// cos and sin of position * inv_freq, times `scale`.  The product and its reduction to a fraction of a turn are in 64
// bits: at position 10^6 a 32-bit product is off by a tenth of a radian.  For what is rounded to 16 or 8 bits behind it the
// fraction goes in float32 (off by up to 2^-26 turns, 9.4e-8) to the sine and cosine instructions, which take turns and are
// good to 1.25e-7 (measured over 2^22 fractions; sincospif is good to 5.1e-8 and takes 40 instructions more).  For float32
// outputs (EXACT), whose half step is 6e-8, both are summed in 64 bits and rounded once: Taylor's series within an eighth of a
// turn of the nearest quarter, good to 1e-11 (sincospi makes a launch of 8191 tokens 72 to 84 us, this one 58 to 60).
__device__ __forceinline__ double turns_of(float inv_freq) { return static_cast<double>(inv_freq) * 0.15915494309189535; }
template <bool EXACT = false>
__device__ __forceinline__ float2 rotation(int64_t position, double turns, float scale) {
  const double whole = static_cast<double>(position) * turns, part = whole - rint(whole);   // -0.5 .. 0.5
  if constexpr (EXACT) {
    const double quarter = rint(4.0 * part), x = (part - 0.25 * quarter) * 6.283185307179586, z = x * x;
    const double s = x + x * z * (-1.0 / 6 + z * (1.0 / 120 + z * (-1.0 / 5040 + z * (1.0 / 362880 + z * (-1.0 / 39916800)))));
    const double c = 1.0 + z * (-0.5 + z * (1.0 / 24 + z * (-1.0 / 720 + z * (1.0 / 40320 + z * (-1.0 / 3628800 + z * (1.0 / 479001600))))));
    const int n = static_cast<int>(quarter);       // -2 .. 2
    const double cosine = n & 1 ? s : c, sine = n & 1 ? c : s;
    return make_float2(static_cast<float>(((n + 1) & 2 ? -cosine : cosine) * scale), static_cast<float>((n & 2 ? -sine : sine) * scale));
  }
  const float turn = static_cast<float>(part);
  return make_float2(__builtin_amdgcn_cosf(turn) * scale, __builtin_amdgcn_sinf(turn) * scale);
}

// Sum over an aligned group of 8, 16 or 32 lanes, in all of them; no LDS.
template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
  v += dpp_f<DPP_QUAD_XOR1>(v);
  v += dpp_f<DPP_QUAD_XOR2>(v);
  v += dpp_f<DPP_ROW_HALF_MIRROR>(v);
  if constexpr (LANES >= 16) v += dpp_f<0x140>(v);          // row_mirror: lane i <-> lane 15-i
  if constexpr (LANES >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(float_to_bits(v), float_to_bits(v), false, false);
    v = bits_to_float(r[0]) + bits_to_float(r[1]);          // one of the two is the lane's own, the other its partner's
  }
  return v;
}

// The first of the pairs that the head dims 8 * slot .. + 7 belong to (8 pairs, or 4 where interleaved).
__device__ __forceinline__ int first_pair(int slot, int rotary_dim, bool interleaved) {
  const int d0 = 8 * slot, pairs = rotary_dim >> 1;
  return interleaved ? d0 >> 1 : d0 < pairs ? d0 : d0 - pairs;
}

// One head's RMS norm and rotation by the D / 8 neighbouring lanes that hold it, 8 values a lane (x: head dims 8 * slot ..).
// turn(i) gives (cos, sin) of the i-th pair from first_pair on.  rotary_dim is a multiple of 16, so a lane's 8 values lie on
// one side of every border and their partners all in one other lane.
template <int D, typename Turn>
__device__ __forceinline__ void norm_rotate8(float (&x)[8], int slot, const float* __restrict__ weight, float eps, Turn turn,
                                             int rotary_dim, bool interleaved) {
  constexpr int LANES = D / 8;
  const int d0 = 8 * slot, pairs = rotary_dim >> 1;
  if (weight) {
    float w[8], sum = 0.0f;
    load8_f32<KIND_F32>(weight, d0, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
    sum = group_sum<LANES>(sum);
    const float r = 1.0f / sqrtf(sum * (1.0f / D) + eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * r * w[i];
  }
  if (d0 >= rotary_dim) return;
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 cs = turn(i);
      const float a = x[2 * i], b = x[2 * i + 1];
      x[2 * i] = fmaf(a, cs.x, -b * cs.y);
      x[2 * i + 1] = fmaf(b, cs.x, a * cs.y);
    }
  } else {
    const bool low = d0 < pairs;
    const int other = low ? d0 + pairs : d0 - pairs, lane = (static_cast<int>(threadIdx.x) & 63 & ~(LANES - 1)) + (other >> 3);
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __shfl(x[i], lane);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 cs = turn(i);
      x[i] = fmaf(x[i], cs.x, (low ? -y[i] : y[i]) * cs.y);
    }
  }
}

}  // namespace hipengine_gfx950
