// RMS norm of every query and key head and the position rotation, in one pass over the activations.
//
//   y = x / sqrt(mean(x^2) + eps) * w          (per head; skipped where the weight is null)
//   (a, b) -> s (a cos t - b sin t, b cos t + a sin t),  t = position * inv_freq[i]
//   over the first rotary_dim values of a head, pairs (i, i + rotary_dim / 2) or (2i, 2i + 1); the rest stays
//
// Statistics and rotation are in float32 and the angle in float64; the result is rounded once, on its way out.
// A launch reads and writes every value once, so HBM (or, for a few tokens, the launch) is what bounds it: 8191 tokens of
// 18 heads of 256 in bf16, 151 MB, take 31 to 36 us, a copy of them 32; one token 3.4 us.

#include "attn_common.hpp"

#include "gguf_init.hpp"

#include "../../include/hipengine_gfx950.h"

namespace {

using namespace hipengine_gfx950;

constexpr int64_t MAX_TOKENS = 4194303;

struct QkArgs {
  const void* q;
  const void* k;
  void* q_out;
  void* k_out;
  const float* q_weight;
  const float* k_weight;
  const int64_t* positions;
  const float* inv_freq;
  int64_t q_stride, k_stride, q_out_stride, k_out_stride;
  int64_t tokens;
  int q_heads, kv_heads, rotary_dim, interleaved;
  float eps, rope_scale;
};

// A workgroup takes every gridDim.x-th token, D / 8 lanes per head and as many heads at once as it has lanes for; the
// angles of a token are computed once and shared by its heads.  The next piece is asked for before this one is worked on:
// with one token a workgroup 8191 tokens of 18 heads of 256 took 46 us, too little being on its way at any time.
template <int IN, int OUT, int D>
__global__ void __launch_bounds__(1024) qk_norm_rope_kernel(QkArgs a) {
  __shared__ float2 turn[2][D / 2];
  constexpr int LANES = D / 8;
  const int heads = a.q_heads + a.kv_heads, pairs = a.rotary_dim / 2;
  const int per_pass = blockDim.x / LANES, slot = threadIdx.x % LANES, first = threadIdx.x / LANES;
  auto load = [&](int64_t t, int head, float (&x)[8]) {
    if (t >= a.tokens || head >= heads) return;
    const bool is_q = head < a.q_heads;
    const int64_t at = is_q ? t * a.q_stride + static_cast<int64_t>(head) * D : t * a.k_stride + static_cast<int64_t>(head - a.q_heads) * D;
    load8_f32<IN>(is_q ? a.q : a.k, at + 8 * slot, x);
  };
  const bool turns = threadIdx.x < static_cast<unsigned>(pairs);
  const double freq = turns ? turns_of(a.inv_freq[threadIdx.x]) : 0.0;
  int64_t position = turns ? a.positions[blockIdx.x] : 0;
  float x[8];
  load(blockIdx.x, first, x);
  int buffer = 0;
  for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x, buffer ^= 1) {
    const int64_t next = t + gridDim.x;
    if (pairs > 0) {
      if (turns) {
        turn[buffer][threadIdx.x] = rotation<OUT == KIND_F32>(position, freq, a.rope_scale);
        position = next < a.tokens ? a.positions[next] : 0;
      }
      __syncthreads();        // (two buffers: who is a token ahead writes the other one, and nobody gets further ahead)
    }
    for (int base = 0; base < heads; base += per_pass) {
      const int head = base + first;
      const bool last = base + per_pass >= heads;
      float ahead[8];
      load(last ? next : t, last ? first : head + per_pass, ahead);
      if (head < heads) {
        const bool is_q = head < a.q_heads;
        const float2* from = turn[buffer] + first_pair(slot, a.rotary_dim, a.interleaved != 0);
        norm_rotate8<D>(x, slot, is_q ? a.q_weight : a.k_weight, a.eps, [&](int i) { return from[i]; }, a.rotary_dim, a.interleaved != 0);
        const int64_t at = is_q ? t * a.q_out_stride + static_cast<int64_t>(head) * D
                                : t * a.k_out_stride + static_cast<int64_t>(head - a.q_heads) * D;
        store8_f32<OUT>(is_q ? a.q_out : a.k_out, at + 8 * slot, x);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = ahead[i];
    }
  }
}

template <int IN, int OUT>
int launch_dim(const QkArgs& a, int64_t tokens, int dim, hipStream_t stream) {
  const int lanes = dim / 8;
  // No fewer threads than pairs: each computes one angle.
  const int64_t values = static_cast<int64_t>(a.q_heads + a.kv_heads) * lanes, want = values > dim / 2 ? values : dim / 2;
  const unsigned threads = static_cast<unsigned>(want >= 1024 ? 1024 : (want + 63) / 64 * 64);
  // As many workgroups as the chip's 256 CUs run at once.
  const int64_t most = 256 * (2048 / threads);
  const dim3 grid(static_cast<unsigned>(tokens < most ? tokens : most));
  switch (dim) {
    case 64: hipLaunchKernelGGL((qk_norm_rope_kernel<IN, OUT, 64>), grid, dim3(threads), 0, stream, a); break;
    case 128: hipLaunchKernelGGL((qk_norm_rope_kernel<IN, OUT, 128>), grid, dim3(threads), 0, stream, a); break;
    default: hipLaunchKernelGGL((qk_norm_rope_kernel<IN, OUT, 256>), grid, dim3(threads), 0, stream, a); break;
  }
  return static_cast<int>(hipGetLastError());
}

template <int IN>
int launch_out(const QkArgs& a, int out_kind, int64_t tokens, int dim, hipStream_t stream) {
  switch (out_kind) {
    case KIND_F32: return launch_dim<IN, KIND_F32>(a, tokens, dim, stream);
    case KIND_BF16: return launch_dim<IN, KIND_BF16>(a, tokens, dim, stream);
    default: return launch_dim<IN, KIND_F16>(a, tokens, dim, stream);
  }
}

}  // namespace

extern "C" int hipengine_gfx950_qk_norm_rope(const void* q, const void* k, const float* q_weight, const float* k_weight,
                                             const int64_t* positions, const float* inv_freq, void* q_out, void* k_out,
                                             int32_t in_kind, int32_t out_kind, int64_t tokens, int64_t q_heads,
                                             int64_t kv_heads, int64_t head_dim, int64_t rotary_dim, int64_t q_stride,
                                             int64_t k_stride, int64_t q_out_stride, int64_t k_out_stride, float eps,
                                             float rope_scale, int32_t interleaved, hipStream_t stream) {
  const int bad = static_cast<int>(hipErrorInvalidValue);
  if (tokens <= 0 || tokens > MAX_TOKENS || q_heads < 0 || kv_heads < 0 || q_heads > 4096 || kv_heads > 4096 ||
      q_heads + kv_heads == 0 || !(head_dim == 64 || head_dim == 128 || head_dim == 256) || in_kind < KIND_F32 ||
      in_kind > KIND_F16 || out_kind < KIND_F32 || out_kind > KIND_F16 || !(eps >= 0.0f))
    return bad;
  if ((q_heads > 0 && (!q || !q_out)) || (kv_heads > 0 && (!k || !k_out))) return bad;
  if (inv_freq ? (!positions || rotary_dim < 16 || rotary_dim > head_dim || rotary_dim % 16 != 0) : rotary_dim != 0) return bad;
  const int64_t qw = q_heads * head_dim, kw = kv_heads * head_dim;
  if (q_stride == 0) q_stride = qw;
  if (k_stride == 0) k_stride = kw;
  if (q_out_stride == 0) q_out_stride = qw;
  if (k_out_stride == 0) k_out_stride = kw;
  if (q_stride < qw || q_out_stride < qw || k_stride < kw || k_out_stride < kw) return bad;
  // In place only where a value keeps its address.
  if (q_heads > 0 && q == q_out && (in_kind != out_kind || q_stride != q_out_stride)) return bad;
  if (kv_heads > 0 && k == k_out && (in_kind != out_kind || k_stride != k_out_stride)) return bad;
  const QkArgs a{q, k, q_out, k_out, q_weight, k_weight, positions, inv_freq, q_stride, k_stride, q_out_stride, k_out_stride,
                 tokens, static_cast<int>(q_heads), static_cast<int>(kv_heads), static_cast<int>(rotary_dim), interleaved, eps, rope_scale};
  const int dim = static_cast<int>(head_dim);
  switch (in_kind) {
    case KIND_F32: return launch_out<KIND_F32>(a, out_kind, tokens, dim, stream);
    case KIND_BF16: return launch_out<KIND_BF16>(a, out_kind, tokens, dim, stream);
    default: return launch_out<KIND_F16>(a, out_kind, tokens, dim, stream);
  }
}

int hipengine_gfx950::qk_norm_rope_load() {
  hipFuncAttributes attr;
  return static_cast<int>(hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(qk_norm_rope_kernel<KIND_BF16, KIND_BF16, 128>)));
}
