// Sampling one token of every row of float32 logits from given uniform numbers: temperature, top-k, top-p, min-p.
//
// Tokens are ordered by logit, the highest first and equal ones by index.  With w = exp((l - l_max) / temperature):
//   top-k   keeps the first k;   top-p keeps, of those, the tokens before which less than p of their total lies (the
//   shortest prefix that holds p);   min-p drops those with w < min_p (the largest w is 1).
// The token is the first one, by index, up to which the kept weights sum to more than u times their total.
//
// Sums are integers: a weight is held as w * 2^40 in 64 bits, so sums do not depend on the order in which they are added, a
// prefix and its border are exact, and the result is the same in every run.  (The argument is computed in float64, exp2
// of its fraction in float32: a weight is good to 2^-23 of itself, or 2^-40 of the largest.)  Nothing is sorted.
//
// A row is read three times by many workgroups, each on a chunk of 4096 logits (the second and third time from the
// caches): 1. its maximum; 2. the chunk's weights (with top-k: counts) in 512 bins of an eighth of an octave of w, as sums
// over the bins, from which one workgroup a row then finds the bin B that holds the border; 3. the tokens of B in a list
// (with top-k, all tokens down to B).  4. One workgroup a row finds the exact border inside the list, then the chunk that
// holds the token by the chunks' weights up to B, and the token in it.
// A list that would not fit (a row so flat that one bin holds over 16384 tokens) is replaced by the row itself, which one
// workgroup then reads once for every digit: one such row of 151936 takes 740 us, 64 of them 1010.
//
// What bounds it.  One row of 151936 with top-k 50: four launches of 4 to 8 us, each a few steps that wait for each other.
// Nothing but a temperature: one row 22 us by the clock, 64 rows 38.
// 64 rows with top-p 0.9 (39 MB): 11 + 16 + 5 + 15 + 16 us; the passes over the logits stand at what such a launch takes to
// read them (11) plus 4 us for 10^7 weights in the second, and pass 4 at its barriers.  Sums of bins through global
// atomics, and a counter beside the neighbouring rows', cost 15 us more: additions to one line wait for each other.

#include "gguf_common.hpp"

#include "gguf_init.hpp"

#include "../../include/hipengine_gfx950.h"

namespace {

using namespace hipengine_gfx950;

constexpr int CHUNK = 4096;              // logits of a workgroup in passes 1 to 3
constexpr int THREADS = 256;
constexpr int LAST = 1024;               // threads of pass 4
constexpr int BINS = 512;
constexpr int LIST = 16384;
constexpr int FEW = 128;
constexpr int NOTHING = 8 * 42;          // from this bin on a weight is less than 2^-40
constexpr int CACHED = 2048;             // tokens of a list that pass 4 keeps in LDS
constexpr int LINE = 32;
// rows * chunks^2 up to which pass 3's workgroups each find their row's borders (and read all its sums): one launch less
// (8 rows of 32003: 25.3 us against 27.2, 1 of 151936: 25.9 against 27.3, 4 of 151936: no difference, 16 of 151936: 33
// against 30, 1 of 10^6: 38 against 35).
constexpr int64_t SHARED_CUTS = 4096;
constexpr int64_t MAX_VOCAB = 1 << 22;   // 1024 chunks; 2^22 weights of 2^40 stay under 2^63
constexpr int MAX_CHUNKS = static_cast<int>(MAX_VOCAB / CHUNK);

struct Cut;

struct Args {
  const float* logits;
  int64_t stride;
  const float* uniform;
  const float* temperature;   // null: 1
  const int32_t* top_k;       // null, 0 or less: all
  const float* top_p;         // null, 1 or more: all
  const float* min_p;         // null, 0 or less: all
  int32_t* ids;
  float* logprobs;            // or null
  int vocab, chunks;
  int cap;                    // tokens that a row's list holds
  // workspace
  uint64_t* best;             // [rows][chunks] key << 32 | ~index of the chunk's first token in the order
  uint64_t* sums;             // [rows][chunks] weight of a chunk, where nothing is cut
  uint64_t* before;           // [rows][chunks][BINS] weight, or with top-k number, of a chunk's tokens in the bins before one
  Cut* cuts;                  // [rows]
  uint64_t* list;             // [rows][cap] key << 32 | ~index
  uint32_t* listed;           // [rows], a line each: the chunks' additions to one line wait for each other
};

// The order as one number, higher is earlier: the logit's bits made to order like unsigned integers, then the index
// downwards.  0 where the token cannot be chosen (-infinity, NaN).  -0 is made 0, infinity the largest number.
__device__ __forceinline__ uint32_t key_of(float l) {
  l = fminf(l + 0.0f, 3.4028234663852886e+38f);
  if (!(l >= -3.4028234663852886e+38f)) return 0;      // (fminf gave the number for a NaN: looked at by the caller)
  const uint32_t u = float_to_bits(l);
  return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ uint64_t order_of(float l, int index) {
  const uint32_t key = l != l ? 0 : key_of(l);
  return key ? (static_cast<uint64_t>(key) << 32) | static_cast<uint32_t>(~index) : 0;
}
__device__ __forceinline__ float logit_of(uint64_t order) {
  const uint32_t k = static_cast<uint32_t>(order >> 32);
  return bits_to_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ int index_of(uint64_t order) { return static_cast<int>(~static_cast<uint32_t>(order)); }

// A row's settings as they are given.  Loaded at once and first of all: which array is null is only asked afterwards (the
// uniform numbers stand in for it), since loads behind branches wait for each other, a microsecond each in a short call.
struct Given {
  float t, p, m;
  int k;
};
__device__ __forceinline__ Given given(const Args& a, int64_t row) {
  auto at = [&](const void* from) { return static_cast<const uint32_t*>(from ? from : a.uniform)[row]; };
  const uint32_t t = at(a.temperature), k = at(a.top_k), p = at(a.top_p), m = at(a.min_p);
  return {a.temperature ? bits_to_float(t) : 1.0f, a.top_p ? bits_to_float(p) : 1.0f, a.min_p ? bits_to_float(m) : 0.0f,
          a.top_k ? static_cast<int>(k) : 0};
}

struct Row {
  float top;             // largest logit
  double per;            // octaves of weight per unit of logit: log2(e) / temperature
  float per8;            // bins
  bool greedy;
  int k;                 // 0: all
  double p;              // 1: all
  double octaves;        // min-p's border; infinity: none
};

__device__ __forceinline__ Row row_of(const Args& a, const Given& g, float top) {
  Row r;
  r.top = top;
  const float t = g.t;
  r.greedy = !(t > 0.0f);
  r.per = r.greedy ? 1.0 : 1.4426950408889634 / static_cast<double>(fmaxf(t, 4.70197740e-38f));   // 2^-124: per8 is finite
  r.per8 = static_cast<float>(r.per * 8.0);
  r.k = g.k > 0 && g.k < a.vocab ? g.k : 0;
  r.p = g.p < 1.0f ? fmax(static_cast<double>(g.p), 0.0) : 1.0;
  r.octaves = g.m > 0.0f ? -log2(fmin(static_cast<double>(g.m), 1.0)) : __builtin_inf();
  return r;
}
__device__ __forceinline__ bool cuts(const Row& r) { return r.k > 0 || r.p < 1.0 || r.octaves < __builtin_inf(); }

// A logit as it counts, with infinity as the largest number.  What is below MINUS (or NaN) cannot be chosen.
constexpr float MINUS = -3.4028234663852886e+38f;
__device__ __forceinline__ float finite(float l) { return fminf(l, -MINUS); }

// Octaves below the largest weight, exactly enough for weights and for min-p.
__device__ __forceinline__ double depth(const Row& r, float l) {
  return (static_cast<double>(r.top) - static_cast<double>(l)) * r.per;
}
// A bin need not be exact, only monotonous in the logit: float32.
__device__ __forceinline__ int bin_of(const Row& r, float l) {
  return static_cast<int>(fminf(fminf(r.top - l, 3e38f) * r.per8, static_cast<float>(BINS - 1)));
}
__device__ __forceinline__ uint64_t weight(double y) {   // 2^-y * 2^40, downwards
  const double n = rint(fmin(y, 100.0));
  const uint32_t e = float_to_bits(__builtin_amdgcn_exp2f(static_cast<float>(n - y)));   // 0.7 .. 1.42 (0 behind 100)
  const uint32_t m = (e & 0x7FFFFFu) | 0x800000u;
  return (static_cast<uint64_t>(m) << 18) >> min(static_cast<int>(n) + 128 - static_cast<int>(e >> 23), 63);
}

// 64-bit values of a wave joined, or summed up to each lane, by moves between registers: through LDS every step would wait
// some hundred clocks, and a short call consists of such steps. All lanes have to be active.
__device__ __forceinline__ uint64_t whole(uint32_t lo, uint32_t hi) { return (static_cast<uint64_t>(hi) << 32) | lo; }
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t moved(uint64_t v) {      // 0 where nothing comes from
  const int lo = static_cast<int>(v), hi = static_cast<int>(v >> 32);
  return whole(__builtin_amdgcn_update_dpp(0, lo, CTRL, ROWS, 0xf, false), __builtin_amdgcn_update_dpp(0, hi, CTRL, ROWS, 0xf, false));
}
template <typename F>
__device__ __forceinline__ uint64_t wave_join(uint64_t v, F f) {
  v = f(v, moved<DPP_QUAD_XOR1, 0xf>(v));
  v = f(v, moved<DPP_QUAD_XOR2, 0xf>(v));
  v = f(v, moved<DPP_ROW_HALF_MIRROR, 0xf>(v));
  v = f(v, moved<0x140, 0xf>(v));                            // row_mirror
  const uint32_t lo = static_cast<uint32_t>(v), hi = static_cast<uint32_t>(v >> 32);
  const auto l = __builtin_amdgcn_permlane16_swap(lo, lo, false, false), h = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
  v = f(whole(l[0], h[0]), whole(l[1], h[1]));
  const uint32_t lo2 = static_cast<uint32_t>(v), hi2 = static_cast<uint32_t>(v >> 32);
  const auto l2 = __builtin_amdgcn_permlane32_swap(lo2, lo2, false, false), h2 = __builtin_amdgcn_permlane32_swap(hi2, hi2, false, false);
  return f(whole(l2[0], h2[0]), whole(l2[1], h2[1]));
}
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
  return wave_join(v, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
}
__device__ __forceinline__ uint64_t wave_sum(uint64_t v) {
  return wave_join(v, [](uint64_t a, uint64_t b) { return a + b; });
}
__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {  // with the lane's own
  v += moved<0x111, 0xf>(v);                                 // row_shr 1, 2, 4, 8
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);                                 // lane 15 of rows 0 and 2 to rows 1 and 3
  return v + moved<0x143, 0xc>(v);                           // lane 31 to rows 2 and 3
}

template <int N>
__device__ __forceinline__ uint64_t block_max(uint64_t v, uint64_t* lds) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < N / 64; ++w) v = lds[w] > v ? lds[w] : v;
  return v;
}
template <int N>
__device__ __forceinline__ uint64_t block_sum(uint64_t v, uint64_t* lds) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < N / 64; ++w) v += lds[w];
  return v;
}


// A thread's 16 logits of a chunk: groups of 4 at (g * 256 + thread) * 4.  Behind the row's end: NaN.
__device__ __forceinline__ int chunk_index(int chunk, int i) {
  return chunk * CHUNK + ((i >> 2) * THREADS + static_cast<int>(threadIdx.x)) * 4 + (i & 3);
}
__device__ __forceinline__ void load_chunk(const Args& a, int64_t row, int chunk, float (&l)[16]) {
  const float* src = a.logits + row * a.stride;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int at = chunk_index(chunk, 4 * g);
    if (at + 4 <= a.vocab) {
      __builtin_memcpy(&l[4 * g], __builtin_assume_aligned(src + at, 4), 16);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) l[4 * g + j] = at + j < a.vocab ? src[at + j] : __builtin_nanf("");
    }
  }
}

// Pass 1; also clears what pass 3 adds to.
__global__ void __launch_bounds__(THREADS) sample_max_kernel(Args a) {
  __shared__ uint64_t lds[THREADS / 64];
  const int64_t row = blockIdx.y;
  const int chunk = blockIdx.x;
  float l[16];
  load_chunk(a, row, chunk, l);
  uint64_t v = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint64_t o = order_of(l[i], chunk_index(chunk, i));
    v = o > v ? o : v;
  }
  v = block_max<THREADS>(v, lds);
  if (threadIdx.x == 0) a.best[row * a.chunks + chunk] = v;
  if (chunk == 0 && threadIdx.x == 0) a.listed[row * LINE] = 0;
}

// Pass 2.
__global__ void __launch_bounds__(THREADS) sample_histogram_kernel(Args a) {
  __shared__ uint64_t lds[THREADS / 64];
  __shared__ unsigned long long weights[BINS];
  const int64_t row = blockIdx.y;
  const int chunk = blockIdx.x;
  float l[16];
  const Given g = given(a, row);
  load_chunk(a, row, chunk, l);
  uint64_t best = 0;
  for (int c = threadIdx.x; c < a.chunks; c += THREADS) {
    const uint64_t o = a.best[row * a.chunks + c];
    best = o > best ? o : best;
  }
  best = block_max<THREADS>(best, lds);
  const Row r = row_of(a, g, logit_of(best));
  if (best == 0 || r.greedy || !cuts(r)) return;
  // With top-k the border is found by counting, else by weight: one addition a token.
  const bool count = r.k > 0;
  for (int i = threadIdx.x; i < BINS; i += THREADS) weights[i] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if (!(l[i] >= MINUS)) continue;
    const float x = finite(l[i]);
    const int bin = bin_of(r, x);
    if (count) {
      atomicAdd(&weights[bin], 1ull);
    } else if (bin < NOTHING) {
      atomicAdd(&weights[bin], static_cast<unsigned long long>(weight(depth(r, x))));
    }
  }
  __syncthreads();
  // Sums over the bins, as the next kernel needs them for the row (it adds the chunks') and pass 4 for the chunk.
  const int b = 2 * threadIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t first = weights[b], own = first + weights[b + 1];
  uint64_t run = wave_scan(own);
  if (lane == 63) lds[wave] = run;
  __syncthreads();
  run -= own;
  for (int w = 0; w < wave; ++w) run += lds[w];
  const uint64_t before[2] = {run, run + first};
  __builtin_memcpy(__builtin_assume_aligned(a.before + (row * a.chunks + chunk) * BINS + b, 8), before, 16);
}

enum Mode : int { ALL, BOUND, PREFIX, FULL };

// What is known of a row before pass 3.
struct Cut {
  Row row;
  uint64_t best;        // the first token in the order; 0: there is none
  uint64_t above;       // weight of the bins before B (BOUND)
  uint64_t need;        // top-p: a token stays if less than this lies before it (BOUND)
  int mode;
  int bin, last;        // B; min-p's border may lie in either of two bins
  int reached;          // whether `need` is reached within B (else min-p's border is there)
};

__device__ __forceinline__ uint64_t border(double p, uint64_t total) {   // smallest whole number >= p * total
  return static_cast<uint64_t>(ceil(p * static_cast<double>(total)));
}

// Between passes 2 and 3 a workgroup of N threads adds up the row's chunks, two neighbouring bins a thread; then one wave
// looks for the borders, 8 bins a lane.
template <int N>
struct CutLds {
  static constexpr int PARTS = N / (BINS / 2);
  uint64_t before[PARTS][BINS];
  Cut cut;
};
template <int N>
__device__ __forceinline__ void find_cut(const Args& a, int64_t row, CutLds<N>& lds) {
  constexpr int PARTS = CutLds<N>::PARTS;
  auto& before = lds.before;
  const int lane = threadIdx.x & 63;
  const Given g = given(a, row);
  uint64_t best = 0, sum[2] = {0, 0};
  const int pair = 2 * (threadIdx.x % (BINS / 2)), part = __builtin_amdgcn_readfirstlane(threadIdx.x / (BINS / 2));
  if (g.t > 0.0f && (g.k > 0 || g.p < 1.0f || g.m > 0.0f)) {   // (what no histogram was written for is not used)
    // Loads on their way, the last few too: not a loop over the rest. 20 make two rounds of the 38 chunks of 151936 logits, 16
    // made three (one row: 7.3 us for the pass against 7.8).
    constexpr int AHEAD = 20;
    for (int c0 = part; c0 < a.chunks; c0 += AHEAD * PARTS) {
      uint64_t v[AHEAD][2] = {};
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (c0 + i * PARTS < a.chunks)
          __builtin_memcpy(v[i], __builtin_assume_aligned(a.before + (row * a.chunks + c0 + i * PARTS) * BINS + pair, 8), 16);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        sum[0] += v[i][0];
        sum[1] += v[i][1];
      }
    }
  }
  for (int c = lane; c < a.chunks; c += 64) {
    const uint64_t o = a.best[row * a.chunks + c];
    best = o > best ? o : best;
  }
  best = wave_max(best);
  const Row r = row_of(a, g, logit_of(best));
  Cut cut{r, best, 0, 0, ALL, BINS, BINS, 0};
  if (best != 0 && !r.greedy && cuts(r)) {
    before[part][pair] = sum[0];
    before[part][pair + 1] = sum[1];
    __syncthreads();
    if constexpr (PARTS > 1) {
      if (threadIdx.x < BINS) {
        uint64_t all = 0;
#pragma unroll
        for (int p = 0; p < PARTS; ++p) all += before[p][threadIdx.x];
        before[0][threadIdx.x] = all;
      }
      __syncthreads();
    }
    if (threadIdx.x >= 64) return;
    // (Nothing in the last bin counts: it has no weight, and top-k is taken to end in it where it is not reached before.)
    auto up_to = [&](int bin) { return before[0][min(bin + 1, BINS - 1)]; };
    const uint64_t total = before[0][BINS - 1];
    const uint64_t need = r.p < 1.0 ? border(r.p, total) : ~uint64_t{0};
    // First bin up to which k tokens, or `need`, are reached.
    const uint64_t goal = r.k > 0 ? static_cast<uint64_t>(r.k) : need;
    int reached = BINS - 1;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (up_to(lane * 8 + i) >= goal) reached = min(reached, lane * 8 + i);
    const unsigned long long some = __ballot(reached < BINS - 1);      // (sums only grow: the first lane has it)
    reached = some ? __builtin_amdgcn_readlane(reached, __builtin_ctzll(some)) : BINS - 1;
    cut.need = need;
    if (r.k > 0) {
      // A border in the last bin cuts nothing (its weights are 0); what top-p and min-p then cut is not known by weight.
      cut.bin = cut.last = reached;
      if (reached < BINS - 1) cut.mode = up_to(reached) <= static_cast<uint64_t>(a.cap) ? PREFIX : FULL;
      else cut.mode = r.p < 1.0 || r.octaves < __builtin_inf() ? FULL : ALL;
    } else {
      // Bins below min_bin lie on this side of min-p's border whatever float32 makes of it, those above max_bin behind it.
      const int min_bin = static_cast<int>(fmin(r.octaves * 8.0 * (1.0 - 1e-6), BINS - 1.0));
      const int max_bin = static_cast<int>(fmin(r.octaves * 8.0 * (1.0 + 1e-6), BINS - 1.0));
      cut.bin = min(reached, min_bin);
      cut.last = reached < min_bin ? reached : min(reached, max_bin);
      cut.reached = reached <= cut.last;
      cut.above = before[0][cut.bin];
      cut.mode = cut.bin < BINS - 1 ? BOUND : ALL;
    }
    if (cut.mode == ALL) cut.bin = cut.last = BINS;
  }
  if (threadIdx.x == 0) lds.cut = cut;
}

__global__ void __launch_bounds__(LAST) sample_cut_kernel(Args a) {
  __shared__ CutLds<LAST> cut_lds;
  find_cut(a, blockIdx.x, cut_lds);
  if (threadIdx.x == 0) a.cuts[blockIdx.x] = cut_lds.cut;
}

// Pass 3; with CUT every workgroup finds the borders for itself.
template <bool CUT>
__global__ void __launch_bounds__(THREADS) sample_collect_kernel(Args a) {
  __shared__ uint64_t lds[THREADS / 64];
  __shared__ CutLds<CUT ? THREADS : BINS / 2> cut_lds;
  __shared__ uint32_t here, base;
  const int64_t row = blockIdx.y;
  const int chunk = blockIdx.x;
  float l[16];
  load_chunk(a, row, chunk, l);
  if constexpr (CUT) {
    find_cut(a, row, cut_lds);
    __syncthreads();
    if (chunk == 0 && threadIdx.x == 0) a.cuts[row] = cut_lds.cut;
  }
  const Cut cut = CUT ? cut_lds.cut : a.cuts[row];
  const Row r = cut.row;
  if (cut.best == 0 || r.greedy || cut.mode == FULL) return;
  if (threadIdx.x == 0) here = 0;
  __syncthreads();
  // A logit that lies more than half a bin behind B's end is passed over by one comparison.
  const float floor = cut.last < BINS - 1 ? static_cast<float>(static_cast<double>(r.top) - (cut.last + 1.5) * 0.125 / r.per)
                                         : MINUS;
  uint64_t sum = 0;
  uint32_t slot[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    slot[i] = ~0u;
    if (!(l[i] >= fmaxf(floor, MINUS))) continue;
    const float x = finite(l[i]);
    const int bin = bin_of(r, x);
    if (cut.mode == ALL) {
      if (bin < NOTHING) sum += weight(depth(r, x));
    } else if ((cut.mode == PREFIX || bin >= cut.bin) && bin <= cut.last) {
      slot[i] = atomicAdd(&here, 1u);
    }
  }
  if (cut.mode == ALL) {
    sum = block_sum<THREADS>(sum, lds);
    if (threadIdx.x == 0) a.sums[row * a.chunks + chunk] = sum;
  }
  __syncthreads();
  if (here == 0) return;
  if (threadIdx.x == 0) base = atomicAdd(&a.listed[row * LINE], here);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (slot[i] != ~0u && base + slot[i] < static_cast<uint32_t>(a.cap)) a.list[row * a.cap + base + slot[i]] = order_of(l[i], chunk_index(chunk, i));
}

// ---- pass 4 ------------------------------------------------------------------------------------------------------

struct Digits {
  unsigned long long weights[256];
  uint32_t counts[256];
  uint64_t before;       // found: weight (or count) of the buckets before the one
  uint64_t in;           // found: tokens in it
  unsigned long long some, all;
  int digit;
};

// The tokens that pass 4 looks through: a list (with its weights, where it is kept in LDS), or the whole row.
struct Tokens {
  const Row& r;
  const uint64_t* list;
  const uint64_t* weights;
  const float* logits;
  int n;
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    for (int i = threadIdx.x; i < n; i += LAST) {
      const uint64_t o = list ? list[i] : order_of(logits[i], i);
      if (o) f(o, [&] { return weights ? weights[i] : weight(depth(r, logit_of(o))); });
    }
  }
};

// Walks down a number digit by digit (8 bits) to the token at which a running sum first exceeds `before` (the sum up to and
// including it is more than that).  value(order): the number, larger is earlier, no two tokens' the same.  add(order, weight):
// what the token adds (0: not among them).  Counts or weights: any whole numbers.  Returns the number.  Leading bits that all
// tokens have in common are passed over, and it ends early where one token is left.
template <typename V, typename A>
__device__ __forceinline__ uint64_t walk(const Tokens& t, Digits& d, uint64_t before, V value, A add) {
  uint64_t some = 0, all = ~uint64_t{0};
  t.each([&](uint64_t o, auto) {
    const uint64_t v = value(o);
    some |= v;
    all &= v;
  });
  some = wave_join(some, [](uint64_t x, uint64_t y) { return x | y; });
  all = wave_join(all, [](uint64_t x, uint64_t y) { return x & y; });
  if (threadIdx.x == 0) { d.some = 0; d.all = ~0ull; }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    atomicOr(&d.some, static_cast<unsigned long long>(some));
    atomicAnd(&d.all, static_cast<unsigned long long>(all));
  }
  __syncthreads();
  some = d.some;
  const uint64_t differ = some & ~d.all;
  int high = differ ? 64 - __builtin_clzll(differ) : 0;       // bits still to be found
  uint64_t prefix = high < 64 ? some >> high : 0;
  while (high > 0) {
    const int low = high > 8 ? high - 8 : 0;
    const uint64_t mask = (1u << (high - low)) - 1;
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += LAST) { d.weights[i] = 0; d.counts[i] = 0; }
    __syncthreads();
    t.each([&](uint64_t o, auto w_of) {
      const uint64_t v = value(o);
      if (high < 64 && (v >> high) != prefix) return;
      const uint64_t w = add(o, w_of);
      if (w == 0) return;
      const int digit = static_cast<int>((v >> low) & mask);
      atomicAdd(&d.weights[digit], static_cast<unsigned long long>(w));
      atomicAdd(&d.counts[digit], 1u);
    });
    __syncthreads();
    if (threadIdx.x < 64) {      // lane 0 holds the largest digits
      const int lane = threadIdx.x;
      uint64_t w[4], s = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) { w[i] = d.weights[255 - 4 * lane - i]; s += w[i]; }
      uint64_t run = wave_scan(s);
      const unsigned long long over = __ballot(run > before);
      const int owner = over ? __builtin_ctzll(over) : 63;
      if (lane == owner) {
        run -= s;
        int i = 0;
        while (i < 3 && !(run + w[i] > before)) run += w[i++];
        d.digit = 255 - 4 * lane - i;
        d.before = run;
        d.in = d.counts[d.digit];
      }
    }
    __syncthreads();
    prefix = (prefix << (high - low)) | static_cast<uint64_t>(d.digit);
    before -= d.before;
    high = low;
    if (d.in == 1 && high > 0) {     // the one token's remaining digits
      __syncthreads();
      t.each([&](uint64_t o, auto w_of) {
        const uint64_t v = value(o);
        if ((v >> high) == prefix && add(o, w_of)) d.before = v;
      });
      __syncthreads();
      prefix = d.before;
      high = 0;
    }
  }
  __syncthreads();                   // `d` may be used again
  return prefix;
}

__device__ __forceinline__ void answer(const Args& a, int64_t row, const Row& r, int id, float l, uint64_t total) {
  a.ids[row] = id;
  if (!a.logprobs) return;
  a.logprobs[row] = static_cast<float>(-((static_cast<double>(r.top) - static_cast<double>(l)) * r.per +
                                         log2(static_cast<double>(total)) - 40.0) * 0.6931471805599453);
}

__device__ __forceinline__ uint64_t target_of(float u, uint64_t total) {
  const uint64_t target = static_cast<uint64_t>((u > 0.0f ? fmin(static_cast<double>(u), 1.0) : 0.0) * static_cast<double>(total));
  return target < total ? target : total - 1;      // the largest weight is 2^40, so there is a total
}

// Top-k has left a list of at most 128 tokens: each is compared with every other one, 8 threads a token.
struct Few {
  uint64_t order[FEW], weight[FEW];
  unsigned long long before[FEW], by_index[FEW];    // weight of the tokens earlier in the order; of the kept ones of lower index
  uint32_t rank[FEW];
  unsigned long long total, kept;
};

__device__ __forceinline__ void choose_of_few(const Args& a, int64_t row, const Row& r, uint64_t order, int n, float u, Few& f) {
  const int i = threadIdx.x % FEW, part = threadIdx.x / FEW;
  const bool mine = i < n;
  uint64_t w = 0;
  double y = 0.0;
  if (!mine) order = 0;
  if (mine) {
    y = depth(r, logit_of(order));
    w = weight(y);
  }
  if (part == 0) {
    f.order[i] = order;
    f.weight[i] = w;
    f.before[i] = f.by_index[i] = 0;
    f.rank[i] = 0;
    if (i == 0) f.total = f.kept = 0;
  }
  __syncthreads();
  uint32_t rank = 0;
  uint64_t before = 0;
  for (int j = part; j < n; j += LAST / FEW) {
    const bool earlier = f.order[j] > order;
    rank += earlier ? 1 : 0;
    before += earlier ? f.weight[j] : 0;
  }
  if (mine && rank) {
    atomicAdd(&f.rank[i], rank);
    atomicAdd(&f.before[i], static_cast<unsigned long long>(before));
  }
  __syncthreads();
  bool keep = mine && f.rank[i] < static_cast<uint32_t>(r.k);
  if (part == 0) {
    const uint64_t sum = wave_sum(keep ? w : 0);
    if ((threadIdx.x & 63) == 0) atomicAdd(&f.total, static_cast<unsigned long long>(sum));
  }
  __syncthreads();
  const uint64_t need = r.p < 1.0 ? border(r.p, f.total) : ~uint64_t{0};
  keep = keep && (f.before[i] < need || f.rank[i] == 0) && y <= r.octaves;
  __syncthreads();
  if (part == 0) {
    if (!keep) f.weight[i] = 0;
    const uint64_t sum = wave_sum(keep ? w : 0);
    if ((threadIdx.x & 63) == 0) atomicAdd(&f.kept, static_cast<unsigned long long>(sum));
  }
  __syncthreads();
  uint64_t lower = 0;
  for (int j = part; j < n; j += LAST / FEW)
    if (static_cast<uint32_t>(f.order[j]) > static_cast<uint32_t>(order)) lower += f.weight[j];   // (complement of the index)
  if (mine && lower) atomicAdd(&f.by_index[i], static_cast<unsigned long long>(lower));
  __syncthreads();
  const uint64_t target = target_of(u, f.kept);
  if (part == 0 && keep && f.by_index[i] <= target && target < f.by_index[i] + w)
    answer(a, row, r, index_of(order), logit_of(order), f.kept);
}

__global__ void __launch_bounds__(LAST) sample_choose_kernel(Args a) {
  __shared__ uint64_t lds[LAST / 64];
  __shared__ Digits digits;
  __shared__ unsigned long long chunk_sum[MAX_CHUNKS];
  __shared__ int chosen_chunk;
  __shared__ Few few;
  __shared__ uint64_t kept_order[CACHED], kept_weight[CACHED];
  __shared__ uint64_t rest;
  const int64_t row = blockIdx.x;
  Cut cut = a.cuts[row];
  const uint32_t listed = a.listed[row * LINE];
  const float u = a.uniform[row];
  const uint64_t order = a.list[row * a.cap + min(static_cast<int>(threadIdx.x) % FEW, a.cap - 1)];   // (for choose_of_few)
  const uint64_t best = cut.best;
  const Row r = cut.row;
  if (best == 0 || r.greedy) {
    if (threadIdx.x == 0) {
      a.ids[row] = best ? index_of(best) : -1;
      if (a.logprobs) a.logprobs[row] = best ? 0.0f : -__builtin_inff();
    }
    return;
  }
  if (listed > static_cast<uint32_t>(a.cap)) cut.mode = FULL;   // (BOUND: the bin did not fit the list)
  const float* logits = a.logits + row * a.stride;
  if (cut.mode == PREFIX && listed <= FEW) {
    choose_of_few(a, row, r, order, static_cast<int>(listed), u, few);
    return;
  }
  Tokens t{r, cut.mode == BOUND || cut.mode == PREFIX ? a.list + row * a.cap : nullptr, nullptr, logits,
           cut.mode == FULL ? a.vocab : cut.mode == ALL ? 0 : static_cast<int>(listed)};
  const bool by_chunk = cut.mode == ALL || cut.mode == BOUND;
  if (by_chunk) {
    for (int c = threadIdx.x; c < a.chunks; c += LAST)
      chunk_sum[c] = cut.mode == ALL ? a.sums[row * a.chunks + c] : a.before[(row * a.chunks + c) * BINS + cut.bin];
  }
  if (t.list && t.n <= CACHED) {
    for (int i = threadIdx.x; i < t.n; i += LAST) {
      const uint64_t o = t.list[i];
      kept_order[i] = o;
      kept_weight[i] = weight(depth(r, logit_of(o)));
    }
    t.list = kept_order;
    t.weights = kept_weight;
  }
  __syncthreads();
  const uint64_t above = cut.mode == BOUND ? cut.above : 0;
  auto self = [](uint64_t o) { return o; };

  // Borders: a token stays if its order is `least` or more and its weight min-p's or more.
  uint64_t least = 0;
  if (cut.mode != ALL) {
    uint64_t total = 0;      // of the tokens that top-k leaves
    if (cut.mode != BOUND) {
      if (r.k > 0) {
        uint64_t there = 0;
        t.each([&](uint64_t, auto) { ++there; });
        there = block_sum<LAST>(there, lds);
        if (there > static_cast<uint64_t>(r.k))
          least = walk(t, digits, static_cast<uint64_t>(r.k) - 1, self, [](uint64_t, auto) { return uint64_t{1}; });
      }
      t.each([&](uint64_t o, auto w_of) { if (o >= least) total += w_of(); });
      total = block_sum<LAST>(total, lds);
    }
    if (r.p < 1.0) {
      const uint64_t need = cut.mode == BOUND ? cut.need : border(r.p, total);
      if (need == 0) {
        least = best;            // p = 0: the first token
      } else {
        // The token up to which the sum reaches `need`, that is exceeds need - 1: there is one, unless min-p's border
        // comes first.
        if (cut.mode != BOUND || cut.reached) {
          const uint64_t from = least;
          least = walk(t, digits, need - above - 1, self,
                       [&](uint64_t o, auto w_of) { return o >= from ? w_of() : uint64_t{0}; });
        }
      }
    }
  }
  const bool by_depth = r.octaves < __builtin_inf();
  auto stays = [&](uint64_t o) { return o >= least && (!by_depth || depth(r, logit_of(o)) <= r.octaves); };
  auto weight_left = [&](uint64_t o, auto w_of) { return stays(o) ? w_of() : uint64_t{0}; };

  uint64_t total = 0;
  if (by_chunk) {
    t.each([&](uint64_t o, auto w_of) {
      const uint64_t w = weight_left(o, w_of);
      if (w) atomicAdd(&chunk_sum[index_of(o) / CHUNK], static_cast<unsigned long long>(w));
    });
    __syncthreads();
    for (int c = threadIdx.x; c < a.chunks; c += LAST) total += chunk_sum[c];
  } else {
    t.each([&](uint64_t o, auto w_of) { total += weight_left(o, w_of); });
  }
  total = block_sum<LAST>(total, lds);
  const uint64_t target = target_of(u, total);
  if (by_chunk) {
    if (threadIdx.x < 64) {
      const int lane = threadIdx.x;
      uint64_t passed = 0;
      for (int c0 = 0; c0 < a.chunks; c0 += 64) {
        const uint64_t s = c0 + lane < a.chunks ? chunk_sum[c0 + lane] : 0;
        const uint64_t run = wave_scan(s);
        const unsigned long long over = __ballot(passed + run > target);
        if (over) {
          const int owner = __builtin_ctzll(over);
          if (lane == owner) { chosen_chunk = c0 + lane; rest = target - (passed + run - s); }
          break;
        }
        passed += __shfl(static_cast<unsigned long long>(run), 63);
      }
    }
    __syncthreads();
    // The chunk's tokens, 4 neighbours a thread, in index order.
    const int first = chosen_chunk * CHUNK + static_cast<int>(threadIdx.x) * 4;
    uint64_t w[4], s = 0;
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = first + i < a.vocab ? logits[first + i] : __builtin_nanf("");
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = 0;
      const uint64_t o = order_of(x[i], first + i);
      if (o) {
        const float l = logit_of(o);
        const int bin = bin_of(r, l);
        if (bin < cut.bin || (bin <= cut.last && stays(o))) w[i] = weight(depth(r, l));
      }
      s += w[i];
    }
    uint64_t run = wave_scan(s);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();
    if (lane == 63) lds[wave] = run;
    __syncthreads();
    for (int v = 0; v < wave; ++v) run += lds[v];
    if (run > rest && run - s <= rest) {            // one thread
      uint64_t at = run - s;
      int i = 0;
      while (i < 3 && !(at + w[i] > rest)) at += w[i++];
      answer(a, row, r, first + i, finite(x[i]), total);
    }
  } else {
    // Smaller indices first: the complement of the index orders them so, in 24 bits.
    const uint64_t v = walk(t, digits, target, [](uint64_t o) { return o & 0xFFFFFFu; }, weight_left);
    const int id = static_cast<int>(~static_cast<uint32_t>(v) & 0xFFFFFFu);
    if (threadIdx.x == 0) answer(a, row, r, id, finite(logits[id]), total);
  }
}

constexpr int BAD = static_cast<int>(hipErrorInvalidValue);

bool shape_ok(int64_t rows, int64_t vocab) { return rows > 0 && rows <= 65535 && vocab > 0 && vocab <= MAX_VOCAB; }
int64_t chunks_of(int64_t vocab) { return (vocab + CHUNK - 1) / CHUNK; }
int64_t cap_of(int64_t vocab) { return vocab < LIST ? vocab : LIST; }
int64_t workspace_of(int64_t rows, int64_t vocab) {
  return rows * ((16 + 8 * BINS) * chunks_of(vocab) + static_cast<int64_t>(sizeof(Cut)) + 8 * cap_of(vocab) + 4 * LINE);
}

}  // namespace

extern "C" int hipengine_gfx950_sample_f32_rows_i32_workspace_bytes(int64_t rows, int64_t vocab_size, int64_t* bytes) {
  if (!bytes || !shape_ok(rows, vocab_size)) return BAD;
  *bytes = workspace_of(rows, vocab_size);
  return 0;
}

extern "C" int hipengine_gfx950_sample_f32_rows_i32(const float* logits, int64_t logits_stride, const float* uniform,
                                                    const float* temperature, const int32_t* top_k, const float* top_p,
                                                    const float* min_p, int32_t* out_ids, float* out_logprobs, int64_t rows,
                                                    int64_t vocab_size, void* workspace, int64_t workspace_bytes,
                                                    hipStream_t stream) {
  if (!logits || !uniform || !out_ids || !shape_ok(rows, vocab_size) || !workspace ||
      workspace_bytes < workspace_of(rows, vocab_size) || (reinterpret_cast<uintptr_t>(workspace) & 7) != 0)
    return BAD;
  if (logits_stride == 0) logits_stride = vocab_size;
  if (logits_stride < vocab_size) return BAD;
  const int64_t chunks = chunks_of(vocab_size);
  uint64_t* w = static_cast<uint64_t*>(workspace);
  Args a{logits, logits_stride, uniform, temperature, top_k, top_p, min_p, out_ids, out_logprobs, static_cast<int>(vocab_size),
         static_cast<int>(chunks), static_cast<int>(cap_of(vocab_size)), nullptr, nullptr, nullptr, nullptr, nullptr, nullptr};
  a.before = w;
  a.best = a.before + rows * chunks * BINS;
  a.sums = a.best + rows * chunks;
  a.cuts = reinterpret_cast<Cut*>(a.sums + rows * chunks);
  a.list = reinterpret_cast<uint64_t*>(a.cuts + rows);
  a.listed = reinterpret_cast<uint32_t*>(a.list + rows * a.cap);
  const dim3 grid(static_cast<unsigned>(chunks), static_cast<unsigned>(rows)), threads(THREADS);
  hipLaunchKernelGGL(sample_max_kernel, grid, threads, 0, stream, a);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return static_cast<int>(err);
  hipLaunchKernelGGL(sample_histogram_kernel, grid, threads, 0, stream, a);
  if ((err = hipGetLastError()) != hipSuccess) return static_cast<int>(err);
  if (rows * chunks * chunks <= SHARED_CUTS) {
    hipLaunchKernelGGL(sample_collect_kernel<true>, grid, threads, 0, stream, a);
  } else {
    hipLaunchKernelGGL(sample_cut_kernel, dim3(static_cast<unsigned>(rows)), dim3(LAST), 0, stream, a);
    if ((err = hipGetLastError()) != hipSuccess) return static_cast<int>(err);
    hipLaunchKernelGGL(sample_collect_kernel<false>, grid, threads, 0, stream, a);
  }
  if ((err = hipGetLastError()) != hipSuccess) return static_cast<int>(err);
  hipLaunchKernelGGL(sample_choose_kernel, dim3(static_cast<unsigned>(rows)), dim3(LAST), 0, stream, a);
  return static_cast<int>(hipGetLastError());
}

int hipengine_gfx950::sample_rows_load() {
  hipFuncAttributes attr;
  return static_cast<int>(hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(sample_choose_kernel)));
}
