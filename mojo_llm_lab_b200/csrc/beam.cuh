// Beam search's selection: of all continuations (beam w, token v) of a batch
// entry, the n of highest score
//   score[w][v] = cum[w] + x[w][v] - log(sum over u of exp(x[w][u])),
// ties to the lower beam, in a beam to the larger logit (far below the beam's
// best, fp64 scores of different logits meet), then to the lower token.  Within a beam the order is that of the
// logits, so one pass over them finds both the n best of every chunk and the
// chunk's part of the sum; a second, small kernel joins them in fp64.
//
// Logits: NaN counts as -inf, +inf as the largest finite fp32, and -inf is
// no candidate (nor is anything of a beam whose cum is -inf or NaN).
#pragma once

#include "paged.cuh"

namespace mllb {

constexpr int kBeamThreads = 256;
constexpr int kBeamWarps = kBeamThreads / 32;
constexpr int kBeamPer = 32;                            // logits a thread holds in registers
constexpr int kBeamChunk = kBeamThreads * kBeamPer;     // logits a CTA holds
constexpr int kBeamMost = 64;                           // beams, and candidates returned
constexpr int kBeamTokenBits = 26;                      // vocabularies of up to 2^26
constexpr int kBeamList = 512;                          // keys that reach the threshold, as a rule 20 to 60

// fp32 -> uint32 in the same order (the framework's packed argmax key, decode.cuh).
__device__ __forceinline__ uint32_t ordered_bits(float x) {
  const uint32_t b = __float_as_uint(x);
  return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float ordered_value(uint32_t b) {
  return __uint_as_float(b ^ (b >> 31 ? 0x80000000u : 0xffffffffu));
}
// fp64 -> uint64 in the same order.
__device__ __forceinline__ unsigned long long ordered_bits64(double x) {
  const unsigned long long b = __double_as_longlong(x);
  return b ^ (b >> 63 ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ double ordered_value64(unsigned long long b) {
  return __longlong_as_double(b ^ (b >> 63 ? 1ull << 63 : ~0ull));
}

struct BeamChunkSum {
  double sum;  // sum of exp(x - top) over the chunk
  float top;   // its largest logit, -inf if it has none
  float pad;
};

struct BeamArgs {
  const void* logits;        // [batch][beams][vocab], strides in elements
  const float* scores;       // [batch][beams]
  const uint8_t* done;       // [batch][beams] or nullptr
  unsigned long long* keys;  // [batch * beams][chunks][n]
  BeamChunkSum* sums;        // [batch * beams][chunks]
  float* out_scores;         // [batch][n]
  int32_t* out_tokens;
  int32_t* out_parents;
  long long batch_stride, beam_stride;
  int batch, beams, vocab, chunks, n, end_token;
};

// A value that at least n of the CTA's keys reach, from the threads' own
// largest ordered values (0: none): every warp's k-th largest lane with
// k = ceil(n / warps), and the least of those.  Few more than n reach it
// unless the large ones sit in one warp.  All threads call it.
__device__ __forceinline__ uint32_t beam_threshold(uint32_t mine, int n, uint32_t* warp_kth) {
  const int k = (n + kBeamWarps - 1) / kBeamWarps;
  uint32_t kth = 0;
  for (int i = 0; i < k; ++i) {
    kth = __reduce_max_sync(0xffffffffu, mine);
    if (mine == kth) mine = 0;  // equal lanes leave together: the next one is lower still
  }
  if ((threadIdx.x & 31) == 0) warp_kth[threadIdx.x >> 5] = kth;
  __syncthreads();
  uint32_t least = warp_kth[0];
#pragma unroll
  for (int i = 1; i < kBeamWarps; ++i) least = min(least, warp_kth[i]);
  return max(least, 1u);
}

// CTA (chunk, batch * beams + beam): the n largest logits of the chunk, with
// ties to the lower index, and its part of the sum of exponentials.  Key of a
// logit: its ordered bits above the complement of its index; 0 is no
// candidate.  The logits stay in registers; those that reach a threshold
// (beam_threshold) are listed and ranked by counting.
// Bound: 2 or 4 bytes a logit from HBM, but also 8 instructions (unpack, two
// clamps, maximum, difference, product, ex2, sum) and one special-function
// slot, about as much; 16-byte loads, and 8192 logits a CTA so that the
// reductions are a tenth of its time.
template <int kType, bool kVector>
__global__ void __launch_bounds__(kBeamThreads) beam_scan_kernel(const BeamArgs a) {
  __shared__ unsigned long long list[kBeamList];
  __shared__ unsigned long long warp_best[kBeamWarps];
  __shared__ uint32_t warp_kth[kBeamWarps];
  __shared__ float warp_top[kBeamWarps];
  __shared__ double warp_sum[kBeamWarps];
  __shared__ int count;
  pdl_wait_prerequisite();
  pdl_launch_dependents();
  const int chunk = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (a.done && a.done[row]) return;
  const long long base = (row / a.beams) * a.batch_stride + (row % a.beams) * a.beam_stride;
  const int v0 = chunk * kBeamChunk;
  constexpr int kWide = kVector ? (kType == kTypeF32 ? 4 : 8) : 1;  // values of one load
  float x[kBeamPer];
  auto index = [&](int i) { return v0 + ((i / kWide) * kBeamThreads + tid) * kWide + i % kWide; };
  auto load_one = [&](int v) {
    if (v >= a.vocab) return -INFINITY;
    if constexpr (kType == kTypeF32)
      return static_cast<const float*>(a.logits)[base + v];
    else
      return unpack16<kType == kTypeBf16>(static_cast<const uint16_t*>(a.logits)[base + v]).x;
  };
#pragma unroll
  for (int i = 0; i < kBeamPer; i += kWide) {
    if constexpr (kVector) {
      float f[kWide];
      if (index(i) + kWide <= a.vocab) {
        load_values<kType, kWide>(a.logits, base + index(i), f);
#pragma unroll
        for (int j = 0; j < kWide; ++j) x[i + j] = f[j];
      } else {
#pragma unroll
        for (int j = 0; j < kWide; ++j) x[i + j] = load_one(index(i) + j);
      }
    } else {
      x[i] = load_one(index(i));
    }
  }
  if (tid == 0) count = 0;
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kBeamPer; ++i) {
    x[i] = fminf(fmaxf(x[i], -INFINITY), FLT_MAX);  // a maximum with NaN is the other value
    top = fmaxf(top, x[i]);
  }
  const float wtop = warp_max_float(top);
  if (lane == 0) warp_top[warp] = wtop;
  // (+ 0: zeros of either sign are one value.)
  const uint32_t mine = top == -INFINITY ? 0u : ordered_bits(top + 0.0f);
  const uint32_t least = beam_threshold(mine, a.n, warp_kth);
  if (mine >= least) {
#pragma unroll
    for (int i = 0; i < kBeamPer; ++i) {
      const uint32_t o = ordered_bits(x[i] + 0.0f);
      if (x[i] != -INFINITY && o >= least) {
        const int at = atomicAdd(&count, 1);
        if (at < kBeamList) list[at] = static_cast<unsigned long long>(o) << 32 | (0xffffffffu - index(i));
      }
    }
  }
  // Differences to the chunk's largest, so that the largest weighs exactly 1;
  // terms and a thread's sum in fp32, the threads' sums in fp64.
  top = warp_top[0];
#pragma unroll
  for (int i = 1; i < kBeamWarps; ++i) top = fmaxf(top, warp_top[i]);
  float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const float zero = top == -INFINITY ? 0.0f : top;
#pragma unroll
  for (int i = 0; i < kBeamPer; ++i) part[i & 3] += ex2((x[i] - zero) * 1.4426950408889634f);
  const double sum = warp_sum_double((part[0] + part[1]) + (part[2] + part[3]));
  if (lane == 0) warp_sum[warp] = sum;
  __syncthreads();
  const int found = count;
  unsigned long long* out = a.keys + (static_cast<long long>(row) * a.chunks + chunk) * a.n;
  if (found <= kBeamList) {
    for (int i = tid; i < found; i += kBeamThreads) {
      const unsigned long long k = list[i];
      int r = 0;
      for (int j = 0; j < found; ++j) r += list[j] > k;
      if (r < a.n) out[r] = k;
    }
    for (int i = found + tid; i < a.n; i += kBeamThreads) out[i] = 0;
  } else {
    // More than the list holds (equal logits, as a rule): one maximum below the last at a time.
    unsigned long long last = ~0ull;
    for (int r = 0; r < a.n; ++r) {
      unsigned long long best = 0;
#pragma unroll
      for (int i = 0; i < kBeamPer; ++i) {
        const unsigned long long k =
            x[i] == -INFINITY ? 0ull
                              : static_cast<unsigned long long>(ordered_bits(x[i] + 0.0f)) << 32 | (0xffffffffu - index(i));
        if (k < last) best = max(best, k);
      }
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, d));
      if (lane == 0) warp_best[warp] = best;
      __syncthreads();
      best = warp_best[0];
#pragma unroll
      for (int i = 1; i < kBeamWarps; ++i) best = max(best, warp_best[i]);
      last = best;
      if (tid == 0) out[r] = best;
      __syncthreads();
    }
  }
  if (tid == 0) {
    double total = 0.0;
    for (int i = 0; i < kBeamWarps; ++i) total += warp_sum[i];
    a.sums[static_cast<long long>(row) * a.chunks + chunk] = {total, top, 0.0f};
  }
}

// CTA per batch entry: the log-sum of every beam, then the n best of the
// beams' chunk lists by (fp64 score, place), found as in the scan.  fp64: two
// beams' candidates can lie closer than fp32 tells apart.  Bound: a chain of
// latencies (sums, exp and log, keys, threshold, ranks).
__global__ void __launch_bounds__(kBeamThreads) beam_pick_kernel(const BeamArgs a) {
  // score = cum + ((x - top) - log(sum of exp(x - top))), from the inside out:
  // x - top is exact or small beside cum, whatever the logits' size.
  __shared__ double beam_top[kBeamMost], beam_log[kBeamMost];
  __shared__ double beam_cum[kBeamMost];  // -inf: no candidates
  __shared__ uint32_t warp_kth[kBeamWarps];
  __shared__ unsigned long long list_score[kBeamList], list_place[kBeamList];
  __shared__ unsigned long long best_score[kBeamThreads], best_place[kBeamThreads];
  __shared__ int count;
  const int entry = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row0 = entry * a.beams;
  if (tid == 0) count = 0;
  pdl_wait_prerequisite();
  pdl_launch_dependents();
  for (int w = warp; w < a.beams; w += kBeamWarps) {
    const double cum = a.scores[row0 + w];
    double live = -INFINITY;
    if (!(a.done && a.done[row0 + w])) {
      const BeamChunkSum* sums = a.sums + static_cast<long long>(row0 + w) * a.chunks;
      float top = -INFINITY;
      for (int i = lane; i < a.chunks; i += 32) top = fmaxf(top, sums[i].top);
      top = warp_max_float(top);
      double sum = 0.0;
      for (int i = lane; i < a.chunks; i += 32)
        if (sums[i].top != -INFINITY) sum += sums[i].sum * exp(static_cast<double>(sums[i].top) - top);
      sum = warp_sum_double(sum);
      if (top != -INFINITY && cum == cum) live = cum;
      if (lane == 0) {
        beam_top[w] = top;
        beam_log[w] = log(sum);
      }
    }
    if (lane == 0) beam_cum[w] = live;
  }
  __syncthreads();
  // Candidate i of this entry: (score, place), score 0 if there is none.  A
  // place holds, from the top, the complement of the beam (6 bits), the
  // logit's ordered bits and the complement of the token, so that the larger
  // pair comes first.
  constexpr unsigned long long kTokens = (1ull << kBeamTokenBits) - 1;
  const int per_beam = a.chunks * a.n, total = a.beams * per_beam;
  auto place_of = [&](int w, unsigned long long logit, uint32_t token) {
    return static_cast<unsigned long long>(kBeamMost - 1 - w) << (32 + kBeamTokenBits) | logit << kBeamTokenBits |
           (kTokens - token);
  };
  auto candidate = [&](int i, unsigned long long* score, unsigned long long* place) {
    const int w = i / per_beam;
    *score = 0;
    *place = 0;
    if (a.done && a.done[row0 + w]) {
      const float cum = a.scores[row0 + w];
      if (i == w * per_beam && cum > -INFINITY) {
        *score = ordered_bits64(cum);
        *place = place_of(w, 0, a.end_token);
      }
      return;
    }
    const double cum = beam_cum[w];
    const unsigned long long key = a.keys[static_cast<long long>(row0) * per_beam + i];
    if (key == 0 || cum == -INFINITY) return;
    *score = ordered_bits64(cum + (ordered_value(static_cast<uint32_t>(key >> 32)) - beam_top[w] - beam_log[w]));
    *place = place_of(w, key >> 32, 0xffffffffu - static_cast<uint32_t>(key));
  };
  // The threshold on the scores' upper halves: in the same order, ties apart.
  uint32_t mine = 0;
#pragma unroll 4
  for (int i = tid; i < total; i += kBeamThreads) {
    unsigned long long s, p;
    candidate(i, &s, &p);
    mine = max(mine, static_cast<uint32_t>(s >> 32));
  }
  const uint32_t least = beam_threshold(mine, a.n, warp_kth);
  if (mine >= least) {
    for (int i = tid; i < total; i += kBeamThreads) {
      unsigned long long s, p;
      candidate(i, &s, &p);
      if (static_cast<uint32_t>(s >> 32) >= least) {
        const int k = atomicAdd(&count, 1);
        if (k < kBeamList) {
          list_score[k] = s;
          list_place[k] = p;
        }
      }
    }
  }
  __syncthreads();
  int found = count;
  auto write = [&](int r, unsigned long long s, unsigned long long p) {
    const bool any = s != 0;
    a.out_scores[entry * a.n + r] = any ? static_cast<float>(ordered_value64(s)) : -INFINITY;
    a.out_tokens[entry * a.n + r] = any ? static_cast<int32_t>(kTokens - (p & kTokens)) : -1;
    a.out_parents[entry * a.n + r] = any ? kBeamMost - 1 - static_cast<int32_t>(p >> (32 + kBeamTokenBits)) : -1;
  };
  if (found <= kBeamList) {
    for (int i = tid; i < found; i += kBeamThreads) {
      const unsigned long long s = list_score[i], p = list_place[i];
      int r = 0;
      for (int j = 0; j < found; ++j) r += list_score[j] > s || (list_score[j] == s && list_place[j] > p);
      if (r < a.n) write(r, s, p);
    }
    for (int i = found + tid; i < a.n; i += kBeamThreads) write(i, 0, 0);
  } else {
    // More than the list holds: one maximum below the last at a time.
    unsigned long long last_s = ~0ull, last_p = ~0ull;
    for (int r = 0; r < a.n; ++r) {
      unsigned long long bs = 0, bp = 0;
      for (int i = tid; i < total; i += kBeamThreads) {
        unsigned long long s, p;
        candidate(i, &s, &p);
        if ((s < last_s || (s == last_s && p < last_p)) && (s > bs || (s == bs && p > bp))) bs = s, bp = p;
      }
      __syncthreads();
      best_score[tid] = bs;
      best_place[tid] = bp;
      __syncthreads();
      for (int i = 0; i < kBeamThreads; ++i)
        if (best_score[i] > bs || (best_score[i] == bs && best_place[i] > bp)) bs = best_score[i], bp = best_place[i];
      last_s = bs;
      last_p = bp;
      if (tid == 0) write(r, bs, bp);
    }
  }
}

}  // namespace mllb
