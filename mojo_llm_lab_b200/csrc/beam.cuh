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
constexpr int kBeamPer = 16;                            // logits a thread holds in registers
constexpr int kBeamChunk = kBeamThreads * kBeamPer;     // logits a CTA holds
constexpr int kBeamMost = 64;                           // beams, and candidates returned
constexpr int kBeamTokenBits = 26;                      // vocabularies of up to 2^26
constexpr int kBeamList = kBeamMost * kBeamPer;         // keys that can reach the threshold (see below)

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

// CTA (chunk, batch * beams + beam).  Key of a logit: its ordered bits above
// the complement of its index, so keys are distinct and their order is "value
// down, index up"; 0 is no candidate.  The n-th largest of the 256 threads'
// own maxima is a threshold that at least n keys reach and that only the n
// threads above it can reach: at most 16 n keys are ranked (by counting).
template <int kType, bool kVector>
__global__ void __launch_bounds__(kBeamThreads) beam_scan_kernel(const BeamArgs a) {
  __shared__ unsigned long long best[kBeamThreads];
  __shared__ unsigned long long list[kBeamList];
  __shared__ unsigned long long threshold;
  __shared__ int count;
  __shared__ float warp_top[kBeamThreads / 32];
  __shared__ double warp_sum[kBeamThreads / 32];
  pdl_wait_prerequisite();
  pdl_launch_dependents();
  const int chunk = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (a.done && a.done[row]) return;
  const long long base = (row / a.beams) * a.batch_stride + (row % a.beams) * a.beam_stride;
  const int v0 = chunk * kBeamChunk;
  constexpr int kWide = kVector ? (kType == kTypeF32 ? 4 : 8) : 1;  // values of one load
  float x[kBeamPer];
#pragma unroll
  for (int i = 0; i < kBeamPer / kWide; ++i) {
    const int v = v0 + (i * kBeamThreads + tid) * kWide;
    if constexpr (kVector) {
      float f[kWide];
      if (v + kWide <= a.vocab) {
        load_values<kType, kWide>(a.logits, base + v, f);
      } else {
#pragma unroll
        for (int j = 0; j < kWide; ++j) {
          f[j] = -INFINITY;
          if (v + j < a.vocab) {
            if constexpr (kType == kTypeF32) {
              f[j] = static_cast<const float*>(a.logits)[base + v + j];
            } else {
              f[j] = unpack16<kType == kTypeBf16>(static_cast<const uint16_t*>(a.logits)[base + v + j]).x;
            }
          }
        }
      }
#pragma unroll
      for (int j = 0; j < kWide; ++j) x[i * kWide + j] = f[j];
    } else {
      x[i] = -INFINITY;
      if (v < a.vocab) {
        if constexpr (kType == kTypeF32) {
          x[i] = static_cast<const float*>(a.logits)[base + v];
        } else {
          x[i] = unpack16<kType == kTypeBf16>(static_cast<const uint16_t*>(a.logits)[base + v]).x;
        }
      }
    }
  }
  if (tid == 0) {
    threshold = 1;
    count = 0;
  }
  auto index = [&](int i) { return v0 + ((i / kWide) * kBeamThreads + tid) * kWide + i % kWide; };
  auto key_of = [&](int i) {
    return x[i] == -INFINITY ? 0ull
                             : static_cast<unsigned long long>(ordered_bits(x[i])) << 32 | (0xffffffffu - index(i));
  };
  float top = -INFINITY;
  unsigned long long mine = 0;
#pragma unroll
  for (int i = 0; i < kBeamPer; ++i) {
    x[i] = isnan(x[i]) ? -INFINITY : fminf(x[i], FLT_MAX) + 0.0f;  // + 0: a zero of either sign is one value
    top = fmaxf(top, x[i]);
    mine = max(mine, key_of(i));
  }
  best[tid] = mine;
  const float wtop = warp_max_float(top);
  if (lane == 0) warp_top[warp] = wtop;
  __syncthreads();
  top = warp_top[0];
#pragma unroll
  for (int i = 1; i < kBeamThreads / 32; ++i) top = fmaxf(top, warp_top[i]);
  // exp in fp32 of each term, the sum in fp64.
  if (top != -INFINITY) {
    float part = 0.0f;
#pragma unroll
    for (int i = 0; i < kBeamPer; ++i) part += expf(x[i] - top);
    const double sum = warp_sum_double(part);
    if (lane == 0) warp_sum[warp] = sum;
  } else if (lane == 0) {
    warp_sum[warp] = 0.0;
  }
  int rank = 0;
  for (int i = 0; i < kBeamThreads; ++i) rank += best[i] > mine;
  if (mine && rank == a.n - 1) threshold = mine;
  __syncthreads();
  const unsigned long long least = threshold;
  if (mine >= least) {
#pragma unroll
    for (int i = 0; i < kBeamPer; ++i) {
      const unsigned long long k = key_of(i);
      if (k >= least) list[atomicAdd(&count, 1)] = k;
    }
  }
  __syncthreads();
  const int found = count;
  unsigned long long* out = a.keys + (static_cast<long long>(row) * a.chunks + chunk) * a.n;
  for (int i = tid; i < found; i += kBeamThreads) {
    const unsigned long long k = list[i];
    int r = 0;
    for (int j = 0; j < found; ++j) r += list[j] > k;
    if (r < a.n) out[r] = k;
  }
  for (int i = found + tid; i < a.n; i += kBeamThreads) out[i] = 0;
  if (tid == 0) {
    double sum = 0.0;
    for (int i = 0; i < kBeamThreads / 32; ++i) sum += warp_sum[i];
    a.sums[static_cast<long long>(row) * a.chunks + chunk] = {sum, top, 0.0f};
  }
}

// CTA per batch entry: the log-sum of every beam, then the n best of the
// beams' chunk lists by (fp64 score, place), found as in the scan.  fp64: two
// beams' candidates can lie closer than fp32 tells apart.
__global__ void __launch_bounds__(kBeamThreads) beam_pick_kernel(const BeamArgs a) {
  // score = cum + ((x - top) - log(sum of exp(x - top))), from the inside out:
  // x - top is exact or small beside cum, whatever the logits' size.
  __shared__ double beam_top[kBeamMost], beam_log[kBeamMost];
  __shared__ double beam_cum[kBeamMost];  // -inf: no candidates
  __shared__ unsigned long long best_score[kBeamThreads];
  __shared__ unsigned long long best_place[kBeamThreads];
  __shared__ unsigned long long list_score[kBeamList];
  __shared__ unsigned long long list_place[kBeamList];
  __shared__ unsigned long long least_score;
  __shared__ unsigned long long least_place;
  __shared__ int count;
  pdl_wait_prerequisite();
  pdl_launch_dependents();
  const int entry = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row0 = entry * a.beams;
  for (int w = warp; w < a.beams; w += kBeamThreads / 32) {
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
  if (tid == 0) {
    least_score = 1;
    least_place = 0;
    count = 0;
  }
  __syncthreads();
  // Candidate i of this entry: (score, place), score 0 if there is none.  A
  // place holds, from the top, the complement of the beam (6 bits), the
  // logit's ordered bits and the complement of the token, so that the larger
  // pair comes first.
  constexpr unsigned long long kTokens = (1ull << kBeamTokenBits) - 1;
  auto place_of = [&](int w, unsigned long long logit, uint32_t token) {
    return static_cast<unsigned long long>(kBeamMost - 1 - w) << (32 + kBeamTokenBits) | logit << kBeamTokenBits |
           (kTokens - token);
  };
  const int per_beam = a.chunks * a.n, total = a.beams * per_beam;
  auto candidate = [&](int i, unsigned long long* score, unsigned long long* place) {
    const int w = i / per_beam;
    *score = 0;
    *place = 0;
    if (a.done && a.done[row0 + w]) {
      const float cum = a.scores[row0 + w];
      if (i % per_beam == 0 && cum > -INFINITY) {
        *score = ordered_bits64(cum);
        *place = place_of(w, 0, a.end_token);
      }
      return;
    }
    const double cum = beam_cum[w];
    const unsigned long long key = a.keys[static_cast<long long>(row0) * per_beam + i];
    if (key == 0 || cum == -INFINITY) return;
    const uint32_t token = 0xffffffffu - static_cast<uint32_t>(key);
    *score = ordered_bits64(cum + (ordered_value(static_cast<uint32_t>(key >> 32)) - beam_top[w] - beam_log[w]));
    *place = place_of(w, key >> 32, token);
  };
  unsigned long long mine = 0, at = 0;
  for (int i = tid; i < total; i += kBeamThreads) {
    unsigned long long s, p;
    candidate(i, &s, &p);
    if (s > mine || (s == mine && p > at)) mine = s, at = p;
  }
  best_score[tid] = mine;
  best_place[tid] = at;
  __syncthreads();
  int rank = 0;
  for (int i = 0; i < kBeamThreads; ++i)
    rank += best_score[i] > mine || (best_score[i] == mine && best_place[i] > at);
  if (mine && rank == a.n - 1) {
    least_score = mine;
    least_place = at;
  }
  __syncthreads();
  const unsigned long long ls = least_score;
  const unsigned long long lp = least_place;
  if (mine > ls || (mine == ls && at >= lp)) {
    for (int i = tid; i < total; i += kBeamThreads) {
      unsigned long long s, p;
      candidate(i, &s, &p);
      if (s > ls || (s == ls && p >= lp)) {
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
    a.out_scores[entry * a.n + r] = static_cast<float>(ordered_value64(s));
    a.out_tokens[entry * a.n + r] = static_cast<int32_t>(kTokens - (p & kTokens));
    a.out_parents[entry * a.n + r] = kBeamMost - 1 - static_cast<int32_t>(p >> (32 + kBeamTokenBits));
  };
  if (found <= kBeamList) {
    for (int i = tid; i < found; i += kBeamThreads) {
      const unsigned long long s = list_score[i];
      const unsigned long long p = list_place[i];
      int r = 0;
      for (int j = 0; j < found; ++j) r += list_score[j] > s || (list_score[j] == s && list_place[j] > p);
      if (r < a.n) write(r, s, p);
    }
  } else {
    // More keys than the list holds (a few threads' shares hold nearly all the
    // large ones): one maximum below the last at a time.
    unsigned long long last_s = ~0ull, last_p = ~0ull;
    for (int r = 0; r < a.n; ++r) {
      mine = 0;
      at = 0;
      for (int i = tid; i < total; i += kBeamThreads) {
        unsigned long long s, p;
        candidate(i, &s, &p);
        if ((s < last_s || (s == last_s && p < last_p)) && (s > mine || (s == mine && p > at))) mine = s, at = p;
      }
      __syncthreads();
      best_score[tid] = mine;
      best_place[tid] = at;
      __syncthreads();
      for (int i = 0; i < kBeamThreads; ++i)
        if (best_score[i] > mine || (best_score[i] == mine && best_place[i] > at)) mine = best_score[i], at = best_place[i];
      last_s = mine;
      last_p = at;
      if (tid == 0) write(r, mine, at);
    }
    found = a.n;
  }
  for (int i = found + tid; i < a.n; i += kBeamThreads) {
    a.out_scores[entry * a.n + i] = -INFINITY;
    a.out_tokens[entry * a.n + i] = -1;
    a.out_parents[entry * a.n + i] = -1;
  }
}

}  // namespace mllb
