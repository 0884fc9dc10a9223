// Beam search's selection: of all continuations (beam w, token v) of a batch
// entry, the n of highest score
//   score[w][v] = cum[w] + x[w][v] - log(sum over u of exp(x[w][u])),
// ties to the lower beam, in a beam to the larger logit (far below the beam's
// best, fp64 scores of different logits meet), then to the lower token.  Within
// a beam the order is that of the logits, so one pass over them finds both the n
// best of every chunk and the chunk's part of the sum; a second, small kernel
// joins them in fp64.  The scan's exponentials are fp32 (ex2, and 16 terms at a
// time): a log-sum may be off by 2^-20.
//
// Logits: NaN counts as -inf, +inf as the largest finite fp32, and -inf is
// no candidate (nor is anything of a beam whose cum is -inf or NaN).
#pragma once

#include "paged.cuh"

namespace mllb {

constexpr int kBeamThreads = 256;
constexpr int kBeamWarps = kBeamThreads / 32;
constexpr int kBeamPer = 16;                            // logits of a step that a thread holds in registers
constexpr int kBeamStep = kBeamThreads * kBeamPer;      // logits of a step
constexpr int kBeamStepsMost = 36;                      // steps of a chunk: 36 KB of maxima
constexpr int kPickThreads = 512;                       // of the joining kernel
constexpr int kPickWarps = kPickThreads / 32;
constexpr int kBeamMost = 64;                           // beams, and candidates returned
constexpr int kBeamTokenBits = 26;                      // vocabularies of up to 2^26
constexpr int kBeamList = 512;                          // keys at or above a threshold, as a rule 20 to 60

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
  int batch, beams, vocab, chunks, steps, n, end_token;  // a chunk is `steps` steps
};

// A value that at least n of the CTA's keys reach, from the threads' own
// largest ordered values (0: none); 1 if they do not show one.  Each warp
// shows its t = ceil(n / 4) largest, and the n-th of those is it: exact unless
// more than a quarter of the n best are in one warp.  All threads of kWarps
// warps call it; `words`: kWarps * kBeamShown + 1, free again after the
// caller's next barrier.
constexpr int kBeamShown = kBeamMost / 4;
template <int kWarps>
__device__ __forceinline__ uint32_t beam_threshold(uint32_t mine, int n, uint32_t* words) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int t = (n + 3) / 4, shown = kWarps * t;
  uint32_t* least = words + kWarps * kBeamShown;
  if (tid == 0) *least = 1;
  for (int got = 0; got < t;) {  // equal lanes are shown together
    const uint32_t top = __reduce_max_sync(0xffffffffu, mine);
    const unsigned with = __ballot_sync(0xffffffffu, mine == top);
    if (mine == top) mine = 0;
    const int at = got + __popc(with & ((1u << lane) - 1));
    if ((with >> lane & 1) && at < t) words[warp * t + at] = top;
    got += __popc(with);  // (with top 0 all lanes are left: zeros fill up)
  }
  __syncthreads();
  if (tid < shown) {
    const uint32_t v = words[tid];
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < shown; ++i) rank += words[i] > v || (words[i] == v && i < tid);
    if (v && rank == n - 1) *least = v;
  }
  __syncthreads();
  return *least;
}

// Key of a logit (+ 0: zeros of either sign are one value).
__device__ __forceinline__ unsigned long long beam_key(float x, int index) {
  return static_cast<unsigned long long>(ordered_bits(x + 0.0f)) << 32 | (0xffffffffu - static_cast<uint32_t>(index));
}

// Of the keys key_of(0 .. total), the n largest in descending order into
// kept[0..n) (0 where there are fewer); keys are distinct or 0.  Those that
// reach a threshold (beam_threshold) are listed and ranked by counting, a key
// a warp; if the list does not hold them (equal values, as a rule) the n are
// found one maximum below the last at a time.  All threads call it.
struct BeamScratch {
  unsigned long long list[kBeamList], best[kBeamWarps];
  uint32_t words[kBeamWarps * kBeamShown + 1];
  int count;
};
template <typename KeyOf>
__device__ __forceinline__ void beam_best(BeamScratch& sh, int total, int n, unsigned long long* kept, KeyOf key_of) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned long long mine = 0;
  for (int i = tid; i < total; i += kBeamThreads) mine = max(mine, key_of(i));
  if (tid == 0) sh.count = 0;
  const uint32_t least = beam_threshold<kBeamWarps>(static_cast<uint32_t>(mine >> 32), n, sh.words);
  if (static_cast<uint32_t>(mine >> 32) >= least) {
    for (int i = tid; i < total; i += kBeamThreads) {
      const unsigned long long k = key_of(i);
      if (static_cast<uint32_t>(k >> 32) >= least) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kBeamList) sh.list[at] = k;
      }
    }
  }
  __syncthreads();
  const int held = sh.count;
  if (held <= kBeamList) {
    for (int i = warp; i < held; i += kBeamWarps) {
      const unsigned long long k = sh.list[i];
      int r = 0;
      for (int j = lane; j < held; j += 32) r += sh.list[j] > k;
      r = __reduce_add_sync(0xffffffffu, r);
      if (lane == 0 && r < n) kept[r] = k;
    }
    for (int i = held + tid; i < n; i += kBeamThreads) kept[i] = 0;
  } else {
    unsigned long long last = ~0ull;
    for (int r = 0; r < n; ++r) {
      unsigned long long best = 0;
      for (int i = tid; i < total; i += kBeamThreads) {
        const unsigned long long k = key_of(i);
        if (k < last) best = max(best, k);
      }
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, d));
      if (lane == 0) sh.best[warp] = best;
      __syncthreads();
      best = sh.best[0];
#pragma unroll
      for (int i = 1; i < kBeamWarps; ++i) best = max(best, sh.best[i]);
      last = best;
      if (tid == 0) kept[r] = best;
      __syncthreads();
    }
  }
  __syncthreads();
}

// CTA (chunk, batch * beams + beam): the n largest logits of the chunk, with
// ties to the lower index, and its part of the sum of exponentials.
//
// One pass over the logits, in steps of 4096: a thread takes 16 in a row, adds
// their exponentials to its own running sum and leaves their maximum in shared
// memory; nothing else, and no barrier.  The n best logits lie in the n groups
// of 16 with the best (maximum, place), so afterwards those are found among
// the maxima and read again, and the n best of their 16 n logits taken.
// Groups are in the order of their logits, so ties come out right.
// Key of a logit: its ordered bits above the complement of its index; 0 is no
// candidate.  No unit is full (32 x 8 rows: issue slots 54 %, exponentials 39 %,
// DRAM 23 %): about 8 slots a logit while the scan runs (unpack, NaN, maximum,
// difference, product, ex2, sum), then the barriers of two selections, when most
// warps wait; for short chunks those are all.  Both kernels, 32 x 8 rows of
// 151936 in bf16: n = 8 33 us, n = 16 with some of the beams done 39; the
// bytes alone 12.  4 rows in fp32: 11.
template <int kType, bool kVector>
__global__ void __launch_bounds__(kBeamThreads, 4) beam_scan_kernel(const BeamArgs a) {
  constexpr int kWide = kVector ? (kType == kTypeF32 ? 4 : 8) : 1;  // values of one load
  constexpr int kWords = kType == kTypeF32 ? kBeamPer : kBeamPer / 2;
  constexpr float kLog2e = 1.4426950408889634f;
  extern __shared__ float maxima[];  // [steps][threads]
  __shared__ BeamScratch sh;
  __shared__ unsigned long long kept[kBeamMost];
  __shared__ float warp_top[kBeamWarps];
  __shared__ double warp_sum[kBeamWarps];
  pdl_wait_prerequisite();
  pdl_launch_dependents();
  const int chunk = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (a.done && a.done[row]) return;
  const uint8_t* logits = static_cast<const uint8_t*>(a.logits) +
                          ((row / a.beams) * a.batch_stride + (row % a.beams) * a.beam_stride) * (kType == kTypeF32 ? 4 : 2);
  const int begin = chunk * a.steps * kBeamStep, end = min(begin + a.steps * kBeamStep, a.vocab);
  // Vectors that end inside the row; the up to seven logits behind them come last, one a thread.
  const int vectors_end = kVector ? begin + (end - begin) / kWide * kWide : end;
  auto logit = [&](int v) {
    float y;
    if constexpr (kType == kTypeF32)
      y = reinterpret_cast<const float*>(logits)[v];
    else
      y = unpack16<kType == kTypeBf16>(reinterpret_cast<const uint16_t*>(logits)[v]).x;
    return fminf(fmaxf(y, -INFINITY), FLT_MAX);  // a maximum with NaN is the other value
  };
  constexpr uint32_t kNone = kType == kTypeF32 ? 0xff800000u : kType == kTypeF16 ? 0xfc00fc00u : 0xff80ff80u;  // -inf
  uint32_t raw[kWords];
  auto load = [&](int v) {  // 16 logits from v on
    if constexpr (kVector) {
      constexpr int kLoads = kBeamPer / kWide;
      const uint4* from = reinterpret_cast<const uint4*>(logits + static_cast<long long>(v) * (16 / kWide));
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        uint4 w = make_uint4(kNone, kNone, kNone, kNone);
        if (v + i * kWide < vectors_end) w = from[i];
        raw[4 * i] = w.x, raw[4 * i + 1] = w.y, raw[4 * i + 2] = w.z, raw[4 * i + 3] = w.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kBeamPer; ++i) {
        if constexpr (kType == kTypeF32) {
          raw[i] = v + i < end ? reinterpret_cast<const uint32_t*>(logits)[v + i] : kNone;
        } else {
          const uint32_t w = v + i < end ? reinterpret_cast<const uint16_t*>(logits)[v + i] : kNone & 0xffffu;
          raw[i / 2] = i % 2 ? raw[i / 2] | w << 16 : w;
        }
      }
    }
  };
  load(begin + tid * kBeamPer);
  float top = -INFINITY;  // this thread's largest so far
  double sum = 0.0;       // of exp(x - top)
  int steps = 0;
  for (int v = begin + tid * kBeamPer; v - tid * kBeamPer < vectors_end; v += kBeamStep, ++steps) {
    float x[kBeamPer];
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      if constexpr (kType == kTypeF32) {
        x[w] = __uint_as_float(raw[w]);
      } else {
        const float2 f = unpack16<kType == kTypeBf16>(raw[w]);
        x[2 * w] = f.x, x[2 * w + 1] = f.y;
      }
    }
    load(min(v + kBeamStep, end));
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kBeamPer; i += 2) {
      x[i] = fmaxf(x[i], -INFINITY);
      x[i + 1] = fmaxf(x[i + 1], -INFINITY);
      m = fmaxf(fmaxf(m, x[i]), x[i + 1]);
    }
    if (m == INFINITY) {
#pragma unroll
      for (int i = 0; i < kBeamPer; ++i) x[i] = fminf(x[i], FLT_MAX);
      m = FLT_MAX;
    }
    maxima[steps * kBeamThreads + tid] = m;
    // Differences to the largest, so that it weighs exactly 1; terms and a
    // step's sum in fp32, the steps' sums in fp64.
    const float now = fmaxf(top, m), zero = now == -INFINITY ? 0.0f : now;
    float2 part[2] = {};
#pragma unroll
    for (int i = 0; i < kBeamPer; i += 2) {
      float2 d = __fadd2_rn(make_float2(x[i], x[i + 1]), make_float2(-zero, -zero));
      d = __fmul2_rn(d, make_float2(kLog2e, kLog2e));
      d.x = ex2(d.x);
      d.y = ex2(d.y);
      part[i >> 1 & 1] = __fadd2_rn(part[i >> 1 & 1], d);
    }
    part[0] = __fadd2_rn(part[0], part[1]);
    const float before = sum != 0.0 ? ex2((top - zero) * kLog2e) : 0.0f;
    sum = sum * before + (part[0].x + part[0].y);
    top = now;
  }
  const int behind = vectors_end + tid;  // this thread's logit behind the vectors
  if (kVector && behind < end) {
    const float y = logit(behind), now = fmaxf(top, y), zero = now == -INFINITY ? 0.0f : now;
    sum = sum * ex2((top - zero) * kLog2e) + ex2((y - zero) * kLog2e);
    top = now;
  }
  const float wtop = warp_max_float(top);
  if (lane == 0) warp_top[warp] = wtop;
  __syncthreads();
  float all = warp_top[0];
#pragma unroll
  for (int i = 1; i < kBeamWarps; ++i) all = fmaxf(all, warp_top[i]);
  sum = warp_sum_double(top == -INFINITY ? 0.0 : sum * ex2((top - all) * kLog2e));
  if (lane == 0) warp_sum[warp] = sum;
  // The n best groups, then the n best of their logits and of those behind the vectors.
  beam_best(sh, steps * kBeamThreads, a.n, kept, [&](int i) {
    return maxima[i] == -INFINITY ? 0ull : beam_key(maxima[i], i);
  });
  unsigned long long* out = a.keys + (static_cast<long long>(row) * a.chunks + chunk) * a.n;
  beam_best(sh, a.n * kBeamPer + (end - vectors_end), a.n, out, [&](int i) {
    int v = vectors_end + i - a.n * kBeamPer;
    if (i < a.n * kBeamPer) {
      const unsigned long long group = kept[i / kBeamPer];
      v = begin + static_cast<int>(0xffffffffu - static_cast<uint32_t>(group)) * kBeamPer + i % kBeamPer;
      if (group == 0 || v >= vectors_end) return 0ull;
    }
    const float y = logit(v);
    return y == -INFINITY ? 0ull : beam_key(y, v);
  });
  if (warp == 0) {
    double total = lane < kBeamWarps ? warp_sum[lane] : 0.0;
#pragma unroll
    for (int d = kBeamWarps / 2; d >= 1; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    if (lane == 0) a.sums[static_cast<long long>(row) * a.chunks + chunk] = {total, all, 0.0f};
  }
}

// CTA per batch entry: the log-sum of every beam, then the n best of the
// beams' chunk lists by (fp64 score, place), found as in the scan.  fp64: two
// beams' candidates can lie closer than fp32 tells apart.  Bound: a chain of
// latencies (sums, exp and log, keys, threshold, ranks).
__global__ void __launch_bounds__(kPickThreads) beam_pick_kernel(const BeamArgs a) {
  // score = cum + ((x - top) - log(sum of exp(x - top))), from the inside out:
  // x - top is exact or small beside cum, whatever the logits' size.
  __shared__ double beam_top[kBeamMost], beam_log[kBeamMost];
  __shared__ double beam_cum[kBeamMost];  // -inf: no candidates
  __shared__ bool beam_done[kBeamMost];
  __shared__ uint32_t scratch[kPickWarps * kBeamShown + 1];
  __shared__ unsigned long long list_score[kBeamList], list_place[kBeamList];
  __shared__ unsigned long long best_score[kPickWarps], best_place[kPickWarps];
  __shared__ int count;
  const int entry = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row0 = entry * a.beams;
  if (tid == 0) count = 0;
  pdl_wait_prerequisite();
  pdl_launch_dependents();
  for (int w = warp; w < a.beams; w += kPickWarps) {
    const double cum = a.scores[row0 + w];
    const bool done = a.done && a.done[row0 + w];
    double live = cum > -INFINITY ? cum : -INFINITY;  // NaN: none
    if (!done) {
      const BeamChunkSum* sums = a.sums + static_cast<long long>(row0 + w) * a.chunks;
      float top = -INFINITY;
      for (int i = lane; i < a.chunks; i += 32) top = fmaxf(top, sums[i].top);
      top = warp_max_float(top);
      double sum = 0.0;
      for (int i = lane; i < a.chunks; i += 32)
        if (sums[i].top != -INFINITY) sum += sums[i].sum * exp(static_cast<double>(sums[i].top) - top);
      sum = warp_sum_double(sum);
      if (top == -INFINITY) live = -INFINITY;
      if (lane == 0) {
        beam_top[w] = top;
        beam_log[w] = log(sum);
      }
    }
    if (lane == 0) {
      beam_cum[w] = live;
      beam_done[w] = done;
    }
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
    const double cum = beam_cum[w];
    if (beam_done[w]) {
      if (i == w * per_beam && cum > -INFINITY) {
        *score = ordered_bits64(cum);
        *place = place_of(w, 0, a.end_token);
      }
      return;
    }
    const unsigned long long key = a.keys[static_cast<long long>(row0) * per_beam + i];
    if (key == 0 || cum == -INFINITY) return;
    *score = ordered_bits64(cum + (ordered_value(static_cast<uint32_t>(key >> 32)) - beam_top[w] - beam_log[w]));
    *place = place_of(w, key >> 32, 0xffffffffu - static_cast<uint32_t>(key));
  };
  // The threshold on the scores' upper halves: in the same order, ties apart.
  uint32_t mine = 0;
#pragma unroll 4
  for (int i = tid; i < total; i += kPickThreads) {
    unsigned long long s, p;
    candidate(i, &s, &p);
    mine = max(mine, static_cast<uint32_t>(s >> 32));
  }
  const uint32_t least = beam_threshold<kPickWarps>(mine, a.n, scratch);
  if (mine >= least) {
    for (int i = tid; i < total; i += kPickThreads) {
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
    for (int i = warp; i < found; i += kPickWarps) {
      const unsigned long long s = list_score[i], p = list_place[i];
      int r = 0;
      for (int j = lane; j < found; j += 32) r += list_score[j] > s || (list_score[j] == s && list_place[j] > p);
      r = __reduce_add_sync(0xffffffffu, r);
      if (lane == 0 && r < a.n) write(r, s, p);
    }
    for (int i = found + tid; i < a.n; i += kPickThreads) write(i, 0, 0);
  } else {
    // More than the list holds: one maximum below the last at a time.
    unsigned long long last_s = ~0ull, last_p = ~0ull;
    for (int r = 0; r < a.n; ++r) {
      unsigned long long bs = 0, bp = 0;
      for (int i = tid; i < total; i += kPickThreads) {
        unsigned long long s, p;
        candidate(i, &s, &p);
        if ((s < last_s || (s == last_s && p < last_p)) && (s > bs || (s == bs && p > bp))) bs = s, bp = p;
      }
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) {
        const unsigned long long os = __shfl_xor_sync(0xffffffffu, bs, d), op = __shfl_xor_sync(0xffffffffu, bp, d);
        if (os > bs || (os == bs && op > bp)) bs = os, bp = op;
      }
      __syncthreads();
      if (lane == 0) {
        best_score[warp] = bs;
        best_place[warp] = bp;
      }
      __syncthreads();
      for (int i = 0; i < kPickWarps; ++i)
        if (best_score[i] > bs || (best_score[i] == bs && best_place[i] > bp)) bs = best_score[i], bp = best_place[i];
      last_s = bs;
      last_p = bp;
      if (tid == 0) write(r, bs, bp);
    }
  }
}

}  // namespace mllb
