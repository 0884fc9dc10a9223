// A KV cache in pages: the append with q/k norms and rotary positions, and
// the reordering of page tables by parent beam.
//
// Cache: pages of page_size rows (a power of two) for every KV head, fp16 or
// bf16, addressed by element strides (page, head, row; the head_dim elements
// of a row are contiguous), so both [pages][kv_heads][page_size][D] and
// [pages][page_size][kv_heads][D] are the same code.  Sequence b's row r is
// row r % page_size of page page_table[b][r / page_size].
#pragma once

#include <cfloat>
#include <cuda_bf16.h>

#include "common.cuh"

namespace mllb {

struct PagedCache {
  uint16_t* k;
  uint16_t* v;
  long long page_stride, head_stride, row_stride, layer_stride;  // elements
  int pages, kv_heads, page_shift, layers;
};

// 16-bit types of a cache: rounding to nearest even from fp32, two at a time
// (the lower half of the word is the first value).
template <bool kBf16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if constexpr (kBf16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

template <bool kBf16>
__device__ __forceinline__ float2 unpack16(uint32_t w) {
  if constexpr (kBf16) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
}

// 2^x by the special-function unit (2 units in the last place).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Element types of activations and logits (MLLB_TYPE_* of the public header).
enum : int { kTypeF32 = 0, kTypeF16 = 1, kTypeBf16 = 2 };

// N consecutive values of a row as fp32 (N x the type's size: 4, 8 or 16 bytes, aligned to that).
template <int kType, int N>
__device__ __forceinline__ void load_values(const void* base, long long index, float (&x)[N]) {
  constexpr int kWords = kType == kTypeF32 ? N : N / 2;
  uint32_t w[kWords];
  const uint32_t* p = reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(base) +
                                                        index * (kType == kTypeF32 ? 4 : 2));
  if constexpr (kWords == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (kWords == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *p;
  }
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    if constexpr (kType == kTypeF32) {
      x[i] = __uint_as_float(w[i]);
    } else {
      const float2 f = unpack16<kType == kTypeBf16>(w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}

template <bool kBf16, int N>
__device__ __forceinline__ void store_values16(uint16_t* p, const float (&x)[N]) {
  if constexpr (N == 4)
    *reinterpret_cast<uint2*>(p) = make_uint2(pack16<kBf16>(x[0], x[1]), pack16<kBf16>(x[2], x[3]));
  else
    *reinterpret_cast<uint32_t*>(p) = pack16<kBf16>(x[0], x[1]);
}

struct AppendArgs {
  const void* qkv;          // [tokens][q_heads + 2 kv_heads][D], row stride qkv_stride
  const int32_t* positions; // [tokens] rotary positions
  const int32_t* rows;      // [tokens] row of the sequence, negative: padding
  const int32_t* seq;       // [tokens] sequence, nullptr: token t is sequence t's
  const int32_t* table;     // [seqs][width]
  const float* q_gamma;     // [D] or nullptr (no norm)
  const float* k_gamma;
  const double* freqs;      // [rot / 2] radians per position
  uint16_t* q_out;          // [tokens][q_heads][D]
  PagedCache cache;
  long long qkv_stride;
  int tokens, q_heads, seqs, width, rot, interleaved;
  int heads_per_warp, warps_per_token;
  float eps, magnitude;
};

constexpr int kAppendWarps = 8;

// A warp takes heads_per_warp heads of one token, one at a time; a lane holds
// D / 32 consecutive elements.
//   norm:     y = x / sqrt(sum(x^2) / D + eps) * gamma            (fp32)
//   rotation: y'_e = y_e c_e + y_partner(e) s_e,  c = m cos, s = -+ m sin
// The angle position * freq is taken in fp64 as turns and reduced to half a
// turn before the fp32 sine and cosine: at position 1e6 an fp32 product would
// be off by up to 0.06 rad.  A lane keeps the cosines and sines of its
// elements for all its heads; warps share nothing, so none waits for another
// (with a table made once a CTA and token, 8190 tokens of 48 heads took 86 us,
// now 60: those CTAs were too short for their latencies).
// Bound: HBM for prompts, one value in, one 16-bit value out; a warp has two
// heads' loads on their way, the first before the sines are made (8190 tokens of
// 48 fp32 heads: 60 us, 5.0 TB/s).  One token: the chain row -> page -> stores
// and the launch (2.5 us).
template <int D, int kType, bool kBf16>
__global__ void __launch_bounds__(kAppendWarps * 32, 4) paged_append_kernel(const AppendArgs a) {
  constexpr int N = D / 32, kAhead = 2;
  __shared__ float exchange[kAppendWarps][D];
  pdl_wait_prerequisite();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int unit = blockIdx.x * kAppendWarps + warp, token = unit / a.warps_per_token;
  if (token >= a.tokens) return;
  const int kv_heads = a.cache.kv_heads, heads = a.q_heads + 2 * kv_heads;
  const int head0 = unit % a.warps_per_token * a.heads_per_warp, head1 = min(head0 + a.heads_per_warp, heads);
  float x[kAhead][N];
  auto load = [&](int first) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (first + i < head1) load_values<kType, N>(a.qkv, token * a.qkv_stride + (first + i) * D + lane * N, x[i]);
  };
  load(head0);
  const int row = a.rows[token];
  if (row < 0) return;  // padding: nothing is stored
  const int half = a.rot >> 1;
  const int seq = a.seq ? a.seq[token] : token;
  const int slot = row >> a.cache.page_shift;
  int page = -1;
  if (seq >= 0 && seq < a.seqs && slot < a.width) page = a.table[static_cast<long long>(seq) * a.width + slot];
  const bool stored = page >= 0 && page < a.cache.pages;
  if (!stored && lane == 0 && head0 == 0) record_error(kErrBadPage);
  const long long cache_row = stored ? page * a.cache.page_stride +
                                           (row & ((1 << a.cache.page_shift) - 1)) * a.cache.row_stride : 0;
  float gq[N], gk[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    gq[j] = a.q_gamma ? a.q_gamma[lane * N + j] : 1.0f;
    gk[j] = a.k_gamma ? a.k_gamma[lane * N + j] : 1.0f;
  }
  // Pairs lane * kPairs + q of the rotation: made here, handed round below.
  constexpr int kPairs = D / 64;
  float pc[kPairs], ps[kPairs];
  const double position = a.positions[token] * 0.15915494309189533577;  // x freq: turns
#pragma unroll
  for (int q = 0; q < kPairs; ++q) {
    const int pair = lane * kPairs + q;
    const double turns = pair < half ? position * a.freqs[pair] : 0.0;
    float sn, cs;
    sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &sn, &cs);
    pc[q] = cs * a.magnitude;
    ps[q] = sn * a.magnitude;
  }
  // This lane's cosines and signed sines, and where each element's partner is:
  // in the lane (interleaved), at the same place of another lane (half a
  // rotation is a whole number of lanes), or anywhere.
  float c[N], s[N];
  int partner[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int e = lane * N + j;
    const bool turns = e < a.rot, second = a.interleaved ? (e & 1) : e >= half;
    const int pair = !turns ? 0 : a.interleaved ? e >> 1 : (second ? e - half : e);
    float cs = __shfl_sync(0xffffffffu, pc[0], pair / kPairs), sn = __shfl_sync(0xffffffffu, ps[0], pair / kPairs);
    if constexpr (kPairs == 2) {
      const float c1 = __shfl_sync(0xffffffffu, pc[1], pair / 2), s1 = __shfl_sync(0xffffffffu, ps[1], pair / 2);
      if (pair & 1) cs = c1, sn = s1;
    }
    c[j] = turns ? cs : 1.0f;
    s[j] = !turns ? 0.0f : second ? sn : -sn;
    partner[j] = !turns ? e : a.interleaved ? e ^ 1 : (second ? e - half : e + half);
  }
  const bool by_lane = half % N == 0;
  for (int first = head0; first < head1; first += kAhead) {
    float y[kAhead][N];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) y[i][j] = x[i][j];
    load(first + kAhead);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int head = first + i;
      if (head >= head1) break;
      const bool is_q = head < a.q_heads, is_v = head >= a.q_heads + kv_heads;
      if (!is_v) {
        if (is_q ? a.q_gamma : a.k_gamma) {
          float sum = 0.0f;
#pragma unroll
          for (int j = 0; j < N; ++j) sum = fmaf(y[i][j], y[i][j], sum);
          const float scale = rsqrtf(warp_sum_float_butterfly(sum) * (1.0f / D) + a.eps);
#pragma unroll
          for (int j = 0; j < N; ++j) y[i][j] = y[i][j] * scale * (is_q ? gq[j] : gk[j]);
        }
        float other[N];
        if (a.interleaved) {
#pragma unroll
          for (int j = 0; j < N; ++j) other[j] = y[i][j ^ 1];
        } else if (by_lane) {
#pragma unroll
          for (int j = 0; j < N; ++j) other[j] = __shfl_sync(0xffffffffu, y[i][j], partner[j] / N);
        } else {
          float* ex = exchange[warp];
          __syncwarp();
#pragma unroll
          for (int j = 0; j < N; ++j) ex[lane * N + j] = y[i][j];
          __syncwarp();
#pragma unroll
          for (int j = 0; j < N; ++j) other[j] = ex[partner[j]];
        }
#pragma unroll
        for (int j = 0; j < N; ++j) y[i][j] = fmaf(other[j], s[j], y[i][j] * c[j]);
      }
      if (is_q) {
        store_values16<kBf16, N>(a.q_out + (static_cast<long long>(token) * a.q_heads + head) * D + lane * N, y[i]);
      } else if (stored) {
        const int h = head - a.q_heads - (is_v ? kv_heads : 0);
        store_values16<kBf16, N>((is_v ? a.cache.v : a.cache.k) + cache_row + h * a.cache.head_stride + lane * N, y[i]);
      }
    }
  }
}

struct ReorderArgs {
  const int32_t* parents;  // [batch][beams] beam of the same batch entry, negative: the row ends
  const int32_t* table;    // [batch * beams][width]
  const int32_t* lens;     // [batch * beams]
  const int32_t* fresh;    // [batch * beams] a free page for each row
  int32_t* table_out;
  int32_t* lens_out;
  int32_t* used;
  PagedCache cache;
  int beams, width, row_bytes;
};

constexpr int kReorderWarps = 8;
constexpr int kReorderAhead = 8;

// CTA (x, row): the pages of its rows and the length come from its parent's row;
// the first CTA writes them.  Columns behind stay the row's own, pages that its
// caller reserved ahead: the parent's would be every child's, who would write
// over one another.  Where the row's own rows were is no such page (a sibling may
// hold it), so those columns become -1.  A page that is part full goes on being
// written by its beam, so only the first child of a parent keeps it: the others take
// fresh[row], and the CTAs copy the rows held so far, one (layer, K or V,
// head) a warp, 16 bytes a lane.  Bound: HBM where there is much to copy, as
// many bytes in as out (16 x 8 beams, 36 layers of 8 heads, 13 rows of a page:
// 52 us, 78 % of the copy rate).  4 beams: latency (2.9 us).
__global__ void __launch_bounds__(kReorderWarps * 32) beam_reorder_kernel(const ReorderArgs a) {
  pdl_wait_prerequisite();
  pdl_launch_dependents();
  const int row = blockIdx.y, beam = row % a.beams, first = row - beam;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int parent = a.parents[row];
  const bool leads = blockIdx.x == 0;
  if (parent < 0 || parent >= a.beams) {
    if (leads) {
      for (int i = threadIdx.x; i < a.width; i += blockDim.x) a.table_out[static_cast<long long>(row) * a.width + i] = -1;
      if (threadIdx.x == 0) {
        a.lens_out[row] = 0;
        a.used[row] = 0;
        if (parent >= a.beams) record_error(kErrBadParent);
      }
    }
    return;
  }
  bool further = false;  // an earlier row has the same parent
  for (int i = lane; i < beam; i += 32) further |= a.parents[first + i] == parent;
  further = __any_sync(0xffffffffu, further);
  const int32_t* from = a.table + static_cast<long long>(first + parent) * a.width;
  const int len = a.lens[first + parent];
  const int part = len & ((1 << a.cache.page_shift) - 1), slot = len >> a.cache.page_shift;
  const bool valid = len >= 0 && slot + (part > 0) <= a.width;
  const int source = valid && part > 0 ? from[slot] : -1, target = a.fresh[row];
  const bool wants = valid && further && part > 0;
  const bool copies = wants && source >= 0 && source < a.cache.pages && target >= 0 && target < a.cache.pages;
  if (leads) {
    const int32_t* mine = a.table + static_cast<long long>(row) * a.width;
    const int held = len < 0 ? 0 : slot + (part > 0), len0 = a.lens[row];
    const int past = len0 < 0 ? a.width : (len0 >> a.cache.page_shift) + ((len0 & ((1 << a.cache.page_shift) - 1)) > 0);
    for (int i = threadIdx.x; i < a.width; i += blockDim.x)
      a.table_out[static_cast<long long>(row) * a.width + i] =
          i < held ? (copies && i == slot ? target : from[i]) : i < past ? -1 : mine[i];
    if (threadIdx.x == 0) {
      a.lens_out[row] = len;
      a.used[row] = copies;
      if (!valid || wants != copies) record_error(kErrBadPage);
    }
  }
  if (!copies) return;
  const int units = a.row_bytes / 16, triples = a.cache.layers * 2 * a.cache.kv_heads;
  for (int w = blockIdx.x * kReorderWarps + warp; w < triples; w += gridDim.x * kReorderWarps) {
    const int h = w % a.cache.kv_heads, kv = w / a.cache.kv_heads & 1, layer = w / a.cache.kv_heads / 2;
    uint16_t* base = (kv ? a.cache.v : a.cache.k) + layer * a.cache.layer_stride + h * a.cache.head_stride;
    const uint16_t* src = base + source * a.cache.page_stride;
    uint16_t* dst = base + target * a.cache.page_stride;
    // (units is 8 or 16: head_dim 64 or 128.)  Eight 16-byte loads a lane on their way.
    const int shift = units == 16 ? 4 : 3, all = part << shift;
    for (int u0 = lane; u0 < all; u0 += 32 * kReorderAhead) {
      uint4 v[kReorderAhead];
      long long at[kReorderAhead];
#pragma unroll
      for (int i = 0; i < kReorderAhead; ++i) {
        const int u = u0 + 32 * i;
        at[i] = static_cast<long long>(u >> shift) * a.cache.row_stride + (u & (units - 1)) * 8;
        if (u < all) v[i] = *reinterpret_cast<const uint4*>(src + at[i]);
      }
#pragma unroll
      for (int i = 0; i < kReorderAhead; ++i)
        if (u0 + 32 * i < all) *reinterpret_cast<uint4*>(dst + at[i]) = v[i];
    }
  }
}

}  // namespace mllb
