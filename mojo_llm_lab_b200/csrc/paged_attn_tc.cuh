// Attention over the paged cache where a key serves many query rows (a long
// prefix under a batch's queries, prompts): the products run on the
// 5th-generation tensor cores.
//
// One persistent CTA per SM walks its share of the line (paged_attn.cuh) with
// R = 256 rows an item, as two streams of 128 rows (a TMEM lane each) that use
// the same key tiles of 128:
//   warps 0-3, 4-7  softmax of stream 0, 1: a thread is a row
//   warp 8          TMA copies of K and V tiles into a ring
//   warp 9          issues the matrix instructions, owns TMEM
//   warp 10         walks the line ahead, posts the segments, fetches their queries
//   warp 11         fills the warpgroup, whose registers the softmax takes
// S = Q K^T goes to 128 TMEM columns a stream; the softmax reads it, writes
// P over it in 16 bits, and P V adds to the stream's D columns of O, with P
// read from TMEM and V from shared memory as it lies in the cache (MN-major).
// While one stream's softmax runs, the tensor cores work for the other.  P is
// handed over in two halves, so that the first is multiplied while the second
// is made.
//
// The running maximum is moved, and O rescaled, only when a row's scores
// outgrow it by 2^8: until then its weights are up to 2^8 instead of up to 1
// (2^15 with fp16's lift of 7), which the 16-bit types hold as well and fp32
// sums too.  After the first tiles O is hardly ever touched by the softmax
// warps.  The price is that the largest weight is not 1, which has no rounding:
// prompts in bf16 are 2.3e-3 off the exact values (rounding the result alone is
// 1.7e-3), ragged sequences in the few-row kernel, whose maxima always move, 1.8e-3.
//
// Where an item ends, the next one's queries and first keys are on their way
// already: warp 10 posts segments two ahead and lets TMA bring their queries
// once the last scores of the one before are made (read by the softmax warps
// themselves, they cost 10 000 cycles an item: prompts 180 -> 151 us).  Results
// go through registers so that stores cover whole lines (transpose8).
//
// Bound: a key tile of 256 rows takes the tensor cores 2048 cycles and the
// exponentials as many (16 a cycle), the rest of the softmax issue slots beside
// them; the two streams hide less of one behind the other than they might, and
// the clock falls under this load.  4 prompts of up to 1024 tokens behind a
// prefix of 1500 rows (119 GFLOP): 150 us on changing inputs, 0.79 PFLOP/s, 130
// us replayed on one; one of 8000 tokens, replayed, 447 to 490 (it goes by the
// clock), 1.07 to 1.17.  With heads of 128 the 168 registers do not quite do
// (52 to 56 bytes of spill stores a thread).
#pragma once

#include "paged_attn.cuh"
#include "prefill.cuh"

namespace mllb {

template <int D>
struct AttnMany {
  static constexpr int kRows = 256, kKeys = 128;
  static constexpr int kThreads = 384;            // three warpgroups
  // Registers a thread: the launch's, then the softmax warpgroups' and the
  // third's (setmaxnreg moves them; the sum must not exceed the launch's).
  static constexpr int kRegs = 168, kSoftmaxRegs = 208, kOtherRegs = 88;
  static_assert(2 * kSoftmaxRegs + kOtherRegs <= 3 * kRegs, "register split");
  static constexpr int kQTile = 128 * D * 2;      // one stream's queries
  static constexpr int kTile = kKeys * D * 2;     // a K or V tile: a ring slot
  static constexpr int kSlots = D == 128 ? 5 : 8;
  static constexpr int kRingOff = 2 * kQTile;
  static constexpr int kBarOff = kRingOff + kSlots * kTile;
  static constexpr int kPosts = 2;                // segments posted ahead
  static constexpr int kBars = 2 * kSlots + 6 * 2 + 1 + 2 * kPosts;
  static constexpr int kPostOff = kBarOff + (kBars + 1) * 8;
  static constexpr int kSmem = kPostOff + kPosts * static_cast<int>(sizeof(AttnSegment));
  static constexpr int kTmemCols = 512;           // S (P over it) 2 x 128, O 2 x D
  static constexpr uint32_t kSCol = 0, kOCol = 256;
  static_assert(kSmem <= 227 * 1024, "shared memory");
  static_assert(kSlots * kTile >= (2 * (kAttnMaxEntities + 1) + 64) * 4, "the scan fits in the ring");
};

// Shared-memory descriptor, 128-byte swizzle.  K-major (Q, K): 8-row groups at
// sbo; MN-major (V): 8-key groups at sbo, blocks of 64 elements at lbo.
__device__ __forceinline__ uint64_t attn_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return pf_smem_desc(saddr, lbo, sbo) | (2ull << 61);
}

// kind::f16 instruction descriptor: D fp32, A and B of the cache's type, M = 128.
template <bool kBf16>
__host__ __device__ constexpr uint32_t attn_idesc(int n, bool b_mn_major) {
  return (1u << 4) | (kBf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn_major ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(n >> 3) << 17) | ((128u >> 4) << 24);
}

// Matrix instruction and commit by one elected lane: all lanes of the warp call
// them with the same operands.
__device__ __forceinline__ void tc_mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add)
      : "memory");
}
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add)
      : "memory");
}
__device__ __forceinline__ void tc_commit_elected(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
      ::"r"(smem_addr(bar))
      : "memory");
}

// 32 TMEM columns of this thread's lane (issue only), and 16 columns back.
__device__ __forceinline__ void tc_ld32(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
        "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Eight 16-byte pieces of this lane's row -> piece `lane % 8` of the rows of the
// eight lanes around it, so that a store covers 128 bytes of four rows and not
// 16 of 32.
__device__ __forceinline__ void transpose8(uint4 (&v)[8], int lane) {
#pragma unroll
  for (int d = 1; d < 8; d <<= 1) {
    const bool upper = lane & d;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j & d) continue;
      uint4 give = upper ? v[j] : v[j | d];
      give.x = __shfl_xor_sync(0xffffffffu, give.x, d);
      give.y = __shfl_xor_sync(0xffffffffu, give.y, d);
      give.z = __shfl_xor_sync(0xffffffffu, give.z, d);
      give.w = __shfl_xor_sync(0xffffffffu, give.w, d);
      if (upper) v[j] = give; else v[j | d] = give;
    }
  }
}

template <int D, bool kBf16>
__global__ void __launch_bounds__(384, 1)
    paged_attn_many_kernel(const AttnArgs a, const AttnPass pass, const __grid_constant__ CUtensorMap kmap,
                           const __grid_constant__ CUtensorMap vmap, const __grid_constant__ CUtensorMap qmap,
                           const int q_by_tma) {
  using C = AttnMany<D>;
  constexpr int R = C::kRows, KT = C::kKeys, NS = C::kSlots;
  constexpr float kLift = attn_lift(kBf16, 7);  // weights reach 2^8 above the running maximum's
  extern __shared__ __align__(1024) uint8_t attn_smem[];
  uint8_t* ring = attn_smem + C::kRingOff;
  uint64_t* full = reinterpret_cast<uint64_t*>(attn_smem + C::kBarOff);  // [NS] a tile has landed
  uint64_t* empty = full + NS;                                            // [NS] its products are done
  uint64_t* q_full = empty + NS;                                          // [2] a stream's queries are in shared memory
  uint64_t* s_full = q_full + 2;                                          // [2] its scores are in TMEM
  uint64_t* p_full = s_full + 2;                                          // [2][2 halves] its weights are, and O is at their scale
  uint64_t* o_done = p_full + 4;                                          // [2] its products with V are done
  uint64_t* drained = o_done + 2;
  uint64_t* q_empty = drained + 1;                                        // [2] a segment's last scores are made
  uint64_t* post_full = q_empty + 2;                                      // [kPosts] a segment is posted
  uint64_t* post_empty = post_full + C::kPosts;                           // [kPosts] all warps have read it
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(post_empty + C::kPosts);
  AttnSegment* posts = reinterpret_cast<AttnSegment*>(attn_smem + C::kPostOff);
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], q_by_tma ? 1 : 4);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&o_done[i], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&p_full[i], 4);
    for (int i = 0; i < C::kPosts; ++i) {
      mbar_init(&post_full[i], 1);
      mbar_init(&post_empty[i], 10);
    }
    mbar_init(drained, 1);
    fence_mbar_init();
    tma_prefetch_map(&kmap);
    tma_prefetch_map(&vmap);
    tma_prefetch_map(&qmap);
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                 "r"(C::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait_prerequisite();
  pdl_launch_dependents();
  const AttnCursor start = attn_start<R, KT, C::kThreads>(a, pass, reinterpret_cast<int*>(ring));
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the scan used the ring
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // The posted segments in their order; false behind the last (or when the
  // walk gave up).  Every warp but the walking one takes each.
  int post = 0;
  auto take = [&](AttnSegment* s) {
    const int at = post % C::kPosts;
    if (!mbar_wait_bounded(&post_full[at], (post / C::kPosts) & 1)) {
      record_error(kErrFullWaitTimeout);
      return false;
    }
    *s = posts[at];
    __syncwarp();
    if (lane == 0) mbar_arrive(&post_empty[at]);
    ++post;
    return s->of > 0;
  };
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kOtherRegs));
    if (warp == 10) {
      // ------------------------------------------------ the walk along the line, ahead of the others
      AttnWalk<R, KT> walk(a, pass, start);
      AttnSegment s = {}, last = {};
      int segments = 0, fetched[2] = {0, 0};
      for (bool more = true; more; ++post) {
        more = walk.next(&s);
        if (more) {
          ++segments;
          last = s;
          if (lane == 0) {
            if (pass.dense)
              attn_leave_item(pass, s);
            else if (pass.by_item)
              attn_leave_cut(a, pass, start, s, segments, false, R);
          }
        } else {
          s.of = 0;
        }
        const int at = post % C::kPosts;
        if (post >= C::kPosts && !mbar_wait_bounded(&post_empty[at], (post / C::kPosts - 1) & 1)) {
          record_error(kErrEmptyWaitTimeout);
          break;
        }
        if (lane == 0) {
          posts[at] = s;
          mbar_arrive(&post_full[at]);
        }
        __syncwarp();
        if (!more || !q_by_tma) continue;
        // The queries, as soon as the segment before is through with its own.
        // Rows behind the entity's are other tokens' (or zeros): their results
        // go nowhere.
        for (int i = 0; i < 2; ++i) {
          if (i && s.ent.ntok * a.ratio - s.t * R <= 128) break;
          if (fetched[i] && !mbar_wait_bounded(&q_empty[i], (fetched[i] - 1) & 1)) {
            record_error(kErrEmptyWaitTimeout);
            more = false;
            break;
          }
          ++fetched[i];
          if (lane == 0) mbar_arrive_expect_tx(&q_full[i], C::kQTile);
          __syncwarp();
          if (lane < D / 64)
            tma_load_4d(attn_smem + i * C::kQTile + lane * (128 * 128), &qmap, lane * 64, 0, s.h,
                        s.ent.tok0 + (s.t * R + i * 128) / a.ratio, &q_full[i]);
        }
      }
      for (int i = 0; i < 2; ++i)  // the last copies land before the CTA's shared memory is given back
        if (fetched[i] && !mbar_wait_bounded(&q_full[i], (fetched[i] - 1) & 1)) record_error(kErrDrainTimeout);
      if (!pass.dense && !pass.by_item && lane == 0) attn_leave_cut(a, pass, start, last, segments, true, R);
    } else if (warp == 8) {
      // ------------------------------------------------ copies: K and V tiles in turn, a box a lane
      AttnSegment s;
      const int box_rows = min(1 << a.page_shift, KT), per_tile = KT / box_rows;
      constexpr int kHalves = D / 64;
      const int boxes = per_tile * kHalves;
      int n = 0;
      bool stuck = false;
      while (!stuck && take(&s)) {
        for (int k = s.begin; k < s.end && !stuck; ++k) {
          const AttnTile tile = attn_tile<KT>(s.ent, k);
          const int p = lane % per_tile, half = lane / per_tile;
          int page = 0;
          if (lane < boxes) page = attn_page(a, tile, p * box_rows);
          const int in_page = (tile.row0 + p * box_rows) & ((1 << a.page_shift) - 1);
#pragma unroll
          for (int is_v = 0; is_v < 2; ++is_v) {
            const int st = n % NS;
            if (n >= NS && !mbar_wait_bounded(&empty[st], (n / NS - 1) & 1)) {
              record_error(kErrEmptyWaitTimeout);
              stuck = true;
              break;
            }
            if (lane == 0) mbar_arrive_expect_tx(&full[st], C::kTile);
            __syncwarp();
            if (lane < boxes)
              tma_load_4d(ring + st * C::kTile + half * (KT * 128) + p * box_rows * 128, is_v ? &vmap : &kmap, half * 64,
                          in_page, s.h, page, &full[st]);
            ++n;
          }
        }
      }
      for (int i = max(n - NS, 0); i < n; ++i)
        if (!mbar_wait_bounded(&full[i % NS], (i / NS) & 1)) record_error(kErrDrainTimeout);
    } else if (warp == 9) {
      // ------------------------------------------------ matrix instructions
      AttnSegment s;
      constexpr uint32_t kQk = attn_idesc<kBf16>(KT, false), kPv = attn_idesc<kBf16>(D, true);
      const uint64_t q_desc = attn_desc(smem_addr(attn_smem), 16, 1024), k_desc = attn_desc(smem_addr(ring), 16, 1024),
                     v_desc = attn_desc(smem_addr(ring), KT * 128, 1024);
      int n = 0;  // ring position of the next K tile to use
      int qn = 0, pn = 0, qn1 = 0, pn1 = 0;
      bool ok = true;
      auto wait = [&](uint64_t* bar, int phase) {
        if (ok && !mbar_wait_bounded(bar, phase & 1)) {
          record_error(kErrFullWaitTimeout);
          ok = false;
        }
        ok = __all_sync(0xffffffffu, ok);
        return ok;
      };
      auto scores = [&](int stream, int pos) {
        const uint64_t qd = q_desc + stream * (C::kQTile >> 4), kd = k_desc + (pos % NS) * (C::kTile >> 4);
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          const int off = ((c >> 2) * (128 * 128) + (c & 3) * 32) >> 4;  // 64 elements a swizzled row, 32 bytes a step
          tc_mma_f16_ss(tmem + C::kSCol + stream * 128, qd + off, kd + off, kQk, c > 0);
        }
        tc_commit_elected(&s_full[stream]);
      };
      while (ok && take(&s)) {
        const bool both = s.ent.ntok * a.ratio - s.t * R > 128;
        const int tiles = s.end - s.begin;
        wait(&q_full[0], qn++);
        if (both) wait(&q_full[1], qn1++);
        wait(&full[n % NS], n / NS);
        if (!ok) break;
        tc_fence_after();
        scores(0, n);
        if (tiles == 1) tc_commit_elected(&q_empty[0]);
        if (both) {
          scores(1, n);
          if (tiles == 1) tc_commit_elected(&q_empty[1]);
        }
        tc_commit_elected(&empty[n % NS]);
        for (int k = 0; k < tiles; ++k, n += 2) {
          const int vpos = n + 1, kpos = n + 2;
          const bool more = k + 1 < tiles;
          wait(&full[vpos % NS], vpos / NS);
          if (more) wait(&full[kpos % NS], kpos / NS);
          const uint64_t vd = v_desc + (vpos % NS) * (C::kTile >> 4);
          auto products = [&](int stream, int phase) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {  // the second half's weights come while the first is multiplied
              if (!wait(&p_full[2 * stream + half], phase)) return;
              tc_fence_after();
#pragma unroll
              for (int c = half * (KT / 32); c < (half + 1) * (KT / 32); ++c)
                tc_mma_f16_ts(tmem + C::kOCol + stream * 128, tmem + C::kSCol + stream * 128 + c * 8, vd + c * (2048 >> 4),
                              kPv, k > 0 || c > 0);
            }
            tc_commit_elected(&o_done[stream]);
            if (more) scores(stream, kpos);  // over P, which the products before it have read: they run in order
            if (k + 2 == tiles) tc_commit_elected(&q_empty[stream]);
          };
          products(0, pn++);
          if (both) products(1, pn1++);
          if (!ok) break;
          tc_commit_elected(&empty[vpos % NS]);
          if (more) tc_commit_elected(&empty[kpos % NS]);
        }
      }
      // Nothing is in flight when TMEM is given back.
      tc_commit_elected(drained);
      if (!mbar_wait_bounded(drained, 0)) record_error(kErrDrainTimeout);
      __syncwarp();
    }
  } else {
    // ------------------------------------------------ softmax: this thread's row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kSoftmaxRegs));
    const int stream = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t s_col = lanes + C::kSCol + stream * 128, o_col = lanes + C::kOCol + stream * 128;  // P over S
    const float scale = fmaxf(fabsf(a.scale_log2), 1e-30f);  // q carries the sign; 0 x a masked -inf must not come up
    const uint32_t flip = a.scale_log2 < 0.0f ? 0x80008000u : 0u;
    int sn = 0, ring_pos = 0;
    bool first = true, stuck = false;
    auto wait = [&](uint64_t* bar, int phase) {
      if (!stuck && !mbar_wait_bounded(bar, phase & 1)) {
        record_error(kErrFullWaitTimeout);
        stuck = true;
      }
    };
    struct Row {
      int token, head, limit;  // token -1: no such row
    };
    // The thread's row of a segment; its queries brought to shared memory where
    // the copies do not (a ratio that does not divide 128, a negative scale).
    auto load_queries = [&](const AttnSegment& s) {
      const int at = s.t * R + stream * 128 + r;
      const bool there = at < s.ent.ntok * a.ratio;
      const int j = there ? at / a.ratio : 0;
      const Row row = {there ? s.ent.tok0 + j : -1, s.h * a.ratio + (there ? at - j * a.ratio : 0),
                       there ? attn_limit(s.ent, j) : 0};
      if (!q_by_tma) {
        const uint4* src = reinterpret_cast<const uint4*>(a.q + max(row.token, 0) * a.q_token + row.head * a.q_head);
        uint8_t* dst = attn_smem + stream * C::kQTile + r * 128;
#pragma unroll 4
        for (int c = 0; c < D / 8; ++c) {
          uint4 v = there ? src[c] : make_uint4(0, 0, 0, 0);
          v.x ^= flip, v.y ^= flip, v.z ^= flip, v.w ^= flip;
          *reinterpret_cast<uint4*>(dst + (c >> 3) * (128 * 128) + (((c & 7) ^ (r & 7)) << 4)) = v;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[stream]);
      }
      return row;
    };
    // The next segment with rows of this stream; the tiles of those without pass by.
    auto take_own = [&](AttnSegment* s) {
      for (;; ring_pos += 2 * (s->end - s->begin), first = false) {
        if (!take(s)) return false;
        if (!stream || s->ent.ntok * a.ratio - s->t * R > 128) return true;
      }
    };
    AttnSegment s;
    Row row = {};
    bool more = take_own(&s);
    if (more) row = load_queries(s);
    while (more && !stuck) {
      // Rows that do not exist are other tokens' (being written, where out is q):
      // nothing outgrows their maximum, so they have no say in when the warp's move.
      float top = row.token >= 0 ? -INFINITY : INFINITY, sum = 0.0f;
      for (int k = s.begin; k < s.end; ++k, ++sn) {
        const AttnTile tile = attn_tile<KT>(s.ent, k);
        const int held = tile.rows - tile.row0;
        if (stream == 0 && held < KT) {
          // V rows behind the end may hold anything, and a weight of zero does
          // not make NaN vanish: they become zero before the products.
          const int pos = ring_pos + 2 * (k - s.begin) + 1;
          wait(&full[pos % NS], pos / NS);
          uint8_t* vt = ring + (pos % NS) * C::kTile;
          for (int i = threadIdx.x; i < (KT - held) * (D / 8); i += 128) {
            const int key = held + i / (D / 8), c = i % (D / 8);
            *reinterpret_cast<uint4*>(vt + (c >> 3) * (KT * 128) + key * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        wait(&s_full[stream], sn);
        tc_fence_after();
        float x[KT];
#pragma unroll
        for (int c = 0; c < KT; c += 32) tc_ld32(s_col + c, x + c);
        tc_wait_ld();
        const int end = min(tile.own ? row.limit : tile.rows, tile.rows) - tile.row0;
        if (__any_sync(0xffffffffu, end < KT)) {
#pragma unroll
          for (int c = 0; c < KT; ++c) x[c] = c < end ? x[c] : -INFINITY;
        }
        // Four chains of three-input maxima.
        float mc[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int c = 4; c + 8 <= KT; c += 8)
#pragma unroll
          for (int i = 0; i < 4; ++i) mc[i] = fmaxf(fmaxf(mc[i], x[c + i]), x[c + 4 + i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) mc[i] = fmaxf(mc[i], x[KT - 4 + i]);
        const float m = fmaxf(fmaxf(mc[0], mc[1]), fmaxf(mc[2], mc[3])) * scale;
        if (__any_sync(0xffffffffu, m > top + 8.0f)) {
          const float z = fmaxf(m, top), f = z == -INFINITY ? 0.0f : ex2(top - z);
          top = z;
          sum *= f;
          if (k > s.begin) {
            wait(&o_done[stream], sn - 1);
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < D; c += 32) {
              float o[32];
              tc_ld32(o_col + c, o);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] *= f;
              tc_st16(o_col + c, reinterpret_cast<uint32_t*>(o));
              tc_st16(o_col + c + 16, reinterpret_cast<uint32_t*>(o) + 16);
            }
          }
        }
        const float z = top == -INFINITY ? 0.0f : top - kLift;
        float2 part[4] = {};
        // P in the cache's type: half a step off at most, in fp16 from 2^-21 of
        // the running maximum's weight on, and 2^-32 of that one below; the sum
        // keeps the unrounded weights.
#pragma unroll
        for (int c = 0; c < KT; c += 32) {
          uint32_t p[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float2 w = __ffma2_rn(make_float2(x[c + 2 * i], x[c + 2 * i + 1]), make_float2(scale, scale), make_float2(-z, -z));
            w.x = ex2(w.x);
            w.y = ex2(w.y);
            part[i & 3] = __fadd2_rn(part[i & 3], w);
            p[i] = pack16<kBf16>(w.x, w.y);
          }
          tc_st16(s_col + c / 2, p);
          if ((c + 32) % (KT / 2) == 0) {  // a half is complete
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[2 * stream + c / (KT / 2)]);
          }
        }
        part[0] = __fadd2_rn(__fadd2_rn(part[0], part[1]), __fadd2_rn(part[2], part[3]));
        sum += part[0].x + part[0].y;
      }
      // The next segment's queries can come in now (this one's last scores are
      // made), so that its first scores are there when O has been read.
      const bool whole = s.begin == 0 && s.end == s.of;
      const bool direct = whole && !pass.dense;
      const int slot = pass.dense ? static_cast<int>(blockIdx.x) + s.item : 2 * static_cast<int>(blockIdx.x) + !first;
      const Row mine = row;
      ring_pos += 2 * (s.end - s.begin);
      first = false;
      more = take_own(&s);
      if (more) row = load_queries(s);
      wait(&o_done[stream], sn - 1);
      tc_fence_after();
      const bool fits = slot < pass.slots, keeps = !direct && fits && mine.token >= 0;
      if (!direct && !fits) record_error(kErrBadPage);
      const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
      const long long at = static_cast<long long>(slot) * R + stream * 128 + r;
      if (keeps) pass.stats[at] = make_float2(top - kLift, sum);
      const int near = lane & ~7, piece = lane & 7;
      if (direct) {
        const long long place = mine.token * a.out_token + mine.head * a.out_head;
#pragma unroll 1
        for (int c = 0; c < D; c += 64) {
          uint4 v[8];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float o[32];
            tc_ld32(o_col + c + 32 * h, o);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 4; ++i)
              v[4 * h + i] = make_uint4(pack16<kBf16>(o[8 * i] * inv, o[8 * i + 1] * inv),
                                        pack16<kBf16>(o[8 * i + 2] * inv, o[8 * i + 3] * inv),
                                        pack16<kBf16>(o[8 * i + 4] * inv, o[8 * i + 5] * inv),
                                        pack16<kBf16>(o[8 * i + 6] * inv, o[8 * i + 7] * inv));
          }
          transpose8(v, lane);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const long long to = __shfl_sync(0xffffffffu, place, near + i);
            const bool there = __shfl_sync(0xffffffffu, mine.token, near + i) >= 0;
            if (there) *reinterpret_cast<uint4*>(a.out + to + c + piece * 8) = v[i];
          }
        }
      } else if (fits) {
        float* row0 = pass.acc + (at - lane + near) * D + piece * 4;
        const unsigned rows = __ballot_sync(0xffffffffu, keeps) >> near;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          float o[32];
          tc_ld32(o_col + c, o);
          tc_wait_ld();
          uint4 v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            v[i] = make_uint4(__float_as_uint(o[4 * i]), __float_as_uint(o[4 * i + 1]), __float_as_uint(o[4 * i + 2]),
                              __float_as_uint(o[4 * i + 3]));
          transpose8(v, lane);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (rows >> i & 1) *reinterpret_cast<uint4*>(row0 + i * D + c) = v[i];
        }
      }
      tc_fence_before();  // the next item's products write O
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmemCols) : "memory");
  }
}

}  // namespace mllb
