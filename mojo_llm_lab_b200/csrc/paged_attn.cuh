// Attention of a batch of sequences over a paged cache, with prefixes that
// several sequences share.
//
//   out[t][h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - max)
//
// over the prefix of the token's group and the sequence's own rows up to the
// token's.  Work comes as entities: a sequence (its own rows, or its prefix
// and its own rows), or a group (its prefix under the queries of ALL its
// sequences, so that the prefix is read once).  An entity's query rows are
// (token, query head of a KV head), cut into tiles of R rows; a (row tile, KV
// head) is an item, and its keys are cut into tiles of KT.  The (item, key
// tile) pairs of all entities, in order, are one line that is cut into equal
// shares, one per CTA, whatever the lengths: no CTA idles because one context
// is long, and short ones are not padded.  The lengths are read on the device
// (each CTA adds them up for itself), so a captured graph stays right while
// they grow.
//
// A CTA's share of an item is a segment.  Where an item's rows get nothing from
// elsewhere, an item of one segment is written to out at once; other segments
// leave (maximum, sum, unnormalised accumulator) in fp32 in the workspace.
// paged_join_kernel joins the items that were cut (at most one for each CTA);
// where prefixes and own rows run apart, paged_merge_kernel joins all of a
// row's segments.
#pragma once

#include <cuda.h>

#include "paged.cuh"

namespace mllb {

enum : int {
  kAttnOwn = 0,     // entities: sequences, own rows only
  kAttnConcat = 1,  // entities: sequences, prefix then own rows
  kAttnBoth = 2,    // entities: groups' prefixes, then sequences' own rows
  kAttnPrefix = 3,  // entities: groups' prefixes
};

constexpr int kAttnMaxEntities = 2048;

struct AttnArgs {
  const uint16_t* q;  // [tokens][q_heads][D], strides in elements
  uint16_t* out;
  long long q_token, q_head, out_token, out_head;
  const int32_t* table;         // [seqs][width]
  const int32_t* lens;          // [seqs]
  const int32_t* prefix_table;  // [groups][prefix_width]
  const int32_t* prefix_lens;   // [groups]
  const int32_t* group_start;   // [groups + 1], nullptr: one group of all sequences
  const int32_t* q_start;       // [seqs + 1], nullptr: token b is sequence b's
  int width, prefix_width, seqs, groups, tokens, kv_heads, ratio, page_shift, pages;
  float scale_log2;  // scale x log2(e): the softmax runs on powers of two
};

// One launch's line of work and where its segments go.
struct AttnPass {
  int mode, entities, ctas;
  int dense;       // 1: segment of CTA c and item i at slot c + i; 0: at 2 c (a CTA's first) or 2 c + 1
  int slots;       // capacity of the workspace
  int rows, keys;  // R and KT of the kernel that ran it (for the merge)
  // For the kernel that joins.  dense: [entities] items before each entity, 1
  // (0: the starts descend, nothing was done), then int2 [items] first and last
  // CTA of an item; otherwise AttnCut, the number of records first (as segments),
  // then one an item (by_item: there are no more items than CTAs) or one a CTA.
  int32_t* plan;
  int by_item;
  float* acc;      // [slots][R][D]
  float2* stats;   // [slots][R] (maximum in powers of two, sum)
};

// An item that CTA `cta` began and others went on with (segments 0: none): how
// many segments, the slot of that CTA's, the item's first row of its entity's
// `rows`, its KV head and the entity's first token.
struct AttnCut {
  int segments, slot, row0, rows, h, tok0, cta, pad;
};

struct AttnEntity {
  int tok0, ntok, plen, len, causal;  // ntok < 0: starts that descend (attn_start: no work at all)
  const int32_t* ptab;
  const int32_t* tab;
};

__device__ __forceinline__ int attn_clamp_len(int len, int width, int page_shift) {
  const int most = width << page_shift;
  if (len < 0 || len > most) record_error(kErrBadPage);
  return min(max(len, 0), most);
}

__device__ __forceinline__ int attn_token_start(const AttnArgs& a, int seq) {
  if (!a.q_start) return min(max(seq, 0), a.tokens);
  return min(max(a.q_start[min(max(seq, 0), a.seqs)], 0), a.tokens);
}

// The group of a sequence, -1 if it has none.
__device__ __forceinline__ int attn_group_of(const AttnArgs& a, int seq) {
  if (a.groups == 0) return -1;
  if (!a.group_start) return 0;
  int lo = 0, hi = a.groups;  // group_start[lo] <= seq < group_start[hi], if any
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.group_start[mid] <= seq) lo = mid; else hi = mid;
  }
  return a.group_start[lo] <= seq && seq < a.group_start[lo + 1] ? lo : -1;
}

__device__ __forceinline__ AttnEntity attn_entity(const AttnArgs& a, int mode, int e) {
  AttnEntity n;
  n.plen = 0;
  n.ptab = nullptr;
  if (mode == kAttnPrefix || (mode == kAttnBoth && e < a.groups)) {
    const int s0 = a.group_start ? a.group_start[e] : 0, s1 = a.group_start ? a.group_start[e + 1] : a.seqs;
    n.tok0 = attn_token_start(a, s0);
    n.ntok = attn_token_start(a, s1) - n.tok0;
    n.len = attn_clamp_len(a.prefix_lens[e], a.prefix_width, a.page_shift);
    n.tab = a.prefix_table + static_cast<long long>(e) * a.prefix_width;
    n.causal = 0;
    return n;
  }
  const int seq = mode == kAttnBoth ? e - a.groups : e;
  n.tok0 = attn_token_start(a, seq);
  n.ntok = attn_token_start(a, seq + 1) - n.tok0;
  n.len = attn_clamp_len(a.lens[seq], a.width, a.page_shift);
  n.tab = a.table + static_cast<long long>(seq) * a.width;
  n.causal = 1;
  if (mode == kAttnConcat) {
    const int g = attn_group_of(a, seq);
    if (g >= 0) {
      n.plen = attn_clamp_len(a.prefix_lens[g], a.prefix_width, a.page_shift);
      n.ptab = a.prefix_table + static_cast<long long>(g) * a.prefix_width;
    }
  }
  return n;
}

// Own rows that the entity's token j sees.
__device__ __forceinline__ int attn_limit(const AttnEntity& n, int j) {
  return n.causal ? min(max(n.len - n.ntok + j + 1, 0), n.len) : n.len;
}

__device__ __forceinline__ int attn_row_tiles(const AttnEntity& n, int ratio, int R) {
  return (n.ntok * ratio + R - 1) / R;
}

// Key tiles of row tile t: the prefix's, then the own rows' up to the last
// token's limit.  least 1 makes an item of rows that see nothing, too (one
// masked tile), so that their zeros are written like other rows.
__device__ __forceinline__ int attn_key_tiles(const AttnEntity& n, int ratio, int t, int R, int KT, int least) {
  const int last = min(n.ntok * ratio, (t + 1) * R) - 1;
  return max((n.plen + KT - 1) / KT + (attn_limit(n, last / ratio) + KT - 1) / KT, least);
}

// An item's length on the line: its key tiles, and what its start and end cost
// beside them, on the tensor cores about as long as two key tiles (queries, first
// scores, results).  Without that the CTAs of short items end last: one prompt of
// 8000 tokens, whose first row tiles see one key tile, 638 -> 451 us (counted as
// one tile 515, as three 454), of 1000 tokens 41 -> 32.
__host__ __device__ constexpr int attn_ends(int R) { return R > 64 ? 2 : 0; }
__device__ __forceinline__ int attn_cost(int key_tiles, int R) { return key_tiles > 0 ? key_tiles + attn_ends(R) : 0; }

// First place of CTA c's share.  No more CTAs take part than there are places,
// so every one of an item's CTAs, first to last with a key tile, has a segment.
__device__ __forceinline__ int attn_share(int total, int ctas, int c) {
  return static_cast<int>(static_cast<long long>(total) * c / ctas);
}

// Where a CTA's share starts, and how far it goes.
struct AttnCursor {
  int total;       // all pairs
  int left;        // key tiles left in the share
  int e, t, h;     // entity, row tile, KV head
  int begin;       // where the share starts in the item
  int item;        // number of the item on the line
};

// Entity e's length on the line (attn_cost of its items) and its items; 0 past
// the last.  False where its starts descend.
template <int R, int KT>
__device__ __forceinline__ bool attn_work(const AttnArgs& a, const AttnPass& pass, int e, int* pairs, int* items) {
  int w = 0, t = 0;
  bool ascends = true;
  if (e < pass.entities) {
    const AttnEntity ent = attn_entity(a, pass.mode, e);
    ascends = ent.ntok >= 0;
    t = ascends ? attn_row_tiles(ent, a.ratio, R) : 0;
    if (ent.causal && ent.ntok > 1) {
      for (int i = 0; i < t; ++i) w += attn_cost(attn_key_tiles(ent, a.ratio, i, R, KT, !pass.dense), R);
    } else if (t > 0) {
      w = t * attn_cost(attn_key_tiles(ent, a.ratio, 0, R, KT, !pass.dense), R);
    }
  }
  *pairs = w * a.kv_heads;
  *items = t * a.kv_heads;
  return ascends;
}

// Starts outside the call's tokens or sequences count as their ends, and starts
// that descend as no call; either is flagged.
template <int kThreads>
__device__ __forceinline__ void attn_check_starts(const AttnArgs& a) {
  for (int i = threadIdx.x; a.q_start && i <= a.seqs; i += kThreads)
    if (a.q_start[i] < (i ? max(a.q_start[i - 1], 0) : 0) || a.q_start[i] > a.tokens) record_error(kErrBadPage);
  for (int i = threadIdx.x; a.group_start && i <= a.groups; i += kThreads)
    if (a.group_start[i] < (i ? max(a.group_start[i - 1], 0) : 0) || a.group_start[i] > a.seqs) record_error(kErrBadPage);
}

// This CTA's share, which starts `rest` pairs into entity e (whose first item is `item0`).
template <int R, int KT>
__device__ __forceinline__ AttnCursor attn_locate(const AttnArgs& a, const AttnPass& pass, int total, int e, int rest,
                                                  int item0) {
  AttnCursor c = {};
  c.total = total;
  const int ctas = min(pass.ctas, total), cta = blockIdx.x;
  if (cta >= ctas) return c;
  c.left = attn_share(total, ctas, cta + 1) - attn_share(total, ctas, cta);
  c.e = e;
  const AttnEntity ent = attn_entity(a, pass.mode, e);
  int k = attn_cost(attn_key_tiles(ent, a.ratio, 0, R, KT, !pass.dense), R);
  if (ent.causal && ent.ntok > 1) {
    while (rest >= a.kv_heads * k) {
      rest -= a.kv_heads * k;
      k = attn_cost(attn_key_tiles(ent, a.ratio, ++c.t, R, KT, !pass.dense), R);
    }
  } else {
    c.t = rest / (a.kv_heads * k);
    rest -= c.t * a.kv_heads * k;
  }
  c.h = rest / k;
  c.begin = rest - c.h * k;
  c.item = item0 + c.t * a.kv_heads + c.h;
  return c;
}

// Adds up all entities' work and finds this CTA's share.  All threads of the
// CTA call it; `scan` is shared scratch of 2 (entities + 1) + 64 ints.  CTA 0
// leaves the numbers of items, or of records, in pass.plan.
//
// Starts that ascend share out the call's tokens, whatever their values, so the
// sums stay below the 2^31 that the host has checked.  Descending ones count
// tokens many times over, and a sum that wraps would send attn_locate after a
// place that does not exist: then the pass has no work.
template <int R, int KT, int kThreads>
__device__ __forceinline__ AttnCursor attn_start(const AttnArgs& a, const AttnPass& pass, int* scan) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int kWarps = kThreads / 32;
  if (blockIdx.x == 0) attn_check_starts<kThreads>(a);
  if (pass.entities <= 32) {
    // Few entities: every warp adds them up for itself, a lane each.
    int w, n;
    const bool ascends = __all_sync(0xffffffffu, attn_work<R, KT>(a, pass, lane, &w, &n));
    int ws = w, ns = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int wu = __shfl_up_sync(0xffffffffu, ws, d), nu = __shfl_up_sync(0xffffffffu, ns, d);
      if (lane >= d) ws += wu, ns += nu;
    }
    if (blockIdx.x == 0 && warp == 0) {
      if (!pass.dense && lane == 31) pass.plan[0] = !ascends ? 0 : pass.by_item ? ns : pass.ctas;
      if (pass.dense && lane < pass.entities) pass.plan[lane] = ns - n;
      if (pass.dense && lane == 0) pass.plan[pass.entities] = ascends;
    }
    const int total = ascends ? __shfl_sync(0xffffffffu, ws, 31) : 0, ctas = min(pass.ctas, total);
    const int w0 = attn_share(total, max(ctas, 1), blockIdx.x);
    // The entity that holds pair w0: the first whose sum passes it.
    const unsigned past = __ballot_sync(0xffffffffu, ws > w0);
    const int e = past ? __ffs(past) - 1 : 0;
    return attn_locate<R, KT>(a, pass, total, e, w0 - __shfl_sync(0xffffffffu, ws - w, e), __shfl_sync(0xffffffffu, ns - n, e));
  }
  int* tiles = scan;
  int* items = scan + pass.entities + 1;
  int* part = items + pass.entities + 1;  // [2][kWarps]
  int tiles_before = 0, items_before = 0, descends = 0;
  for (int e0 = 0; e0 < pass.entities; e0 += kThreads) {
    int w, n;
    const bool ascends = attn_work<R, KT>(a, pass, e0 + tid, &w, &n);
    int ws = w, ns = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int wu = __shfl_up_sync(0xffffffffu, ws, d), nu = __shfl_up_sync(0xffffffffu, ns, d);
      if (lane >= d) ws += wu, ns += nu;
    }
    if (lane == 31) part[warp] = ws, part[kWarps + warp] = ns;
    descends |= __syncthreads_or(!ascends);
    int wb = tiles_before, nb = items_before;
    for (int i = 0; i < kWarps; ++i) {
      if (i < warp) wb += part[i], nb += part[kWarps + i];
      tiles_before += part[i];
      items_before += part[kWarps + i];
    }
    if (e0 + tid < pass.entities) {
      tiles[e0 + tid] = wb + ws - w;
      items[e0 + tid] = nb + ns - n;
    }
    __syncthreads();
  }
  if (tid == 0) {
    tiles[pass.entities] = tiles_before;
    items[pass.entities] = items_before;
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    if (!pass.dense && tid == 0) pass.plan[0] = descends ? 0 : pass.by_item ? items_before : pass.ctas;
    if (pass.dense)
      for (int i = tid; i <= pass.entities; i += kThreads) pass.plan[i] = i < pass.entities ? items[i] : !descends;
  }
  if (descends) return {};
  const int w0 = attn_share(tiles_before, max(min(pass.ctas, tiles_before), 1), blockIdx.x);
  int lo = 0, hi = pass.entities;  // tiles[lo] <= w0 < tiles[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tiles[mid] <= w0) lo = mid; else hi = mid;
  }
  const AttnCursor c = attn_locate<R, KT>(a, pass, tiles_before, lo, w0 - tiles[lo], items[lo]);
  __syncthreads();
  return c;
}

// The segments of a share, one after the other.
struct AttnSegment {
  AttnEntity ent;
  int t, h, begin, end;  // row tile, KV head, key tiles [begin, end) of `of`
  int of, item;
};

template <int R, int KT>
struct AttnWalk {
  const AttnArgs& a;
  int mode, entities, least;
  AttnCursor c;
  AttnEntity ent;
  __device__ AttnWalk(const AttnArgs& args, const AttnPass& pass, const AttnCursor& start)
      : a(args), mode(pass.mode), entities(pass.entities), least(!pass.dense), c(start) {
    if (c.left > 0) ent = attn_entity(a, mode, c.e);
  }
  __device__ bool next(AttnSegment* s) {
    while (c.left > 0) {
      int k = 0;
      for (;;) {  // skip row tiles that see nothing and entities without rows
        const int tiles = attn_row_tiles(ent, a.ratio, R);
        if (c.t < tiles) {
          k = attn_key_tiles(ent, a.ratio, c.t, R, KT, least);
          if (k > 0) break;
          ++c.t;
          c.item += a.kv_heads;
        } else {
          if (++c.e >= entities) return false;
          c.t = 0;
          ent = attn_entity(a, mode, c.e);
        }
      }
      // The key tiles stand behind the item's start on the line; a share that
      // ends before them leaves the item to the next CTA.
      const int end = min(attn_cost(k, R), c.begin + c.left);
      const int first = max(c.begin - attn_ends(R), 0), past = max(end - attn_ends(R), 0);
      const int t = c.t, h = c.h, item = c.item;
      c.left -= end - c.begin;
      c.begin = 0;
      ++c.item;
      if (++c.h == a.kv_heads) c.h = 0, ++c.t;
      if (first >= past) continue;
      s->ent = ent;
      s->t = t;
      s->h = h;
      s->begin = first;
      s->end = past;
      s->of = k;
      s->item = item;
      return true;
    }
    return false;
  }
};

__device__ __forceinline__ int attn_owner(int total, int ctas, int w) {
  int c = static_cast<int>(static_cast<long long>(w) * ctas / total);
  while (c + 1 < ctas && attn_share(total, ctas, c + 1) <= w) ++c;
  while (c > 0 && attn_share(total, ctas, c) > w) --c;
  return c;
}

// What a CTA leaves for paged_join_kernel behind segment s, its `segments`-th
// (last: there is none behind it).  An item's first CTA writes the item's
// record; by CTA, each writes one, of its last segment.
__device__ __forceinline__ void attn_leave_cut(const AttnArgs& a, const AttnPass& pass, const AttnCursor& start,
                                               const AttnSegment& s, int segments, bool last, int R) {
  const bool begins = segments > 0 && s.begin == 0;
  if (pass.by_item ? !begins || s.item >= pass.ctas : !last) return;
  AttnCut cut = {};
  if (begins && s.end < s.of) {
    const int c = blockIdx.x, ctas = min(pass.ctas, start.total);
    const int end = attn_owner(start.total, ctas, attn_share(start.total, ctas, c + 1) + s.of - s.end - 1);
    cut = {end - c + 1, 2 * c + (segments > 1), s.t * R, s.ent.ntok * a.ratio, s.h, s.ent.tok0, c, 0};
  }
  reinterpret_cast<AttnCut*>(pass.plan)[1 + (pass.by_item ? s.item : static_cast<int>(blockIdx.x))] = cut;
}

// What it leaves for paged_merge_kernel: the items that it begins or ends.
__device__ __forceinline__ void attn_leave_item(const AttnPass& pass, const AttnSegment& s) {
  int2* items = reinterpret_cast<int2*>(pass.plan + (pass.entities + 2) / 2 * 2);
  if (s.item >= pass.slots) return;
  if (s.begin == 0) items[s.item].x = blockIdx.x;
  if (s.end == s.of) items[s.item].y = blockIdx.x;
}

// Key tile k of an entity: which table, its first row there, and how many rows that table's part has.
struct AttnTile {
  const int32_t* tab;
  int row0, rows, own;
};
template <int KT>
__device__ __forceinline__ AttnTile attn_tile(const AttnEntity& n, int k) {
  const int before = (n.plen + KT - 1) / KT;
  if (k < before) return {n.ptab, k * KT, n.plen, 0};
  return {n.tab, (k - before) * KT, n.len, 1};
}

// The page of tile row `row` (a multiple of the page size or inside a page);
// rows behind the end and bad entries give page number `pages`, which the
// copies fill with zeros.
__device__ __forceinline__ int attn_page(const AttnArgs& a, const AttnTile& tile, int row) {
  const int r = tile.row0 + row;
  if (r >= tile.rows) return a.pages;
  const int page = tile.tab[r >> a.page_shift];
  if (page >= 0 && page < a.pages) return page;
  record_error(kErrBadPage);
  return a.pages;
}

// TMA box (64 elements x box rows of one page and head) into a 128-byte-swizzled tile.
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(smem_addr(dst)),
      "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_addr(bar))
      : "memory");
}
__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool kBf16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kBf16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Weights of a row are 2^(x - maximum + lift).  fp16 rounds to zero what is
// below 2^-25, so without a lift a long tail 17.5 nats below one key vanished
// from the products while the sum counted it (4000 such keys: 1e-4 of the
// result).  2^15 is fp16's largest power of two.  Sums and accumulators carry
// the same factor, which the division takes out; a segment's statistics are
// (maximum - lift, sum).  bf16 has fp32's exponents and needs none.
__host__ __device__ constexpr float attn_lift(bool bf16, int most) { return bf16 ? 0.0f : static_cast<float>(most); }

// ------------------------------------------------------------ few rows a key
//
// Row tiles of R = 16, 32 or 64: a key is used for at most R rows, so HBM
// bounds it (2 R flops a byte; the warp-level matrix instructions do R = 64
// in the time the tile takes to arrive) and what matters is copies in flight.
// Four warps compute: R / 16 of them side by side over the rows, the rest
// over the keys of a tile (each with its own maximum and sum, joined once per
// segment through shared memory).  A fifth issues the copies: a ring of
// three K + V tiles of 64 keys, so two CTAs per SM keep 100 KB or more in
// flight.  48 sequences of 1 to 5000 rows, 8 KV heads of 128: 117 us with the
// join, 93 % of the copy rate.  One sequence of 4096 rows: 12.4 us, latencies
// (lengths and pages, the first tiles, the segments' join) and not the 2.6 us of
// its bytes.  R = 64 with heads of 128 spills 340 to 352 bytes a thread.
template <int D, int R>
struct AttnFew {
  static constexpr int kKeys = 64;
  static constexpr int kStages = 3;
  static constexpr int kThreads = 160;
  static constexpr int kTile = kKeys * D * 2;            // bytes of a K or V tile
  static constexpr int kStage = 2 * kTile;
  static constexpr int kRowWarps = R / 16, kKeyWarps = 4 / kRowWarps, kWarpKeys = kKeys / kKeyWarps;
  static constexpr int kJoin = 64 * D * 4 / 2;           // fp32 accumulators of two warps
  static constexpr int kStatsOff = kStages * kStage + (kKeyWarps > 1 ? kJoin : 0);
  static constexpr int kBarOff = kStatsOff + 4 * 16 * 8;
  static constexpr int kSmem = kBarOff + 64;
  static_assert(kStages * kStage >= (2 * (kAttnMaxEntities + 1) + 64) * 4, "the scan fits in the ring");
};

template <int D, int R, bool kBf16>
__global__ void __launch_bounds__(160, 2)
    paged_attn_few_kernel(const AttnArgs a, const AttnPass pass, const __grid_constant__ CUtensorMap kmap,
                          const __grid_constant__ CUtensorMap vmap) {
  using C = AttnFew<D, R>;
  constexpr int KT = C::kKeys;
  constexpr float kLift = attn_lift(kBf16, 15);
  extern __shared__ __align__(1024) uint8_t attn_smem[];
  uint8_t* ring = attn_smem;
  float* join = reinterpret_cast<float*>(attn_smem + C::kStages * C::kStage);
  float2* row_stats = reinterpret_cast<float2*>(attn_smem + C::kStatsOff);  // [4 warps][16]
  uint64_t* full = reinterpret_cast<uint64_t*>(attn_smem + C::kBarOff);
  uint64_t* empty = full + C::kStages;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);
    }
    fence_mbar_init();
    tma_prefetch_map(&kmap);
    tma_prefetch_map(&vmap);
  }
  pdl_wait_prerequisite();
  pdl_launch_dependents();
  const AttnCursor start = attn_start<R, KT, C::kThreads>(a, pass, reinterpret_cast<int*>(ring));
  // The scan used the ring through the generic proxy; the copies come through the async one.
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncthreads();
  AttnWalk<R, KT> walk(a, pass, start);
  AttnSegment s;

  if (warp == 4) {
    // ------------------------------------------------ copies
    // Lanes take one box each: page p of the tile, half of the head, K or V.
    const int box_rows = min(1 << a.page_shift, KT), per_tile = KT / box_rows;
    constexpr int kHalves = D / 64;
    const int boxes = per_tile * kHalves * 2;
    int n = 0, segments = 0;
    bool stuck = false;
    s = {};
    while (!stuck && walk.next(&s)) {
      ++segments;
      if (lane == 0) {
        if (pass.dense)
          attn_leave_item(pass, s);
        else if (pass.by_item)
          attn_leave_cut(a, pass, start, s, segments, false, R);
      }
      for (int k = s.begin; k < s.end; ++k, ++n) {
        const AttnTile tile = attn_tile<KT>(s.ent, k);
        const int p = lane % per_tile, rest = lane / per_tile, half = rest % kHalves, is_v = rest / kHalves;
        int page = 0;
        if (lane < boxes) page = attn_page(a, tile, p * box_rows);
        const int in_page = (tile.row0 + p * box_rows) & ((1 << a.page_shift) - 1);
        const int st = n % C::kStages;
        if (n >= C::kStages && !mbar_wait_bounded(&empty[st], (n / C::kStages - 1) & 1)) {
          record_error(kErrEmptyWaitTimeout);
          stuck = true;
          break;
        }
        if (lane == 0) mbar_arrive_expect_tx(&full[st], C::kStage);
        __syncwarp();
        if (lane < boxes)
          tma_load_4d(ring + st * C::kStage + is_v * C::kTile + half * (KT * 128) + p * box_rows * 128,
                      is_v ? &vmap : &kmap, half * 64, in_page, s.h, page, &full[st]);
      }
    }
    if (!pass.dense && !pass.by_item && lane == 0) attn_leave_cut(a, pass, start, s, segments, true, R);
    // The last copies land before the CTA's shared memory is given back.
    for (int i = max(n - C::kStages, 0); i < n; ++i)
      if (!mbar_wait_bounded(&full[i % C::kStages], (i / C::kStages) & 1)) record_error(kErrDrainTimeout);
    return;
  }

  // -------------------------------------------------- products
  const int rw = warp % C::kRowWarps, kw = warp / C::kRowWarps;
  const int g = lane >> 2, tq = lane & 3;
  int n = 0;
  bool first = true, stuck = false;
  while (walk.next(&s)) {
    const int rows = s.ent.ntok * a.ratio;
    int row[2], token[2], head[2], limit[2];
    uint32_t q[D / 16][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      row[i] = s.t * R + rw * 16 + g + i * 8;
      const bool there = row[i] < rows;
      const int j = there ? row[i] / a.ratio : 0;
      token[i] = there ? s.ent.tok0 + j : -1;
      head[i] = s.h * a.ratio + (there ? row[i] - j * a.ratio : 0);
      limit[i] = there ? attn_limit(s.ent, j) : 0;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(a.q + max(token[i], 0) * a.q_token + head[i] * a.q_head);
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        q[c][i] = there ? src[c * 8 + tq] : 0u;
        q[c][i + 2] = there ? src[c * 8 + 4 + tq] : 0u;
      }
    }
    float acc[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};

    for (int k = s.begin; k < s.end; ++k, ++n) {
      const AttnTile tile = attn_tile<KT>(s.ent, k);
      const int st = n % C::kStages;
      if (!stuck && !mbar_wait_bounded(&full[st], (n / C::kStages) & 1)) {
        record_error(kErrFullWaitTimeout);  // finish on what is there: the other warps wait at barriers
        stuck = true;
      }
      const uint32_t kbase = smem_addr(ring + st * C::kStage), vbase = kbase + C::kTile;
      constexpr int NT = C::kWarpKeys / 8;
      const int key0 = kw * C::kWarpKeys;
      float x[NT][4];
#pragma unroll
      for (int i = 0; i < NT; ++i) x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.0f;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
#pragma unroll
        for (int i = 0; i < NT; i += 2) {
          // Two 8-key blocks x two 8-element halves of the 16-element step.
          const int r = key0 + i * 8 + (lane & 7) + ((lane >> 4) << 3);
          const int chunk = c * 2 + ((lane >> 3) & 1);
          uint32_t b[4];
          ldsm4(kbase + (chunk >> 3) * (KT * 128) + r * 128 + (((chunk & 7) ^ (r & 7)) << 4), b);
          mma16816<kBf16>(x[i], q[c], b[0], b[1]);
          mma16816<kBf16>(x[i + 1], q[c], b[2], b[3]);
        }
      }
      // Keys a row does not see weigh nothing, whatever their scores are.
      const int end0 = min(tile.own ? limit[0] : tile.rows, tile.rows) - tile.row0;
      const int end1 = min(tile.own ? limit[1] : tile.rows, tile.rows) - tile.row0;
      float m0 = top[0], m1 = top[1];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int key = key0 + i * 8 + tq * 2;
        x[i][0] = key < end0 ? x[i][0] * a.scale_log2 : -INFINITY;
        x[i][1] = key + 1 < end0 ? x[i][1] * a.scale_log2 : -INFINITY;
        x[i][2] = key < end1 ? x[i][2] * a.scale_log2 : -INFINITY;
        x[i][3] = key + 1 < end1 ? x[i][3] * a.scale_log2 : -INFINITY;
        m0 = fmaxf(m0, fmaxf(x[i][0], x[i][1]));
        m1 = fmaxf(m1, fmaxf(x[i][2], x[i][3]));
      }
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, d));
        m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, d));
      }
      const float f0 = ex2(top[0] - (m0 == -INFINITY ? 0.0f : m0)), f1 = ex2(top[1] - (m1 == -INFINITY ? 0.0f : m1));
      const float z0 = m0 == -INFINITY ? 0.0f : m0 - kLift, z1 = m1 == -INFINITY ? 0.0f : m1 - kLift;
      top[0] = m0;
      top[1] = m1;
      sum[0] *= f0;
      sum[1] *= f1;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        acc[i][0] *= f0;
        acc[i][1] *= f0;
        acc[i][2] *= f1;
        acc[i][3] *= f1;
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        x[i][0] = ex2(x[i][0] - z0);
        x[i][1] = ex2(x[i][1] - z0);
        x[i][2] = ex2(x[i][2] - z1);
        x[i][3] = ex2(x[i][3] - z1);
        sum[0] += x[i][0] + x[i][1];
        sum[1] += x[i][2] + x[i][3];
      }
      // P in the cache's type: off by half a step, a factor 1 +- 2^-11 or 2^-8 at
      // most, in fp16 from 2^-29 of the largest weight on and 2^-40 of that one
      // below (attn_lift); the sums keep the unrounded weights.  V rows behind the
      // end of a sequence are anything at all, NaN too: those registers become zero.
      const int held = tile.rows - tile.row0;
#pragma unroll
      for (int i = 0; i < NT; i += 2) {
        uint32_t p[4] = {pack16<kBf16>(x[i][0], x[i][1]), pack16<kBf16>(x[i][2], x[i][3]),
                         pack16<kBf16>(x[i + 1][0], x[i + 1][1]), pack16<kBf16>(x[i + 1][2], x[i + 1][3])};
        const int k0 = key0 + i * 8 + tq * 2;
        const uint32_t lo = (k0 < held ? 0xffffu : 0u) | (k0 + 1 < held ? 0xffff0000u : 0u);
        const uint32_t hi = (k0 + 8 < held ? 0xffffu : 0u) | (k0 + 9 < held ? 0xffff0000u : 0u);
#pragma unroll
        for (int c = 0; c < D / 8; c += 2) {
          const int r = key0 + i * 8 + (lane & 15);
          const int chunk = c + (lane >> 4);
          uint32_t b[4];
          ldsm4t(vbase + (chunk >> 3) * (KT * 128) + r * 128 + (((chunk & 7) ^ (r & 7)) << 4), b);
          mma16816<kBf16>(acc[c], p, b[0] & lo, b[1] & hi);
          mma16816<kBf16>(acc[c + 1], p, b[2] & lo, b[3] & hi);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
      sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], d);
      sum[1] += __shfl_xor_sync(0xffffffffu, sum[1], d);
    }

    if constexpr (C::kKeyWarps > 1) {
      // Join the warps that share rows: scale to the common maximum, then add
      // the accumulators, the upper half of the warps to the lower, until one is left.
      if (tq == 0) {
        row_stats[warp * 16 + g] = make_float2(top[0], sum[0]);
        row_stats[warp * 16 + g + 8] = make_float2(top[1], sum[1]);
      }
      named_barrier(1, 128);
      float f[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int w = 0; w < C::kKeyWarps; ++w) m = fmaxf(m, row_stats[(w * C::kRowWarps + rw) * 16 + g + i * 8].x);
        const float z = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int w = 0; w < C::kKeyWarps; ++w) {
          const float2 st = row_stats[(w * C::kRowWarps + rw) * 16 + g + i * 8];
          l = fmaf(st.y, ex2(st.x - z), l);
        }
        f[i] = ex2(top[i] - z);
        top[i] = m;
        sum[i] = l;
      }
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        acc[i][0] *= f[0];
        acc[i][1] *= f[0];
        acc[i][2] *= f[1];
        acc[i][3] *= f[1];
      }
#pragma unroll
      for (int step = C::kKeyWarps / 2; step >= 1; step >>= 1) {
        // Element i of lane l at i * 32 + l: no bank is hit twice.
        if (kw >= step && kw < 2 * step) {
          float* dst = join + ((kw - step) * C::kRowWarps + rw) * (16 * D);
#pragma unroll
          for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) dst[(i * 4 + j) * 32 + lane] = acc[i][j];
        }
        named_barrier(1, 128);
        if (kw < step) {
          const float* src = join + (kw * C::kRowWarps + rw) * (16 * D);
#pragma unroll
          for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] += src[(i * 4 + j) * 32 + lane];
        }
        named_barrier(1, 128);
      }
    }
    if (kw == 0) {
      const bool whole = s.begin == 0 && s.end == s.of;
      const bool direct = whole && !pass.dense;
      if (direct) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (token[i] < 0) continue;
          const float inv = sum[i] > 0.0f ? 1.0f / sum[i] : 0.0f;
          uint32_t* dst = reinterpret_cast<uint32_t*>(a.out + token[i] * a.out_token + head[i] * a.out_head);
#pragma unroll
          for (int c = 0; c < D / 8; ++c)
            dst[c * 4 + tq] = pack16<kBf16>(acc[c][2 * i] * inv, acc[c][2 * i + 1] * inv);
        }
      } else {
        const int slot = pass.dense ? static_cast<int>(blockIdx.x) + s.item : 2 * static_cast<int>(blockIdx.x) + !first;
        if (slot < pass.slots) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (token[i] < 0) continue;
            const long long r = static_cast<long long>(slot) * R + rw * 16 + g + i * 8;
            if (tq == 0) pass.stats[r] = make_float2(top[i] - kLift, sum[i]);
            float2* dst = reinterpret_cast<float2*>(pass.acc + r * D);
#pragma unroll
            for (int c = 0; c < D / 8; ++c) dst[c * 4 + tq] = make_float2(acc[c][2 * i], acc[c][2 * i + 1]);
          }
        } else {
          record_error(kErrBadPage);  // starts that overlap: more items than there are tokens
        }
      }
    }
    first = false;
  }
}

// ------------------------------------------------------------ joining segments

// What a dense pass left of one row: segments of CTAs c0 to c1, at slots c + item.
struct AttnRowParts {
  int c0, c1, item, row;  // c1 < c0: nothing
};

__device__ __forceinline__ AttnRowParts attn_row_parts(const AttnArgs& a, const AttnPass& pass, int e, int token, int h,
                                                       int hr) {
  AttnRowParts p = {0, -1, 0, 0};
  const int before = pass.plan[e];
  const AttnEntity ent = attn_entity(a, pass.mode, e);
  const int row = (token - ent.tok0) * a.ratio + hr;
  if (row < 0 || row >= ent.ntok * a.ratio) return p;
  const int t = row / pass.rows;
  if (attn_key_tiles(ent, a.ratio, t, pass.rows, pass.keys, 0) == 0) return p;
  p.row = row - t * pass.rows;
  p.item = before + t * a.kv_heads + h;
  if (p.item < 0 || p.item >= pass.slots) return p;
  const int2 ctas = reinterpret_cast<const int2*>(pass.plan + (pass.entities + 2) / 2 * 2)[p.item];
  p.c1 = max(min(ctas.y, pass.ctas - 1), -1);
  p.c0 = min(max(ctas.x, 0), p.c1 + 1);
  return p;
}

// Where a segment of a row lies (nullptr: outside the workspace).
struct AttnSlot {
  const float2* stats;
  const float* acc;
};
template <int D>
__device__ __forceinline__ AttnSlot attn_slot(const AttnPass& pass, int slot, int row) {
  if (slot < 0 || slot >= pass.slots) return {nullptr, nullptr};
  const long long r = static_cast<long long>(slot) * pass.rows + row;
  return {pass.stats + r, pass.acc + r * D};
}

// A row's segments joined by `parts` warps (1 or 4) of a CTA: warp `part` takes
// every parts-th.  The lanes first read 32 segments' statistics at once (lane
// i: segment i), so that the accumulators, D / 32 elements a lane, load
// without waiting for one another.
template <int D>
struct AttnJoin {
  static constexpr int N = D / 32;
  float top = -INFINITY, sum = 0.0f, acc[N] = {};

  // Segments i < n, i % parts == part, at row row_of(i) of slot_of(i).  Four
  // accumulators load at a time, the first four beside the statistics.
  template <typename At>
  __device__ __forceinline__ void add(int n, int lane, int part, int parts, At at) {
    for (int base = 0; base < n; base += 32 * parts) {
      const int i = base + lane * parts + part;
      AttnSlot mine = {nullptr, nullptr};
      if (i < n) mine = at(i);
      float2 st = make_float2(-INFINITY, 0.0f);
      if (mine.stats) st = *mine.stats;
      const int here = min((n - base - part + parts - 1) / parts, 32);
      float x[4][N];
      auto load = [&](int k) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const auto from = reinterpret_cast<const float*>(
              __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine.acc), (k + u) & 31));
#pragma unroll
          for (int e = 0; e < N; ++e) x[u][e] = 0.0f;
          if (k + u < here && from) load_values<kTypeF32, N>(from, lane * N, x[u]);
        }
      };
      load(0);
      const float m = fmaxf(top, warp_max_float(st.x)), z = m == -INFINITY ? 0.0f : m;
      const float f = ex2(top - z), w = ex2(st.x - z);
      sum = fmaf(sum, f, warp_sum_float_butterfly(st.y * w));
      top = m;
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] *= f;
      for (int k = 0; k < here; k += 4) {
        if (k) load(k);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float ws = __shfl_sync(0xffffffffu, w, (k + u) & 31);
#pragma unroll
          for (int e = 0; e < N; ++e) acc[e] = k + u < here ? fmaf(x[u][e], ws, acc[e]) : acc[e];
        }
      }
    }
  }

  // The warps of a row together, in the last of them (the others return false).
  // `shared`: 256 / 32 x (D + 2) floats.
  __device__ __forceinline__ bool gather(float* shared, int warp, int lane, int part, int parts) {
    if (parts == 1) return true;
    float* mine = shared + warp * (D + 2);
#pragma unroll
    for (int e = 0; e < N; ++e) mine[lane * N + e] = acc[e];
    if (lane == 0) mine[D] = top, mine[D + 1] = sum;
    __syncthreads();
    if (part) return false;
    float m = top;
    for (int p = 1; p < parts; ++p) m = fmaxf(m, mine[p * (D + 2) + D]);
    const float z = m == -INFINITY ? 0.0f : m, f = ex2(top - z);
    sum *= f;
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] *= f;
    for (int p = 1; p < parts; ++p) {
      const float* other = mine + p * (D + 2);
      const float fx = ex2(other[D] - z);
      sum = fmaf(other[D + 1], fx, sum);
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] = fmaf(other[lane * N + e], fx, acc[e]);
    }
    return true;
  }
};

// The result of a row's segments; zeros where there was nothing to see.
template <int D, bool kBf16>
__device__ __forceinline__ void attn_store_row(const AttnArgs& a, int token, int head, int lane, float sum,
                                               float (&acc)[D / 32]) {
  constexpr int N = D / 32;
  const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] *= inv;
  store_values16<kBf16, N>(a.out + token * a.out_token + head * a.out_head + lane * N, acc);
}

// Joins an item that one CTA began and others went on with: their segments of
// it are the first ones of their shares.  Grid (record, rows in turn); a row's
// loads take about a microsecond, so as many warps as fit run beside one
// another and a CTA takes several rows rather than the SMs several waves of CTAs.
template <int D, bool kBf16>
__global__ void __launch_bounds__(256, 4) paged_join_kernel(const AttnArgs a, const AttnPass pass, int parts) {
  __shared__ float shared[8 * (D + 2)];
  pdl_wait_prerequisite();
  pdl_launch_dependents();
  const AttnCut cut = reinterpret_cast<const AttnCut*>(pass.plan)[1 + blockIdx.x];
  if (static_cast<int>(blockIdx.x) >= pass.plan[0] || cut.segments == 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % parts;
  for (int row0 = blockIdx.y * (8 / parts); row0 < pass.rows; row0 += gridDim.y * (8 / parts)) {
    const int row = row0 + warp / parts, at = cut.row0 + row;
    const bool there = at < cut.rows;
    if (cut.row0 + row0 >= cut.rows) return;
    AttnJoin<D> join;
    if (there)
      join.add(min(cut.segments, pass.ctas), lane, part, parts,
               [&](int i) { return attn_slot<D>(pass, i == 0 ? cut.slot : 2 * (cut.cta + i), row); });
    if (join.gather(shared, warp, lane, part, parts) && there) {
      const int j = at / a.ratio;
      if (cut.tok0 + j < a.tokens) attn_store_row<D, kBf16>(a, cut.tok0 + j, cut.h * a.ratio + at - j * a.ratio, lane, join.sum, join.acc);
    }
    if (parts > 1) __syncthreads();  // `shared` is free again
  }
}

// Prefixes apart from own rows: `parts` warps per (token, query head) join all
// segments of both.  Rows that see nothing become zeros.  first: the prefixes'
// pass, or the one of both; second: the own rows' pass where there are two.
template <int D, bool kBf16>
__global__ void __launch_bounds__(256)
    paged_merge_kernel(const AttnArgs a, const AttnPass first, const AttnPass second, int parts) {
  __shared__ float shared[8 * (D + 2)];
  pdl_wait_prerequisite();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % parts, q_heads = a.kv_heads * a.ratio;
  const long long w = static_cast<long long>(blockIdx.x) * (8 / parts) + warp / parts;
  bool there = w < static_cast<long long>(a.tokens) * q_heads;
  const int token = there ? static_cast<int>(w / q_heads) : 0, head = static_cast<int>(w % q_heads);
  const int h = head / a.ratio, hr = head - h * a.ratio;
  int seq = token;
  if (a.q_start) {
    there = there && token >= a.q_start[0] && token < a.q_start[a.seqs];  // rows behind the last sequence stay
    int lo = 0, hi = a.seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.q_start[mid] <= token) lo = mid; else hi = mid;
    }
    seq = lo;
  }
  AttnJoin<D> join;
  // Loaded beside the parts, looked at before the store.
  const bool two = first.mode != kAttnBoth;
  const int done = first.plan[first.entities], done_own = two ? second.plan[second.entities] : 1;
  if (there) {
    const int g = attn_group_of(a, seq);
    AttnRowParts pre = {0, -1, 0, 0};
    const bool both = first.mode == kAttnBoth;
    const AttnPass& own_pass = both ? first : second;
    const AttnRowParts own = attn_row_parts(a, own_pass, both ? a.groups + seq : seq, token, h, hr);
    if (g >= 0) pre = attn_row_parts(a, first, g, token, h, hr);
    const int shared_segments = pre.c1 - pre.c0 + 1;
    join.add(shared_segments + own.c1 - own.c0 + 1, lane, part, parts, [&](int i) {
      return i < shared_segments ? attn_slot<D>(first, pre.c0 + i + pre.item, pre.row)
                                 : attn_slot<D>(own_pass, own.c0 + i - shared_segments + own.item, own.row);
    });
  }
  if (!join.gather(shared, warp, lane, part, parts) || !there || !(done & done_own)) return;
  attn_store_row<D, kBf16>(a, token, head, lane, join.sum, join.acc);
}

}  // namespace mllb
