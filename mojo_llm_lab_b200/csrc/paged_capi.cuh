// extern "C" launchers of the paged-cache operators (paged.cuh,
// paged_attn.cuh, beam.cuh); part of the library's one translation unit,
// included by capi.cu behind its helpers.
#pragma once

#include <algorithm>

#include "beam.cuh"
#include "paged.cuh"
#include "paged_attn.cuh"
#include "paged_attn_tc.cuh"

namespace {

// All launches here carry the programmatic-serialisation attribute: the kernels
// touch global memory only behind griddepcontrol.wait, so they may always be
// scheduled while the preceding kernel runs (MLLB_LAUNCH_PDL changes nothing).
constexpr bool kEarly = true;

int log2_exact(int64_t n) {
  int s = 0;
  while ((1ll << s) < n) ++s;
  return s;
}

// Memory that a call reads or writes.
struct Span {
  const void* at;
  int64_t bytes;
};
bool meet(const Span& a, const Span& b) {
  const auto x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
  return x < y + b.bytes && y < x + a.bytes;
}

// Whether two of the rows of d elements at t * token + h * head, t < tokens, h < heads, have an element in common.
bool rows_overlap(int64_t tokens, int64_t token, int64_t heads, int64_t head, int64_t d) {
  if ((tokens > 1 && token < d) || (heads > 1 && head < d)) return true;
  if (tokens == 1 || heads == 1 || token >= (heads - 1) * head + d || head >= (tokens - 1) * token + d) return false;
  for (int64_t h = 1; h < heads; ++h) {  // row (0, h) lies between rows (t, 0) and (t + 1, 0), or behind all
    const int64_t at = h * head, t = at / token, behind = at - t * token;
    if ((t < tokens && behind < d) || (t + 1 < tokens && token - behind < d)) return true;
  }
  return false;
}

// Whether a row of out has an element in common with a row of q, both of d
// elements at t * token + h * head from their bases.  Rows of one buffer taken
// in turn have the same token stride; with others, rows in the same range count
// as shared.
bool out_overlaps_q(const mllb_paged_attn* p, int64_t d) {
  const int64_t tokens = p->tokens - 1, heads = p->q_heads - 1;
  const auto q = reinterpret_cast<uintptr_t>(p->q), out = reinterpret_cast<uintptr_t>(p->out);
  const uintptr_t q_end = q + 2 * (tokens * p->q_token_stride + heads * p->q_head_stride + d);
  const uintptr_t out_end = out + 2 * (tokens * p->out_token_stride + heads * p->out_head_stride + d);
  if (q_end <= out || out_end <= q) return false;
  if (tokens && p->q_token_stride != p->out_token_stride) return true;
  const int64_t base = (static_cast<int64_t>(out) - static_cast<int64_t>(q)) / 2, token = tokens ? p->out_token_stride : 0;
  // Whether rows that lie x apart, or whole token strides more or less, meet.
  auto near_zero = [&](int64_t x) {
    const int64_t near = tokens ? std::min(std::max(x / token, -tokens), tokens) : 0;
    for (int64_t t = std::max(near - 1, -tokens); t <= std::min(near + 1, tokens); ++t)
      if (x - t * token > -d && x - t * token < d) return true;
    return false;
  };
  if (heads == 0 || p->q_head_stride == p->out_head_stride) {
    for (int64_t h = -heads; h <= heads; ++h)
      if (near_zero(base + h * p->out_head_stride)) return true;
    return false;
  }
  for (int64_t h = 0; h <= heads; ++h)
    for (int64_t g = 0; g <= heads; ++g)
      if (near_zero(base + h * p->out_head_stride - g * p->q_head_stride)) return true;
  return false;
}

// Checks a cache description and turns it into the kernels' form.
int paged_cache(const mllb_paged_cache* c, mllb::PagedCache* out) {
  if (!c || !c->k || !c->v) return fail(MLLB_EINVAL, "null pointer: cache");
  if (c->type != MLLB_TYPE_F16 && c->type != MLLB_TYPE_BF16) return fail(MLLB_EINVAL, "cache type must be fp16 or bf16");
  if (c->head_dim != 64 && c->head_dim != 128)
    return fail(MLLB_EUNSUPPORTED, "head_dim=%lld is not 64 or 128", static_cast<long long>(c->head_dim));
  if (c->pages <= 0 || c->pages > (1 << 30)) return fail(MLLB_EINVAL, "pages=%lld out of range", static_cast<long long>(c->pages));
  if (c->kv_heads <= 0 || c->kv_heads > 1024)
    return fail(MLLB_EINVAL, "kv_heads=%lld out of range", static_cast<long long>(c->kv_heads));
  if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)))
    return fail(MLLB_EINVAL, "page_size=%lld is not a power of two from 16 to 1024", static_cast<long long>(c->page_size));
  if (c->layers <= 0 || c->layers > 65535) return fail(MLLB_EINVAL, "layers=%lld out of range", static_cast<long long>(c->layers));
  const int64_t strides[4] = {c->page_stride, c->head_stride, c->row_stride, c->layers > 1 ? c->layer_stride : 8};
  for (int64_t s : strides) {
    if (s <= 0 || s >= (1ll << 38)) return fail(MLLB_EINVAL, "cache strides must be positive and below 2^38 elements");
    if (s % 8) return fail(MLLB_EALIGN, "cache strides must be multiples of 8 elements (16 bytes)");
  }
  if (c->row_stride < c->head_dim) return fail(MLLB_EINVAL, "cache rows overlap");
  if (!aligned(c->k, 16) || !aligned(c->v, 16)) return fail(MLLB_EALIGN, "caches must be 16-byte aligned");
  out->k = static_cast<uint16_t*>(c->k);
  out->v = static_cast<uint16_t*>(c->v);
  out->page_stride = c->page_stride;
  out->head_stride = c->head_stride;
  out->row_stride = c->row_stride;
  out->layer_stride = c->layers > 1 ? c->layer_stride : 0;
  out->pages = static_cast<int>(c->pages);
  out->kv_heads = static_cast<int>(c->kv_heads);
  out->page_shift = log2_exact(c->page_size);
  out->layers = static_cast<int>(c->layers);
  return MLLB_OK;
}

template <int D, int kType>
cudaError_t launch_append(const mllb::AppendArgs& a, bool bf16, unsigned grid, cudaStream_t stream) {
  auto kernel = bf16 ? mllb::paged_append_kernel<D, kType, true> : mllb::paged_append_kernel<D, kType, false>;
  return launch(kernel, dim3(grid), dim3(mllb::kAppendWarps * 32), 0, stream, kEarly, a);
}

template <int kType>
cudaError_t launch_scan(const mllb::BeamArgs& a, bool vector, cudaStream_t stream) {
  auto kernel = vector ? mllb::beam_scan_kernel<kType, true> : mllb::beam_scan_kernel<kType, false>;
  return launch(kernel, dim3(static_cast<unsigned>(a.chunks), static_cast<unsigned>(a.batch * a.beams)),
                dim3(mllb::kBeamThreads), a.steps * mllb::kBeamThreads * sizeof(float), stream, kEarly, a);
}

int64_t beam_steps(int64_t vocab) { return (vocab + mllb::kBeamStep - 1) / mllb::kBeamStep; }

int check_beams(int64_t batch, int64_t beams, int64_t vocab, int64_t n) {
  if (batch <= 0 || beams <= 0 || vocab <= 0 || n <= 0) return fail(MLLB_EINVAL, "sizes must be positive");
  if (beams > mllb::kBeamMost || n > mllb::kBeamMost)
    return fail(MLLB_EUNSUPPORTED, "at most %d beams and candidates", mllb::kBeamMost);
  if (vocab > (1ll << mllb::kBeamTokenBits)) return fail(MLLB_EINVAL, "vocab above 2^%d", mllb::kBeamTokenBits);
  if (batch > 65535 || batch * beams > 65535) return fail(MLLB_EINVAL, "batch x beams above 65535");
  if (n > beams * vocab) return fail(MLLB_EINVAL, "n above beams x vocab: out of range");
  return MLLB_OK;
}

// The driver's tensor-map encoder, looked up once.
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled tensor_map_encoder() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// Tiles of box_rows rows x 64 elements of one head of one page, 128-byte swizzled.
int paged_map(CUtensorMap* map, const mllb_paged_cache* c, void* base, int box_rows) {
  const EncodeTiled encode = tensor_map_encoder();
  if (!encode) return fail(MLLB_ECUDA, "cuTensorMapEncodeTiled not found");
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(c->head_dim), static_cast<cuuint64_t>(c->page_size),
                              static_cast<cuuint64_t>(c->kv_heads), static_cast<cuuint64_t>(c->pages)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(c->row_stride * 2), static_cast<cuuint64_t>(c->head_stride * 2),
                                 static_cast<cuuint64_t>(c->page_stride * 2)};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_rows), 1, 1}, step[4] = {1, 1, 1, 1};
  const CUresult r = encode(map, c->type == MLLB_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                            4, base, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MLLB_EINVAL, "tensor map refused (error %d): strides or sizes", static_cast<int>(r));
  return MLLB_OK;
}

// How a call is cut into launches; the same from the sizes alone in the
// workspace query and in the call.
struct PagedPlan {
  int passes;
  int mode[2], rows[2], keys[2], ctas[2], entities[2], slots[2], dense[2], by_item[2], records[2];
  int64_t plan_off[2], stats_off[2], acc_off[2], bytes;
};

// What a call's page tables decide of its plan.
enum : unsigned { kPlanRepeat = 1, kPlanLong = 2, kPlanChoices = 4 };

// Row tile for entities of `rows` query rows: up to 64 the kernel for few rows
// a key, in its narrowest shape that holds them; beyond, the tensor cores'.
// 48 sequences of 2000 to 4000 rows, 8 KV heads: 4 query rows 102 us (in tiles of
// 32: 105), 32 109 us (in tiles of 64: 168).  33 to 64 lie between, and the length
// decides: 48 sequences of 16 tokens on 30 to 60 rows take the few-row kernel 20 us
// and the other, whose items start and end dearer, 22; on 350 to 700 rows 53 and
// 48, on 2000 to 4000 172 and 134.
int tile_rows(int64_t rows, bool longs) {
  return rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 && !longs ? 64 : mllb::AttnMany<128>::kRows;
}

// Whether prefix and own rows run as one softmax a sequence (paged_plan).
bool one_softmax(int64_t seq_rows, int64_t seqs, int64_t groups, bool repeat) {
  return groups == 0 || groups >= seqs || seq_rows >= 64 || repeat;
}

// Whether every sequence reads its group's prefix for itself although few rows
// each do so: the prefixes come from L2 after the first time, and one pass has
// less to join and to launch.  By the bytes read again at most, as the tables'
// widths bound them: 64 MB against a pass of prefixes and own rows (fp16, heads
// of 128, own rows 100; 16 sequences of a 1000-row prefix, 60 MB, 18.1 us
// against 19.5; of 4000, 236 MB, 32.4 against 22.7), 192 MB against a pass each
// (40 of 1000, 156 MB, 28.0 against 31.8; of 4000, 614 MB, 63 against 37).
// And whether a sequence's item is long by the same bound: 512 rows and more
// (tile_rows).  The lengths are on the device, so tables far wider than they are
// take the other plan: 22 sequences of 100 rows on a prefix of 30 14.4 us in
// narrow tables, 29.7 in ones of 8192 rows; 111 of 20 on 74 20.3 and 36.1.
unsigned plan_choice(const mllb_paged_attn* p, const mllb_paged_cache* c) {
  const int64_t prefix = p->groups ? p->prefix_width * c->page_size : 0, rows = p->tokens * (p->q_heads / c->kv_heads);
  const int64_t again = (p->seqs - p->groups) * prefix * c->kv_heads * c->head_dim * 4;
  const bool together = p->groups && (rows + p->groups - 1) / p->groups <= 64;
  const bool repeat = p->groups && again <= (together ? 64ll : 192ll) << 20;
  const int64_t keys = p->table_width * c->page_size +
                       (one_softmax((rows + p->seqs - 1) / p->seqs, p->seqs, p->groups, repeat) ? prefix : 0);
  return (repeat ? kPlanRepeat : 0u) | (keys >= 512 ? kPlanLong : 0u);
}

// Mean query rows (tokens x query heads of a KV head) of a sequence and of a
// group decide the shape, for all sequences of the call: a prompt's chunk of 512
// tokens on 8000 rows beside 128 single tokens takes 515 us, the two calls apart
// 69 and 206.  A sequence with a row tile's worth of rows shares
// nothing more by going through its group, so prefix and own rows then run as
// one softmax (no segments to join); so they do where kPlanRepeat says.  Otherwise
// the prefix runs once a group (16 sequences over a prefix of 8000 rows: up to 32
// rows each 49 us, as one softmax 84; up to 128 rows each 98 and 103): in one
// pass with the own rows where a group's rows fit one tile, in a pass of its own
// on the tensor cores beyond.
int paged_plan(int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t seqs, int64_t groups,
               unsigned choice, int dev, PagedPlan* p) {
  const bool repeat = choice & kPlanRepeat, longs = choice & kPlanLong;
  const int64_t ratio = q_heads / kv_heads;
  const int64_t seq_rows = (tokens * ratio + seqs - 1) / seqs;
  const int64_t group_rows = groups ? (tokens * ratio + groups - 1) / groups : 0;
  memset(p, 0, sizeof(*p));
  p->passes = 1;
  if (one_softmax(seq_rows, seqs, groups, repeat)) {
    p->mode[0] = groups ? mllb::kAttnConcat : mllb::kAttnOwn;
    p->rows[0] = tile_rows(seq_rows, longs);
    p->entities[0] = static_cast<int>(seqs);
  } else if (group_rows <= 64) {
    p->mode[0] = mllb::kAttnBoth;
    p->rows[0] = tile_rows(group_rows, false);
    p->entities[0] = static_cast<int>(groups + seqs);
    p->dense[0] = 1;
  } else {
    p->passes = 2;
    p->mode[0] = mllb::kAttnPrefix;
    p->rows[0] = tile_rows(group_rows, false);
    p->entities[0] = static_cast<int>(groups);
    p->mode[1] = mllb::kAttnOwn;
    p->rows[1] = tile_rows(seq_rows, longs);
    p->entities[1] = static_cast<int>(seqs);
    p->dense[0] = p->dense[1] = 1;
  }
  int64_t at = 0;
  for (int i = 0; i < p->passes; ++i) {
    const bool many = p->rows[i] > 64;
    p->keys[i] = many ? mllb::AttnMany<128>::kKeys : mllb::AttnFew<128, 16>::kKeys;
    p->ctas[i] = many ? sm_count(dev) : 2 * sm_count(dev);
    // Items: every entity's last row tile may be part full.
    const int64_t covers = p->mode[i] == mllb::kAttnBoth && groups ? 2 : 1;
    const int64_t items = kv_heads * (covers * ((tokens * ratio + p->rows[i] - 1) / p->rows[i]) + p->entities[i]);
    p->by_item[i] = !p->dense[i] && items <= p->ctas[i];
    p->records[i] = p->by_item[i] ? static_cast<int>(items) : p->ctas[i];
    const int64_t slots = p->dense[i] ? p->ctas[i] + items : 2 * p->ctas[i];
    if (slots > (1 << 30)) return fail(MLLB_EINVAL, "too many tokens x heads");
    p->slots[i] = static_cast<int>(slots);
    p->plan_off[i] = at;
    const int64_t plan = p->dense[i] ? (p->entities[i] + 2) / 2 * 8ll + slots * 8
                                     : (p->ctas[i] + 1) * static_cast<int64_t>(sizeof(mllb::AttnCut));
    at += (plan + 255) / 256 * 256;
    p->stats_off[i] = at;
    at += slots * p->rows[i] * 8;
    p->acc_off[i] = at;
    at += slots * p->rows[i] * head_dim * 4;
  }
  p->bytes = at;
  return MLLB_OK;
}

int check_attn_sizes(int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t seqs, int64_t groups) {
  if (tokens <= 0 || q_heads <= 0 || kv_heads <= 0 || seqs <= 0 || groups < 0) return fail(MLLB_EINVAL, "sizes must be positive");
  if (head_dim != 64 && head_dim != 128)
    return fail(MLLB_EUNSUPPORTED, "head_dim=%lld is not 64 or 128", static_cast<long long>(head_dim));
  if (q_heads % kv_heads) return fail(MLLB_EINVAL, "q_heads is not a multiple of kv_heads");
  if (q_heads > 1024 || tokens > (1 << 24) || tokens * q_heads >= (1ll << 31))
    return fail(MLLB_EINVAL, "q_heads or tokens out of range");
  if (groups > seqs) return fail(MLLB_EINVAL, "more groups than sequences");
  if (seqs > mllb::kAttnMaxEntities || seqs + groups > mllb::kAttnMaxEntities)
    return fail(MLLB_EUNSUPPORTED, "more than %d sequences and groups", mllb::kAttnMaxEntities);
  return MLLB_OK;
}

// What the plan of a call goes by.
int check_attn_call(const mllb_paged_attn* p, const mllb_paged_cache* cache) {
  const int rc = check_attn_sizes(p->tokens, p->q_heads, cache->kv_heads, cache->head_dim, p->seqs, p->groups);
  if (rc) return rc;
  if (p->table_width <= 0 || (p->groups && p->prefix_width <= 0)) return fail(MLLB_EINVAL, "page tables need a width");
  if (p->table_width >= (1 << 30) / cache->page_size || (p->groups && p->prefix_width >= (1 << 30) / cache->page_size))
    return fail(MLLB_EINVAL, "page tables of 2^30 rows or more");
  return MLLB_OK;
}

template <int D, int R>
int launch_few(const mllb::AttnArgs& a, const mllb::AttnPass& pass, const CUtensorMap& k, const CUtensorMap& v, bool bf16,
               int dev, cudaStream_t stream) {
  using C = mllb::AttnFew<D, R>;
  auto kernel = bf16 ? mllb::paged_attn_few_kernel<D, R, true> : mllb::paged_attn_few_kernel<D, R, false>;
  int grid, per_sm, rc;
  if ((rc = stream_grid(kernel, C::kSmem, C::kThreads, dev, pass.ctas, &grid, &per_sm))) return rc;
  return launched(launch(kernel, dim3(static_cast<unsigned>(pass.ctas)), dim3(C::kThreads), C::kSmem, stream, kEarly, a, pass,
                         k, v),
                  "paged attention kernel");
}

template <typename Kernel>
int registers_of(Kernel kernel) {
  cudaFuncAttributes attr = {};
  return cudaFuncGetAttributes(&attr, kernel) == cudaSuccess ? attr.numRegs : 0;
}

// Row tiles of 128 queries (token, head of a KV head) x 64 elements.
template <int D>
int query_map(CUtensorMap* map, const mllb::AttnArgs& a, bool bf16) {
  const EncodeTiled encode = tensor_map_encoder();
  if (!encode) return fail(MLLB_ECUDA, "cuTensorMapEncodeTiled not found");
  const cuuint64_t dims[4] = {D, static_cast<cuuint64_t>(a.ratio), static_cast<cuuint64_t>(a.kv_heads),
                              static_cast<cuuint64_t>(a.tokens)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(a.q_head * 2), static_cast<cuuint64_t>(a.q_head * 2 * a.ratio),
                                 static_cast<cuuint64_t>(a.q_token * 2)};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(a.ratio), 1, static_cast<cuuint32_t>(128 / a.ratio)},
                   step[4] = {1, 1, 1, 1};
  const CUresult r = encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                            const_cast<uint16_t*>(a.q), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MLLB_EINVAL, "tensor map of q refused (error %d)", static_cast<int>(r));
  return MLLB_OK;
}

template <int D>
int launch_many(const mllb::AttnArgs& a, const mllb::AttnPass& pass, const CUtensorMap& k, const CUtensorMap& v, bool bf16,
                int dev, cudaStream_t stream) {
  using C = mllb::AttnMany<D>;
  auto kernel = bf16 ? mllb::paged_attn_many_kernel<D, true> : mllb::paged_attn_many_kernel<D, false>;
  int grid, per_sm, rc;
  if ((rc = stream_grid(kernel, C::kSmem, C::kThreads, dev, pass.ctas, &grid, &per_sm))) return rc;
  // The warpgroups share out the launch's registers; with fewer than that they would wait for more for good.
  static const int regs[2] = {registers_of(mllb::paged_attn_many_kernel<D, false>),
                              registers_of(mllb::paged_attn_many_kernel<D, true>)};
  if (regs[bf16] < C::kRegs) return fail(MLLB_ECUDA, "paged attention kernel built with %d registers", regs[bf16]);
  CUtensorMap q = {};
  const bool by_tma = 128 % a.ratio == 0 && a.scale_log2 >= 0.0f && a.q_head > 0 && a.q_token > 0;
  if (by_tma && (rc = query_map<D>(&q, a, bf16))) return rc;
  return launched(launch(kernel, dim3(static_cast<unsigned>(pass.ctas)), dim3(C::kThreads), C::kSmem, stream, kEarly, a, pass,
                         k, v, by_tma ? q : k, by_tma ? 1 : 0),
                  "paged attention kernel (tensor cores)");
}

template <int D>
int launch_attn(const mllb::AttnArgs& a, const mllb::AttnPass& pass, const CUtensorMap& k, const CUtensorMap& v, bool bf16,
                int dev, cudaStream_t stream) {
  switch (pass.rows) {
    case 16: return launch_few<D, 16>(a, pass, k, v, bf16, dev, stream);
    case 32: return launch_few<D, 32>(a, pass, k, v, bf16, dev, stream);
    case 64: return launch_few<D, 64>(a, pass, k, v, bf16, dev, stream);
    default: return launch_many<D>(a, pass, k, v, bf16, dev, stream);
  }
}

// Warps that join one row: four while all rows' fit on the SMs at once (few rows
// of long contexts have tens of segments each; one sequence of 4096 rows 12.4 us,
// with one warp a row 17.5), otherwise one, which has less to gather (16
// sequences of up to 8 tokens over a prefix of 8000 rows 55 us, with four 68,
// both before the tensor cores' kernel stored whole lines).
int join_parts(const mllb::AttnArgs& a, int dev) {
  return static_cast<int64_t>(a.tokens) * a.kv_heads * a.ratio * 4 <= 32ll * sm_count(dev) ? 4 : 1;
}

template <int D>
cudaError_t launch_join(const mllb::AttnArgs& a, const mllb::AttnPass& pass, int records, bool bf16, int dev,
                        cudaStream_t stream) {
  auto kernel = bf16 ? mllb::paged_join_kernel<D, true> : mllb::paged_join_kernel<D, false>;
  const int parts = join_parts(a, dev);
  const int turns = pass.rows * parts / 8;
  return launch(kernel, dim3(static_cast<unsigned>(records), static_cast<unsigned>(parts > 1 || turns < 8 ? turns : 8)), dim3(256), 0,
                stream, kEarly, a, pass, parts);
}

template <int D>
cudaError_t launch_merge(const mllb::AttnArgs& a, const mllb::AttnPass& p0, const mllb::AttnPass& p1, bool bf16,
                         int dev, cudaStream_t stream) {
  auto kernel = bf16 ? mllb::paged_merge_kernel<D, true> : mllb::paged_merge_kernel<D, false>;
  const int parts = join_parts(a, dev);
  const int64_t warps = static_cast<int64_t>(a.tokens) * a.kv_heads * a.ratio * parts;
  return launch(kernel, dim3(static_cast<unsigned>((warps + 7) / 8)), dim3(256), 0, stream, kEarly, a, p0, p1, parts);
}

}  // namespace

extern "C" {

int mllb_paged_qkv_append(const mllb_paged_append* p, const mllb_paged_cache* cache, unsigned flags, void* stream) {
  if (!p || !p->qkv || !p->positions || !p->rows || !p->page_table || !p->freqs || !p->q_out)
    return fail(MLLB_EINVAL, "null pointer");
  if (!known_flags(flags)) return fail(MLLB_EINVAL, "unknown flags %#x", flags);
  mllb::AppendArgs a = {};
  int rc = paged_cache(cache, &a.cache);
  if (rc) return rc;
  const int64_t d = cache->head_dim;
  if (cache->layers != 1) return fail(MLLB_EINVAL, "the append takes one layer's cache");
  if (p->qkv_type < MLLB_TYPE_F32 || p->qkv_type > MLLB_TYPE_BF16) return fail(MLLB_EINVAL, "unknown qkv type %d", p->qkv_type);
  if (p->tokens <= 0 || p->tokens > (1 << 24) || p->seqs <= 0 || p->seqs > (1 << 24) || p->table_width <= 0 ||
      p->table_width > (1 << 24))
    return fail(MLLB_EINVAL, "tokens, seqs or table width out of range");
  if (p->q_heads <= 0 || p->q_heads > 1024) return fail(MLLB_EINVAL, "q_heads=%lld out of range", static_cast<long long>(p->q_heads));
  if (!p->seq && p->tokens > p->seqs) return fail(MLLB_EINVAL, "without seq, token t is sequence t's: more tokens than sequences");
  if (p->rot_dim < 2 || p->rot_dim > d || p->rot_dim % 2)
    return fail(MLLB_EINVAL, "rot_dim=%lld is not an even number from 2 to head_dim", static_cast<long long>(p->rot_dim));
  const int64_t heads = p->q_heads + 2 * cache->kv_heads, size = p->qkv_type == MLLB_TYPE_F32 ? 4 : 2;
  if (p->tokens > 1 && p->qkv_stride >= (1ll << 38)) return fail(MLLB_EINVAL, "qkv_stride must be below 2^38 elements");
  if (p->tokens > 1 && p->qkv_stride < heads * d) return fail(MLLB_EINVAL, "qkv rows overlap");
  if (!aligned(p->qkv, 16) || (p->qkv_stride * size) % 16) return fail(MLLB_EALIGN, "qkv rows must be 16-byte aligned");
  if (!aligned(p->q_out, 8) || !aligned(p->freqs, 8) || !aligned(p->positions, 4) || !aligned(p->rows, 4) ||
      !aligned(p->page_table, 4) || (p->seq && !aligned(p->seq, 4)) || (p->q_gamma && !aligned(p->q_gamma, 4)) ||
      (p->k_gamma && !aligned(p->k_gamma, 4)))
    return fail(MLLB_EALIGN, "q_out and freqs need 8-byte, the other pointers 4-byte alignment");
  if (!(p->eps >= 0.0)) return fail(MLLB_EINVAL, "eps must not be negative");
  const auto in = reinterpret_cast<uintptr_t>(p->qkv), to = reinterpret_cast<uintptr_t>(p->q_out);
  if (to < in + ((p->tokens - 1) * p->qkv_stride + heads * d) * size && in < to + p->tokens * p->q_heads * d * 2)
    return fail(MLLB_EINVAL, "q_out must not overlap qkv");
  a.qkv = p->qkv;
  a.positions = p->positions;
  a.rows = p->rows;
  a.seq = p->seq;
  a.table = p->page_table;
  a.q_gamma = p->q_gamma;
  a.k_gamma = p->k_gamma;
  a.freqs = p->freqs;
  a.q_out = static_cast<uint16_t*>(p->q_out);
  a.qkv_stride = p->qkv_stride;
  a.tokens = static_cast<int>(p->tokens);
  a.q_heads = static_cast<int>(p->q_heads);
  a.seqs = static_cast<int>(p->seqs);
  a.width = static_cast<int>(p->table_width);
  a.rot = static_cast<int>(p->rot_dim);
  a.interleaved = p->interleaved != 0;
  a.eps = static_cast<float>(p->eps);
  a.magnitude = static_cast<float>(p->magnitude);
  int dev;
  if ((rc = current_device(&dev))) return rc;
  // As many warps a token as run at once with all others (one head each: 77
  // tokens of 48 heads 4.4 us, half a token's each 10.3; 1024 tokens 11.1 us,
  // one head each 30.8), two at least: each makes the token's sines again.
  int64_t warps = 32ll * sm_count(dev) / p->tokens;
  warps = warps < 2 ? 2 : warps > heads ? heads : warps;
  a.heads_per_warp = static_cast<int>((heads + warps - 1) / warps);
  a.warps_per_token = static_cast<int>((heads + a.heads_per_warp - 1) / a.heads_per_warp);
  const unsigned grid = static_cast<unsigned>((p->tokens * a.warps_per_token + mllb::kAppendWarps - 1) / mllb::kAppendWarps);
  const bool bf16 = cache->type == MLLB_TYPE_BF16;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (d == 128)
    e = p->qkv_type == MLLB_TYPE_F32   ? launch_append<128, mllb::kTypeF32>(a, bf16, grid, s)
        : p->qkv_type == MLLB_TYPE_F16 ? launch_append<128, mllb::kTypeF16>(a, bf16, grid, s)
                                       : launch_append<128, mllb::kTypeBf16>(a, bf16, grid, s);
  else
    e = p->qkv_type == MLLB_TYPE_F32   ? launch_append<64, mllb::kTypeF32>(a, bf16, grid, s)
        : p->qkv_type == MLLB_TYPE_F16 ? launch_append<64, mllb::kTypeF16>(a, bf16, grid, s)
                                       : launch_append<64, mllb::kTypeBf16>(a, bf16, grid, s);
  return launched(e, "paged append kernel");
}

int64_t mllb_paged_attention_workspace(int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t seqs,
                                       int64_t groups) {
  int dev, rc;
  if ((rc = check_attn_sizes(tokens, q_heads, kv_heads, head_dim, seqs, groups))) return rc;
  if ((rc = current_device(&dev))) return rc;
  int64_t most = 0;  // of the plans that the page tables decide between
  for (unsigned choice = 0; choice < kPlanChoices; ++choice) {
    PagedPlan plan;
    if ((rc = paged_plan(tokens, q_heads, kv_heads, head_dim, seqs, groups, choice, dev, &plan))) return rc;
    if (plan.bytes > most) most = plan.bytes;
  }
  return most;
}

int64_t mllb_paged_attention_call_workspace(const mllb_paged_attn* p, const mllb_paged_cache* cache) {
  if (!p) return fail(MLLB_EINVAL, "null pointer");
  mllb::PagedCache c;
  PagedPlan plan;
  int dev, rc;
  if ((rc = paged_cache(cache, &c)) || (rc = check_attn_call(p, cache)) || (rc = current_device(&dev)) ||
      (rc = paged_plan(p->tokens, p->q_heads, cache->kv_heads, cache->head_dim, p->seqs, p->groups, plan_choice(p, cache), dev,
                       &plan)))
    return rc;
  return plan.bytes;
}

int mllb_paged_attention(const mllb_paged_attn* p, const mllb_paged_cache* cache, void* workspace, int64_t workspace_bytes,
                         unsigned flags, void* stream) {
  if (!p || !p->q || !p->out || !p->page_table || !p->seq_lens || !workspace) return fail(MLLB_EINVAL, "null pointer");
  if (!known_flags(flags)) return fail(MLLB_EINVAL, "unknown flags %#x", flags);
  mllb::PagedCache c;
  int rc = paged_cache(cache, &c);
  if (rc) return rc;
  if (cache->layers != 1) return fail(MLLB_EINVAL, "attention takes one layer's cache");
  if ((rc = check_attn_call(p, cache))) return rc;
  if (p->groups && (!p->prefix_table || !p->prefix_lens)) return fail(MLLB_EINVAL, "null pointer: prefix table or lengths");
  if (p->groups > 1 && !p->group_start) return fail(MLLB_EINVAL, "null pointer: group_start (needed for several groups)");
  if (!p->q_start && p->tokens != p->seqs) return fail(MLLB_EINVAL, "without q_start every sequence has one token");
  if (!(p->scale == p->scale) || p->scale - p->scale != 0.0) return fail(MLLB_EINVAL, "scale must be finite");
  const int64_t strides[4] = {p->q_token_stride, p->q_head_stride, p->out_token_stride, p->out_head_stride};
  for (int64_t s : strides)
    if (s < 0 || s % 8) return fail(MLLB_EALIGN, "q and out strides must be multiples of 8 elements (16 bytes)");
  for (int64_t s : strides)
    if (s >= (1ll << 38)) return fail(MLLB_EINVAL, "q and out strides must be below 2^38 elements");
  if (rows_overlap(p->tokens, p->out_token_stride, p->q_heads, p->out_head_stride, cache->head_dim))
    return fail(MLLB_EINVAL, "rows of out overlap");
  if (!aligned(p->q, 16) || !aligned(p->out, 16) || !aligned(workspace, 16))
    return fail(MLLB_EALIGN, "q, out and workspace must be 16-byte aligned");
  for (const int32_t* at : {p->page_table, p->seq_lens, p->prefix_table, p->prefix_lens, p->group_start, p->q_start})
    if (at && !aligned(at, 4)) return fail(MLLB_EALIGN, "tables, lengths and starts must be 4-byte aligned");
  const bool in_place = p->q == p->out && (p->tokens == 1 || p->q_token_stride == p->out_token_stride) &&
                        (p->q_heads == 1 || p->q_head_stride == p->out_head_stride);
  if (!in_place && out_overlaps_q(p, cache->head_dim))
    return fail(MLLB_EINVAL, "out must be q or must not overlap its rows");
  int dev;
  if ((rc = current_device(&dev))) return rc;
  PagedPlan plan;
  const unsigned choice = plan_choice(p, cache);
  if ((rc = paged_plan(p->tokens, p->q_heads, cache->kv_heads, cache->head_dim, p->seqs, p->groups, choice, dev, &plan)))
    return rc;
  if (workspace_bytes < plan.bytes)
    return fail(MLLB_EINVAL, "workspace of %lld bytes, %lld needed", static_cast<long long>(workspace_bytes),
                static_cast<long long>(plan.bytes));
  mllb::AttnArgs a = {};
  a.q = static_cast<const uint16_t*>(p->q);
  a.out = static_cast<uint16_t*>(p->out);
  a.q_token = p->q_token_stride;
  a.q_head = p->q_head_stride;
  a.out_token = p->out_token_stride;
  a.out_head = p->out_head_stride;
  a.table = p->page_table;
  a.lens = p->seq_lens;
  a.prefix_table = p->prefix_table;
  a.prefix_lens = p->prefix_lens;
  a.group_start = p->groups ? p->group_start : nullptr;
  a.q_start = p->q_start;
  a.width = static_cast<int>(p->table_width);
  a.prefix_width = static_cast<int>(p->groups ? p->prefix_width : 0);
  a.seqs = static_cast<int>(p->seqs);
  a.groups = static_cast<int>(p->groups);
  a.tokens = static_cast<int>(p->tokens);
  a.kv_heads = c.kv_heads;
  a.ratio = static_cast<int>(p->q_heads / c.kv_heads);
  a.page_shift = c.page_shift;
  a.pages = c.pages;
  a.scale_log2 = static_cast<float>(p->scale * 1.4426950408889634);
  const bool bf16 = cache->type == MLLB_TYPE_BF16;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  mllb::AttnPass pass[2] = {};
  uint8_t* work = static_cast<uint8_t*>(workspace);
  for (int i = 0; i < plan.passes; ++i) {
    // The line of (item, key tile) pairs is counted in 32 bits.
    const int64_t items = cache->kv_heads * ((p->tokens * a.ratio + plan.rows[i] - 1) / plan.rows[i] + plan.entities[i]);
    const int64_t most = ((p->table_width + (p->groups ? p->prefix_width : 0)) * cache->page_size) / plan.keys[i] + 2 + mllb::attn_ends(plan.rows[i]);
    if (items * most >= (1ll << 31)) return fail(MLLB_EUNSUPPORTED, "too many rows x keys for one call");
    pass[i].mode = plan.mode[i];
    pass[i].entities = plan.entities[i];
    pass[i].ctas = plan.ctas[i];
    pass[i].dense = plan.dense[i];
    pass[i].by_item = plan.by_item[i];
    pass[i].slots = plan.slots[i];
    pass[i].rows = plan.rows[i];
    pass[i].keys = plan.keys[i];
    pass[i].plan = reinterpret_cast<int32_t*>(work + plan.plan_off[i]);
    pass[i].stats = reinterpret_cast<float2*>(work + plan.stats_off[i]);
    pass[i].acc = reinterpret_cast<float*>(work + plan.acc_off[i]);
  }
  for (int i = 0; i < plan.passes; ++i) {
    CUtensorMap kmap, vmap;
    const int box = static_cast<int>(cache->page_size < plan.keys[i] ? cache->page_size : plan.keys[i]);
    if ((rc = paged_map(&kmap, cache, cache->k, box)) || (rc = paged_map(&vmap, cache, cache->v, box))) return rc;
    rc = cache->head_dim == 128 ? launch_attn<128>(a, pass[i], kmap, vmap, bf16, dev, s)
                                : launch_attn<64>(a, pass[i], kmap, vmap, bf16, dev, s);
    if (rc) return rc;
  }
  if (!pass[0].dense)
    return launched(cache->head_dim == 128 ? launch_join<128>(a, pass[0], plan.records[0], bf16, dev, s)
                                           : launch_join<64>(a, pass[0], plan.records[0], bf16, dev, s),
                    "paged join kernel");
  return launched(cache->head_dim == 128 ? launch_merge<128>(a, pass[0], pass[1], bf16, dev, s)
                                         : launch_merge<64>(a, pass[0], pass[1], bf16, dev, s),
                  "paged merge kernel");
}

int64_t mllb_beam_select_workspace(int64_t batch, int64_t beams, int64_t vocab, int64_t n) {
  const int rc = check_beams(batch, beams, vocab, n);
  if (rc) return rc;
  return batch * beams * beam_steps(vocab) * (n * 8 + static_cast<int64_t>(sizeof(mllb::BeamChunkSum)));
}

int mllb_beam_select(const mllb_beam_scores* p, float* out_scores, int32_t* out_tokens, int32_t* out_parents,
                     void* workspace, int64_t workspace_bytes, unsigned flags, void* stream) {
  if (!p || !p->logits || !p->scores || !out_scores || !out_tokens || !out_parents || !workspace)
    return fail(MLLB_EINVAL, "null pointer");
  if (!known_flags(flags)) return fail(MLLB_EINVAL, "unknown flags %#x", flags);
  int rc = check_beams(p->batch, p->beams, p->vocab, p->n);
  if (rc) return rc;
  if (p->type < MLLB_TYPE_F32 || p->type > MLLB_TYPE_BF16) return fail(MLLB_EINVAL, "unknown logits type %d", p->type);
  if (p->done && (p->end_token < 0 || p->end_token >= p->vocab)) return fail(MLLB_EINVAL, "end_token outside the vocabulary");
  const int64_t size = p->type == MLLB_TYPE_F32 ? 4 : 2;
  if (!aligned(p->logits, size) || !aligned(p->scores, 4) || !aligned(out_scores, 4) || !aligned(out_tokens, 4) ||
      !aligned(out_parents, 4) || !aligned(workspace, 16))
    return fail(MLLB_EALIGN, "workspace needs 16-byte, the other pointers their type's alignment");
  if (p->batch_stride < 0 || p->beam_stride < 0 || p->batch_stride >= (1ll << 38) || p->beam_stride >= (1ll << 38))
    return fail(MLLB_EINVAL, "strides must not be negative, and below 2^38 elements");
  const int64_t need = mllb_beam_select_workspace(p->batch, p->beams, p->vocab, p->n);
  if (workspace_bytes < need)
    return fail(MLLB_EINVAL, "workspace of %lld bytes, %lld needed", static_cast<long long>(workspace_bytes),
                static_cast<long long>(need));
  // An entry's results are written while other entries' scores, sums and lists are still read.
  const int64_t rows = p->batch * p->beams, picked = p->batch * p->n * 4;
  const Span in[] = {{p->scores, rows * 4}, {p->done ? p->done : workspace, p->done ? rows : 1}, {workspace, need}};
  const Span out[] = {{out_scores, picked}, {out_tokens, picked}, {out_parents, picked}};
  for (int i = 0; i < 3; ++i) {
    for (const Span& s : in)
      if (meet(out[i], s) && !(i == 0 && out_scores == p->scores && s.at == p->scores && p->n == p->beams))
        return fail(MLLB_EINVAL, "results must not overlap scores (but be them, where n is beams), done or the workspace");
    for (int j = 0; j < i; ++j)
      if (meet(out[i], out[j])) return fail(MLLB_EINVAL, "results must not overlap one another");
  }
  mllb::BeamArgs a = {};
  a.logits = p->logits;
  a.scores = p->scores;
  a.done = p->done;
  a.out_scores = out_scores;
  a.out_tokens = out_tokens;
  a.out_parents = out_parents;
  a.batch_stride = p->batch_stride;
  a.beam_stride = p->beam_stride;
  a.batch = static_cast<int>(p->batch);
  a.beams = static_cast<int>(p->beams);
  a.vocab = static_cast<int>(p->vocab);
  // About four CTAs per SM (they fit at once), but no chunk shorter than a
  // step: the fewer chunks, the less is listed and joined (32 x 8 rows of 151936
  // bf16: 33 us, in chunks of one step 81), while few rows want all SMs (1 x 4:
  // 11 us, with one CTA for 36 steps of a row 23).
  int dev;
  if ((rc = current_device(&dev))) return rc;
  const int64_t steps = beam_steps(p->vocab);
  int64_t chunks = 4ll * sm_count(dev) / rows;
  if (chunks < 1) chunks = 1;
  a.steps = static_cast<int>((steps + chunks - 1) / chunks);
  if (a.steps > mllb::kBeamStepsMost) a.steps = mllb::kBeamStepsMost;
  a.chunks = static_cast<int>((steps + a.steps - 1) / a.steps);
  a.n = static_cast<int>(p->n);
  a.end_token = static_cast<int>(p->end_token);
  const int64_t lists = p->batch * p->beams * a.chunks;
  a.sums = static_cast<mllb::BeamChunkSum*>(workspace);
  a.keys = reinterpret_cast<unsigned long long*>(a.sums + lists);
  // 16-byte loads where every row starts on that boundary.
  const bool vector = aligned(p->logits, 16) && (p->batch_stride * size) % 16 == 0 && (p->beam_stride * size) % 16 == 0;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = p->type == MLLB_TYPE_F32   ? launch_scan<mllb::kTypeF32>(a, vector, s)
                        : p->type == MLLB_TYPE_F16 ? launch_scan<mllb::kTypeF16>(a, vector, s)
                                                   : launch_scan<mllb::kTypeBf16>(a, vector, s);
  if ((rc = launched(e, "beam scan kernel"))) return rc;
  return launched(launch(mllb::beam_pick_kernel, dim3(static_cast<unsigned>(a.batch)), dim3(mllb::kPickThreads), 0, s, kEarly, a),
                  "beam pick kernel");
}

int mllb_beam_reorder(const mllb_beam_rows* p, const mllb_paged_cache* cache, int32_t* table_out, int32_t* lens_out,
                      int32_t* used, unsigned flags, void* stream) {
  if (!p || !p->parents || !p->page_table || !p->seq_lens || !p->fresh || !table_out || !lens_out || !used)
    return fail(MLLB_EINVAL, "null pointer");
  if (!known_flags(flags)) return fail(MLLB_EINVAL, "unknown flags %#x", flags);
  mllb::ReorderArgs a = {};
  const int rc = paged_cache(cache, &a.cache);
  if (rc) return rc;
  if (p->batch <= 0 || p->beams <= 0 || p->batch > 65535 || p->beams > 65535 || p->batch * p->beams > 65535)
    return fail(MLLB_EINVAL, "batch x beams out of range");
  if (p->table_width <= 0 || p->table_width > (1 << 24)) return fail(MLLB_EINVAL, "table width out of range");
  const int64_t rows = p->batch * p->beams;
  // Rows are written while others' parents, lines, lengths and fresh pages are still read.
  const Span in[] = {{p->parents, rows * 4}, {p->page_table, rows * p->table_width * 4}, {p->seq_lens, rows * 4}, {p->fresh, rows * 4}};
  const Span out[] = {{table_out, rows * p->table_width * 4}, {lens_out, rows * 4}, {used, rows * 4}};
  for (int i = 0; i < 3; ++i) {
    for (const Span& s : in)
      if (meet(out[i], s)) return fail(MLLB_EINVAL, "the reordered table, lengths and used must not overlap what they come from");
    for (int j = 0; j < i; ++j)
      if (meet(out[i], out[j])) return fail(MLLB_EINVAL, "the reordered table, lengths and used must not overlap one another");
  }
  if (!aligned(p->parents, 4) || !aligned(p->page_table, 4) || !aligned(p->seq_lens, 4) || !aligned(p->fresh, 4) ||
      !aligned(table_out, 4) || !aligned(lens_out, 4) || !aligned(used, 4))
    return fail(MLLB_EALIGN, "pointers must be 4-byte aligned");
  a.parents = p->parents;
  a.table = p->page_table;
  a.lens = p->seq_lens;
  a.fresh = p->fresh;
  a.table_out = table_out;
  a.lens_out = lens_out;
  a.used = used;
  a.beams = static_cast<int>(p->beams);
  a.width = static_cast<int>(p->table_width);
  a.row_bytes = static_cast<int>(cache->head_dim * 2);
  const int64_t triples = 2 * cache->layers * cache->kv_heads;
  const int64_t ctas = (triples + mllb::kReorderWarps - 1) / mllb::kReorderWarps;
  return launched(launch(mllb::beam_reorder_kernel, dim3(static_cast<unsigned>(ctas), static_cast<unsigned>(rows)),
                         dim3(mllb::kReorderWarps * 32), 0, static_cast<cudaStream_t>(stream), kEarly, a),
                  "beam reorder kernel");
}

}  // extern "C"
