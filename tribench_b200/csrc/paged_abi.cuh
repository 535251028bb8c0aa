// paged_abi.cuh — the C entry points of the paged cache (include/sage_sm100.h): validation, tensor
// maps and launches. Included by sage_abi.cu, whose helpers it uses.
#pragma once

namespace {

int check_cache(const sage_paged_cache* c) {
  if (!c) return fail(SAGE_ERR_INVALID_ARG, "cache is NULL");
  if (c->dtype != SAGE_DTYPE_F16 && c->dtype != SAGE_DTYPE_BF16)
    return fail(SAGE_ERR_INVALID_ARG, "dtype %d is neither SAGE_DTYPE_F16 nor SAGE_DTYPE_BF16", c->dtype);
  if (c->storage != SAGE_CACHE_16BIT && c->storage != SAGE_CACHE_INT8)
    return fail(SAGE_ERR_INVALID_ARG, "cache storage %d unknown", c->storage);
  if (c->head_dim != 64 && c->head_dim != 128)
    return fail(SAGE_ERR_INVALID_ARG, "head_dim %lld unsupported (64 or 128)", (long long)c->head_dim);
  const int64_t P = c->page_size;
  if (P < 16 || P > 1024 || (P & (P - 1)))
    return fail(SAGE_ERR_INVALID_ARG, "page_size %lld is not a power of two from 16 to 1024", (long long)P);
  if (c->num_pages <= 0 || c->num_pages > (1LL << 31) - 1 || c->heads_kv <= 0 || c->heads_kv > 65535)
    return fail(SAGE_ERR_INVALID_ARG, "empty or oversized cache: num_pages=%lld heads_kv=%lld",
                (long long)c->num_pages, (long long)c->heads_kv);
  const bool i8 = c->storage == SAGE_CACHE_INT8;
  const int64_t unit = i8 ? 16 : 8;  // elements of 16 bytes
  for (int i = 0; i < 3; ++i) {
    if (c->k_strides[i] <= 0 || c->k_strides[i] % unit || c->v_strides[i] <= 0 || c->v_strides[i] % unit)
      return fail(SAGE_ERR_INVALID_ARG, "cache stride[%d] (k %lld, v %lld) must be a positive multiple of %lld elements",
                  i, (long long)c->k_strides[i], (long long)c->v_strides[i], (long long)unit);
    if (c->k_strides[i] > (1LL << 33) || c->v_strides[i] > (1LL << 33))
      return fail(SAGE_ERR_INVALID_ARG, "cache stride[%d] is too large", i);
  }
  if (!c->k || !c->v || (i8 && (!c->k_scale || !c->v_scale))) return fail(SAGE_ERR_INVALID_ARG, "NULL cache pointer");
  if (!i8 && (c->k_scale || c->v_scale || c->k_mean))
    return fail(SAGE_ERR_INVALID_ARG, "scales and k_mean belong to an INT8 cache");
  if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->k_scale) || !aligned16(c->v_scale) || !aligned16(c->k_mean))
    return fail(SAGE_ERR_INVALID_ARG, "cache tensors must be 16-byte aligned");
  return SAGE_OK;
}

// Checks what append, gather and attention share, and fills the device-side description.
int paged_seqs(const sage_paged_cache* c, const int32_t* page_table, int64_t table_stride, int64_t pages_per_seq,
               const int32_t* seq_lens, const int32_t* cu, int64_t batch, int64_t tokens, int64_t max_new,
               sage::PagedSeqs* s) {
  if (batch > 0 && (!page_table || !seq_lens)) return fail(SAGE_ERR_INVALID_ARG, "page_table or seq_lens is NULL");
  if (((reinterpret_cast<uintptr_t>(page_table) | reinterpret_cast<uintptr_t>(seq_lens) |
        reinterpret_cast<uintptr_t>(cu)) & 3u) != 0)
    return fail(SAGE_ERR_INVALID_ARG, "page_table, seq_lens and cu_seqlens must be 4-byte aligned");
  if (batch < 0 || tokens < 0 || batch > (1 << 20) || tokens > (1LL << 30))
    return fail(SAGE_ERR_INVALID_ARG, "batch=%lld or tokens=%lld out of range", (long long)batch, (long long)tokens);
  if (!cu && tokens != batch)
    return fail(SAGE_ERR_INVALID_ARG, "without cu_seqlens every sequence has one token: %lld tokens for %lld sequences",
                (long long)tokens, (long long)batch);
  if (pages_per_seq <= 0 || pages_per_seq > (1LL << 30) || table_stride < 0 || (batch > 1 && table_stride < pages_per_seq))
    return fail(SAGE_ERR_INVALID_ARG, "pages_per_seq=%lld and table_stride=%lld do not fit", (long long)pages_per_seq,
                (long long)table_stride);
  if (max_new < 1) return fail(SAGE_ERR_INVALID_ARG, "max_seqlen_q=%lld must be positive", (long long)max_new);
  s->cu = cu; s->lens = seq_lens; s->table = page_table; s->table_stride = table_stride;
  s->batch = (int)batch; s->width = (int)pages_per_seq; s->tokens = (int)tokens;
  s->max_new = (int)std::min(max_new, tokens);
  s->cap = (int)std::min<int64_t>(pages_per_seq * c->page_size, 1LL << 30);
  return SAGE_OK;
}

int page_shift(const sage_paged_cache* c) {
  int s = 0;
  while ((1LL << s) < c->page_size) ++s;
  return s;
}

Span cache_span(const sage_paged_cache* c, bool v) {
  return tensor_span(v ? c->v : c->k, v ? c->v_strides : c->k_strides, c->num_pages, c->heads_kv, c->page_size,
                     c->head_dim, c->storage == SAGE_CACHE_INT8 ? 1 : 2);
}
Span scale_span(const sage_paged_cache* c, bool v) {
  return buffer_span(v ? c->v_scale : c->k_scale, static_cast<size_t>(c->num_pages * c->heads_kv * c->page_size) * 4);
}

sage::PagedStore paged_store(const sage_paged_cache* c) {
  sage::PagedStore s{};
  s.k = c->k; s.v = c->v; s.k_scale = c->k_scale; s.v_scale = c->v_scale; s.k_mean = c->k_mean;
  s.k_sp = c->k_strides[0]; s.k_sh = c->k_strides[1]; s.k_st = c->k_strides[2];
  s.v_sp = c->v_strides[0]; s.v_sh = c->v_strides[1]; s.v_st = c->v_strides[2];
  s.pages = (int)c->num_pages; s.page_shift = page_shift(c); s.heads = (int)c->heads_kv;
  return s;
}

template <bool READ>
int paged_move(const sage_paged_cache* c, const void* k, const void* v, const int64_t* ks, const int64_t* vs,
               const int32_t* table, int64_t table_stride, int64_t width, const int32_t* lens, const int32_t* cu,
               int64_t batch, int64_t tokens, void* stream) {
  if (int rc = check_cache(c)) return rc;
  sage::PagedMoveParams p{};
  if (int rc = paged_seqs(c, table, table_stride, width, lens, cu, batch, tokens, 1LL << 30, &p.s)) return rc;
  if (tokens == 0 || batch == 0) return SAGE_OK;
  int64_t k3[3], v3[3];
  if (int rc = packed_strides("k", ks, k3)) return rc;
  if (int rc = packed_strides("v", vs, v3)) return rc;
  if (!k || !v) return fail(SAGE_ERR_INVALID_ARG, "NULL tensor pointer");
  if (!aligned16(k) || !aligned16(v)) return fail(SAGE_ERR_INVALID_ARG, "k/v must be 16-byte aligned");
  for (int i = 0; i < 2; ++i)
    if (ks[i] > (1LL << 33) || vs[i] > (1LL << 33)) return fail(SAGE_ERR_INVALID_ARG, "k/v stride[%d] is too large", i);
  // packed tensors must not share a byte with the cache, nor what is read back with itself
  const Span sk = tensor_span(k, k3, 1, c->heads_kv, tokens, c->head_dim, 2);
  const Span sv = tensor_span(v, v3, 1, c->heads_kv, tokens, c->head_dim, 2);
  const Span held[] = {cache_span(c, false), cache_span(c, true), scale_span(c, false), scale_span(c, true)};
  for (const Span& h : held)
    if (spans_overlap(sk, h) || spans_overlap(sv, h))
      return fail(SAGE_ERR_INVALID_ARG, "k or v overlaps the cache");
  if (READ && spans_overlap(sk, sv)) return fail(SAGE_ERR_INVALID_ARG, "k and v overlap each other");
  if (int rc = check_arch()) return rc;
  p.c = paged_store(c);
  p.k = const_cast<void*>(k); p.v = const_cast<void*>(v);
  p.k_sh = ks[0]; p.k_st = ks[1]; p.v_sh = vs[0]; p.v_st = vs[1];
  // Tokens per block: one, so that few tokens spread over the SMs, up to 32, so that the lookup of a
  // token's page is paid by fewer warps. In between eight blocks of K and of V per SM, or, where the
  // arithmetic of INT8 counts, four (32768 tokens of 8 heads: append 46.0 instead of 48.2 us, with means
  // 52.4 instead of 56.1; of 16 bits eight: 46.9 instead of 48.5).
  const int64_t blocks = 148 * (c->storage == SAGE_CACHE_INT8 ? 4 : 8);
  p.per_shift = 0;
  while (p.per_shift < 5 && tokens >= (blocks << (p.per_shift + 1))) ++p.per_shift;
  const dim3 grid((unsigned)cdiv(tokens, int64_t(1) << p.per_shift), 2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool i8 = c->storage == SAGE_CACHE_INT8, bf = c->dtype == SAGE_DTYPE_BF16;
#define SAGE_MOVE(D, T, I8) sage::paged_move_kernel<D, T, I8, READ><<<grid, sage::kPagedThreads, 0, st>>>(p)
#define SAGE_MOVE_T(D)                                                                                   \
  do {                                                                                                   \
    if (i8) { if (bf) SAGE_MOVE(D, __nv_bfloat16, true); else SAGE_MOVE(D, __half, true); }              \
    else SAGE_MOVE(D, __half, false); /* 16-bit values are copied as they are */                         \
  } while (0)
  if (c->head_dim == 128) SAGE_MOVE_T(128);
  else SAGE_MOVE_T(64);
#undef SAGE_MOVE_T
#undef SAGE_MOVE
  SAGE_CUDA_TRY(cudaGetLastError());
  return SAGE_OK;
}

// ---------------------------------------------------------------- attention over the cache
size_t decode_ws_bytes(int64_t D) {
  const size_t rows = size_t(2) * sage::kDecMaxPieces * sage::kDecMaxRows;
  return align256(rows * D * 4) + align256(rows * 4 * 4) + align256(sizeof(int4) * sage::kDecMaxPieces);
}

// Tensor map of the cache's K or V: [pages][heads][page][D], boxes of at most `rows` tokens.
int cache_map(CUtensorMap* map, const sage_paged_cache* c, bool v, int rows, bool swizzle = true) {
  const int64_t* s = v ? c->v_strides : c->k_strides;
  const void* base = v ? c->v : c->k;
  const uint32_t box = (uint32_t)std::min<int64_t>(rows, c->page_size);
  if (c->storage == SAGE_CACHE_INT8)
    return encode_4d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, base, c->head_dim, c->page_size, c->heads_kv, c->num_pages,
                     s[2], s[1], s[0], (uint32_t)c->head_dim, box,
                     !swizzle ? CU_TENSOR_MAP_SWIZZLE_NONE
                     : c->head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
  return encode_4d(map, c->dtype == SAGE_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                   2, base, c->head_dim, c->page_size, c->heads_kv, c->num_pages, s[2], s[1], s[0], 64, box,
                   CU_TENSOR_MAP_SWIZZLE_128B);
}
// Workspace of the chunk kernel: partial sums as above with 256 rows per item, and the schedule.
struct ChunkWs {
  size_t ml, desc, items, prefix, pieces, bytes;  // offsets; the partial sums come first
};
ChunkWs chunk_ws(int64_t D, int64_t max_items) {
  const size_t rows = size_t(2) * sage::kChunkPieces * sage::kChunkRows;
  ChunkWs w;
  w.ml = align256(rows * D * 4);
  w.desc = w.ml + align256(rows * 4 * 4);
  w.items = w.desc + align256(sizeof(int4) * sage::kChunkPieces);
  w.prefix = w.items + align256(sizeof(sage::ChunkItem) * max_items);
  w.pieces = w.prefix + align256(sizeof(int64_t) * max_items);
  w.bytes = w.pieces + align256(sizeof(sage::ChunkPiece) * sage::kChunkPieces);
  return w;
}
// Rows of a query tile: G heads in `parts` equal parts of at most 128, TT tokens.
struct ChunkTile {
  int64_t parts, Gp, TT;
};
ChunkTile chunk_tile(int64_t G) {
  const int64_t parts = cdiv(G, 128), Gp = cdiv(G, parts);
  return {parts, Gp, 128 / Gp};
}
// Blocks of query rows of a call: a sequence's last block may be partly filled.
int64_t chunk_items(int64_t batch, int64_t total_q, int64_t G) { return total_q / (2 * chunk_tile(G).TT) + batch; }

// Which kernel. sage_decode.cuh streams the cache once per 16 query rows of a key/value head, at HBM's
// rate; sage_chunk.cuh once per 256, at a rate that the softmax of a 128-row tile sets. Above 16 rows the
// second wins over a 16-bit cache (32 rows over 16 sequences of 20000: 239 instead of 392 us), above 32
// over an INT8 one, whose codes cost it more (17 to 32 rows: 341 instead of 311 us; 64: 343 instead of
// 592).
int64_t few_rows(const sage_paged_cache* c) { return (c->storage == SAGE_CACHE_INT8 ? 2 : 1) * sage::kDecMaxRows; }
// Sequences from which two kernels pay: 64 single tokens over up to 8192 beside a chunk of 512, 32/8 heads: 311
// instead of 377 us (INT8 237 instead of 628); 8 sequences 39 instead of 31 us, the price of two more launches.
constexpr int64_t kMixedBatch = 16;
enum class PagedRoute { kFew, kMany, kBoth };
// Of a batch the host knows a bound on the largest sequence's tokens, and their total. Where the bound means
// many rows and what it leaves to the others few on average (single tokens beside a chunk), both kernels
// run, each on the sequences of its kind; else the bound decides. So the bound picks the kernels: with no
// better one than the total (a caller that does not know its largest sequence) nothing is left to the
// others, and from 16 sequences on both kernels run, of which one may find no work; and single tokens
// beside several chunks, whose rows count as the others', go through the many-row kernel.
PagedRoute paged_route(const sage_paged_cache* c, int64_t G, int64_t batch, int64_t total_q, int64_t max_seqlen_q) {
  const int64_t few = few_rows(c), largest = std::min(max_seqlen_q, total_q);  // a bound may be anything above
  if (largest * G <= few) return PagedRoute::kFew;
  const bool mixed = batch >= kMixedBatch && (total_q - largest) * G <= few * (batch - 1);
  return mixed ? PagedRoute::kBoth : PagedRoute::kMany;
}

// Tensor map of the packed queries: boxes of Gp heads by TT tokens by 64 channels.
int query_map(CUtensorMap* map, const void* q, int dtype, int64_t D, int64_t heads, int64_t tokens, int64_t sh, int64_t st,
              const ChunkTile& t) {
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)tokens};
  cuuint64_t strides[2] = {(cuuint64_t)(sh * 2), (cuuint64_t)(st * 2)};
  cuuint32_t box[3] = {64, (cuuint32_t)t.Gp, (cuuint32_t)t.TT};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = g_encode(map, dtype == SAGE_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                              const_cast<void*>(q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(SAGE_ERR_CUDA, "cuTensorMapEncodeTiled failed (CUresult %d)", (int)r);
  return SAGE_OK;
}

struct PagedMaps {
  CUtensorMap q, k, v;
};

// A launch that may start while its predecessor in the stream still runs; the kernel waits for it on
// the device (griddepcontrol.wait) before it reads anything the predecessor writes.
template <typename... A>
int launch_early(void (*kern)(A...), dim3 grid, int threads, int smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  SAGE_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, args...));
  return SAGE_OK;
}

template <int D, bool I8, typename T>
int launch_chunk(const PagedMaps& m, const sage::ChunkParams& p, cudaStream_t st) {
  using C = sage::ChunkCfg<D, I8, T>;
  auto kern = sage::paged_chunk_kernel<D, I8, T>;
  if (int rc = ensure_smem(reinterpret_cast<const void*>(kern), C::SMEM_BYTES)) return rc;
  sage::paged_schedule_kernel<<<1, sage::kScheduleThreads, 0, st>>>(p);
  SAGE_CUDA_TRY(cudaGetLastError());
  if (int rc = launch_early(kern, dim3(sage::kChunkPieces), sage::kChunkThreads, C::SMEM_BYTES, st, m.q, m.k, m.v, p)) return rc;
  const int64_t rows = p.d.s.max_new >= p.d.TT ? sage::kChunkRows : p.d.s.max_new * p.d.Gp;  // of a block, at most
  return launch_early(sage::paged_chunk_join_kernel<D, I8, T>, dim3(sage::kChunkPieces, (unsigned)cdiv(rows, sage::kJoinRows)),
                      sage::kJoinRows * D / 4, 0, st, p.d);
}

template <int D, bool I8, typename T, int NR>
int launch_decode(const PagedMaps& m, const sage::DecodeParams& p, int max_rows, cudaStream_t st) {
  using C = sage::DecodeCfg<D, I8, NR>;
  auto kern = sage::paged_decode_kernel<D, I8, T, NR>;
  constexpr int pieces = C::CTAS * 148;
  static_assert(pieces <= sage::kDecMaxPieces && C::ROWS <= sage::kDecMaxRows, "workspace");
  if (int rc = ensure_smem(reinterpret_cast<const void*>(kern), C::SMEM)) return rc;
  kern<<<pieces, sage::kDecThreads, C::SMEM, st>>>(m.k, m.v, p);
  SAGE_CUDA_TRY(cudaGetLastError());
  return launch_early(sage::paged_combine_kernel<D, I8, T, NR>, dim3(pieces, (unsigned)std::min(max_rows, C::ROWS)),
                      sage::kCombineThreads, 0, st, p);
}

template <int D>
int chunk_dispatch(bool i8, bool bf, const PagedMaps& m, const sage::ChunkParams& p, cudaStream_t st) {
  if (i8) return bf ? launch_chunk<D, true, __nv_bfloat16>(m, p, st) : launch_chunk<D, true, __half>(m, p, st);
  return bf ? launch_chunk<D, false, __nv_bfloat16>(m, p, st) : launch_chunk<D, false, __half>(m, p, st);
}

// Eight query rows where no sequence has more, else sixteen.
template <int D, bool I8, typename T>
int decode_rows(const PagedMaps& m, const sage::DecodeParams& p, int max_rows, cudaStream_t st) {
  return max_rows <= 8 ? launch_decode<D, I8, T, 1>(m, p, max_rows, st) : launch_decode<D, I8, T, 2>(m, p, max_rows, st);
}
template <int D>
int decode_dispatch(bool i8, bool bf, const PagedMaps& m, const sage::DecodeParams& p, int max_rows, cudaStream_t st) {
  if (i8) return bf ? decode_rows<D, true, __nv_bfloat16>(m, p, max_rows, st) : decode_rows<D, true, __half>(m, p, max_rows, st);
  return bf ? decode_rows<D, false, __nv_bfloat16>(m, p, max_rows, st) : decode_rows<D, false, __half>(m, p, max_rows, st);
}

}  // namespace

extern "C" {

int sage_paged_append(const sage_paged_cache* cache, const void* k, const void* v, const int64_t k_strides[2],
                      const int64_t v_strides[2], const int32_t* page_table, int64_t table_stride,
                      int64_t pages_per_seq, const int32_t* seq_lens, const int32_t* cu_seqlens, int64_t batch,
                      int64_t tokens, void* stream) {
  g_last_error.clear();
  return paged_move<false>(cache, k, v, k_strides, v_strides, page_table, table_stride, pages_per_seq, seq_lens,
                           cu_seqlens, batch, tokens, stream);
}

int sage_paged_gather(const sage_paged_cache* cache, void* k, void* v, const int64_t k_strides[2],
                      const int64_t v_strides[2], const int32_t* page_table, int64_t table_stride,
                      int64_t pages_per_seq, const int32_t* seq_lens, const int32_t* cu_seqlens, int64_t batch,
                      int64_t tokens, void* stream) {
  g_last_error.clear();
  return paged_move<true>(cache, k, v, k_strides, v_strides, page_table, table_stride, pages_per_seq, seq_lens,
                          cu_seqlens, batch, tokens, stream);
}

size_t sage_paged_workspace_bytes(const sage_paged_cache* cache, int64_t heads_q, int64_t batch, int64_t total_q,
                                  int64_t max_seqlen_q, int64_t pages_per_seq) {
  if (!cache || heads_q <= 0 || batch <= 0 || total_q <= 0 || max_seqlen_q <= 0 || pages_per_seq <= 0) return 0;
  if (cache->heads_kv <= 0 || heads_q % cache->heads_kv) return 0;
  const int64_t G = heads_q / cache->heads_kv;
  // the two kernels of a mixed batch run one after the other in the same workspace
  const PagedRoute route = paged_route(cache, G, batch, total_q, max_seqlen_q);
  const size_t many = route == PagedRoute::kFew ? 0 : chunk_ws(cache->head_dim, chunk_items(batch, total_q, G)).bytes;
  return std::max(many, route == PagedRoute::kMany ? size_t(0) : decode_ws_bytes(cache->head_dim));
}

int sage_paged_attn_fwd(const sage_paged_cache* cache, const void* q, const int64_t q_strides[2], void* o,
                        const int64_t o_strides[2], int64_t heads_q, const int32_t* page_table, int64_t table_stride,
                        int64_t pages_per_seq, const int32_t* seq_lens, const int32_t* cu_seqlens, int64_t batch,
                        int64_t total_q, int64_t max_seqlen_q, int causal, int64_t window, int64_t sinks,
                        float sm_scale, void* workspace, size_t workspace_bytes, void* stream) {
  g_last_error.clear();
  const sage_paged_cache* c = cache;
  if (int rc = check_cache(c)) return rc;
  if (heads_q <= 0 || heads_q % c->heads_kv != 0)
    return fail(SAGE_ERR_INVALID_ARG, "heads_q=%lld is not a multiple of heads_kv=%lld", (long long)heads_q,
                (long long)c->heads_kv);
  const int64_t G = heads_q / c->heads_kv;
  if (window < 0 || sinks < 0) return fail(SAGE_ERR_INVALID_ARG, "window and sinks must not be negative");
  if (window > 0 && !causal) return fail(SAGE_ERR_INVALID_ARG, "a window needs causal attention");
  if (sinks > 0 && window == 0) return fail(SAGE_ERR_INVALID_ARG, "sinks need a window");
  sage::DecodeParams p{};
  if (int rc = paged_seqs(c, page_table, table_stride, pages_per_seq, seq_lens, cu_seqlens, batch, total_q,
                          max_seqlen_q, &p.s))
    return rc;
  if (total_q * G > (1LL << 30)) return fail(SAGE_ERR_INVALID_ARG, "total_q * heads_q / heads_kv exceeds 2^30");
  if (total_q == 0 || batch == 0) return SAGE_OK;
  int64_t qs[3], os[3];
  if (int rc = packed_strides("q", q_strides, qs)) return rc;
  if (int rc = packed_strides("o", o_strides, os)) return rc;
  if (!q || !o) return fail(SAGE_ERR_INVALID_ARG, "NULL tensor pointer");
  if (!aligned16(q) || !aligned16(o)) return fail(SAGE_ERR_INVALID_ARG, "q/o must be 16-byte aligned");
  const size_t need = sage_paged_workspace_bytes(c, heads_q, batch, total_q, max_seqlen_q, pages_per_seq);
  if (!workspace || workspace_bytes < need)
    return fail(SAGE_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  if (!aligned16(workspace)) return fail(SAGE_ERR_INVALID_ARG, "workspace must be 16-byte aligned");
  const NamedSpan others[] = {{"k", cache_span(c, false)}, {"v", cache_span(c, true)},
                              {"k_scale", scale_span(c, false)}, {"v_scale", scale_span(c, true)},
                              {"workspace", buffer_span(workspace, workspace_bytes)}};
  if (int rc = check_out_alias(o, os, tensor_span(o, os, 1, heads_q, total_q, c->head_dim, 2), q, qs,
                               tensor_span(q, qs, 1, heads_q, total_q, c->head_dim, 2), others, 5))
    return rc;
  if (int rc = check_arch()) return rc;
  const bool i8 = c->storage == SAGE_CACHE_INT8, bf = c->dtype == SAGE_DTYPE_BF16;
  const int64_t D = c->head_dim;
  p.q = q; p.o = o;
  p.q_sh = q_strides[0]; p.q_st = q_strides[1]; p.o_sh = o_strides[0]; p.o_st = o_strides[1];
  p.Hkv = (int)c->heads_kv; p.G = (int)G;
  p.page_shift = page_shift(c);
  p.pages = (int)c->num_pages;
  p.k_scale = c->k_scale; p.v_scale = c->v_scale;
  p.causal = causal ? 1 : 0;
  p.window = (int)std::min<int64_t>(window, 1LL << 30);
  p.sinks = (int)std::min<int64_t>(sinks, 1LL << 30);
  const double s = sm_scale > 0.0f ? static_cast<double>(sm_scale) : 1.0 / std::sqrt(static_cast<double>(D));
  p.scale_log2 = static_cast<float>(s * 1.4426950408889634);
  p.wait_limit_ns = wait_limit_ns();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* w = static_cast<char*>(workspace);
  p.part = reinterpret_cast<float*>(w);
  const PagedRoute route = paged_route(c, G, batch, total_q, max_seqlen_q);
  p.s.group = (int)G;
  if (route != PagedRoute::kMany) {
    if (route == PagedRoute::kBoth) { p.s.rows_lo = 1; p.s.rows_hi = (int)few_rows(c); }
    PagedMaps m;
    if (int rc = cache_map(&m.k, c, false, sage::kDecKeys)) return rc;
    if (int rc = cache_map(&m.v, c, true, sage::kDecKeys)) return rc;
    const size_t rows = size_t(2) * sage::kDecMaxPieces * sage::kDecMaxRows;
    p.part_ml = reinterpret_cast<float*>(w + align256(rows * D * 4));
    p.desc = reinterpret_cast<int4*>(w + align256(rows * D * 4) + align256(rows * 4 * 4));
    // rows of an item, at most: of a mixed batch 8 where a single token's fit (a few tokens' take several items)
    const int max_rows = route == PagedRoute::kBoth ? (G <= 8 ? 8 : sage::kDecMaxRows)
                                                    : (int)std::min<int64_t>(G * p.s.max_new, sage::kDecMaxRows);
    if (int rc = D == 128 ? decode_dispatch<128>(i8, bf, m, p, max_rows, st) : decode_dispatch<64>(i8, bf, m, p, max_rows, st))
      return rc;
  }
  if (route != PagedRoute::kFew) {
    if (route == PagedRoute::kBoth) { p.s.rows_lo = (int)few_rows(c) + 1; p.s.rows_hi = 0x7fffffff; }
    const ChunkTile t = chunk_tile(G);
    PagedMaps m;
    // the kernel widens INT8 codes itself, from rows as they are
    if (int rc = cache_map(&m.k, c, false, 128, false)) return rc;
    if (int rc = cache_map(&m.v, c, true, 128, false)) return rc;
    if (int rc = query_map(&m.q, q, c->dtype, D, heads_q, total_q, q_strides[0], q_strides[1], t)) return rc;
    const int64_t items = chunk_items(batch, total_q, G);
    const ChunkWs o = chunk_ws(D, items);
    p.part_ml = reinterpret_cast<float*>(w + o.ml);
    p.desc = reinterpret_cast<int4*>(w + o.desc);
    p.parts = (int)t.parts; p.Gp = (int)t.Gp; p.TT = (int)t.TT;
    sage::ChunkParams cp{};
    cp.d = p;
    cp.items = reinterpret_cast<sage::ChunkItem*>(w + o.items);
    cp.prefix = reinterpret_cast<int64_t*>(w + o.prefix);
    cp.pieces = reinterpret_cast<sage::ChunkPiece*>(w + o.pieces);
    cp.max_items = (int)items;
    if (i8) cp.c = paged_store(c);
    return D == 128 ? chunk_dispatch<128>(i8, bf, m, cp, st) : chunk_dispatch<64>(i8, bf, m, cp, st);
  }
  return SAGE_OK;
}

}  // extern "C"
