// sage_chunk.cuh — attention of many query rows per key/value head over the paged cache (chunks of
// new prompt tokens, whole prompts, mixed batches) on the tensor cores.
//
// The mathematics is that of sage_decode.cuh; with 256 query rows per tile of keys the products bound
// it (4 D operations per pair), and behind them the softmax's issue slots, as in sage_attn.cuh, whose
// pipeline this is: two 128-row query tiles, S = Q K^T and O += P V as tcgen05.mma into TMEM, one
// softmax warpgroup per query tile, MMA issued by one thread.
//
// Rows. A query tile holds TT = 128 / G tokens times the G query heads of the group (row = token * G +
// head; a few rows stay unused where G does not divide 128), so that all query heads of the group share
// every tile of keys and a short chunk still fills rows. One TMA box of G heads by TT tokens per
// 64 channels is a query tile. A group of more than 128 heads is cut into equal parts, each treated as
// a key/value head of its own. A block is two query tiles.
//
// Work split. Blocks of one sequence need different numbers of key tiles (causal mask, window). A
// one-block kernel (paged_schedule_kernel) lists the blocks with their tiles and cuts the line of all
// tiles (block by block, head by head) into equal pieces, one per SM; each CTA runs through its piece
// segment by segment, the tile ring running on across segments. A block cut between pieces leaves
// fp32 partial sums, joined afterwards in a fixed order, as in sage_decode.cuh.
//
// INT8 cache: helper warps turn the codes into fp16 tiles (exact) in shared memory, in the layout the
// TMA load would give, and the scales stay out of the products: scores are multiplied by k_scale per
// column in fp32, P by v_scale before it is rounded to fp16, in units of a power of two 2^E. Two ways:
// - The tile's visible scales (other than 0) span less than 2^11, the usual case: one E for the tile,
//   2^E <= v_scale < 2^(E + 11), kept from tile to tile while it fits, else moved and O rescaled. P < 2^4 *
//   2^11 stays inside fp16 (hence a maximum less lazy than 16 bit's 2^8), and what it loses below 2^(E - 25)
//   is at most 2^-25 of v_scale.
// - They span more, or E would move by more than 2^30 within a segment: E per query row, 2^E <= the
//   largest P v_scale that the row has met, from the products themselves, for this tile and the rest of
//   the segment. A key weighs by what it contributes to the row, whatever scales other keys have. The
//   softmax loop stays the same: E goes into the exponent, and out of the sum of the tile. What finds it
//   is a pass of its own over S (random scales over 2^20, the chunks below, fp16: 534 us; single
//   tokens have no such case).
// bf16 queries are brought to fp16 by a power of two per row.
//
// Code size counts: the softmax's and the converters' loops run side by side on the same instruction
// cache, and unrolled whole (22 KB of converter) the INT8 kernel took 475 us where the loop took 343
// (two chunks of 1024 over 7168, 32/8 heads, head_dim 128). For the same reason every exponential is
// MUFU.ex2: the polynomial share that sage_attn.cuh computes on the FMA pipe costs more here (12 of 32
// columns: 16 bit 243 -> 231 us, INT8 540 -> 475 us without).
//
// P is rounded to the operand type as in sage_decode.cuh; scores, sums and outputs are fp32.
//
// Measured (B200, two chunks of 1024 tokens over 7168, 32/8 heads, head_dim 128, calls back to back): bf16 226 to
// 232 us, 1111 to 1140 TFLOP/s; INT8 344 us (fp16) and 340 us (bf16); head_dim 64: 195 to 207 us (623 to 661
// TFLOP/s), INT8 333 us (fp16) and 332 us (bf16). Chunks of 512 and 1024 over 8192 and 16384, bf16: 364 to 371 us,
// 954 to 974 TFLOP/s. A tile of 128 keys takes about 4100 clk, the chain S -> softmax -> P V -> next S of the two
// query tiles in turn.
//
// Warps: 0-7 softmax (two warpgroups), 8 TMA producer of K and V, 9 MMA issuer, 10 loads the next
// segment's queries as soon as the last Q K^T of this one has run, 11 puts zeros over rows of V that no
// query sees (an unused row may hold a NaN, which its weight of 0 would not silence). INT8: 8 loads
// the queries too, 10 converts K, 11 converts V and brings the scales.
#pragma once

#include "sage_attn.cuh"
#include "sage_decode.cuh"
#include "sage_inflight.cuh"

namespace sage {

constexpr int kChunkRows = 256;     // query rows per block, the unused ones included
constexpr int kChunkPieces = 148;   // CTAs: one per SM
constexpr int kChunkThreads = 384;

// One block of query rows: the sequence's span, the block's number and its key tiles.
struct ChunkItem {
  int base, n, len, b;
  int blk, ns, tw, count;
};
struct ChunkPiece {
  int item, head, tile;                 // where it starts
  int last_item, last_head, last_tile;  // where the next piece starts
  int count, pad;                       // 0: empty
};
// What a block costs beyond its tiles (queries in, output out, an empty pipeline), in tiles: without
// it, pieces with many short blocks end long after the others (the first rows of a causal prompt).
constexpr int kChunkSetup = 2;

struct ChunkParams {
  DecodeParams d;
  ChunkItem* items;
  int64_t* prefix;      // [items] line length of one head before an item (schedule only)
  ChunkPiece* pieces;   // [kChunkPieces]
  int max_items;
  PagedStore c;         // INT8 only
};

template <int D, bool I8, typename T>
struct ChunkCfg {
  using M = typename std::conditional<I8, __half, T>::type;  // operand type of the products
  static constexpr bool PRE_BIAS = false, QK_F16 = true, PV_FP8 = false;
  static constexpr int BM = 128, BN = 128;
  static constexpr int NS = (D == 128) ? 2 : 4;  // K/V ring stages
  static constexpr int TILE = 128 * D * 2;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = OFF_Q + 2 * TILE;
  static constexpr int OFF_V = OFF_K + NS * TILE;
  static constexpr int OUT_CH = (I8 && D == 128) ? 32 : 64;  // output channels staged at a time
  static constexpr int OUT_BYTES = 32 * OUT_CH * 2;          // per softmax warp: 32 rows of them
  static constexpr int OFF_OUT = OFF_V + NS * TILE;
  static constexpr int OFF_BAR = OFF_OUT + 8 * OUT_BYTES;
  static constexpr int NUM_BARS = 4 + 7 * NS + 12;
  static constexpr int OFF_MISC = OFF_BAR + NUM_BARS * 8;
  static constexpr int OFF_WALK = (OFF_MISC + 8 + 15) / 16 * 16;  // where each warp is in the piece
  static constexpr int WALK_BYTES = 80;
  static constexpr int OFF_SCALE = (OFF_WALK + 12 * WALK_BYTES + 15) / 16 * 16;  // INT8: per stage k_scale, v_scale 2^-E
  static constexpr int OFF_LOG = OFF_SCALE + (I8 ? NS * 1024 : 0);               // log2 v_scale, for units of the rows
  static constexpr int OFF_EXP = OFF_LOG + (I8 ? NS * 512 : 0);                  // and E
  static constexpr int SMEM_BYTES = 1024 + OFF_EXP + (I8 ? 16 : 0);
  static_assert(SMEM_BYTES <= 227 * 1024 && SMEM_BYTES > 114 * 1024, "one CTA per SM");
  // 256 softmax and 128 other threads share 384 x 168 registers; a converter keeps 32 registers of loads in flight.
  // Two chunks of 1024 over 7168, INT8: head_dim 64, fp16, 104 registers for the others 340 us, 120 347; bf16 120 339,
  // 104 350, 88 393; head_dim 128, fp16, 88 364 us, 104 374.
  static constexpr int REGS_OTHER = !I8 ? 72 : D == 128 ? 88 : std::is_same<T, M>::value ? 104 : 120;
  static constexpr int REGS_SOFTMAX = (384 * 168 - 128 * REGS_OTHER) / 256;
  static_assert(256 * REGS_SOFTMAX + 128 * REGS_OTHER <= 384 * 168, "register split");
  static constexpr uint32_t QK_LAYOUT = kLayoutSW128, QK_SBO = 1024;
  static constexpr int QK_STEPS = D / 16;
  static __device__ __forceinline__ uint32_t qk_step_offset(int kk, int rows) {
    return (32 * kk / 128) * rows * 128 + (32 * kk) % 128;
  }
  static constexpr int ATOMS = D / 64;  // 128-byte column atoms
  static constexpr uint32_t V_LBO = BN * 128, V_SBO = 1024;
  static constexpr bool SEP_P = (D == 64);
  static constexpr uint32_t P_COL = SEP_P ? 128 + D : 64;
  static constexpr uint32_t FMT = std::is_same<M, __half>::value ? kFmtF16 : kFmtBF16;
  static constexpr uint32_t IDESC_QK = make_idesc(kFmtD_F32, FMT, FMT, 0, 0, BM, BN);
  static constexpr uint32_t IDESC_PV = make_idesc(kFmtD_F32, FMT, FMT, 0, 1, BM, D);
  static constexpr float LAZY = I8 ? 4.0f : 8.0f;
};
// INT8: the exponents that the scales of a tile of one E may differ by. kRowUnits is added to E where every row
// finds its own unit; E is then kRowRange below the largest scale so far: the row's unit may be kRowRange + 1
// above E and kRowDepth below before an exponential leaves fp32.
constexpr int kUnitSpan = 10, kRowUnits = 1 << 20, kRowRange = 60, kRowDepth = 118;

// ------------------------------------------------------------------ schedule
__device__ __forceinline__ int chunk_blocks(const ChunkParams& p, const PagedSeq& sq) {
  return (sq.n + 2 * p.d.TT - 1) / (2 * p.d.TT);
}

// The tiles of 128 keys that block `blk` of a sequence needs.
__device__ __forceinline__ void chunk_tiles(const ChunkParams& p, const PagedSeq& sq, int blk, ChunkItem* it) {
  const int tok_a = blk * 2 * p.d.TT, last = min(sq.n, tok_a + 2 * p.d.TT) - 1;
  const int first = sq.len - sq.n;
  const int lo = p.d.window ? max(0, first + tok_a - p.d.window + 1) : 0;
  const int hi = p.d.causal ? first + last + 1 : sq.len;
  it->ns = p.d.window ? min((min(p.d.sinks, lo) + 127) / 128, (max(hi, 0) + 127) / 128) : 0;
  it->tw = max(lo / 128, it->ns);
  it->count = max(1, it->ns + max(0, (hi + 127) / 128 - it->tw));
}

constexpr int kScheduleThreads = 512;
constexpr int kSchedulePrefix = 2048;  // blocks whose line positions stay in shared memory
__global__ void __launch_bounds__(kScheduleThreads) paged_schedule_kernel(const ChunkParams p) {
  __shared__ int64_t s_warp[kScheduleThreads / 32];
  __shared__ int64_t s_prefix[kSchedulePrefix];
  __shared__ int s_count[kSchedulePrefix];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto block_scan = [&](int64_t v, int64_t* total) {  // exclusive prefix over the block
    int64_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += up;
    }
    __syncthreads();
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    int64_t w = lane < kScheduleThreads / 32 ? s_warp[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += up;
    }
    *total = __shfl_sync(0xffffffffu, w, 31);
    const int64_t before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
    return x - v + (warp ? before : 0);
  };
  // ---- the list of blocks: a warp writes a sequence's, 32 sequences' offsets at a time from one scan
  int64_t n_items = 0;
  for (int b0 = 0; b0 < p.d.s.batch; b0 += kScheduleThreads) {
    const int b = b0 + tid;
    PagedSeq sq{0, 0, 0};
    if (b < p.d.s.batch) sq = paged_seq(p.d.s, b);
    const int nb = chunk_blocks(p, sq);
    int64_t total = 0;
    const int64_t at = n_items + block_scan(nb, &total);
    for (unsigned todo = __ballot_sync(0xffffffffu, nb > 0); todo; todo &= todo - 1) {
      const int l = __ffs(todo) - 1;
      PagedSeq q;
      q.base = __shfl_sync(0xffffffffu, sq.base, l);
      q.n = __shfl_sync(0xffffffffu, sq.n, l);
      q.len = __shfl_sync(0xffffffffu, sq.len, l);
      const int64_t off = __shfl_sync(0xffffffffu, at, l);
      const int blocks = __shfl_sync(0xffffffffu, nb, l);
      for (int k = lane; k < blocks; k += 32) {
        if (off + k >= p.max_items) break;  // the host's bound holds for any prefix sums; kept as a fence
        ChunkItem it;
        it.base = q.base; it.n = q.n; it.len = q.len; it.b = b0 + warp * 32 + l;
        it.blk = k;
        chunk_tiles(p, q, k, &it);
        p.items[off + k] = it;
        if (off + k < kSchedulePrefix) s_count[off + k] = it.count + kChunkSetup;
      }
    }
    n_items += total;
  }
  if (n_items > p.max_items) n_items = p.max_items;
  __syncthreads();
  // ---- the line: a block takes its tiles and kChunkSetup units before them, for every head
  const int heads = p.d.Hkv * p.d.parts;
  int64_t line = 0;
  for (int64_t i0 = 0; i0 < n_items; i0 += kScheduleThreads) {
    const int64_t i = i0 + tid;
    const int len = i >= n_items ? 0 : i < kSchedulePrefix ? s_count[i] : p.items[i].count + kChunkSetup;
    int64_t total = 0;
    const int64_t at = (line + block_scan(len, &total)) * heads;
    if (i < n_items) {
      if (i < kSchedulePrefix) s_prefix[i] = at;
      else p.prefix[i] = at;
    }
    line += total;
  }
  __syncthreads();
  // ---- equal pieces of it
  if (tid >= kChunkPieces) return;
  const int64_t all = line * heads;
  const int64_t per = max((all + kChunkPieces - 1) / kChunkPieces, (int64_t)1);
  // where a position of the line lies: block, head and tile (0 in the units before the tiles)
  auto find = [&](int64_t at, int* item, int* head, int* tile, int64_t* end) {
    int64_t lo = 0, n = n_items;
    while (n > 1) {
      const int64_t half = n / 2, mid = lo + half;
      if ((mid < kSchedulePrefix ? s_prefix[mid] : p.prefix[mid]) <= at) { lo = mid; n -= half; }
      else n = half;
    }
    const int64_t begin = lo < kSchedulePrefix ? s_prefix[lo] : p.prefix[lo];
    const unsigned len = lo < kSchedulePrefix ? s_count[lo] : p.items[lo].count + kChunkSetup;
    *item = (int)lo;
    *head = (int)((uint64_t)(at - begin) < (1ull << 32) ? (unsigned)(at - begin) / len : (at - begin) / len);
    const int64_t left = at - begin - (int64_t)*head * len;
    *tile = max((int)left - kChunkSetup, 0);
    *end = at - left + len;  // first position behind this head's part
  };
  ChunkPiece c{0, 0, 0, 0};
  int4 cut = make_int4(0, 0, 0, 0);
  const int64_t begin = per * tid, stop = min(begin + per, all);
  if (begin < stop) {
    int64_t end;
    find(begin, &c.item, &c.head, &c.tile, &end);
    c.count = 1;  // not empty; the walk ends at (last_item, last_head, last_tile)
    if (stop < all) find(stop, &c.last_item, &c.last_head, &c.last_tile, &end);
    else { c.last_item = (int)n_items; c.last_head = 0; c.last_tile = 0; }
    // the block that this piece begins and does not end, and how many pieces follow that hold the rest
    if (c.last_tile > 0 && !(c.last_item == c.item && c.last_head == c.head && c.tile > 0)) {
      const ChunkItem it = p.items[c.last_item];
      cut = make_int4(it.b, c.last_head, it.blk, (int)((end - 1) / per) - tid);
    }
  }
  p.pieces[tid] = c;
  p.d.desc[tid] = cut;
}

// ------------------------------------------------------------------ attention
// One segment of a CTA's piece: tiles [t0, t0 + n) of a block for one head.
struct ChunkWalk {
  const ChunkItem* items;
  int item, head, tile, Hkv;
  int last_item, last_head, last_tile;
  bool go;
  ChunkItem it;
  int n;
  ChunkWalk() = default;
  __device__ __forceinline__ ChunkWalk(const ChunkParams& p, int cta) {
    const int4 a = reinterpret_cast<const int4*>(p.pieces + cta)[0], z = reinterpret_cast<const int4*>(p.pieces + cta)[1];
    items = p.items;
    item = a.x; head = a.y; tile = a.z;
    last_item = a.w; last_head = z.x; last_tile = z.y;
    Hkv = p.d.Hkv * p.d.parts;
    go = z.z > 0;
    if (go) load();
    settle();
  }
  __device__ __forceinline__ void load() {
    const int4 a = reinterpret_cast<const int4*>(items + item)[0], z = reinterpret_cast<const int4*>(items + item)[1];
    it.base = a.x; it.n = a.y; it.len = a.z; it.b = a.w;
    it.blk = z.x; it.ns = z.y; it.tw = z.z; it.count = z.w;
  }
  // tiles of the present segment; the piece's last one may be cut short, or be empty
  __device__ __forceinline__ void settle() {
    const bool last = item == last_item && head == last_head;
    n = (last ? last_tile : it.count) - tile;
    if (n <= 0) go = false;
  }
  __device__ __forceinline__ bool more() const { return go; }
  __device__ __forceinline__ bool whole() const { return tile == 0 && n == it.count; }
  __device__ __forceinline__ void next() {
    if (item == last_item && head == last_head) { go = false; return; }
    tile = 0;
    if (++head == Hkv) {
      head = 0;
      ++item;
      if (item > last_item || (item == last_item && last_head == 0 && last_tile == 0)) { go = false; return; }
      load();
    }
    settle();
  }
  // tokens [first_tok, first_tok + toks) of the sequence's new ones
  __device__ __forceinline__ int first_tok(const ChunkParams& p) const { return it.blk * 2 * p.d.TT; }
  __device__ __forceinline__ int toks(const ChunkParams& p) const { return min(2 * p.d.TT, it.n - it.blk * 2 * p.d.TT); }
  __device__ __forceinline__ int key0(int j) const {  // first key of tile `tile + j`
    const int i = tile + j;
    return (i < it.ns ? i : it.tw + i - it.ns) * 128;
  }
};

__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

__device__ __forceinline__ float lg2_approx(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The lowest n bits (n may be anything).
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u); }

__device__ __forceinline__ void st_shared_v4(uint32_t dst, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t src) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(src) : "memory");
  return v;
}
__device__ __forceinline__ void ld_shared_f4(uint32_t src, float2 (&v)[2]) {
  asm volatile("ld.shared.v2.b64 {%0,%1}, [%2];"
               : "=l"(reinterpret_cast<uint64_t&>(v[0])), "=l"(reinterpret_cast<uint64_t&>(v[1])) : "r"(src));
}
// One 16-byte piece of INT8 codes as 16 fp16 values: 32 bytes, as two 16-byte units.
__device__ __forceinline__ void codes_to_half16(const uint4& w, uint4& a, uint4& z) {
  const uint32_t x = w.x ^ 0x80808080u, y = w.y ^ 0x80808080u, u = w.z ^ 0x80808080u, v = w.w ^ 0x80808080u;
  a = make_uint4(biased_to_half2(__byte_perm(x, 0x64646464u, 0x4140)), biased_to_half2(__byte_perm(x, 0x64646464u, 0x4342)),
                 biased_to_half2(__byte_perm(y, 0x64646464u, 0x4140)), biased_to_half2(__byte_perm(y, 0x64646464u, 0x4342)));
  z = make_uint4(biased_to_half2(__byte_perm(u, 0x64646464u, 0x4140)), biased_to_half2(__byte_perm(u, 0x64646464u, 0x4342)),
                 biased_to_half2(__byte_perm(v, 0x64646464u, 0x4140)), biased_to_half2(__byte_perm(v, 0x64646464u, 0x4342)));
}

template <int D, bool I8, typename T>
__global__ void __launch_bounds__(kChunkThreads, 1)
    paged_chunk_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, const ChunkParams cp) {
  using C = ChunkCfg<D, I8, T>;
  using M = typename C::M;
  constexpr bool Q_CONV = I8 && std::is_same<T, __nv_bfloat16>::value;  // queries from bf16 to fp16
  // How far the pass for units of the rows is unrolled: it hardly runs, but where it puts the code behind it in the
  // instruction cache shows (two chunks of 1024 over 7168; rolled, by 2, whole: fp16 359, 365, 351 us, bf16 360, 350, 397)
  constexpr int ROW_PASS = Q_CONV ? 2 : 4;
  const DecodeParams& p = cp.d;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bar_q = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* bar_qfree = bar_q + 1;
  uint64_t* bar_vraw = bar_q + 2;  // [stage]: V landed, rows that no query sees still to be cleared
  uint64_t* bar_kfull = bar_vraw + C::NS;
  uint64_t* bar_vfull = bar_kfull + C::NS;
  uint64_t* bar_kempty = bar_vfull + C::NS;  // K's slot is free after Q K^T, V's a softmax later
  uint64_t* bar_vempty = bar_kempty + C::NS;
  uint64_t* bar_sfull = bar_vempty + C::NS;
  uint64_t* bar_phalf = bar_sfull + 2;
  uint64_t* bar_pfull = bar_phalf + 2;
  uint64_t* bar_odone = bar_pfull + 2;
  uint64_t* bar_sload = bar_odone + 2;
  uint64_t* bar_pvdone = bar_sload + 2;
  uint64_t* bar_sc = bar_pvdone + 2;    // [stage] INT8: the tile's scales are in place
  uint64_t* bar_kraw = bar_sc + C::NS;  // [stage] INT8: K's codes landed (V's: bar_vraw)
  uint64_t* bar_qraw = bar_kraw + C::NS;  // bf16 queries landed, to be converted by the softmax threads
  uint64_t* bar_mma = bar_qraw + 1;       // after a wait ran out: every product has run
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC + 4);
  const uint32_t warp = warp_id(), lane = lane_id();
  const int cta = blockIdx.x;

  if (threadIdx.x == 0) {
    mbar_init(bar_q, Q_CONV ? 256 : 1);
    mbar_init(bar_qraw, 1);
    mbar_init(bar_mma, 1);
    mbar_init(bar_qfree, 1);
    for (int s = 0; s < C::NS; ++s) {
      mbar_init(bar_vraw + s, 1);
      mbar_init(bar_sc + s, 1);
      mbar_init(bar_kraw + s, 1);
      mbar_init(bar_kfull + s, 1);
      mbar_init(bar_vfull + s, 1);
      mbar_init(bar_kempty + s, 1);
      mbar_init(bar_vempty + s, 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(bar_sfull + t, 1);
      mbar_init(bar_phalf + t, 128);
      mbar_init(bar_pfull + t, 128);
      mbar_init(bar_odone + t, 1);
      mbar_init(bar_sload + t, 128);
      mbar_init(bar_pvdone + t, 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the schedule is written
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // The walk through the piece. In the softmax warps, and in those that convert INT8, it lives in shared
  // memory: its registers would spill beside a row of 128 scores, or beside the loads in flight.
  static_assert(sizeof(ChunkWalk) <= C::WALK_BYTES, "walk");
  ChunkWalk* const shared_walk = reinterpret_cast<ChunkWalk*>(smem + C::OFF_WALK + warp * C::WALK_BYTES);
  auto shared_next = [&] {
    __syncwarp();
    if (lane == 0) shared_walk->next();
    __syncwarp();
  };
  if (I8 || warp < 8) {
    if (lane == 0) *shared_walk = ChunkWalk(cp, cta);
    __syncwarp();
  }
  if (warp >= 8) {
    regs_dec<C::REGS_OTHER>();
    ChunkWalk own;
    if constexpr (!I8) own = ChunkWalk(cp, cta);
    ChunkWalk& w = I8 ? *shared_walk : own;
    auto step = [&] {
      if constexpr (I8) shared_next();
      else own.next();
    };
      auto seen = [&](int* hi, int* lo) {
      const int first = w.it.len - w.it.n + w.first_tok(cp);
      *hi = p.causal ? first + w.toks(cp) : w.it.len;
      *lo = p.window ? first - p.window + 1 : 0;
    };
    // a tile that holds rows of V which no query of the block sees
    auto ragged = [&](int key0) {
      int hi, lo;
      seen(&hi, &lo);
      return key0 + 128 > hi || (key0 < lo && key0 + 128 > p.sinks);
    };

    // what this warp has issued, for the case that a wait runs out
    int tiles_k = 0, tiles_v = 0, segments = 0;
    ValueCopies value_copies;

    // the segment's queries: one box per query tile and 64 channels
    auto load_queries = [&] {
      const int nt = w.toks(cp) > p.TT ? 2 : 1, kvh = w.head / p.parts, part = w.head - kvh * p.parts;
      uint64_t* bar = Q_CONV ? bar_qraw : bar_q;
      mbar_arrive_expect_tx(bar, nt * C::ATOMS * 128 * p.TT * p.Gp);
      for (int t = 0; t < nt; ++t)
        for (int x = 0; x < C::ATOMS; ++x)
          tma_load_3d(smem + C::OFF_Q + t * C::TILE + x * (128 * 128), &tmQ, bar, x * 64, kvh * p.G + part * p.Gp,
                      w.it.base + w.first_tok(cp) + t * p.TT);
    };
    const int page = 1 << p.page_shift;
    const int rows = min(page, 128), ppt = 128 / rows;    // rows of a tile in one page, pages of a tile
    const int batch_tiles = 32 / ppt;                     // tiles whose page numbers the 32 lanes hold
    auto page_of = [&](int j) {  // this lane's page of tiles [j, j + batch_tiles) of the segment
      const int tj = j + (int)lane / ppt;
      if (tj >= w.n) return -1;
      const int pg = (w.key0(tj) >> p.page_shift) + (int)lane % ppt;
      return pg < p.s.width ? p.s.table[(int64_t)w.it.b * p.s.table_stride + pg] : -1;
    };
    if (I8 && warp >= 10) {
      // ------------------------------------------------------------ codes to fp16 tiles: K (warp 10), V (warp 11)
      // The codes land in the upper half of their slot and are widened in place: at head_dim 128 row r's
      // codes lie where the upper half of its fp16 values goes; at 64 rows are taken in order, and the
      // values of rows up to r cover codes of rows up to r only. A group of rows is read whole, then
      // written. Codes that nobody sees are finite whatever they are, so their weight of 0 suffices.
      // Warp 11 also brings the scales: k_scale, and v_scale in units of 2^E.
      const bool isv = warp == 11;
      constexpr int LPR = D / 16, RPI = 32 / LPR;  // lanes per row of codes, rows per pass
      constexpr int NG = 128 / (8 * RPI);          // groups of eight passes
      // Lane: 16 codes c of row `sub` of every RPI rows. At head_dim 128 the upper half's lanes take the
      // neighbouring row, so that the eight lanes of a store phase hit eight different 16-byte banks.
      const int c = lane % LPR, sub = (lane / LPR) ^ (D == 128 ? c >> 2 : 0), sh = min(p.page_shift, 7);
      uint64_t* bar_full = isv ? bar_vfull : bar_kfull;
      uint64_t* bar_raw = isv ? bar_vraw : bar_kraw;
      const uint32_t slots = smem_u32(smem + (isv ? C::OFF_V : C::OFF_K));
      const uint32_t src = slots + C::TILE / 2 + sub * D + c * 16;
      // a row's two 16-byte units (2 c, 2 c + 1 of 8 per 128-byte atom), rows of even and odd passes
      const int unit = 2 * (c & 3);
      const uint32_t dst = slots + (c >> 2) * (128 * 128) + sub * 128;
      const uint32_t off0 = (unit ^ (sub & 7)) << 4, off1 = (unit ^ ((RPI + sub) & 7)) << 4;
      int it = 0;
      bool ok = true;
      for (; w.more() && ok; step()) {
        const int n = w.n, kvh = w.head / p.parts;
        int hi, lo, ids = 0;
        int e = -126, e_first = 0;                 // the scales' unit; that of the segment's first tile
        bool has_unit = false, row_units = false;  // e is set; the rows have units of their own
        int unit = -126;                           // what the tile's v_scales are divided by (log2)
        seen(&hi, &lo);
        for (int j = 0; j < n; ++j, ++it) {
          const int s = it % C::NS;
          float k4[4] = {0.f, 0.f, 0.f, 0.f}, v4[4] = {0.f, 0.f, 0.f, 0.f};
          const int key = w.key0(j) + 4 * lane;
          if (isv) {
            if (j % batch_tiles == 0) ids = page_of(j);
            const int id = __shfl_sync(0xffffffffu, ids, (j % batch_tiles) * ppt + ((4 * lane) >> sh));
            if (id >= 0 && id < cp.c.pages) {
              const int64_t at = (((int64_t)id * cp.c.heads + kvh) << p.page_shift) + (key & (page - 1));
              const float4 a = *reinterpret_cast<const float4*>(cp.c.k_scale + at), z = *reinterpret_cast<const float4*>(cp.c.v_scale + at);
              k4[0] = a.x; k4[1] = a.y; k4[2] = a.z; k4[3] = a.w;
              v4[0] = z.x; v4[1] = z.y; v4[2] = z.z; v4[3] = z.w;
            }
          }
          ok = mbar_wait(bar_raw + s, (it / C::NS) & 1, abort_flag, kDevTimeoutProducer, p.wait_limit_ns);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (isv) {  // V's slot is free, so are the scales'
            unsigned top = 0, low = 255;  // exponent fields of the visible scales other than 0 (and subnormal ones)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int kx = key + x;
              if (!(kx < hi && (kx >= lo || kx < p.sinks))) k4[x] = v4[x] = 0.0f;
              const unsigned f = (__float_as_uint(v4[x]) >> 23) & 255u;
              top = max(top, f);
              low = min(low, f ? f : 255u);
            }
            const bool fits = has_unit && !row_units && (int)low >= e + 127 && (int)top <= e + 127 + kUnitSpan;
            if (!__all_sync(0xffffffffu, fits)) {
              top = __reduce_max_sync(0xffffffffu, top);
              low = __reduce_min_sync(0xffffffffu, low);
              const int t_hi = (int)top - 127, t_lo = (int)low - 127;
              if (top == 255u || (top && t_hi - t_lo > kUnitSpan)) {
                row_units = true;
              } else if (top && (!has_unit || t_lo < e || t_hi > e + kUnitSpan)) {
                e = min(max(t_lo - (kUnitSpan - (t_hi - t_lo)) / 2, -126), 121);
                if (!has_unit) e_first = e;
                has_unit = true;
                row_units |= e > e_first + 30 || e < e_first - 30;
              }
              if (!row_units) unit = e;
              else if (top) unit = max(unit, t_hi - kRowRange);  // never below what a row's unit may follow
            }
            const float down = pow2(-unit);
            float4* sc = reinterpret_cast<float4*>(smem + C::OFF_SCALE + s * 1024);
            sc[lane] = make_float4(k4[0], k4[1], k4[2], k4[3]);
            sc[32 + lane] = make_float4(v4[0] * down, v4[1] * down, v4[2] * down, v4[3] * down);
            if (row_units)
              reinterpret_cast<float4*>(smem + C::OFF_LOG + s * 512)[lane] =
                  make_float4(lg2_approx(fabsf(v4[0])), lg2_approx(fabsf(v4[1])), lg2_approx(fabsf(v4[2])), lg2_approx(fabsf(v4[3])));
            if (lane == 0) reinterpret_cast<int*>(smem + C::OFF_EXP)[s] = row_units ? unit + kRowUnits : unit;
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_sc + s);
          }
#pragma unroll 1
          for (int g = 0; g < NG; ++g) {
            uint4 x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] = ld_shared_v4(src + s * C::TILE + (g * 8 + u) * (RPI * D));
            __syncwarp();
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              uint4 a, z;
              codes_to_half16(x[u], a, z);
              const uint32_t o = dst + s * C::TILE + (g * 8 + u) * (RPI * 128) + ((u & 1) ? off1 : off0);
              st_shared_v4(o, a);
              st_shared_v4(o ^ 16, z);
            }
            __syncwarp();
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_full + s);
        }
      }
    } else if (warp == 8) {
      // ------------------------------------------------------------ TMA producer
      // boxes of K, and of V: one per page and 128-byte atom (INT8: per page, into the slot's upper half)
      const int boxes = I8 ? ppt : ppt * C::ATOMS;
      int it = 0, k_ahead = 0;  // k_ahead: gave up between a tile's K and V
      bool ok = true;
      for (int seg = 0; w.more() && ok; step(), ++seg) {
        if constexpr (I8) {  // the queries too: warp 10 converts
          if (seg > 0) ok = mbar_wait(bar_qfree, (seg - 1) & 1, abort_flag, kDevTimeoutProducer, p.wait_limit_ns);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (lane == 0) load_queries();
          __syncwarp();
          segments = seg + 1;
        }
        const int kvh = w.head / p.parts;
        int next = page_of(0);
        for (int j0 = 0; j0 < w.n && ok; j0 += batch_tiles) {
          const int ids = next;
          if (j0 + batch_tiles < w.n) next = page_of(j0 + batch_tiles);
          const int j1 = min(w.n, j0 + batch_tiles);
          for (int j = j0; j < j1; ++j, ++it) {
            const int s = it % C::NS;
            const int key0 = w.key0(j), y = key0 & (page - 1);
            const int sub = lane % ppt, atom = lane / ppt;
            const int id = __shfl_sync(0xffffffffu, ids, (j - j0) * ppt + sub);
            const int dst = s * C::TILE + (I8 ? C::TILE / 2 + sub * rows * D : atom * (128 * 128) + sub * rows * 128);
            const bool raw = I8 || ragged(key0);
            uint64_t* vbar = (raw ? bar_vraw : bar_vfull) + s;
#pragma unroll
            for (int isv = 0; isv < 2; ++isv) {
              if (ok && it >= C::NS)
                ok = mbar_wait((isv ? bar_vempty : bar_kempty) + s, ((it / C::NS) - 1) & 1, abort_flag, kDevTimeoutProducer,
                               p.wait_limit_ns);
              ok = __all_sync(0xffffffffu, ok);
              if (!ok) {
                k_ahead = isv;
                break;
              }
              uint64_t* bar = isv ? vbar : (I8 ? bar_kraw : bar_kfull) + s;
              if (lane == 0) mbar_arrive_expect_tx(bar, I8 ? C::TILE / 2 : C::TILE);
              __syncwarp();
              if (lane < boxes)
                tma_load_4d(smem + (isv ? C::OFF_V : C::OFF_K) + dst, isv ? &tmV : &tmK, bar, atom * 64, y, kvh, id);
            }
            if (!ok) break;
            if constexpr (!I8) value_copies.note(s, it / C::NS, raw);
          }
        }
      }
      tiles_v = it;
      tiles_k = it + k_ahead;
    } else if (warp == 9) {
      // ------------------------------------------------------------ MMA issuer
      if (elect_one()) {
        const uint32_t q_addr = smem_u32(smem + C::OFF_Q);
        const uint32_t k_addr = smem_u32(smem + C::OFF_K);
        const uint32_t v_addr = smem_u32(smem + C::OFF_V);
        int it0 = 0, seg = 0;  // tiles before the segment, segments before it
        int ct0[2] = {0, 0};   // tiles of each query tile before the segment
        bool ok = true;
        for (; w.more() && ok; w.next(), ++seg) {
          const int nt = w.toks(cp) > p.TT ? 2 : 1, n = w.n;
          ok = mbar_wait(bar_q, seg & 1, abort_flag, kDevTimeoutMma, p.wait_limit_ns);
          if (ok) ok = mbar_wait(bar_kfull + it0 % C::NS, (it0 / C::NS) & 1, abort_flag, kDevTimeoutMma, p.wait_limit_ns);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (t >= nt) continue;
            issue_qk<C>(tmem_base + 256 * t, q_addr + t * C::TILE, k_addr + (it0 % C::NS) * C::TILE, 0);
            umma_commit(bar_sfull + t);
          }
          umma_commit(bar_kempty + it0 % C::NS);
          if (n == 1) umma_commit(bar_qfree);
          for (int j = 0; ok && j < n; ++j) {
            const int i = it0 + j, s = i % C::NS, s1 = (i + 1) % C::NS;
            bool v_ready = false, knext_ready = false;
            // Q K^T of tile j + 1 for query tile t
            auto next_qk = [&](int t) {
              if (!knext_ready) {
                if (!mbar_wait(bar_kfull + s1, ((i + 1) / C::NS) & 1, abort_flag, kDevTimeoutMma, p.wait_limit_ns)) return false;
                knext_ready = true;
              }
              tc_fence_after();
              issue_qk<C>(tmem_base + 256 * t, q_addr + t * C::TILE, k_addr + s1 * C::TILE, 0);
              umma_commit(bar_sfull + t);
              if (t + 1 == nt) {
                umma_commit(bar_kempty + s1);
                if (j + 2 == n) umma_commit(bar_qfree);  // the block's queries have been read
              }
              return true;
            };
            if constexpr (C::SEP_P) {
#pragma unroll
              for (int t = 0; t < 2; ++t) {
                if (t >= nt || j + 1 >= n || !ok) continue;
                ok = mbar_wait(bar_sload + t, (ct0[t] + j) & 1, abort_flag, kDevTimeoutMma, p.wait_limit_ns) && next_qk(t);
              }
              if (!ok) break;
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              if (t >= nt || !ok) continue;
              const uint64_t vd = make_smem_desc(v_addr + s * C::TILE, C::V_LBO, C::V_SBO, kLayoutSW128);
              const uint32_t p_tmem = tmem_base + 256 * t + C::P_COL;
              const uint32_t o_tmem = tmem_base + 256 * t + 128;
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                if (!ok) continue;
                ok = mbar_wait((half ? bar_pfull : bar_phalf) + t, (ct0[t] + j) & 1, abort_flag, kDevTimeoutMma, p.wait_limit_ns);
                if (ok && !v_ready) {
                  ok = mbar_wait(bar_vfull + s, (i / C::NS) & 1, abort_flag, kDevTimeoutMma, p.wait_limit_ns);
                  v_ready = true;
                }
                if (!ok) continue;
                tc_fence_after();
#pragma unroll
                for (int kk = half * 4; kk < half * 4 + 4; ++kk)
                  umma_f16_ts(o_tmem, p_tmem + kk * 8, desc_advance(vd, kk * 16 * 128), C::IDESC_PV,
                              (j > 0 || kk > 0) ? 1u : 0u);
              }
              if (!ok) continue;
              if (j + 1 == n) umma_commit(bar_odone + t);
              if constexpr (C::SEP_P) umma_commit(bar_pvdone + t);
              else if (j + 1 < n) ok = next_qk(t);
            }
            if (ok) umma_commit(bar_vempty + s);
          }
          it0 += n;
          ct0[0] += n;
          if (nt == 2) ct0[1] += n;
        }
      }
    } else if (warp == 10) {
      // ------------------------------------------------------------ queries
      if (elect_one()) {
        tma_prefetch_desc(&tmQ);
        bool ok = true;
        for (int seg = 0; w.more() && ok; w.next(), ++seg) {
          if (seg > 0) ok = mbar_wait(bar_qfree, (seg - 1) & 1, abort_flag, kDevTimeoutProducer, p.wait_limit_ns);
          if (!ok) break;
          load_queries();
          segments = seg + 1;
        }
      }
    } else {
      // ------------------------------------------------------------ rows of V that no query sees
      int it = 0;
      uint32_t raw_phase = 0;  // bit s: phase of bar_vraw[s]
      bool ok = true;
      for (; w.more() && ok; step()) {
        int hi, lo;
        seen(&hi, &lo);
        for (int j = 0; j < w.n && ok; ++j, ++it) {
          const int key0 = w.key0(j), s = it % C::NS;
          if (!ragged(key0)) continue;
          ok = mbar_wait(bar_vraw + s, (raw_phase >> s) & 1, abort_flag, kDevTimeoutProducer, p.wait_limit_ns);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          raw_phase ^= 1u << s;
          uint8_t* v = smem + C::OFF_V + s * C::TILE;
          for (int x = lane; x < 128 * C::ATOMS * 8; x += 32) {
            const int atom = x / 1024, r = (x / 8) % 128, key = key0 + r;
            if (!(key < hi && (key >= lo || key < p.sinks)))
              *reinterpret_cast<uint4*>(v + atom * (128 * 128) + r * 128 + (x % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_vfull + s);
        }
      }
    }
    // every warp leaves through barrier 2; the MMA warp frees TMEM after all have arrived
    tc_fence_before();
    if (warp == 11) {
      asm volatile("bar.arrive 2, %0;" ::"n"(kChunkThreads) : "memory");
      return;
    }
    __syncwarp();
    asm volatile("bar.sync 2, %0;" ::"n"(kChunkThreads) : "memory");
    if (*abort_flag) {
      // A wait ran out, so what this warp issued may still be on its way: wait for it, again within the limit.
      auto landed = [&](uint64_t* bar, uint32_t phase) {
        volatile int none = 0;
        (void)mbar_wait(bar, phase, &none, kDevTimeoutProducer, p.wait_limit_ns);
      };
      const CopyLedger k = ring_copies(tiles_k, C::NS), v = I8 ? ring_copies(tiles_v, C::NS) : value_copies.raw;
      for (int s = 0; s < C::NS; ++s) {
        if (k.pending(s)) landed((I8 ? bar_kraw : bar_kfull) + s, k.phase(s));
        if (v.pending(s)) landed(bar_vraw + s, v.phase(s));
        if (value_copies.full.pending(s)) landed(bar_vfull + s, value_copies.full.phase(s));
      }
      if (segments > 0) landed(Q_CONV ? bar_qraw : bar_q, (segments - 1) & 1);
      if (warp == 9 && elect_one()) {
        umma_commit(bar_mma);
        landed(bar_mma, 0);
      }
      __syncwarp();
    }
    if (warp == 9) {
      tc_fence_after();
      tmem_dealloc(tmem_base, 512);
    }
  } else {
    // ------------------------------------------------------------ softmax warpgroups
    regs_inc<C::REGS_SOFTMAX>();
    const int t = warp / 4;
    const int row_in_tile = (warp % 4) * 32 + lane;
    const uint32_t lane_base = ((warp % 4) * 32u) << 16;
    const uint32_t s_tmem = tmem_base + lane_base + 256 * t;
    const uint32_t o_tmem = s_tmem + 128;
    const int row_tok = row_in_tile / p.Gp, row_head = row_in_tile - row_tok * p.Gp;
    int ct = 0, segs = 0;  // tiles and segments of this query tile so far
    int it0 = 0, qseg = 0;  // tiles and segments of the CTA so far
    bool ok = true;
    ChunkWalk& w = *shared_walk;
    for (; ok && w.more(); shared_next()) {
      const int first_tok = w.first_tok(cp) + t * p.TT;           // of this query tile
      const int toks = min(p.TT, w.it.n - first_tok);
      const int n = w.n, it_seg = it0;
      it0 += n;
      float scale = p.scale_log2;
      if constexpr (Q_CONV) {
        // this thread's query row from bf16 to fp16 in place, in units of a power of two
        if (!__all_sync(0xffffffffu, mbar_wait(bar_qraw, qseg++ & 1, abort_flag, kDevTimeoutSoftmax, p.wait_limit_ns))) { ok = false; break; }
        if (toks > 0) {
          uint8_t* q = smem + C::OFF_Q + t * C::TILE + row_in_tile * 128;
          auto piece = [&](int x) { return reinterpret_cast<uint4*>(q + (x >> 3) * (128 * 128) + (((x & 7) ^ (row_in_tile & 7)) << 4)); };
          uint32_t m = 0;
#pragma unroll 2
          for (int x = 0; x < D / 8; ++x) {
            float f[8];
            Half8<T>::to_float(*piece(x), f);
#pragma unroll
            for (int y = 0; y < 8; ++y) m = max(m, abs_bits(f[y]));
          }
          const int e = min(max((int)(m >> 23) - 127, -126), 126);
          const float down = pow2(-e);
          scale *= pow2(e);
#pragma unroll 2
          for (int x = 0; x < D / 8; ++x) {
            float f[8];
            Half8<T>::to_float(*piece(x), f);
#pragma unroll
            for (int y = 0; y < 8; ++y) f[y] *= down;
            *piece(x) = Half8<__half>::from_float(f);
          }
        }
        fence_proxy_async_smem();
        mbar_arrive(bar_q);
      }
      if (toks <= 0) continue;  // uniform over the warpgroup
      const int pos = w.it.len - w.it.n + first_tok + min(row_tok, toks - 1);
      const int hi = p.causal ? pos + 1 : w.it.len;  // this row sees keys [lo, hi) and those of [0, sinks) below hi
      const int lo = p.window ? pos - p.window + 1 : 0;
      // over the rows of this query tile
      const int first = w.it.len - w.it.n + first_tok;
      const int all_hi = p.causal ? first + 1 : w.it.len, all_lo = p.window ? first + toks - p.window : 0;
      float m_run = -INFINITY, l_run = 0.0f;
      int e_run = 0;  // INT8: O is in units of 2^e_run
      int key0 = w.key0(0);
      const int jump = w.it.ns - 1 - w.tile, jump_to = w.it.tw * 128;  // the tile after tile `jump` lies behind the sinks'
      for (int j = 0; j < n; ++j) {
        if (!__all_sync(0xffffffffu, mbar_wait(bar_sfull + t, (ct + j) & 1, abort_flag, kDevTimeoutSoftmax, p.wait_limit_ns))) { ok = false; break; }
        tc_fence_after();
        float shrink = 1.0f;  // INT8: O's factor where the unit moves
        int unit_shift = 0;   // INT8: the exponentials are divided by 2^unit_shift
        float lazy = C::LAZY;
        uint32_t scales = 0;
        const int up = hi - key0, down = lo - key0, sk = p.sinks - key0;
        if constexpr (I8) {
          const int s = (it_seg + j) % C::NS;
          if (!__all_sync(0xffffffffu, mbar_wait(bar_sc + s, ((it_seg + j) / C::NS) & 1, abort_flag, kDevTimeoutSoftmax, p.wait_limit_ns))) { ok = false; break; }
          scales = smem_u32(smem + C::OFF_SCALE) + s * 1024;
          const int e_tile = *reinterpret_cast<const int*>(smem + C::OFF_EXP + 4 * s);
          int e = e_tile;
          if (e_tile >= kRowUnits / 2) {
            // Rare, and kept out of the code below: the row's unit, from its largest product, by a pass over S
            // (32 columns at a time, from TMEM).
            const int et = e_tile - kRowUnits;
            const uint32_t logs = smem_u32(smem + C::OFF_LOG) + s * 512;
            float mx = -INFINITY, mo = -INFINITY;  // largest score (unscaled), largest log2 of a product
#pragma unroll ROW_PASS
            for (int c0 = 0; c0 < 128; c0 += 32) {
              uint32_t sr[32];
              tmem_ld32_sync(s_tmem + c0, sr);
              const uint32_t vis = low_bits(up - c0) & (~low_bits(down - c0) | low_bits(sk - c0));
#pragma unroll
              for (int c = 0; c < 32; c += 4) {
                float2 ks[2], lg[2];
                ld_shared_f4(scales + 4 * (c0 + c), ks);
                ld_shared_f4(logs + 4 * (c0 + c), lg);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                  const int i = c + 2 * x;
                  float2 b = fmul2(make_float2(__uint_as_float(sr[i]), __uint_as_float(sr[i + 1])), ks[x]);
                  if (!((vis >> i) & 1u)) b.x = -INFINITY;
                  if (!((vis >> (i + 1)) & 1u)) b.y = -INFINITY;
                  const float2 y = ffma2(b, make_float2(scale, scale), lg[x]);
                  mx = fmax3(mx, b.x, b.y);
                  mo = fmax3(mo, y.x, y.y);
                }
              }
            }
            const float m = fmaxf(m_run, mx * scale);
            const int top = mo == -INFINITY ? -126 : (int)floorf(fmaxf(mo - m, -126.0f));
            // the weights of before have shrunk by 2^(m - m_run), so may their unit
            const int before = m_run == -INFINITY ? -126 : e_run - (int)ceilf(fminf(m - m_run, 256.0f));
            e = min(max(max(top, before), max(et - kRowDepth, -126)), 121);
            if (m_run == -INFINITY) e_run = e;
            unit_shift = e - et;
            lazy = 0.0f;
          }
          if (j > 0 && e != e_run) shrink = pow2(min(max(e_run - e, -126), 126));
          e_run = e;
        }
        float b[128];
        {
          uint32_t sr[128];
          tmem_ld128_sync(s_tmem, sr);
          if constexpr (C::SEP_P) {
            tc_fence_before();
            mbar_arrive(bar_sload + t);
          }
#pragma unroll
          for (int c = 0; c < 128; ++c) b[c] = __uint_as_float(sr[c]);
        }
        if constexpr (I8) {
          float2 ks4[4][2];
#pragma unroll
          for (int c = 0; c < 128; c += 4) {
            if (c % 16 == 0) {
#pragma unroll
              for (int x = 0; x < 4; ++x) ld_shared_f4(scales + 4 * c + 16 * x, ks4[x]);
            }
            const float2* ks = ks4[c / 4 % 4];
            const float2 x = fmul2(make_float2(b[c], b[c + 1]), ks[0]);
            const float2 y = fmul2(make_float2(b[c + 2], b[c + 3]), ks[1]);
            b[c] = x.x; b[c + 1] = x.y; b[c + 2] = y.x; b[c + 3] = y.y;
          }
        }
        const bool masked = key0 + 128 > all_hi || (key0 < all_lo && key0 + 128 > p.sinks);
        if (masked) {
          uint32_t vis[4];  // bit c % 32 of word c / 32: this row sees key c of the tile
#pragma unroll
          for (int x = 0; x < 4; ++x)
            vis[x] = low_bits(up - 32 * x) & (~low_bits(down - 32 * x) | low_bits(sk - 32 * x));
#pragma unroll
          for (int c = 0; c < 128; ++c)
            if (!((vis[c / 32] >> (c % 32)) & 1u)) b[c] = -INFINITY;
        }
        float hm[2];
#pragma unroll
        for (int h2 = 0; h2 < 2; ++h2) {
          float a[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float* v = b + h2 * 64 + i;
            a[i] = fmaxf(fmax3(fmax3(v[0], v[8], v[16]), v[24], v[32]), fmax3(v[40], v[48], v[56]));
          }
          hm[h2] = fmax3(fmax3(a[0], a[1], a[2]), fmax3(a[3], a[4], a[5]), fmaxf(a[6], a[7]));
        }
        const float tmax = fmaxf(hm[0], hm[1]) * scale;
        const bool upd = tmax > m_run + (I8 ? lazy : C::LAZY);
        const float m_new = upd ? tmax : m_run;
        const float alpha = upd ? ex2_approx(m_run - m_new) : 1.0f;
        float m_use = (m_new == -INFINITY) ? 0.0f : m_new;
        const float2 scv = make_float2(scale, scale);
        if constexpr (I8) m_use += (float)unit_shift;
        const float2 ccv = make_float2(-m_use, -m_use);
        float2 acc[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        const bool rescale = j > 0 && __any_sync(0xffffffffu, upd || (I8 && shrink != 1.0f));
#pragma unroll
        for (int h2 = 0; h2 < 2; ++h2) {
          uint32_t pk[32];
          float2 vs[2][2];  // INT8: v_scale of four columns, and of the next four
          if constexpr (I8) ld_shared_f4(scales + 512 + 256 * h2, vs[0]);
#pragma unroll
          for (int pr = 0; pr < 32; ++pr) {
            const int c = h2 * 64 + 2 * pr;
            if (I8 && pr % 2 == 0 && pr < 30) ld_shared_f4(scales + 528 + 4 * c, vs[(pr / 2 + 1) % 2]);
            const float2 a = ffma2(make_float2(b[c], b[c + 1]), scv, ccv);
            float2 e = make_float2(ex2_approx(a.x), ex2_approx(a.y));
            acc[pr & 3] = fadd2(acc[pr & 3], e);
            if constexpr (I8) e = fmul2(e, vs[pr / 2 % 2][pr % 2]);
            pk[pr] = pack2<M>(e.x, e.y);
          }
          if (h2 == 1) {
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(bar_phalf + t);
          } else if (C::SEP_P && j > 0) {
            if (!__all_sync(0xffffffffu, mbar_wait(bar_pvdone + t, (ct + j - 1) & 1, abort_flag, kDevTimeoutSoftmax, p.wait_limit_ns))) { ok = false; break; }
            tc_fence_after();
          }
          tmem_st32(s_tmem + C::P_COL + 32 * h2, *reinterpret_cast<uint32_t(*)[32]>(&pk[0]));
          if (h2 == 0 && rescale) {
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 32) {
              uint32_t orow[32];
              tmem_ld32_sync(o_tmem + c0, orow);
#pragma unroll
              for (int c = 0; c < 32; ++c) orow[c] = __float_as_uint(__uint_as_float(orow[c]) * (I8 ? alpha * shrink : alpha));
              tmem_st32(o_tmem + c0, orow);
            }
          }
        }
        if (!ok) break;
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(bar_pfull + t);
        const float2 s01 = fadd2(fadd2(acc[0], acc[1]), fadd2(acc[2], acc[3]));
        l_run = I8 ? fmaf(l_run, alpha, (s01.x + s01.y) * pow2(unit_shift)) : fmaf(l_run, alpha, s01.x + s01.y);
        m_run = m_new;
        key0 = j == jump ? jump_to : key0 + 128;
      }
      if (!ok) break;
      if (!__all_sync(0xffffffffu, mbar_wait(bar_odone + t, segs & 1, abort_flag, kDevTimeoutEpilogue, p.wait_limit_ns))) { ok = false; break; }
      tc_fence_after();
      ct += n;
      ++segs;
      const bool whole = w.whole();
      const float inv = m_run == -INFINITY ? 0.0f : (I8 ? pow2(e_run) / l_run : 1.0f / l_run);
      const int64_t slot = 2 * cta + (w.tile == 0 ? 1 : 0);
      const int kvh = w.head / p.parts, part = w.head - kvh * p.parts, heads = min(p.Gp, p.G - part * p.Gp);
      const int row = t * 128 + row_in_tile;
      const bool valid = row_tok < toks && row_head < heads;
      if (whole) {
        // Through the warp's part of shared memory, OUT_CH channels at a time: PR consecutive lanes then
        // store a row's contiguous bytes, where one lane per row would touch 32 lines. Piece c of row r
        // lies at c ^ swizzle(r), against bank conflicts.
        constexpr int PR = C::OUT_CH / 8, SW = 8 / PR;  // pieces per row; rows that share 128 bytes
        uint4* stage = reinterpret_cast<uint4*>(smem + C::OFF_OUT + warp * C::OUT_BYTES);
        T* out = static_cast<T*>(p.o) + (int64_t)(w.it.base + first_tok) * p.o_st +
                 (int64_t)(kvh * p.G + part * p.Gp) * p.o_sh;
        const int piece = lane % PR;
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += C::OUT_CH) {
#pragma unroll
          for (int h2 = 0; h2 < C::OUT_CH / 32; ++h2) {
            uint32_t orow[32];
            tmem_ld32_sync(o_tmem + c0 + 32 * h2, orow);
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              float f[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(orow[8 * v + e]) * inv;
              stage[lane * PR + ((4 * h2 + v) ^ ((lane / SW) % PR))] = Half8<T>::from_float(f);
            }
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < PR; ++i) {
            const int r = i * (32 / PR) + lane / PR;
            const int tok = __shfl_sync(0xffffffffu, row_tok, r), hd = __shfl_sync(0xffffffffu, row_head, r);
            if (tok < toks && hd < heads)
              *reinterpret_cast<uint4*>(out + (int64_t)tok * p.o_st + (int64_t)hd * p.o_sh + c0 + piece * 8) =
                  stage[r * PR + (piece ^ ((r / SW) % PR))];
          }
          __syncwarp();
        }
      } else {
        // channels 4 x .. 4 x + 3 of row r at [x][r], so that a warp's store is contiguous
        float4* dst = reinterpret_cast<float4*>(p.part) + slot * kChunkRows * (D / 4) + row;
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += 32) {
          uint32_t orow[32];
          tmem_ld32_sync(o_tmem + c0, orow);
          if (valid) {
#pragma unroll
            for (int v = 0; v < 8; ++v)
              dst[(c0 / 4 + v) * kChunkRows] =
                  make_float4(__uint_as_float(orow[4 * v]), __uint_as_float(orow[4 * v + 1]),
                              __uint_as_float(orow[4 * v + 2]), __uint_as_float(orow[4 * v + 3]));
          }
        }
        if (valid) *reinterpret_cast<float4*>(p.part_ml + (slot * kChunkRows + row) * 4) = make_float4(m_run, l_run, (float)e_run, 0.0f);
      }
      tc_fence_before();
    }
    tc_fence_before();
    asm volatile("bar.arrive 2, %0;" ::"n"(kChunkThreads) : "memory");
  }
}

// Joins the parts of blocks that the pieces' borders cut, as paged_combine_kernel does: eight rows per
// block, a thread per row and four channels (eight threads read 128 contiguous bytes).
constexpr int kJoinRows = 8;
template <int D, bool I8, typename T>
__global__ void __launch_bounds__(kJoinRows * D / 4) paged_chunk_join_kernel(const DecodeParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 d = p.desc[blockIdx.x];
  if (d.w == 0) return;
  const int row = blockIdx.y * kJoinRows + threadIdx.x % kJoinRows, x = threadIdx.x / kJoinRows;
  const int r = row & 127, rt = r / p.Gp, hd = r - rt * p.Gp;
  const int kvh = d.y / p.parts, part = d.y - kvh * p.parts;
  const PagedSeq sq = paged_seq(p.s, d.x);
  const int tok = (2 * d.z + (row >> 7)) * p.TT + rt;
  if (rt >= p.TT || tok >= sq.n || part * p.Gp + hd >= p.G) return;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float m = I8 ? kNoScore : -INFINITY, l = 0.0f, eo = -126.0f;  // INT8: the outputs are in units of 2^(m + eo)
#pragma unroll 4
  for (int j = 0; j <= d.w; ++j) {
    const int64_t slot = j == 0 ? 2 * blockIdx.x + 1 : 2 * (blockIdx.x + j);
    const float4 ml = *reinterpret_cast<const float4*>(p.part_ml + (slot * kChunkRows + row) * 4);
    const float4 v = reinterpret_cast<const float4*>(p.part)[(slot * (D / 4) + x) * kChunkRows + row];
    const float mn = fmaxf(m, ml.x), use = mn == -INFINITY ? 0.0f : mn;
    float a = ex2_approx(m - use), z = ex2_approx(ml.x - use);
    l = fmaf(l, a, ml.y * z);
    if constexpr (I8) {
      const float en = fmaxf(unit_under(m, eo, mn), unit_under(ml.x, ml.z, mn));
      a = ex2_approx((m - mn) + (eo - en));
      z = ex2_approx((ml.x - mn) + (ml.z - en));
      eo = en;
    }
    m = mn;
    o.x = fmaf(o.x, a, v.x * z);
    o.y = fmaf(o.y, a, v.y * z);
    o.z = fmaf(o.z, a, v.z * z);
    o.w = fmaf(o.w, a, v.w * z);
  }
  const float inv = l == 0.0f ? 0.0f : (I8 ? pow2((int)eo) : 1.0f) / l;
  T* dst = static_cast<T*>(p.o) + (int64_t)(sq.base + tok) * p.o_st + (int64_t)(kvh * p.G + part * p.Gp + hd) * p.o_sh + x * 4;
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
}

}  // namespace sage
